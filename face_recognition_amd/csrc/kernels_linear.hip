// Products behind the embeddings: y = act(x W^T + b) + r for any sizes, the same grouped by row (every row names the matrix
// it goes through), and their gradients.  No counterpart in the reference, whose one linear layer is the network's last.
//
//   forward      z = x W^T + b,  y = act(z) + r         rows of one group against that group's matrix
//   backward     dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum dz;  dslope = sum dy min(z, 0);  dr = dy
//
// A row list (`order`, stable by group) stands between the rows in memory and the tiles: a tile gathers its rows through it
// and scatters its results back, so nothing is permuted in memory.  Sums are fp32; z and dz are rounded once to the product's
// type (they are operands of the matrix instructions / of act' only, the same half step as the outputs').
#include "pj_tile.h"

namespace fra {

enum { PJ_NONE = 0, PJ_RELU = 1, PJ_PRELU = 2, PJ_SILU = 3, PJ_GELU_TANH = 4 };

// 1 / (1 + e^-v).  For 16-bit results the hardware's reciprocal (1 ulp) is far below the final rounding.
template <typename T> __device__ __forceinline__ float pj_sigmoid(float v) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.0f + __expf(-v));
    else return 1.0f / (1.0f + expf(-v));
}
constexpr float GELU_C = 1.5957691216057308f, GELU_A = 0.044715f;       // 2 sqrt(2 / pi)

// comparisons are written so that a NaN goes through
template <typename T> __device__ __forceinline__ float pj_act(int act, float z, float s) {
    switch (act) {
        case PJ_RELU: return z < 0.0f ? 0.0f : z;
        case PJ_PRELU: return z < 0.0f ? z * s : z;
        case PJ_SILU: return z * pj_sigmoid<T>(z);
        case PJ_GELU_TANH: return z * pj_sigmoid<T>(GELU_C * (z + GELU_A * z * z * z));
        default: return z;
    }
}
// one branch for a whole piece
template <typename T, int V> __device__ __forceinline__ void pj_act_all(int act, float (&v)[V], const float (&s)[V]) {
    switch (act) {
#define PJ_CASE(A)                                                \
    case A:                                                       \
        _Pragma("unroll") for (int e = 0; e < V; ++e) v[e] = pj_act<T>(A, v[e], s[e]); \
        break;
        PJ_CASE(PJ_RELU) PJ_CASE(PJ_PRELU) PJ_CASE(PJ_SILU) PJ_CASE(PJ_GELU_TANH)
#undef PJ_CASE
        default: break;
    }
}
template <typename T> __device__ __forceinline__ float pj_act_grad(int act, float z, float s) {
    switch (act) {
        case PJ_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case PJ_PRELU: return z > 0.0f ? 1.0f : s;
        case PJ_SILU: {
            const float q = pj_sigmoid<T>(z);
            return q * (1.0f + z * (1.0f - q));
        }
        case PJ_GELU_TANH: {
            const float q = pj_sigmoid<T>(GELU_C * (z + GELU_A * z * z * z));
            return q + z * q * (1.0f - q) * GELU_C * (1.0f + 3.0f * GELU_A * z * z);
        }
        default: return 1.0f;
    }
}

// what every product kernel knows about its rows
struct RowArgs {
    const int* order;           // nullptr: the rows themselves
    const int4* tiles;          // (group, first list entry, end, -) per row tile; nullptr: one group, tiles of BI rows
    const int* offsets;         // [G + 1] list entries of a group (grouped only)
    int n_tiles, M, G;
};
__device__ __forceinline__ bool row_tile(const RowArgs& a, int t, int bi, int& g, int& begin, int& end) {
    if (a.tiles) {
        const int4 e = a.tiles[t];
        g = e.x; begin = e.y; end = e.z;
        return g >= 0;                                              // entries past the last tile
    }
    g = 0;
    begin = t * bi;
    end = begin + bi < a.M ? begin + bi : a.M;
    return true;
}

struct FwdArgs {
    RowArgs rows;
    const void *x, *w, *bias, *slope, *resid;
    void *z, *y;
    int64_t ldx, ldw, wg, ldr;
    int K, N, act, bias_f32, slope_f32, n_col_tiles;
};

// A lane's columns are the same in all its pieces, so bias and slope sit in registers.
template <typename T> struct ForwardEmit {
    static constexpr int V = 16 / sizeof(T);
    struct Pre {
        int row;                    // -1: past the tile's rows or columns
        typename Elem<T>::Frag r;
    };
    const FwdArgs* a;
    int begin, count, n0, left;     // left: valid columns from the lane's first
    bool live;
    float bi[V], sl[V];
    __device__ __forceinline__ void init(int g, int col) {
        const int n = n0 + col;
        left = a->N - n;
#pragma unroll
        for (int q = 0; q < V; q += 4) {
            float b4[4] = {0, 0, 0, 0}, s4[4] = {0, 0, 0, 0};
            if (a->bias && live) load_param4<T>(a->bias, a->bias_f32, (int64_t)g * a->N + n + q, left - q, b4);
            if (a->slope && live) load_param4<T>(a->slope, a->slope_f32, (int64_t)g * a->N + n + q, left - q, s4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { bi[q + e] = b4[e]; sl[q + e] = s4[e]; }
        }
    }
    __device__ __forceinline__ Pre pre(int i, int j) const {
        Pre p;
        p.row = -1;
#pragma unroll
        for (int e = 0; e < V; ++e) p.r[e] = (T)0.0f;
        if (i < count && left > 0) {
            p.row = a->rows.order ? a->rows.order[begin + i] : begin + i;
            if (a->resid) p.r = load_chunk<T>((const T*)a->resid + (int64_t)p.row * a->ldr + n0 + j, left);
        }
        return p;
    }
    __device__ __forceinline__ void emit(const Pre& p, int, int j, float (&v)[V]) const {
        if (p.row < 0) return;
        const int64_t at = (int64_t)p.row * a->N + n0 + j;
        typename Elem<T>::Frag o;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += bi[e];
        if (a->z && live) {
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = (T)v[e];
            store_chunk<T>((T*)a->z + at, left, o);
        }
        if (!live) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = 0.0f;
        } else {
            pj_act_all<T, V>(a->act, v, sl);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = (T)(v[e] + (float)p.r[e]);
        store_chunk<T>((T*)a->y + at, left, o);
    }
};
template <typename T, typename S, bool DMA> __global__ __launch_bounds__(S::NT) void pj_forward_kernel(FwdArgs a) {
    typedef Operand<T, false, S::BI, S::NT> OA;
    typedef Operand<T, false, S::BJ, S::NT> OB;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int ct = blockIdx.x % a.n_col_tiles, rt = blockIdx.x / a.n_col_tiles;
    int g, begin, end;
    if (!row_tile(a.rows, rt, S::BI, g, begin, end)) return;
    const bool live = g < a.rows.G;                                 // group G: rows of no group
    const int n0 = ct * S::BJ;
    f32x4 acc[S::MI][S::MJ];
    OA A;
    A.base = (const T*)a.x; A.order = a.rows.order; A.ld = a.ldx; A.row0 = begin; A.rows = end - begin; A.klen = a.K; A.cols = 0;
    OB B;
    B.base = (const T*)a.w + (live ? (int64_t)g * a.wg : 0); B.order = nullptr; B.ld = a.ldw; B.row0 = n0; B.rows = a.N - n0; B.klen = a.K; B.cols = 0;
    tile_product<T, false, false, S, DMA>(A, B, live ? a.K : 0, lds, acc);

    ForwardEmit<T> f;
    f.a = &a; f.begin = begin; f.count = end - begin; f.n0 = n0; f.live = live;
    f.init(g, (threadIdx.x >> 6) / S::WI * (S::BJ / S::WJ) + (int)(threadIdx.x & 63) % (S::MJ * 16 / f.V) * f.V);
    tile_emit<T, S>(acc, lds, f);
}

// dx = dz W: rows of dz, W contraction-major
struct DxArgs {
    RowArgs rows;
    const void *dz, *w;
    void* dx;
    int64_t lddz, ldw, wg;
    int K, N, Np, n_col_tiles;  // Np: columns of dz, zeros from N on (its pitch if it lies in the workspace, else N)
};
template <typename T, typename S, bool DMA> __global__ __launch_bounds__(S::NT) void pj_dx_kernel(DxArgs a) {
    typedef Operand<T, false, S::BI, S::NT> OA;
    typedef Operand<T, true, S::BJ, S::NT> OB;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int ct = blockIdx.x % a.n_col_tiles, rt = blockIdx.x / a.n_col_tiles;
    int g, begin, end;
    if (!row_tile(a.rows, rt, S::BI, g, begin, end)) return;
    const bool live = g < a.rows.G;
    const int k0 = ct * S::BJ;
    f32x4 acc[S::MI][S::MJ];
    OA A;
    A.base = (const T*)a.dz; A.order = a.rows.order; A.ld = a.lddz; A.row0 = begin; A.rows = end - begin; A.klen = a.Np; A.cols = 0;
    OB B;
    B.base = (const T*)a.w + (live ? (int64_t)g * a.wg : 0) + k0; B.order = nullptr; B.ld = a.ldw; B.row0 = 0; B.rows = 0; B.klen = a.N; B.cols = a.K - k0;
    tile_product<T, false, true, S, DMA>(A, B, live ? a.Np : 0, lds, acc);

    struct Emit {
        typedef int Pre;
        const DxArgs* a;
        int begin, count, k0;
        __device__ __forceinline__ int pre(int i, int) const { return i < count ? (a->rows.order ? a->rows.order[begin + i] : begin + i) : -1; }
        __device__ __forceinline__ void emit(int row, int, int j, float (&v)[16 / sizeof(T)]) const {
            const int left = a->K - k0 - j;
            if (row < 0 || left <= 0) return;
            typename Elem<T>::Frag o;
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(T); ++e) o[e] = (T)v[e];
            store_chunk<T>((T*)a->dx + (int64_t)row * a->K + k0 + j, left, o);
        }
    } f = {&a, begin, end - begin, k0};
    tile_emit<T, S>(acc, lds, f);
}

// dW[g] = sum over the group's rows of dz^T x: both operands contraction-major.  `splits` workgroups share a group's rows
// and leave fp32 partial sums [split][G][N][K], which pj_join_kernel adds in order; one split writes dW itself.
struct DwArgs {
    RowArgs rows;
    const void *dz, *x;
    void* dw;                   // T [G][N][K], or float partial sums if splits > 1
    int64_t lddz, ldx;
    int K, N, Np, n_ti, n_tj, splits;
};
template <typename O> struct DwEmit {
    typedef int Pre;
    O* out;
    int N, K, n0, k0;
    __device__ __forceinline__ int pre(int, int) const { return 0; }
    __device__ __forceinline__ void emit(int, int i, int j, float (&v)[16 / sizeof(O)]) const {
        const int n = n0 + i, left = K - k0 - j;
        if (n >= N || left <= 0) return;
        typename Elem<O>::Frag o;
#pragma unroll
        for (int e = 0; e < 16 / (int)sizeof(O); ++e) o[e] = (O)v[e];
        store_chunk<O>(out + (int64_t)n * K + k0 + j, left, o);
    }
};
template <typename T, typename S, bool DMA> __global__ __launch_bounds__(S::NT) void pj_dw_kernel(DwArgs a) {
    typedef Operand<T, true, S::BI, S::NT> OA;
    typedef Operand<T, true, S::BJ, S::NT> OB;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    unsigned b = blockIdx.x;
    const int tj = b % a.n_tj; b /= a.n_tj;
    const int ti = b % a.n_ti; b /= a.n_ti;
    const int s = b % a.splits, g = b / a.splits;
    int begin = a.rows.offsets ? a.rows.offsets[g] : 0, end = a.rows.offsets ? a.rows.offsets[g + 1] : a.rows.M;
    if (a.splits > 1) {                                             // whole steps per split
        const int steps = (end - begin + Elem<T>::KSTEP - 1) / Elem<T>::KSTEP;
        const int per = (steps + a.splits - 1) / a.splits * Elem<T>::KSTEP;
        const int64_t b0 = (int64_t)begin + (int64_t)s * per, e0 = b0 + per;
        begin = b0 < end ? (int)b0 : end;
        end = e0 < end ? (int)e0 : end;
    }
    const int n0 = ti * S::BI, k0 = tj * S::BJ;
    f32x4 acc[S::MI][S::MJ];
    OA A;
    A.base = (const T*)a.dz + n0; A.order = a.rows.order; A.ld = a.lddz; A.row0 = begin; A.rows = 0; A.klen = end - begin; A.cols = a.Np - n0;
    OB B;
    B.base = (const T*)a.x + k0; B.order = a.rows.order; B.ld = a.ldx; B.row0 = begin; B.rows = 0; B.klen = end - begin; B.cols = a.K - k0;
    tile_product<T, true, true, S, DMA>(A, B, end - begin, lds, acc);

    const int64_t plane = (int64_t)a.N * a.K;
    if (a.splits > 1) {
        DwEmit<float> f = {(float*)a.dw + ((int64_t)s * a.rows.G + g) * plane, a.N, a.K, n0, k0};
        tile_emit<float, S>(acc, lds, f);
    } else {
        DwEmit<T> f = {(T*)a.dw + (int64_t)g * plane, a.N, a.K, n0, k0};
        tile_emit<T, S>(acc, lds, f);
    }
}
// out[e] = sum over splits of part[s][e], s ascending
template <typename T> __global__ __launch_bounds__(256) void pj_join_kernel(const float* part, T* out, int64_t n, int splits) {
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (e >= n) return;
    float v[4] = {0, 0, 0, 0}, o[4];
    const int left = n - e < 4 ? (int)(n - e) : 4;
    for (int s = 0; s < splits; ++s) {
        load_four<float>(part + (int64_t)s * n + e, left, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += o[i];
    }
    store_four<T>(out + e, left, v);
}

// dz = dy act'(z) and, per row tile, the column sums of dz and of dy min(z, 0).  A workgroup takes one row tile x 256 columns,
// wave w its rows w, w + 4, ...; the waves' sums meet in LDS.
struct DzArgs {
    RowArgs rows;
    const void *dy, *z, *slope;
    void* dz;                   // [M][Np], zeros from column N on; nullptr: dz = dy, only the sums are wanted
    float *part_b, *part_s;     // [tiles][N], nullptr where not wanted
    int64_t lddy;
    int N, Np, act, slope_f32, tile_rows, n_col_tiles;
};
template <typename T> __global__ __launch_bounds__(256) void pj_dz_kernel(DzArgs a) {
    __shared__ f32x4 sums[2][4][64];
    const int ct = blockIdx.x % a.n_col_tiles, rt = blockIdx.x / a.n_col_tiles;
    int g, begin, end;
    if (!row_tile(a.rows, rt, a.tile_rows, g, begin, end) || g >= a.rows.G) return;     // the same for the whole workgroup
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = ct * 256 + lane * 4, left = a.N - n;
    float sb[4] = {0, 0, 0, 0}, ss[4] = {0, 0, 0, 0}, sl[4] = {0, 0, 0, 0};
    if (n < a.Np) {
        if (a.slope) load_param4<T>(a.slope, a.slope_f32, (int64_t)g * a.N + n, left, sl);
        for (int at = begin + wave; at < end; at += 4) {
            const int64_t row = a.rows.order ? a.rows.order[at] : at;
            float dy[4], z[4] = {0, 0, 0, 0}, d[4];
            load_four<T>((const T*)a.dy + row * a.lddy + n, left, dy);
            if (a.act != PJ_NONE) load_four<T>((const T*)a.z + row * a.N + n, left, z);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d[e] = a.act != PJ_NONE ? dy[e] * pj_act_grad<T>(a.act, z[e], sl[e]) : dy[e];
                sb[e] += d[e];
                ss[e] += z[e] > 0.0f ? 0.0f : dy[e] * z[e];
            }
            if (a.dz) store_four<T>((T*)a.dz + row * a.Np + n, 4, d);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) { sums[0][wave][lane][e] = sb[e]; sums[1][wave][lane][e] = ss[e]; }
    __syncthreads();
    if (wave < 2 && left > 0) {
        float* part = wave == 0 ? a.part_b : a.part_s;
        if (part) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = (sums[wave][0][lane][e] + sums[wave][1][lane][e]) + (sums[wave][2][lane][e] + sums[wave][3][lane][e]);
            store_four<float>(part + (int64_t)rt * a.N + n, left, v);
        }
    }
}
// out[g][n] = sum of part[t][n] over the group's tiles, in order: 4 waves take every fourth tile of 64 columns
template <typename T> __global__ __launch_bounds__(256) void pj_colsum_kernel(const float* part, const int* tile_offsets, int n_tiles,
                                                                             int N, int n_col_tiles, void* out, int out_f32) {
    __shared__ float sums[4][64];
    const int ct = blockIdx.x % n_col_tiles, g = blockIdx.x / n_col_tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = ct * 64 + lane;
    const int t0 = tile_offsets ? tile_offsets[g] : 0, t1 = tile_offsets ? tile_offsets[g + 1] : n_tiles;
    float v = 0.0f;
    if (n < N)
        for (int t = t0 + wave; t < t1; t += 4) v += part[(int64_t)t * N + n];
    sums[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && n < N) {
        v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
        if (out_f32) ((float*)out)[(int64_t)g * N + n] = v;
        else ((T*)out)[(int64_t)g * N + n] = (T)v;
    }
}

// ---- rows by group: a stable counting sort --------------------------------------------------------------------------
// key = id, or G where id is outside [0, G).  Workgroup b of `nb` owns rows [b R, (b + 1) R), its four waves consecutive
// quarters of them.  A wave walks over 64 rows at a time: lanes with the same key find each other by ballots over the key's
// bits, so a row's rank among its wave's rows of the key is the wave's running count plus the equal lanes below, without
// atomics, and the order does not depend on timing.
constexpr int GR_MAX_GROUPS = 4096;
struct GroupArgs {
    const void* ids;
    int ids64, M, G, nb, rows_per_block, tile_rows, n_tiles;
    int* counts;                // [nb][G + 1]: a block's rows of a key; after the scan: list entries of the key before the block
    int *order, *offsets, *tile_offsets;    // [M], [G + 1], [G + 2]
    int4* tiles;
};
__device__ __forceinline__ int group_key(const GroupArgs& a, int row) {
    const int64_t id = a.ids64 ? ((const int64_t*)a.ids)[row] : ((const int*)a.ids)[row];
    return id >= 0 && id < a.G ? (int)id : a.G;
}
// running counts of this wave in cnt[key]; place == true: writes order[] at cnt[key] + rank, cnt then holding list positions
template <bool PLACE> __device__ __forceinline__ void group_walk(const GroupArgs& a, int begin, int end, int bits, int* cnt, int lane) {
    for (int r0 = begin; r0 < end; r0 += 64) {
        const int row = r0 + lane;
        const bool in = row < end;
        const int key = in ? group_key(a, row) : 0;
        unsigned long long same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long m = __ballot((key >> b) & 1);
            same &= ((key >> b) & 1) ? m : ~m;
        }
        const int below = __popcll(same & ((1ull << lane) - 1)), all = __popcll(same);
        int at = 0;
        if (in) at = cnt[key];
        if (PLACE && in) a.order[at + below] = row;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (in && below == 0) cnt[key] = at + all;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the next rows' lanes read what this row's leader wrote
    }
}
// exclusive sums over 256 threads' values; returns this thread's, total to every thread
__device__ __forceinline__ int block_scan(int v, int* tmp, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) base += w < wave ? tmp[w] : 0;
    total = tmp[0] + tmp[1] + tmp[2] + tmp[3];
    return base + x - v;
}
// totals[key] -> offsets, tile_offsets, the tile table and (in totals) every key's first list entry
__device__ __forceinline__ void group_tables(const GroupArgs& a, int* totals, int* tofs, int* tmp) {
    const int keys = a.G + 1;
    int base = 0, tbase = 0;
    for (int k0 = 0; k0 < keys; k0 += 256) {
        const int k = k0 + threadIdx.x;
        const int c = k < keys ? totals[k] : 0, tc = (c + a.tile_rows - 1) / a.tile_rows;
        int tot, ttot;
        const int o = base + block_scan(c, tmp, tot), to = tbase + block_scan(tc, tmp, ttot);
        if (k < keys) {
            totals[k] = o;
            tofs[k] = to;
            a.offsets[k] = o;
            a.tile_offsets[k] = to;
        }
        base += tot;
        tbase += ttot;
    }
    if (threadIdx.x == 0) a.tile_offsets[keys] = tbase;
    __syncthreads();
    for (int t = threadIdx.x; t < a.n_tiles; t += 256) {
        int4 e = {-1, 0, 0, 0};
        if (t < tbase) {
            int lo = 0, hi = keys - 1;                              // the last key whose first tile is <= t
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (tofs[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            const int first = totals[lo] + (t - tofs[lo]) * a.tile_rows;
            const int end = lo + 1 < keys ? totals[lo + 1] : a.M;
            e.x = lo;
            e.y = first;
            e.z = first + a.tile_rows < end ? first + a.tile_rows : end;
        }
        a.tiles[t] = e;
    }
}
__device__ __forceinline__ void wave_range(const GroupArgs& a, int b, int wave, int& begin, int& end) {
    const int64_t lo = (int64_t)b * a.rows_per_block, q = a.rows_per_block / 4;
    const int64_t e = lo + (wave + 1) * q, s = lo + wave * q;
    begin = s < a.M ? (int)s : a.M;
    end = e < a.M ? (int)e : a.M;
}
// MODE 0: everything in one workgroup; 1: a block's counts; 2: place, after pj_group_scan_kernel
template <int MODE> __global__ __launch_bounds__(256) void pj_group_kernel(GroupArgs a, int bits) {
    extern __shared__ int cnt[];                                    // [4][keys], mode 0: + totals[keys], tofs[keys]
    __shared__ int tmp[4];
    const int keys = a.G + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int begin, end;
    wave_range(a, blockIdx.x, wave, begin, end);
    for (int i = threadIdx.x; i < 4 * keys; i += 256) cnt[i] = 0;
    __syncthreads();
    group_walk<false>(a, begin, end, bits, cnt + wave * keys, lane);
    __syncthreads();
    if (MODE == 1) {
        for (int k = threadIdx.x; k < keys; k += 256)
            a.counts[(int64_t)blockIdx.x * keys + k] = cnt[k] + cnt[keys + k] + cnt[2 * keys + k] + cnt[3 * keys + k];
        return;
    }
    if (MODE == 0) {
        int* totals = cnt + 4 * keys;
        for (int k = threadIdx.x; k < keys; k += 256) totals[k] = cnt[k] + cnt[keys + k] + cnt[2 * keys + k] + cnt[3 * keys + k];
        __syncthreads();
        group_tables(a, totals, totals + keys, tmp);
        __syncthreads();
    }
    for (int k = threadIdx.x; k < keys; k += 256) {                 // counts -> the wave's first list entry of the key
        int at = MODE == 0 ? cnt[4 * keys + k] : a.offsets[k] + a.counts[(int64_t)blockIdx.x * keys + k];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int c = cnt[w * keys + k];
            cnt[w * keys + k] = at;
            at += c;
        }
    }
    __syncthreads();
    group_walk<true>(a, begin, end, bits, cnt + wave * keys, lane);
}
// counts[b][key] -> exclusive sums over b; totals -> tables
__global__ __launch_bounds__(256) void pj_group_scan_kernel(GroupArgs a) {
    extern __shared__ int cnt[];
    __shared__ int tmp[4];
    const int keys = a.G + 1;
    for (int k = threadIdx.x; k < keys; k += 256) {
        int sum = 0;
        for (int b = 0; b < a.nb; ++b) {
            const int c = a.counts[(int64_t)b * keys + k];
            a.counts[(int64_t)b * keys + k] = sum;
            sum += c;
        }
        cnt[k] = sum;
    }
    __syncthreads();
    group_tables(a, cnt, cnt + keys, tmp);
}

// ---- launchers ------------------------------------------------------------------------------------------------------

// dynamic LDS of a product kernel: two buffers of both operands' tiles
template <typename S> constexpr int product_lds() { return 2 * (S::BI + S::BJ) * 128; }

// rows at `p`, `pitches` (one, or several or-ed together) elements apart and `len` long, consist of whole aligned chunks
template <typename T> static bool dma_ok(const void* p, int64_t pitches, int64_t len) {
    return ((uintptr_t)p & 15) == 0 && ((pitches | len) & (16 / (int64_t)sizeof(T) - 1)) == 0;
}

template <typename K> static int raise_lds(K kernel, int bytes, std::atomic<uint64_t>& done) {
    return ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes, done);
}
#define PJ_LAUNCH(KERNEL, GRID, NT, LDS, STREAM, ARGS)                                   \
    do {                                                                                 \
        static std::atomic<uint64_t> lds_done{0};                                        \
        const int rc__ = raise_lds(KERNEL, LDS, lds_done);                               \
        if (rc__ != FRA_OK) return rc__;                                                 \
        hipLaunchKernelGGL(KERNEL, dim3((unsigned)(GRID)), dim3(NT), LDS, STREAM, ARGS); \
        FRA_HIP(hipGetLastError());                                                      \
    } while (0)

typedef Shape<128, 128, 2, 2> Big;
typedef Shape<64, 64, 2, 2> Small;

static int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

static int check_desc(const fra_linear_desc* d, const char* what) {
    FRA_REQUIRE(d, FRA_ERR_ARG, "%s: null descriptor", what);
    FRA_REQUIRE(d->dtype == FRA_F32 || d->dtype == FRA_BF16 || d->dtype == FRA_F16, FRA_ERR_ARG, "%s: dtype %d unsupported", what, d->dtype);
    FRA_REQUIRE(d->M >= 0 && d->M <= 2147483647LL - 1024, FRA_ERR_ARG, "%s: %lld rows (0 to 2^31 - 1025)", what, (long long)d->M);
    FRA_REQUIRE(d->K >= 1 && d->N >= 1 && d->K <= (1 << 24) && d->N <= (1 << 24), FRA_ERR_ARG, "%s: K = %d, N = %d (1 to 2^24)", what, d->K, d->N);
    FRA_REQUIRE(d->act >= PJ_NONE && d->act <= PJ_GELU_TANH, FRA_ERR_ARG, "%s: activation %d unknown", what, d->act);
    FRA_REQUIRE((d->act == PJ_PRELU) == (d->slope != nullptr), FRA_ERR_ARG, "%s: slopes go with the activation FRA_ACT_PRELU, and only with it", what);
    FRA_REQUIRE(!d->bias || d->bias_dtype == d->dtype || d->bias_dtype == FRA_F32, FRA_ERR_ARG, "%s: bias dtype %d (fp32 or the product's)", what, d->bias_dtype);
    FRA_REQUIRE(!d->slope || d->slope_dtype == d->dtype || d->slope_dtype == FRA_F32, FRA_ERR_ARG, "%s: slope dtype %d (fp32 or the product's)", what, d->slope_dtype);
    FRA_REQUIRE(d->w && (d->x || d->M == 0), FRA_ERR_ARG, "%s: null pointer", what);
    FRA_REQUIRE(d->ldx >= d->K && d->ldw >= d->K, FRA_ERR_ARG, "%s: row pitches %lld, %lld below K = %d", what, (long long)d->ldx, (long long)d->ldw, d->K);
    FRA_REQUIRE(!d->resid || d->ldr >= d->N, FRA_ERR_ARG, "%s: residual pitch %lld below N = %d", what, (long long)d->ldr, d->N);
    if (const fra_row_groups* g = d->groups) {
        FRA_REQUIRE(g->rows == d->M, FRA_ERR_ARG, "%s: groups of %lld rows, product of %lld", what, (long long)g->rows, (long long)d->M);
        FRA_REQUIRE(g->n_groups >= 1 && g->n_groups <= GR_MAX_GROUPS, FRA_ERR_ARG, "%s: %d groups (1 to %d)", what, g->n_groups, GR_MAX_GROUPS);
        FRA_REQUIRE(g->tile_rows == fra_group_tile_rows(g->rows, g->n_groups) && g->n_tiles == fra_group_tiles(g->rows, g->n_groups),
                    FRA_ERR_ARG, "%s: a tile table of %d entries of %d rows is not fra_group_rows' own", what, g->n_tiles, g->tile_rows);
        FRA_REQUIRE(g->offsets && g->tiles && g->tile_offsets && (g->order || d->M == 0), FRA_ERR_ARG, "%s: null pointer in the groups", what);
        FRA_REQUIRE(d->w_group_stride >= 0, FRA_ERR_ARG, "%s: group stride %lld", what, (long long)d->w_group_stride);
    }
    return FRA_OK;
}
static RowArgs row_args(const fra_linear_desc* d, int tile_rows) {
    RowArgs r;
    const fra_row_groups* g = d->groups;
    r.order = g ? g->order : nullptr;
    r.tiles = g ? (const int4*)g->tiles : nullptr;
    r.offsets = g ? g->offsets : nullptr;
    r.n_tiles = g ? g->n_tiles : cdiv(d->M, tile_rows);
    r.M = (int)d->M;
    r.G = g ? g->n_groups : 1;
    return r;
}
static int check_grid(int64_t blocks, const char* what) {
    FRA_REQUIRE(blocks < 2147483647LL, FRA_ERR_ARG, "%s: %lld workgroups", what, (long long)blocks);
    return FRA_OK;
}
// 128 x 128 tiles once they fill the 256 compute units, else 64 x 64
static bool big_tiles(int64_t rows, int64_t cols) { return (int64_t)cdiv(rows, 128) * cdiv(cols, 128) >= 256; }

template <typename T> static int forward_t(const fra_linear_desc* d, void* z, void* y, hipStream_t s) {
    FwdArgs a;
    const bool big = d->groups ? d->groups->tile_rows == 128 : big_tiles(d->M, d->N);
    const int bi = big ? 128 : 64;
    a.rows = row_args(d, bi);
    a.x = d->x; a.w = d->w; a.bias = d->bias; a.slope = d->slope; a.resid = d->resid; a.z = z; a.y = y;
    a.ldx = d->ldx; a.ldw = d->ldw; a.wg = d->w_group_stride; a.ldr = d->ldr;
    a.K = d->K; a.N = d->N; a.act = d->act; a.bias_f32 = d->bias_dtype == FRA_F32; a.slope_f32 = d->slope_dtype == FRA_F32;
    a.n_col_tiles = cdiv(d->N, bi);
    const int64_t blocks = (int64_t)a.rows.n_tiles * a.n_col_tiles;
    if (int rc = check_grid(blocks, "fra_linear")) return rc;
    const bool dma = dma_ok<T>(d->x, d->ldx, d->K) && dma_ok<T>(d->w, d->ldw | d->w_group_stride, d->K);
    if (big && dma) PJ_LAUNCH((pj_forward_kernel<T, Big, true>), blocks, Big::NT, product_lds<Big>(), s, a);
    else if (big) PJ_LAUNCH((pj_forward_kernel<T, Big, false>), blocks, Big::NT, product_lds<Big>(), s, a);
    else if (dma) PJ_LAUNCH((pj_forward_kernel<T, Small, true>), blocks, Small::NT, product_lds<Small>(), s, a);
    else PJ_LAUNCH((pj_forward_kernel<T, Small, false>), blocks, Small::NT, product_lds<Small>(), s, a);
    return FRA_OK;
}

// ---- backward: what goes where in the workspace
struct BackwardPlan {
    bool need_dz, need_sums;
    int dz_rows, n_tiles, splits, Np;
    size_t off_dz, off_b, off_s, off_part, bytes;
};
static BackwardPlan backward_plan(const fra_linear_desc* d, bool dx, bool dw, bool db, bool ds) {
    BackwardPlan p;
    const int64_t es = d->dtype == FRA_F32 ? 4 : 2;
    const fra_row_groups* g = d->groups;
    const int G = g ? g->n_groups : 1;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    // dz gets rows of whole 16-byte chunks, so that the products can fetch it by DMA: without activation, a copy of dy where
    // N does not give it such rows
    const int epc = (int)(16 / es);
    p.Np = (d->N + epc - 1) / epc * epc;
    p.need_dz = (d->act != PJ_NONE || p.Np != d->N) && (dx || dw);
    p.need_sums = db || ds;
    p.dz_rows = g ? g->tile_rows : 64;
    p.n_tiles = g ? g->n_tiles : cdiv(d->M, p.dz_rows);
    // workgroups of dW: enough to fill the chip twice, each with at least four steps of its group's average share
    const int64_t tiles = (int64_t)cdiv(d->N, 128) * cdiv(d->K, 128) * G;
    const int64_t steps = cdiv(cdiv(d->M, G), d->dtype == FRA_F32 ? 32 : 64);
    int64_t sp = (512 + tiles - 1) / tiles;
    if (sp > steps / 4) sp = steps / 4;
    p.splits = dw && sp > 1 ? (int)sp : 1;
    size_t at = 0;
    p.off_dz = at; if (p.need_dz) at += up((size_t)d->M * p.Np * es);
    p.off_b = at; if (db) at += up((size_t)p.n_tiles * d->N * 4);
    p.off_s = at; if (ds) at += up((size_t)p.n_tiles * d->N * 4);
    p.off_part = at; if (p.splits > 1) at += up((size_t)p.splits * G * d->N * d->K * 4);
    p.bytes = at;
    return p;
}

template <typename T>
static int backward_t(const fra_linear_desc* d, const BackwardPlan& p, const void* z, const void* dy, int64_t lddy, void* dx, void* dw,
                      void* db, void* ds, char* ws, hipStream_t s) {
    const fra_row_groups* g = d->groups;
    const int G = g ? g->n_groups : 1;
    if ((p.need_dz || p.need_sums) && d->M > 0) {
        DzArgs a;
        a.rows = row_args(d, p.dz_rows);
        a.dy = dy; a.z = z; a.slope = d->slope;
        a.dz = p.need_dz ? ws + p.off_dz : nullptr;
        a.part_b = db ? (float*)(ws + p.off_b) : nullptr;
        a.part_s = ds ? (float*)(ws + p.off_s) : nullptr;
        a.lddy = lddy; a.N = d->N; a.Np = p.Np; a.act = d->act; a.slope_f32 = d->slope_dtype == FRA_F32;
        a.tile_rows = p.dz_rows; a.n_col_tiles = cdiv(p.Np, 256);
        const int64_t blocks = (int64_t)a.rows.n_tiles * a.n_col_tiles;
        if (int rc = check_grid(blocks, "fra_linear_backward")) return rc;
        hipLaunchKernelGGL((pj_dz_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, a);
        FRA_HIP(hipGetLastError());
    }
    for (int which = 0; which < 2; ++which) {
        void* out = which == 0 ? db : ds;
        if (!out) continue;
        const int ct = cdiv(d->N, 64);
        if (int rc = check_grid((int64_t)ct * G, "fra_linear_backward")) return rc;
        hipLaunchKernelGGL((pj_colsum_kernel<T>), dim3((unsigned)ct * G), dim3(256), 0, s, (const float*)(ws + (which == 0 ? p.off_b : p.off_s)),
                           g ? (const int*)g->tile_offsets : nullptr, p.n_tiles, d->N, ct, out,
                           (int)((which == 0 ? d->bias_dtype : d->slope_dtype) == FRA_F32));
        FRA_HIP(hipGetLastError());
    }
    const void* dz = p.need_dz ? ws + p.off_dz : dy;
    const int64_t lddz = p.need_dz ? p.Np : lddy;
    const int Np = p.need_dz ? p.Np : d->N;
    if (dx && d->M > 0) {
        DxArgs a;
        const bool big = g ? g->tile_rows == 128 : big_tiles(d->M, d->K);
        const int bi = big ? 128 : 64;
        a.rows = row_args(d, bi);
        a.dz = dz; a.w = d->w; a.dx = dx; a.lddz = lddz; a.ldw = d->ldw; a.wg = d->w_group_stride; a.K = d->K; a.N = d->N; a.Np = Np;
        a.n_col_tiles = cdiv(d->K, bi);
        const int64_t blocks = (int64_t)a.rows.n_tiles * a.n_col_tiles;
        if (int rc = check_grid(blocks, "fra_linear_backward")) return rc;
        const bool dma = dma_ok<T>(dz, lddz, Np) && dma_ok<T>(d->w, d->ldw | d->w_group_stride, d->K);
        if (big && dma) PJ_LAUNCH((pj_dx_kernel<T, Big, true>), blocks, Big::NT, product_lds<Big>(), s, a);
        else if (big) PJ_LAUNCH((pj_dx_kernel<T, Big, false>), blocks, Big::NT, product_lds<Big>(), s, a);
        else if (dma) PJ_LAUNCH((pj_dx_kernel<T, Small, true>), blocks, Small::NT, product_lds<Small>(), s, a);
        else PJ_LAUNCH((pj_dx_kernel<T, Small, false>), blocks, Small::NT, product_lds<Small>(), s, a);
    }
    if (dw) {
        DwArgs a;
        a.rows = row_args(d, 128);
        a.dz = dz; a.x = d->x; a.dw = p.splits > 1 ? (void*)(ws + p.off_part) : dw; a.lddz = lddz; a.ldx = d->ldx; a.K = d->K; a.N = d->N; a.Np = Np;
        a.n_ti = cdiv(d->N, 128); a.n_tj = cdiv(d->K, 128); a.splits = p.splits;
        const int64_t blocks = (int64_t)a.n_ti * a.n_tj * a.splits * G;
        if (int rc = check_grid(blocks, "fra_linear_backward")) return rc;
        if (dma_ok<T>(dz, lddz, Np) && dma_ok<T>(d->x, d->ldx, d->K)) PJ_LAUNCH((pj_dw_kernel<T, Big, true>), blocks, Big::NT, product_lds<Big>(), s, a);
        else PJ_LAUNCH((pj_dw_kernel<T, Big, false>), blocks, Big::NT, product_lds<Big>(), s, a);
        if (p.splits > 1) {
            const int64_t n = (int64_t)G * d->N * d->K, jb = (n + 1023) / 1024;
            if (int rc = check_grid(jb, "fra_linear_backward")) return rc;
            hipLaunchKernelGGL((pj_join_kernel<T>), dim3((unsigned)jb), dim3(256), 0, s, (const float*)(ws + p.off_part), (T*)dw, n, p.splits);
            FRA_HIP(hipGetLastError());
        }
    }
    return FRA_OK;
}

static int group_blocks(int64_t M, int& rows_per_block) {
    // one workgroup up to 4096 rows; beyond, at most 512 of at least 2048 rows
    int64_t per = M <= 4096 ? 4096 : (M + 511) / 512;
    if (M > 4096 && per < 2048) per = 2048;
    per = (per + 255) / 256 * 256;
    rows_per_block = (int)per;
    return M > 0 ? cdiv(M, per) : 1;
}

}  // namespace fra

using namespace fra;

extern "C" {

int fra_linear(const fra_linear_desc* d, void* preact, void* out, fra_stream stream) {
    if (int rc = check_desc(d, "fra_linear")) return rc;
    if (d->M == 0) return FRA_OK;
    FRA_REQUIRE(out, FRA_ERR_ARG, "fra_linear: null output");
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == FRA_F32) return forward_t<float>(d, preact, out, s);
    if (d->dtype == FRA_BF16) return forward_t<bf16>(d, preact, out, s);
    return forward_t<f16>(d, preact, out, s);
}

int fra_linear_backward_workspace_bytes(const fra_linear_desc* d, int want_dx, int want_dw, int want_dbias, int want_dslope, size_t* bytes) {
    FRA_REQUIRE(bytes, FRA_ERR_ARG, "fra_linear_backward_workspace_bytes: null pointer");
    if (int rc = check_desc(d, "fra_linear_backward_workspace_bytes")) return rc;
    *bytes = backward_plan(d, want_dx, want_dw, want_dbias, want_dslope).bytes;
    return FRA_OK;
}

int fra_linear_backward(const fra_linear_desc* d, const void* preact, const void* dy, int64_t lddy, void* dx, void* dw, void* dbias,
                        void* dslope, void* workspace, size_t workspace_bytes, fra_stream stream) {
    if (int rc = check_desc(d, "fra_linear_backward")) return rc;
    FRA_REQUIRE(dy || d->M == 0, FRA_ERR_ARG, "fra_linear_backward: null gradient");
    FRA_REQUIRE(lddy >= d->N, FRA_ERR_ARG, "fra_linear_backward: gradient pitch %lld below N = %d", (long long)lddy, d->N);
    FRA_REQUIRE(preact || d->act == PJ_NONE || d->M == 0, FRA_ERR_ARG, "fra_linear_backward: the activation needs the values fra_linear left in preact");
    FRA_REQUIRE(!dslope || d->act == PJ_PRELU, FRA_ERR_ARG, "fra_linear_backward: slope gradient without slopes");
    FRA_REQUIRE(!dbias || d->bias_dtype == d->dtype || d->bias_dtype == FRA_F32, FRA_ERR_ARG, "fra_linear_backward: bias dtype %d", d->bias_dtype);
    const BackwardPlan p = backward_plan(d, dx, dw, dbias, dslope);
    FRA_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0), FRA_ERR_WORKSPACE,
                "fra_linear_backward: workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (d->dtype == FRA_F32) return backward_t<float>(d, p, preact, dy, lddy, dx, dw, dbias, dslope, ws, s);
    if (d->dtype == FRA_BF16) return backward_t<bf16>(d, p, preact, dy, lddy, dx, dw, dbias, dslope, ws, s);
    return backward_t<f16>(d, p, preact, dy, lddy, dx, dw, dbias, dslope, ws, s);
}

// rows of a tile: 128 where a group has that many rows on average, else 64
int fra_group_tile_rows(int64_t rows, int n_groups) {
    return n_groups >= 1 && rows / n_groups >= 128 ? 128 : 64;
}
int fra_group_tiles(int64_t rows, int n_groups) {
    if (rows < 0 || n_groups < 1 || n_groups > GR_MAX_GROUPS) return 0;
    return (int)(rows / fra_group_tile_rows(rows, n_groups)) + n_groups + 1;
}
int fra_group_rows_workspace_bytes(int64_t rows, int n_groups, size_t* bytes) {
    FRA_REQUIRE(bytes, FRA_ERR_ARG, "fra_group_rows_workspace_bytes: null pointer");
    FRA_REQUIRE(rows >= 0 && rows <= 2147483647LL - 1024 && n_groups >= 1 && n_groups <= GR_MAX_GROUPS, FRA_ERR_ARG,
                "fra_group_rows_workspace_bytes: %lld rows, %d groups (1 to %d)", (long long)rows, n_groups, GR_MAX_GROUPS);
    int per;
    const int nb = group_blocks(rows, per);
    *bytes = nb > 1 ? (size_t)nb * (n_groups + 1) * 4 : 0;
    return FRA_OK;
}
int fra_group_rows(const void* ids, int ids_are_64bit, const fra_row_groups* g, void* workspace, size_t workspace_bytes, fra_stream stream) {
    FRA_REQUIRE(g, FRA_ERR_ARG, "fra_group_rows: null groups");
    size_t need = 0;
    if (int rc = fra_group_rows_workspace_bytes(g->rows, g->n_groups, &need)) return rc;
    FRA_REQUIRE((ids && g->order) || g->rows == 0, FRA_ERR_ARG, "fra_group_rows: null pointer");
    FRA_REQUIRE(g->offsets && g->tiles && g->tile_offsets, FRA_ERR_ARG, "fra_group_rows: null pointer");
    FRA_REQUIRE(g->tile_rows == fra_group_tile_rows(g->rows, g->n_groups) && g->n_tiles == fra_group_tiles(g->rows, g->n_groups), FRA_ERR_ARG,
                "fra_group_rows: tile_rows / n_tiles are not those of fra_group_tile_rows / fra_group_tiles");
    FRA_REQUIRE(workspace_bytes >= need && (workspace || need == 0), FRA_ERR_WORKSPACE, "fra_group_rows: workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
    GroupArgs a;
    a.ids = ids; a.ids64 = ids_are_64bit != 0; a.M = (int)g->rows; a.G = g->n_groups; a.tile_rows = g->tile_rows; a.n_tiles = g->n_tiles;
    a.nb = group_blocks(g->rows, a.rows_per_block);
    a.counts = (int*)workspace;
    a.order = g->order; a.offsets = g->offsets; a.tile_offsets = g->tile_offsets; a.tiles = (int4*)g->tiles;
    const int keys = a.G + 1;
    int bits = 0;
    while ((1 << bits) < keys) ++bits;
    hipStream_t s = (hipStream_t)stream;
    static std::atomic<uint64_t> done0{0}, done1{0}, done2{0};
    if (a.nb == 1) {
        const int lds = 6 * keys * 4;
        if (int rc = raise_lds(pj_group_kernel<0>, 6 * (GR_MAX_GROUPS + 1) * 4, done0)) return rc;
        hipLaunchKernelGGL((pj_group_kernel<0>), dim3(1), dim3(256), lds, s, a, bits);
        FRA_HIP(hipGetLastError());
        return FRA_OK;
    }
    const int lds = 4 * keys * 4;
    if (int rc = raise_lds(pj_group_kernel<1>, 4 * (GR_MAX_GROUPS + 1) * 4, done1)) return rc;
    if (int rc = raise_lds(pj_group_kernel<2>, 4 * (GR_MAX_GROUPS + 1) * 4, done2)) return rc;
    hipLaunchKernelGGL((pj_group_kernel<1>), dim3(a.nb), dim3(256), lds, s, a, bits);
    FRA_HIP(hipGetLastError());
    hipLaunchKernelGGL(pj_group_scan_kernel, dim3(1), dim3(256), 2 * keys * 4, s, a);
    FRA_HIP(hipGetLastError());
    hipLaunchKernelGGL((pj_group_kernel<2>), dim3(a.nb), dim3(256), lds, s, a, bits);
    FRA_HIP(hipGetLastError());
    return FRA_OK;
}

}  // extern "C"
