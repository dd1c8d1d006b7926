// Products behind the embeddings: y = act(x W^T + b) + r for any sizes, the same grouped by row (every row names the matrix
// it goes through), and their gradients.  No counterpart in the reference, whose one linear layer is the network's last.
//
//   forward      z = x W^T + b,  y = act(z) + r         rows of one group against that group's matrix
//   backward     dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum dz;  dslope = sum dy min(z, 0);  dr = dy
//
// A row list (`order`, stable by group) stands between the rows in memory and the tiles: a tile of the forward product gathers
// its rows through it and scatters its results back.  The backward pass sorts once, while it reads anyway: dz lies in list
// order, x is copied into it for dW, and both gradients' products then run over contiguous rows.  Sums are fp32; z and dz are
// rounded once to the product's type (they are operands of the matrix instructions / of act' only, the same half step as the
// outputs').  What that costs, bf16 with gelu, dx and dW against 64 bits: 0.0017 of the norm is the outputs' own rounding, 0.0023 with
// dz's, 0.0024 with both; a dz in two bf16 halves would double the products, a z in fp32 the bytes kept between the passes.
#include "pj_tile.h"

namespace fra {

enum { PJ_NONE = 0, PJ_RELU = 1, PJ_PRELU = 2, PJ_SILU = 3, PJ_GELU_TANH = 4 };

// 1 / (1 + 2^-t): the sigmoid of t ln 2, so that callers fold log2(e) into their constants.  For 16-bit results the hardware's
// exponential and reciprocal (1 ulp each) are far below the final rounding; the epilogues run on the vector ALU beside the
// matrix cores, where these two cost four slots each.
constexpr float LOG2E = 1.4426950408889634f, GELU_C = 1.5957691216057308f, GELU_A = 0.044715f;      // GELU_C: 2 sqrt(2 / pi)
template <typename T> __device__ __forceinline__ float pj_sigmoid2(float t) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-t));
    else return 1.0f / (1.0f + exp2f(-t));
}

// comparisons are written so that a NaN goes through
template <typename T> __device__ __forceinline__ float pj_act(int act, float z, float s) {
    switch (act) {
        case PJ_RELU: return z < 0.0f ? 0.0f : z;
        case PJ_PRELU: return z < 0.0f ? z * s : z;
        case PJ_SILU: return z * pj_sigmoid2<T>(LOG2E * z);
        case PJ_GELU_TANH: return z * pj_sigmoid2<T>(z * (LOG2E * GELU_C + LOG2E * GELU_C * GELU_A * (z * z)));
        default: return z;
    }
}
// dy act'(z)
template <typename T> __device__ __forceinline__ float pj_dz(int act, float dy, float z, float s) {
    switch (act) {
        case PJ_RELU: return z > 0.0f ? dy : 0.0f;                  // no product: an infinite dy does not reach what relu holds back
        case PJ_PRELU: return z > 0.0f ? dy : dy * s;
        // beyond +-200 the sigmoid q is 0 or 1 exactly and the derivative with it; the other factors are held back there, so that
        // they meet the zero (of q or 1 - q) finite.  A NaN comes through q.
        case PJ_SILU: {
            const float q = pj_sigmoid2<T>(LOG2E * z), c = __builtin_amdgcn_fmed3f(z, -200.0f, 200.0f);
            return dy * (q * (1.0f + c * (1.0f - q)));
        }
        case PJ_GELU_TANH: {
            const float q = pj_sigmoid2<T>(z * (LOG2E * GELU_C + LOG2E * GELU_C * GELU_A * (z * z))), c = __builtin_amdgcn_fmed3f(z, -200.0f, 200.0f);
            return dy * (q * (1.0f + c * (1.0f - q) * (GELU_C + 3.0f * GELU_A * GELU_C * (c * c))));
        }
        default: return dy;
    }
}

// what every product kernel knows about its rows
struct RowArgs {
    const int* order;           // nullptr: the rows themselves
    const int4* tiles;          // (group, first list entry, end, -) per row tile; nullptr: one group, tiles of BI rows
    const int* tile_offsets;    // [G + 2], the last one the number of tiles in use (grouped only)
    int n_tiles, M, G;
    int sub;                    // tiles a table entry is cut into (a kernel's tiles may be shorter than the table's)
};
__device__ __forceinline__ int tiles_in_use(const RowArgs& a) { return a.tiles ? a.tile_offsets[a.G + 1] * a.sub : a.n_tiles; }
__device__ __forceinline__ bool row_tile(const RowArgs& a, int t, int bi, int& g, int& begin, int& end) {
    if (a.tiles) {
        const int part = a.sub > 1 ? t % a.sub : 0;
        const int4 e = a.tiles[a.sub > 1 ? t / a.sub : t];
        g = e.x; begin = e.y; end = e.z;
        if (a.sub > 1) {
            begin += part * bi;
            if (begin >= end) return false;
            end = end - begin > bi ? begin + bi : end;
        }
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

// A lane's columns are the same in all its pieces, so bias and slope sit in registers, sent for before the product (as they lie
// in memory: a conversion there would wait for them) and converted after it.
template <typename T> struct LaneParam {
    static constexpr int V = 16 / sizeof(T);
    f32x4 raw[V / 4];
    __device__ __forceinline__ void load(const void* p, int is_f32, int64_t at, int left) {
        if (is_f32) {
#pragma unroll
            for (int q = 0; q < V / 4; ++q) raw[q] = load_chunk<float>((const float*)p + at + 4 * q, left - 4 * q);
        } else {
            raw[0] = __builtin_bit_cast(f32x4, load_chunk<T>((const T*)p + at, left));
        }
    }
    __device__ __forceinline__ void get(bool there, int is_f32, float (&o)[V]) const {
        const typename Elem<T>::Frag h = __builtin_bit_cast(typename Elem<T>::Frag, raw[0]);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = !there ? 0.0f : is_f32 ? raw[e / 4][e % 4] : (float)h[e];
    }
};
// FULL: the tile's columns are all inside and ACT is the activation, so that the pieces are straight-line code whose loads and
// arithmetic overlap; otherwise everything is checked, and ACT is not used.
template <typename T, int ACT, bool FULL> struct ForwardEmit {
    static constexpr int V = 16 / sizeof(T);
    typedef typename Elem<T>::Frag Frag, Pre;
    const T* resid;
    T *z, *y;
    int64_t ldr, N;
    const int* order;
    int begin, count, n0, left, act;    // left: valid columns from the lane's first
    bool live;
    float bi[V], sl[V];
    // list entry of tile row i, the last row's past the end; -1 - entry where nothing is stored
    __device__ __forceinline__ int row(int i) const {
        const int at = begin + (i < count ? i : count - 1);
        const int r = order ? order[at] : at;
        return i < count && (FULL || left > 0) ? r : -1 - r;
    }
    __device__ __forceinline__ Frag pre(int row, int j) const {
        Frag r = {};
        if (resid) r = load_chunk<T>(resid + (int64_t)(row < 0 ? -1 - row : row) * ldr + n0 + j, FULL ? V : left);
        return r;
    }
    __device__ __forceinline__ void emit(int row, int j, const Frag& r, float (&v)[V]) const {
        const int64_t at = (int64_t)row * N + n0 + j;
        const int n = FULL ? V : left;
        Frag o;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += bi[e];
        if (z && live && row >= 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = (T)v[e];
            store_chunk<T>(z + at, n, o);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if constexpr (FULL) v[e] = pj_act<T>(ACT, v[e], sl[e]);
            else v[e] = live ? pj_act<T>(act, v[e], sl[e]) : 0.0f;
        }
        if (resid) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += (float)r[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = (T)v[e];
        if (row >= 0) store_chunk<T>(y + at, n, o);
    }
};
// A tile of rows x columns as the product kernels see it
struct Tile {
    int g, begin, end, c0;
    bool live;                      // false: rows of no group
};
__device__ __forceinline__ bool next_tile(const RowArgs& a, unsigned b, int n_col_tiles, int bi, int bj, Tile& t) {
    int rt, ct;
    if (!tile_of_block(b, tiles_in_use(a), n_col_tiles, rt, ct) || !row_tile(a, rt, bi, t.g, t.begin, t.end)) return false;
    t.c0 = ct * bj;
    t.live = t.g < a.G;
    return true;
}

// z = x W^T + b, y = act(z) + r.  One tile per workgroup.  Bound, by size: large K by the matrix cores (8192^3 in bf16 826 us, 1.33
// PFLOP/s; the library's plain product 1.45); K = 512 by what surrounds a tile's eight steps -- of the 12.7 us of a 128 x 128 tile
// two such workgroups on a compute unit spend 7.4 in the steps, 2.8 before the first one's data are there and 2.5 on the results
// (4.2 with a residual and a sigmoid), and neither walking over tiles with the next one's data ahead (the registers do not hold it)
// nor a deeper pipeline shortened that.  Aligned 256 x 256 tiles fill the register file: 16 registers of a lane are spilled (68 bytes).
// Calls in a row: 262144 x 512 x 512 f16 with silu and residual 242 us (3.3 TB/s of its 806 MB), 1024 x 40961 x 512 bf16 72 us (595
// TFLOP/s; in a captured graph 63, of which 6 are the odd column's: 57 with 40960), 4096 x 2048 x 1024 bf16 with gelu 23.6 us in a graph
// (728 TFLOP/s), 30001 x 768 x 512 in 37 groups 45 us under the profiler, fp32 4096^3 1.07 to 1.15 ms (120 to 128 TFLOP/s of the
// library's 141).
template <typename T, typename S, bool DMA> __global__ __launch_bounds__(S::NT, S::WAVES) void pj_forward_kernel(FwdArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef Product<T, false, false, S, DMA> P;
    constexpr int V = 16 / sizeof(T);
    f32x4 acc[S::MI][S::MJ];
    P p;
    Tile t;
    if (!next_tile(a.rows, blockIdx.x, a.n_col_tiles, S::BI, S::BJ, t)) return;
    p.A.base = (const T*)a.x; p.A.order = a.rows.order; p.A.ld = a.ldx; p.A.row0 = t.begin; p.A.rows = t.end - t.begin; p.A.klen = a.K; p.A.cols = 0;
    p.B.base = (const T*)a.w + (t.live ? (int64_t)t.g * a.wg : 0); p.B.order = nullptr; p.B.ld = a.ldw; p.B.row0 = t.c0; p.B.rows = a.N - t.c0; p.B.klen = a.K; p.B.cols = 0;
    p.start(t.live ? a.K : 0, lds);
    const int col = (threadIdx.x >> 6) / S::WI * (S::BJ / S::WJ) + (int)(threadIdx.x & 63) % (S::MJ * 16 / V) * V;
    const int left = a.N - t.c0 - col;
    const int64_t at = (int64_t)t.g * a.N + t.c0 + col;
    const bool has_bias = a.bias && t.live, has_slope = a.slope && t.live;
    LaneParam<T> bias, slope;
    if (has_bias) bias.load(a.bias, a.bias_f32, at, left);
    if (has_slope) slope.load(a.slope, a.slope_f32, at, left);
    p.run(lds, acc);
    auto finish = [&](auto f) {
        f.resid = (const T*)a.resid; f.z = (T*)a.z; f.y = (T*)a.y; f.ldr = a.ldr; f.N = a.N; f.order = a.rows.order;
        f.begin = t.begin; f.count = t.end - t.begin; f.n0 = t.c0; f.left = left; f.act = a.act; f.live = t.live;
        bias.get(has_bias, a.bias_f32, f.bi);
        slope.get(has_slope, a.slope_f32, f.sl);
        tile_emit<T, S>(acc, lds, f);
    };
    switch (t.live && t.c0 + S::BJ <= a.N ? a.act : -1) {
#define PJ_CASE(A) \
    case A: finish(ForwardEmit<T, A, true>()); break;
        PJ_CASE(PJ_NONE) PJ_CASE(PJ_RELU) PJ_CASE(PJ_PRELU) PJ_CASE(PJ_SILU) PJ_CASE(PJ_GELU_TANH)
#undef PJ_CASE
        default: finish(ForwardEmit<T, 0, false>());
    }
}

// The same for few rows (tiles of 16 MT): a workgroup takes 16 columns, its eight waves every eighth group of k (K = 512 is one
// trip to memory), and their sums meet in LDS, added in a fixed order.  Bound by the latency of one trip to memory (1 x 512 x 512
// f16: 3.2 us in a captured graph, on tiles 4.9), or by W's bytes (1 x 40961 x 512: 9.6 us, 4.4 TB/s): a column's weights are read once,
// straight into MFMA operands, in pieces of 64 bytes of sixteen rows whose neighbours the other waves take.
template <typename T, int MT> __global__ __launch_bounds__(512) void pj_few_rows_kernel(FwdArgs a) {
    typedef typename Elem<T>::Frag Frag;
    constexpr int KG = Elem<T>::KG, EPC = Elem<T>::EPC, U = 4, NW = 8;
    __shared__ float red[NW][MT][16][17];
    const int ct = blockIdx.x % a.n_col_tiles, rt = blockIdx.x / a.n_col_tiles;
    int g, begin, end;
    if (!row_tile(a.rows, rt, 16 * MT, g, begin, end)) return;
    const bool live = g < a.rows.G;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4, n0 = ct * 16;
    if (live) {
        f32x4 acc[MT];
        const T* xr[MT];
        const T* wr = (const T*)a.w + (int64_t)g * a.wg + (int64_t)(n0 + m < a.N ? n0 + m : a.N - 1) * a.ldw + q * EPC;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
            acc[i] = zero;
            const int at = begin + 16 * i + m < end ? begin + 16 * i + m : end - 1;
            xr[i] = (const T*)a.x + (int64_t)(a.rows.order ? a.rows.order[at] : at) * a.ldx + q * EPC;
        }
        for (int k0 = wave * KG; k0 < a.K; k0 += NW * KG * U) {
            Frag w[U], x[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * NW * KG, left = a.K - k - q * EPC;
                w[u] = load_chunk<T>(wr + k, left);
#pragma unroll
                for (int i = 0; i < MT; ++i) x[u][i] = load_chunk<T>(xr[i] + k, left);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i] = pj_mma<T>(w[u], x[u][i], acc[i]);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave][i][m][4 * q + e] = acc[i][e];
    }
    __syncthreads();
    const int c = threadIdx.x & 15, r = (threadIdx.x >> 4) & 15, n = n0 + c;
    if (n >= a.N) return;
    float bi = 0.0f, sl = 0.0f;
    if (live && a.bias) bi = a.bias_f32 ? ((const float*)a.bias)[(int64_t)g * a.N + n] : (float)((const T*)a.bias)[(int64_t)g * a.N + n];
    if (live && a.slope) sl = a.slope_f32 ? ((const float*)a.slope)[(int64_t)g * a.N + n] : (float)((const T*)a.slope)[(int64_t)g * a.N + n];
    for (int i = threadIdx.x >> 8; i < MT; i += 2) {
        const int at = begin + 16 * i + r;
        if (at >= end) continue;
        const int64_t row = a.rows.order ? a.rows.order[at] : at;
        float v = 0.0f;
        if (live) {
            v = ((red[0][i][r][c] + red[1][i][r][c]) + (red[2][i][r][c] + red[3][i][r][c])) +
                ((red[4][i][r][c] + red[5][i][r][c]) + (red[6][i][r][c] + red[7][i][r][c])) + bi;
            if (a.z) ((T*)a.z)[row * a.N + n] = (T)v;
            v = pj_act<T>(a.act, v, sl);
        }
        if (a.resid) v += (float)((const T*)a.resid)[row * a.ldr + n];
        ((T*)a.y)[row * a.N + n] = (T)v;
    }
}

// ---- backward: everything the products read lies in rows of whole aligned chunks, in list order

// dx = dz W, scattered back to the rows.  W is read as it lies (its rows are the contraction): the fragments come out of LDS through
// the transposing read.  4096 x 1024 x 2048 bf16 26 us (660 TFLOP/s; the library's plain product 28.6).
struct DxArgs {
    RowArgs rows;
    const void *dz, *w;
    void* dx;
    int64_t lddz, ldw, wg;
    int K, Kp, N, Np, n_col_tiles;      // Np, Kp: columns of dz and W, zeros past N and K
};
template <typename T, typename S> __device__ __forceinline__ void dx_tile(const DxArgs& a, unsigned block, char* lds) {
    typedef Product<T, false, true, S, true> P;
    struct Emit {
        struct Pre {};
        const DxArgs& a;
        Tile t;
        __device__ __forceinline__ int row(int i) const { return t.begin + i < t.end ? (a.rows.order ? a.rows.order[t.begin + i] : t.begin + i) : -1; }
        __device__ __forceinline__ Pre pre(int, int) const { return {}; }
        __device__ __forceinline__ void emit(int row, int j, Pre, float (&v)[16 / sizeof(T)]) const {
            const int left = a.K - t.c0 - j;
            if (row < 0 || left <= 0) return;
            typename Elem<T>::Frag o;
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(T); ++e) o[e] = (T)v[e];
            store_chunk<T>((T*)a.dx + (int64_t)row * a.K + t.c0 + j, left, o);
        }
    };
    f32x4 acc[S::MI][S::MJ];
    P p;
    Tile t;
    if (!next_tile(a.rows, block, a.n_col_tiles, S::BI, S::BJ, t)) return;
    p.A.base = (const T*)a.dz; p.A.order = nullptr; p.A.ld = a.lddz; p.A.row0 = t.begin; p.A.rows = t.end - t.begin; p.A.klen = a.Np; p.A.cols = 0;
    p.B.base = (const T*)a.w + (t.live ? (int64_t)t.g * a.wg : 0) + t.c0; p.B.order = nullptr; p.B.ld = a.ldw; p.B.row0 = 0; p.B.rows = 0; p.B.klen = a.N; p.B.cols = a.Kp - t.c0;
    p.start(t.live ? a.Np : 0, lds);
    p.run(lds, acc);
    tile_emit<T, S>(acc, lds, Emit{a, t});
}
template <typename T, typename S> __global__ __launch_bounds__(S::NT, S::WAVES) void pj_dx_kernel(DxArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    dx_tile<T, S>(a, blockIdx.x, lds);
}

// dW[g] = sum over the group's rows of dz^T x: both operands k-major.  Several workgroups share the rows of a tile; what is not
// the whole sum is left in fp32 and added in order by pj_finish_kernel.  Without groups: `splits` shares of the rows, partial sums
// [split][N][K].  With groups: pieces of about so many rows, made from the groups' sizes on the device (a group may hold any part of
// the batch), equal ones of a group so that none is a remainder (with remainders 16 groups of about 512 rows, pieces of 512: the whole
// backward pass 60 us, 53 without); a group of one piece, or none, is written at once, the pieces of the others are numbered through.
// By itself 2048 x 1024 x 4096 bf16 25 us with 5 for the joining (the library's plain product 39).
struct DwArgs {
    RowArgs rows;
    const void *dz, *x;
    void* dw;                   // T [G][N][K]
    float* part;                // [splits or pieces][N][K]
    const int4* pieces;         // (group, first list entry, end, number among the partial sums or -1); group -1: unused entry
    int64_t lddz, ldx;
    int K, Kp, N, Np, n_ti, n_tj, splits;
};
struct PieceArgs {
    const int* offsets;
    int4* pieces;               // [n_pieces]
    int* slots;                 // [G + 1]: a group's first partial sum
    int G, rows, n_pieces;      // rows: of a piece, up to half as many more
    unsigned blocks;            // 1, or 0: no groups
};
template <typename O> struct DwEmit {
    struct Pre {};
    O* out;
    int N, K, n0, k0;
    __device__ __forceinline__ int row(int i) const { return n0 + i; }
    __device__ __forceinline__ Pre pre(int, int) const { return {}; }
    __device__ __forceinline__ void emit(int n, int j, Pre, float (&v)[16 / sizeof(O)]) const {
        const int left = K - k0 - j;
        if (n >= N || left <= 0) return;
        typename Elem<O>::Frag o;
#pragma unroll
        for (int e = 0; e < 16 / (int)sizeof(O); ++e) o[e] = (O)v[e];
        store_chunk<O>(out + (int64_t)n * K + k0 + j, left, o);
    }
};
template <typename T, typename S> __device__ __forceinline__ void dw_tile(const DwArgs& a, unsigned block, unsigned share, char* lds) {
    int ti, tj;
    if (!tile_of_block(block, a.n_ti, a.n_tj, ti, tj)) return;
    int begin = 0, end = a.rows.M, g = 0, slot = -1;
    if (a.pieces) {
        const int4 e = a.pieces[share];
        if (e.x < 0) return;
        g = e.x; begin = e.y; end = e.z; slot = e.w;
    } else if (a.splits > 1) {                                      // whole steps per split
        const int step = S::KS * Elem<T>::KG, steps = (end + step - 1) / step;
        const int64_t per = (int64_t)((steps + a.splits - 1) / a.splits) * step, b0 = share * per;
        begin = b0 < end ? (int)b0 : end;
        end = b0 + per < end ? (int)(b0 + per) : end;
        slot = share;
    }
    const int n0 = ti * S::BI, k0 = tj * S::BJ;
    typedef Product<T, true, true, S, true> P;
    f32x4 acc[S::MI][S::MJ];
    P p;
    p.A.base = (const T*)a.dz + n0; p.A.order = nullptr; p.A.ld = a.lddz; p.A.row0 = begin; p.A.rows = 0; p.A.klen = end - begin; p.A.cols = a.Np - n0;
    p.B.base = (const T*)a.x + k0; p.B.order = nullptr; p.B.ld = a.ldx; p.B.row0 = begin; p.B.rows = 0; p.B.klen = end - begin; p.B.cols = a.Kp - k0;
    p.start(end - begin, lds);
    p.run(lds, acc);
    const int64_t plane = (int64_t)a.N * a.K;
    if (slot >= 0) {
        DwEmit<float> f = {a.part + slot * plane, a.N, a.K, n0, k0};
        tile_emit<float, S>(acc, lds, f);
    } else {
        DwEmit<T> f = {(T*)a.dw + (int64_t)g * plane, a.N, a.K, n0, k0};
        tile_emit<T, S>(acc, lds, f);
    }
}
// Both gradients' products in one launch: neither waits for the other, and one's last tiles run beside the other's (4096 x 2048 x 1024
// bf16 44 us, 52 one after the other; 8192 rows of 16 groups, 1024 x 512: 34 and 45; 1000 x 301 x 500 fp32 15.4 and 21).
// dx first, whose tiles' sums (over N) are the longer ones more often than not: fp32 2999 x 513 x 250 41 us in all, 45 behind dW.
struct GradArgs {
    DxArgs dx;
    DwArgs dw;
    unsigned dx_blocks, dw_blocks;          // dx's, then those of every share of dW: multiples of 8 (tile_of_block)
};
template <typename T, typename S> __global__ __launch_bounds__(S::NT, S::WAVES) void pj_grads_kernel(GradArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if (blockIdx.x < a.dx_blocks) {
        dx_tile<T, S>(a.dx, blockIdx.x, lds);
    } else {
        const unsigned b = blockIdx.x - a.dx_blocks, share = b / a.dw_blocks;
        dw_tile<T, S>(a.dw, b - share * a.dw_blocks, share, lds);
    }
}

// dz = dy act'(z) in list order and, per row tile, the column sums of dz and of dy min(z, 0).  A workgroup takes one row tile x
// `lpr` 16-byte pieces of columns (lpr lanes side by side, a power of two up to 16, so that narrow pieces make many workgroups;
// 256 / lpr rows at a time); four rows per lane are requested together.  Bound by HBM and, with a sigmoid, by the vector ALU
// nearly as much: 4096 x 2048 bf16 with gelu 11 us, 4.6 TB/s of dy and z in and dz out (27 us with a workgroup per 256 columns and
// a guard around every access).
struct DzArgs {
    RowArgs rows;
    const void *dy, *z, *slope;
    void* dz;                   // [M][Np], zeros from column N on; nullptr: dz = dy, only the sums are wanted
    float *part_b, *part_s;     // [tiles][N], nullptr where not wanted
    int64_t lddy;
    int N, Np, act, slope_f32, tile_rows, n_col_tiles, lpr_log2;
};
// ACT: the activation; FULL: every piece is whole (N = Np)
template <typename T, int ACT, bool FULL> __device__ __forceinline__ void dz_rows(const DzArgs& a, int g, int begin, int end, int n, int sub, int nsub,
                                                                                float (&sb)[Elem<T>::EPC], float (&ss)[Elem<T>::EPC]) {
    typedef typename Elem<T>::Frag Frag;
    constexpr int V = Elem<T>::EPC, U = 4;
    const int have = FULL ? V : a.N - n;
    LaneParam<T> slope;
    float sl[V];
    if (ACT == PJ_PRELU) slope.load(a.slope, a.slope_f32, (int64_t)g * a.N + n, have);
    for (int at0 = begin + sub; at0 < end; at0 += nsub * U) {
        Frag dy[U], z[U];
        int row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = at0 + u * nsub;
            row[u] = at < end ? at : at0;                           // rows past the end repeat the first, unused
        }
        if (a.rows.order) {
#pragma unroll
            for (int u = 0; u < U; ++u) row[u] = a.rows.order[row[u]];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            dy[u] = load_chunk<T>((const T*)a.dy + (int64_t)row[u] * a.lddy + n, have);
            if (ACT != PJ_NONE) z[u] = load_chunk<T>((const T*)a.z + (int64_t)row[u] * a.N + n, have);
        }
        if (ACT == PJ_PRELU) slope.get(true, a.slope_f32, sl);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = at0 + u * nsub;
            if (at >= end) continue;
            Frag d = dy[u];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float y = (float)dy[u][e], zv = ACT != PJ_NONE ? (float)z[u][e] : 0.0f;
                const float dz = pj_dz<T>(ACT, y, zv, sl[e]);
                sb[e] += dz;
                if (ACT == PJ_PRELU) ss[e] += zv > 0.0f ? 0.0f : y * zv;
                if (ACT != PJ_NONE) d[e] = (T)dz;
            }
            if (a.dz) *reinterpret_cast<Frag*>((T*)a.dz + (int64_t)at * a.Np + n) = d;
        }
    }
}
template <typename T> __device__ __forceinline__ void dz_tile(const DzArgs& a, unsigned block, float (&sums)[256][Elem<T>::EPC + 1]) {
    constexpr int V = Elem<T>::EPC;
    const int ct = block % a.n_col_tiles, rt = block / a.n_col_tiles;
    int g, begin, end;
    if (!row_tile(a.rows, rt, a.tile_rows, g, begin, end) || g >= a.rows.G) return;     // the same for the whole workgroup
    const int lpr = 1 << a.lpr_log2, lane = threadIdx.x & (lpr - 1), sub = threadIdx.x >> a.lpr_log2, nsub = 256 >> a.lpr_log2;
    const int n = (ct * lpr + lane) * V;
    float sb[V], ss[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sb[e] = ss[e] = 0.0f;
    if (n < a.Np) {
        const bool full = a.N == a.Np;
        switch (a.act) {
#define PJ_CASE(A)                                                               \
    case A:                                                                      \
        if (full) dz_rows<T, A, true>(a, g, begin, end, n, sub, nsub, sb, ss);   \
        else dz_rows<T, A, false>(a, g, begin, end, n, sub, nsub, sb, ss);       \
        break;
            PJ_CASE(PJ_NONE) PJ_CASE(PJ_RELU) PJ_CASE(PJ_PRELU) PJ_CASE(PJ_SILU) PJ_CASE(PJ_GELU_TANH)
#undef PJ_CASE
        }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* part = which == 0 ? a.part_b : a.part_s;
        if (!part) continue;                                        // the same for the whole workgroup
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) sums[threadIdx.x][e] = which == 0 ? sb[e] : ss[e];
        __syncthreads();
        for (int c = threadIdx.x; c < lpr * V; c += 256) {
            const int col = ct * lpr * V + c;
            if (col >= a.N) continue;
            float v = 0.0f;
            for (int s = 0; s < nsub; ++s) v += sums[(s << a.lpr_log2) + c / V][c % V];
            part[(int64_t)rt * a.N + col] = v;
        }
    }
}
// rows of `src` (through `order`, or row r of group r / per_group) to rows of whole aligned chunks, zeros past `cols`
struct PackArgs {
    const void* src;
    void* dst;
    const int* order;
    const int* count;           // rows to copy (device), nullptr: `rows`
    int64_t ld, gs;
    int rows, per_group, cols, cpr;     // cpr: chunks per row of dst
    unsigned blocks;            // workgroups that share the rows, 0: nothing to copy
};
template <typename T> __device__ __forceinline__ void pack_rows(const PackArgs& a, unsigned block) {
    typedef typename Elem<T>::Frag Frag;
    const int64_t n = (int64_t)(a.count ? *a.count : a.rows) * a.cpr, stride = (int64_t)a.blocks * 256;
    for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < n; i += stride) {
        const int r = (int)(i / a.cpr), c = (int)(i - (int64_t)r * a.cpr) * Elem<T>::EPC;
        const T* p = (const T*)a.src;
        if (a.order) p += (int64_t)a.order[r] * a.ld;
        else if (a.per_group) p += (int64_t)(r / a.per_group) * a.gs + (int64_t)(r % a.per_group) * a.ld;
        else p += (int64_t)r * a.ld;
        reinterpret_cast<Frag*>(a.dst)[i] = load_chunk<T>(p + c, a.cols - c);
    }
}
// Everything the gradients' products wait for, in one launch: dz and the column sums, x in list order, W in aligned rows.
struct PrepArgs {
    DzArgs dz;
    PackArgs x, w;
    PieceArgs pieces;
    unsigned dz_blocks;
};
// exclusive sums over the workgroup's values; returns this thread's, `total` to every thread
__device__ __forceinline__ int block_scan(int v, int* tmp, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
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
    total = 0;
    for (int w = 0; w < nw; ++w) {
        base += w < wave ? tmp[w] : 0;
        total += tmp[w];
    }
    return base + x - v;
}
// cuts the groups' rows into pieces, a group into equal ones (one workgroup)
__device__ __forceinline__ void cut_pieces(const PieceArgs& a, int* tmp) {
    int base = 0, sbase = 0;
    for (int g0 = 0; g0 < a.G; g0 += 256) {
        const int g = g0 + threadIdx.x;
        const int first = g < a.G ? a.offsets[g] : 0, end = g < a.G ? a.offsets[g + 1] : 0;
        const int rows = end - first, n = g < a.G ? (rows > a.rows + a.rows / 2 ? (rows + a.rows / 2) / a.rows : 1) : 0, multi = n > 1 ? n : 0;
        int total, stotal;
        const int at = base + block_scan(n, tmp, total), slot = sbase + block_scan(multi, tmp, stotal);
        if (g < a.G) a.slots[g] = slot;
        const int len = n > 1 ? (rows + n - 1) / n : rows;
        for (int i = 0; i < n; ++i) {
            const int64_t b = (int64_t)i * len, e = b + len;
            int4 v = {g, first + (int)(b < rows ? b : rows), first + (int)(e < rows ? e : rows), multi ? slot + i : -1};
            a.pieces[at + i] = v;
        }
        base += total;
        sbase += stotal;
    }
    if (threadIdx.x == 0) a.slots[a.G] = sbase;
    for (int i = base + threadIdx.x; i < a.n_pieces; i += 256) {
        const int4 none = {-1, 0, 0, -1};
        a.pieces[i] = none;
    }
}
template <typename T> __global__ __launch_bounds__(256) void pj_prep_kernel(PrepArgs a) {
    __shared__ float sums[256][Elem<T>::EPC + 1];
    unsigned b = blockIdx.x;
    if (b < a.pieces.blocks) {
        cut_pieces(a.pieces, reinterpret_cast<int*>(sums));
        return;
    }
    b -= a.pieces.blocks;
    if (b < a.dz_blocks) dz_tile<T>(a.dz, b, sums);
    else if (b < a.dz_blocks + a.x.blocks) pack_rows<T>(a.x, b - a.dz_blocks);
    else pack_rows<T>(a.w, b - a.dz_blocks - a.x.blocks);
}

// The sums that the passes before left in parts, in one launch:
//   workgroups 0 .. n_join:  dw[e] = sum over splits of part[s][e], s ascending; with groups dw[g][e] = sum over the group's
//                            pieces, for groups of more than one (a workgroup belongs to one group, join_each to each);
//   the others:              out[g][n] = sum of part[t][n] over the group's tiles, for bias and slope: 16 waves take every sixteenth
//                            tile of 64 columns, their sums are added in order.
// 4 us where only the latter is to do, 7 us with four partial sums of 2048 x 1024.  One workgroup for 64 columns' sums, whatever the
// rows: with 262144 of them and 40 columns (4096 tiles' sums, and 128 of dW's shares) 39 us bf16, 47 fp32.
struct FinishArgs {
    const float* dw_part;
    void* dw;
    int64_t n_dw;               // N K
    const int* slots;           // nullptr: no groups
    int splits;
    unsigned n_join, join_each;
    const float* part[2];
    void* out[2];
    int out_f32[2];
    const int* tile_offsets;
    int n_tiles, N, n_col_tiles, both;      // both: bias and slope, else the one that is there
};
template <typename T> __global__ __launch_bounds__(1024) void pj_finish_kernel(FinishArgs a) {
    __shared__ float sums[16][64];
    if (blockIdx.x < a.n_join) {
        const unsigned g = blockIdx.x / a.join_each;
        const int64_t e = ((int64_t)(blockIdx.x - g * a.join_each) * 1024 + threadIdx.x) * 4;
        const int first = a.slots ? a.slots[g] : 0, end = a.slots ? a.slots[g + 1] : a.splits;
        if (first == end || e >= a.n_dw) return;
        float v[4] = {0, 0, 0, 0};
        const int left = a.n_dw - e < 4 ? (int)(a.n_dw - e) : 4;
#pragma unroll 4
        for (int s = first; s < end; ++s) {
            float o[4];
            load_four<float>(a.dw_part + (int64_t)s * a.n_dw + e, left, o);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += o[i];
        }
        store_four<T>((T*)a.dw + g * a.n_dw + e, left, v);
        return;
    }
    unsigned b = blockIdx.x - a.n_join;
    int which = a.out[0] ? 0 : 1;
    if (a.both) {
        which = b & 1;
        b >>= 1;
    }
    const int ct = b % a.n_col_tiles, g = b / a.n_col_tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = ct * 64 + lane;
    const int t0 = a.tile_offsets ? a.tile_offsets[g] : 0, t1 = a.tile_offsets ? a.tile_offsets[g + 1] : a.n_tiles;
    float v = 0.0f;
    if (n < a.N) {
#pragma unroll 4
        for (int t = t0 + wave; t < t1; t += 16) v += a.part[which][(int64_t)t * a.N + n];
    }
    sums[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && n < a.N) {
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; ++w) v += sums[w][lane];
        if (a.out_f32[which]) ((float*)a.out[which])[(int64_t)g * a.N + n] = v;
        else ((T*)a.out[which])[(int64_t)g * a.N + n] = (T)v;
    }
}
// ---- rows by group: a stable counting sort --------------------------------------------------------------------------
// key = id, or G where id is outside [0, G).  A workgroup of NW waves owns NW * 64 KEYS consecutive rows, a wave 64 KEYS of them,
// kept as KEYS keys per lane: four, or eight where that makes it one workgroup (and one launch).  Eight waves, whose barriers and
// sums over waves are short (9 rows 4.2 us, with sixteen 5.3; 12000 rows of 16 groups 10.0 and 12.5; 30001 of 37 11.0 and 13.3), but
// sixteen for very many rows, whose workgroups' counts are added up (1000000 rows of 100 groups 33 us, with eight 41).  Lanes with the same key find each other by ballots over the
// key's bits, so a row's rank among its wave's rows of the key is the wave's running count plus the equal lanes below: no atomics,
// and the order does not depend on timing.  One launch for one workgroup; else the counts of all workgroups first.  Bound by
// latency: a launch alone is two of the 4.2 us.
constexpr int GR_MAX_GROUPS = 4096;
constexpr int GR_WIDE_KEYS = 1025;          // up to this many keys eight and sixteen waves' counters fit in LDS, beyond it four waves'
constexpr int GR_MANY_ROWS = 1 << 18;       // sixteen waves beyond this
constexpr int GR_INLINE_SCAN = 8192;        // counters up to which every workgroup adds the others' counts itself
struct GroupArgs {
    const void* ids;
    int ids64, M, G, nb, bits, tile_rows, n_tiles, scanned;
    int* counts;                // [nb][G + 1]: a workgroup's rows of a key (scanned: list entries of the key before it), then totals
    int *order, *offsets, *tile_offsets;    // [M], [G + 1], [G + 2]
    int4* tiles;
};
// ranks the wave's rows among its rows of the same key; cnt[key] ends as the count
template <int KEYS> __device__ __forceinline__ void group_rank(const GroupArgs& a, int64_t first, int* cnt, int lane, int (&key)[KEYS], int (&rank)[KEYS]) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        const int64_t row = first + 64 * i + lane;
        key[i] = -1;
        if (row < a.M) {
            const int64_t id = a.ids64 ? ((const int64_t*)a.ids)[row] : ((const int*)a.ids)[row];
            key[i] = id >= 0 && id < a.G ? (int)id : a.G;
        }
    }
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        const bool in = key[i] >= 0;
        unsigned long long same = __ballot(in);
        if (!same) break;
        for (int b = 0; b < a.bits; ++b) {
            const unsigned long long m = __ballot((key[i] >> b) & 1);
            same &= ((key[i] >> b) & 1) ? m : ~m;
        }
        const int below = __popcll(same & ((1ull << lane) - 1));
        const int at = in ? cnt[key[i]] : 0;
        rank[i] = at + below;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (in && below == 0) cnt[key[i]] = at + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the next rows' lanes read what this row's leader wrote
    }
}
// totals[key] -> every key's first list entry (in place), tofs[key] its first tile; WRITE: offsets, tile_offsets and the tiles
template <bool WRITE> __device__ __forceinline__ void group_tables(const GroupArgs& a, int* totals, int* tofs, int* tmp) {
    const int keys = a.G + 1, nt = blockDim.x;
    int base = 0, tbase = 0;
    for (int k0 = 0; k0 < keys; k0 += nt) {
        const int k = k0 + threadIdx.x;
        const int c = k < keys ? totals[k] : 0, tc = (c + a.tile_rows - 1) / a.tile_rows;
        int tot, ttot = 0, to = 0;
        const int o = base + block_scan(c, tmp, tot);
        if (WRITE) to = tbase + block_scan(tc, tmp, ttot);
        if (k < keys) {
            totals[k] = o;
            if (WRITE) {
                tofs[k] = to;
                a.offsets[k] = o;
                a.tile_offsets[k] = to;
            }
        }
        base += tot;
        tbase += ttot;
    }
    __syncthreads();
    if (!WRITE) return;
    if (threadIdx.x == 0) a.tile_offsets[keys] = tbase;
    for (int t = threadIdx.x; t < a.n_tiles; t += nt) {
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
            e.z = end - first > a.tile_rows ? first + a.tile_rows : end;
        }
        a.tiles[t] = e;
    }
}
// COUNT: a workgroup's counts; else place (the only workgroup, or after the counts, or after pj_group_scan_kernel)
template <int NW, int KEYS, bool COUNT> __global__ __launch_bounds__(64 * NW) void pj_group_kernel(GroupArgs a) {
    extern __shared__ int cnt[];                                    // [NW][keys]; place: + totals[keys], before[keys] (= tofs), not scanned: + counts[nb][keys]
    __shared__ int tmp[NW];
    const int keys = a.G + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nt = 64 * NW;
    int key[KEYS], rank[KEYS];
    const int64_t first = ((int64_t)blockIdx.x * NW + wave) * (64 * KEYS);
    for (int i = threadIdx.x; i < NW * keys; i += nt) cnt[i] = 0;
    __syncthreads();
    group_rank(a, first, cnt + wave * keys, lane, key, rank);
    __syncthreads();
    int* totals = cnt + NW * keys;
    int* before = totals + keys;
    if (COUNT || a.nb == 1) {
        for (int k = threadIdx.x; k < keys; k += nt) {
            int c = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) c += cnt[w * keys + k];
            if (COUNT) a.counts[(int64_t)blockIdx.x * keys + k] = c;
            else totals[k] = c;
        }
        if (COUNT) return;
        __syncthreads();
        group_tables<true>(a, totals, before, tmp);
        __syncthreads();
        for (int k = threadIdx.x; k < keys; k += nt) before[k] = 0;
    } else if (a.scanned) {
        for (int k = threadIdx.x; k < keys; k += nt) {
            totals[k] = a.offsets[k];
            before[k] = a.counts[(int64_t)blockIdx.x * keys + k];
        }
    } else {
        int* all = before + keys;                                   // [nb][keys]
        for (int i = threadIdx.x; i < a.nb * keys; i += nt) all[i] = a.counts[i];
        __syncthreads();
        for (int k = threadIdx.x; k < keys; k += nt) {
            int sum = 0;
            for (int b = 0; b < a.nb; ++b) sum += all[b * keys + k];
            totals[k] = sum;
        }
        __syncthreads();
        if (blockIdx.x == 0) group_tables<true>(a, totals, before, tmp);
        else group_tables<false>(a, totals, before, tmp);
        __syncthreads();
        for (int k = threadIdx.x; k < keys; k += nt) {
            int mine = 0;
            for (int b = 0; b < (int)blockIdx.x; ++b) mine += all[b * keys + k];
            before[k] = mine;
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < keys; k += nt) {                  // counts -> the wave's first list entry of the key
        int at = totals[k] + before[k];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const int c = cnt[w * keys + k];
            cnt[w * keys + k] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
        if (key[i] >= 0) a.order[cnt[wave * keys + key[i]] + rank[i]] = (int)(first + 64 * i + lane);
}
// counts[b][key] -> exclusive sums over b; totals -> tables
__global__ __launch_bounds__(1024) void pj_group_scan_kernel(GroupArgs a) {
    extern __shared__ int cnt[];                                    // totals[keys], tofs[keys]
    __shared__ int tmp[16];
    const int keys = a.G + 1;
    for (int k = threadIdx.x; k < keys; k += 1024) {
        int sum = 0, b = 0;
        for (; b + 8 <= a.nb; b += 8) {
            int c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = a.counts[(int64_t)(b + i) * keys + k];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a.counts[(int64_t)(b + i) * keys + k] = sum;
                sum += c[i];
            }
        }
        for (; b < a.nb; ++b) {
            const int c = a.counts[(int64_t)b * keys + k];
            a.counts[(int64_t)b * keys + k] = sum;
            sum += c;
        }
        cnt[k] = sum;
    }
    __syncthreads();
    group_tables<true>(a, cnt, cnt + keys, tmp);
}

// ---- launchers ------------------------------------------------------------------------------------------------------

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
        hipLaunchKernelGGL(KERNEL, (GRID), dim3(NT), LDS, STREAM, ARGS); \
        FRA_HIP(hipGetLastError());                                                      \
    } while (0)

typedef Shape<256, 256, 2, 4, 2, 2> Huge;       // 16-bit types only
typedef Shape<128, 128, 4, 2, 2, 2> Big;
typedef Shape<64, 64, 2, 2, 2, 3> Small;
typedef Shape<32, 32, 2, 1, 2, 4> Tiny;

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
        FRA_REQUIRE(((uintptr_t)g->tiles & 15) == 0, FRA_ERR_ARG, "%s: the groups' tiles are not 16-byte aligned", what);
        FRA_REQUIRE(d->w_group_stride >= 0, FRA_ERR_ARG, "%s: group stride %lld", what, (long long)d->w_group_stride);
    }
    return FRA_OK;
}
static RowArgs row_args(const fra_linear_desc* d, int tile_rows) {
    RowArgs r;
    const fra_row_groups* g = d->groups;
    r.order = g ? g->order : nullptr;
    r.tiles = g ? (const int4*)g->tiles : nullptr;
    r.tile_offsets = g ? g->tile_offsets : nullptr;
    r.sub = g && g->tile_rows > tile_rows ? g->tile_rows / tile_rows : 1;
    r.n_tiles = g ? g->n_tiles * r.sub : cdiv(d->M, tile_rows);
    r.M = (int)d->M;
    r.G = g ? g->n_groups : 1;
    return r;
}
// a launch's threads are counted in 32 bits
static int check_grid(int64_t blocks, int threads, const char* what) {
    FRA_REQUIRE(blocks <= 4294967295LL / threads, FRA_ERR_ARG, "%s: %lld workgroups of %d are more than one launch", what, (long long)blocks, threads);
    return FRA_OK;
}
// The side of a product's tiles.  256 x 256 moves half the bytes per product of 128 x 128 through the caches (8192 x 8192 x 8192:
// 826 against 977 us) but holds one workgroup per compute unit, so it takes rounds that are nearly full (4096 x 2048 x 1024, half a
// round: 37 against 24 us), and 16-bit operands: fp32 tiles are bound by the matrix cores at any size.  128 from one tile per unit
// on, 64 from half of that on (2999 x 513 x 250 in fp32: 423 tiles of 64 15.5 us, 1598 of 32 21.3), below it 32 (1000 x 301 x 500 is
// 80 tiles of 64 on 256 units).  The columns have to fill the tiles: 256 to seven eighths (262144 x 300 x 512 bf16 161 us on 128 x 128,
// 217 on 256 x 256; 262144 x 512 x 512 219 and 185), 128 to more than half (262144 x 64 x 512 bf16 59 us on 64 x 64; fp32 171, on
// 128 x 128 289), and for fp32, which the matrix cores bound, 64 it is where they are a twentieth fewer (262144 x 130 x 512: 452 us
// against 587).  Rows in groups: at most the table's tiles (`most`).
static int tile_side(int64_t rows, int64_t cols, bool f32, int most = 256) {
    auto tiles = [&](int side) { return (int64_t)cdiv(rows, side) * cdiv(cols, side); };
    const int64_t huge = tiles(256);
    if (most >= 256 && !f32 && cols * 8 >= (int64_t)cdiv(cols, 256) * 256 * 7 && huge >= 512 && huge * 10 >= (huge + 255) / 256 * 256 * 9) return 256;
    if (most >= 128 && cols > 64 && tiles(128) >= 256 && !(f32 && cdiv(cols, 64) * 21 <= cdiv(cols, 128) * 40)) return 128;
    return most >= 64 && tiles(64) >= 128 ? 64 : 32;
}

template <typename T> static bool forward_dma(const fra_linear_desc* d) {
    return dma_ok<T>(d->x, d->ldx, d->K) && dma_ok<T>(d->w, d->ldw | d->w_group_stride, d->K);
}
template <typename T, typename S> static int launch_forward(const fra_linear_desc* d, FwdArgs& a, hipStream_t s) {
    a.n_col_tiles = cdiv(d->N, S::BJ);
    const int64_t blocks = ((int64_t)a.rows.n_tiles * a.n_col_tiles + 7) / 8 * 8;
    if (int rc = check_grid(blocks, S::NT, "fra_linear")) return rc;
    if (forward_dma<T>(d))
        PJ_LAUNCH((pj_forward_kernel<T, S, true>), dim3((unsigned)blocks), S::NT, S::LDS, s, a);
    else
        PJ_LAUNCH((pj_forward_kernel<T, S, false>), dim3((unsigned)blocks), S::NT, S::LDS, s, a);
    return FRA_OK;
}
template <typename T, int MT> static int launch_few_rows(const fra_linear_desc* d, FwdArgs& a, hipStream_t s) {
    a.n_col_tiles = cdiv(d->N, 16);
    const int64_t blocks = (int64_t)a.rows.n_tiles * a.n_col_tiles;
    if (int rc = check_grid(blocks, 512, "fra_linear")) return rc;
    hipLaunchKernelGGL((pj_few_rows_kernel<T, MT>), dim3((unsigned)blocks), dim3(512), 0, s, a);
    FRA_HIP(hipGetLastError());
    return FRA_OK;
}
template <typename T> static int forward_t(const fra_linear_desc* d, void* z, void* y, hipStream_t s) {
    FwdArgs a;
    // Few rows, or so few columns that tiles would be empty, have a kernel of their own.  (Its sums are in another order, so beyond 64
    // rows a value does not depend on the number of rows beside it: there the columns alone decide.)  Times in a captured graph, here and
    // on tiles.  Columns: up to 16, the kernel's own, as far as its launch goes (fp32 262144 x 16 x 512 133 us and 163, x 5 127 and 164,
    // 1000 x 12 x 512 4.3 and 10.1; bf16 55 and 53, 51 and 59, 3.4 and 5.8).  Rows: fp32 up to 64 (64 x 40961 x 512 65 us and 76, 50 x
    // 333 x 512 4.5 and 10.2), 16 bits up to 16 (1 x 40961 x 512 9.6 and 13.2), and up to 64 by what a compute unit fetches, in rows of
    // k: this kernel's tiles are smaller, the others' read a wide product's operands less often (f16 50 x 333 x 512 3.6 us and 5.8; 64 x
    // 4096 x 2048 13.1 and 10.6).  What DMA cannot take stays longer in the tiles' steps, for which it gets two rows of sixteen in advance.
    const int most = d->groups ? d->groups->tile_rows : 256, side = tile_side(d->M, d->N, sizeof(T) == 4, most);
    auto fetched = [&](int bi, int bj) { return ((int64_t)cdiv(d->M, bi) * cdiv(d->N, bj) + 255) / 256 * ((bi + bj) / 16); };
    int mt = 1;                                                     // tiles of 16 rows: as many as fetch least
    for (int i = 2; i <= 4; i *= 2)
        if (16 * i <= most && fetched(16 * i, 16) < fetched(16 * mt, 16)) mt = i;
    const bool few = most == 16 || (d->N <= 16 && d->M <= 1 << 28) || d->M <= (sizeof(T) == 4 ? 64 : 16) ||
                     (d->M <= 64 && fetched(16 * mt, 16) < fetched(side, side) + (forward_dma<T>(d) ? 0 : 2));
    const int bi = few ? 16 * mt : side;
    a.rows = row_args(d, bi);
    a.x = d->x; a.w = d->w; a.bias = d->bias; a.slope = d->slope; a.resid = d->resid; a.z = z; a.y = y;
    a.ldx = d->ldx; a.ldw = d->ldw; a.wg = d->w_group_stride; a.ldr = d->ldr;
    a.K = d->K; a.N = d->N; a.act = d->act; a.bias_f32 = d->bias_dtype == FRA_F32; a.slope_f32 = d->slope_dtype == FRA_F32;
    if (few) {
        if (bi == 16) return launch_few_rows<T, 1>(d, a, s);
        return bi == 32 ? launch_few_rows<T, 2>(d, a, s) : launch_few_rows<T, 4>(d, a, s);
    }
    if constexpr (sizeof(T) == 2) {
        if (bi == 256) return launch_forward<T, Huge>(d, a, s);
    }
    return bi == 128 ? launch_forward<T, Big>(d, a, s) : bi == 64 ? launch_forward<T, Small>(d, a, s) : launch_forward<T, Tiny>(d, a, s);
}

// ---- backward: what goes where in the workspace
struct BackwardPlan {
    bool need_dz, need_sums, pack_x, pack_w;
    int dz_rows, n_tiles, splits, piece_rows, n_pieces, n_parts, dx_side, dw_side, Np, Kp;
    size_t off_dz, off_x, off_w, off_b, off_s, off_part, off_pieces, off_slots, bytes;
};
template <typename T> static BackwardPlan backward_plan_t(const fra_linear_desc* d, bool dx, bool dw, bool db, bool ds) {
    BackwardPlan p;
    const int64_t es = sizeof(T), epc = Elem<T>::EPC;
    const fra_row_groups* g = d->groups;
    const int G = g ? g->n_groups : 1;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    // the products' operands have rows of whole aligned chunks: dz always, a copy of dy included where N does not give it such
    // rows; copies of x (in list order with groups) and W only where theirs are not
    p.Np = (int)((d->N + epc - 1) / epc * epc);
    p.Kp = (int)((d->K + epc - 1) / epc * epc);
    p.need_dz = dx || dw;
    p.need_sums = db || ds;
    p.pack_x = dw && (g || !dma_ok<T>(d->x, d->ldx, d->K));
    p.pack_w = dx && !dma_ok<T>(d->w, d->ldw | d->w_group_stride, d->K);
    p.dz_rows = g ? g->tile_rows : 64;
    p.n_tiles = g ? g->n_tiles : cdiv(d->M, p.dz_rows);
    // dW: enough workgroups to fill the chip twice, each with at least 128 rows; tiles of 64 where tiles of 128 cannot be that many
    // (forward and gradients, 4096 x 2048 x 1024 bf16 87 us, with 64 98; fp32 469 and 476).  How far N and K fill the tiles is not
    // weighed, which narrow products pay for (262144 x 40 x 512 fp32 984 us, with 64 579; bf16 268 and 253; 16384 x 130 x 512 134 and 119, 64
    // and 52).
    // With groups a piece has at most four times the average group's rows as well, so that a batch whose rows are nearly all of one
    // group does not leave the chip to that group's tiles.
    const int64_t share = d->M / G / 128 > 1 ? d->M / G / 128 : 1;
    p.dw_side = (int64_t)cdiv(d->N, 128) * cdiv(d->K, 128) * G * share >= 256 ? 128 : 64;
    const int64_t tiles = (int64_t)cdiv(d->N, p.dw_side) * cdiv(d->K, p.dw_side);
    int64_t sp = (512 + tiles - 1) / tiles;
    // dx's tiles as the forward product's; 64 instead of 32 if that lets them into dW's launch (200 x 300 x 250 bf16: 12.5 us for the
    // whole backward pass, 15.6 apart; fp32 64 x 512 x 512: 19.5 against 19.1)
    p.dx_side = dx && d->M > 0 ? tile_side(d->M, d->K, sizeof(T) == 4, g ? g->tile_rows : 256) : 0;
    if (p.dx_side == 32 && dw && p.dw_side == 64 && (!g || g->tile_rows >= 64)) p.dx_side = 64;
    // where one round of workgroups holds dx and dW together, as many shares of dW as fill it, if they are no longer than dx's sums:
    // 4096 x 1024 x 1024 bf16 36.9 us (dW in twice as many shares 46.4), fp32 165 (202).  A group adds half a tile of rows to dx and
    // half a piece to dW on average (8192 rows of 2 groups, 512 x 512, bf16 33 us, fp32 111; 43 and 124 without; without the allowance
    // 37 and 134)
    if (dw && p.dx_side == p.dw_side) {
        const int side = p.dx_side, half = g ? G / 2 : 0;
        const int64_t dx_tiles = (int64_t)(cdiv(d->M, side) + half) * cdiv(d->K, side);
        const int64_t fit = (256 * (side == 128 ? Big::PER_CU : Small::PER_CU) - dx_tiles) / tiles - half;
        if (fit >= 1 && d->M <= fit * d->N * 5 / 4) sp = fit;
    }
    p.splits = 1;
    p.piece_rows = p.n_pieces = p.n_parts = 0;
    if (dw && g) {
        const int64_t want = sp > (G + 3) / 4 ? sp : (G + 3) / 4;
        int64_t rows = (d->M + want - 1) / want;
        rows = rows < 128 ? 128 : (rows + 63) / 64 * 64;
        p.piece_rows = (int)rows;
        p.n_pieces = (int)(d->M / rows) + G;
        p.n_parts = (int)(2 * d->M / rows);     // a group of n > 1 pieces has more than n / 2 times as many
    } else if (dw) {
        if (sp > share) sp = share;
        if (sp > 1) p.splits = (int)sp;
        if (sp > 1) p.n_parts = (int)sp;
    }
    size_t at = 0;
    p.off_dz = at; if (p.need_dz) at += up((size_t)d->M * p.Np * es);      // also where an aligned dy will serve as dz: it is not known yet
    p.off_x = at; if (p.pack_x) at += up((size_t)d->M * p.Kp * es);
    p.off_w = at; if (p.pack_w) at += up((size_t)G * d->N * p.Kp * es);
    p.off_b = at; if (db) at += up((size_t)p.n_tiles * d->N * 4);
    p.off_s = at; if (ds) at += up((size_t)p.n_tiles * d->N * 4);
    p.off_part = at; at += up((size_t)p.n_parts * d->N * d->K * 4);
    p.off_pieces = at; at += up((size_t)p.n_pieces * 16);
    p.off_slots = at; if (p.n_pieces) at += up((size_t)(G + 1) * 4);
    p.bytes = at;
    return p;
}
static BackwardPlan backward_plan(const fra_linear_desc* d, bool dx, bool dw, bool db, bool ds) {
    return d->dtype == FRA_F32 ? backward_plan_t<float>(d, dx, dw, db, ds) : backward_plan_t<f16>(d, dx, dw, db, ds);
}

template <typename T, typename S> static int launch_dx(DxArgs& a, hipStream_t s) {
    a.n_col_tiles = cdiv(a.K, S::BJ);
    const int64_t blocks = ((int64_t)a.rows.n_tiles * a.n_col_tiles + 7) / 8 * 8;
    if (int rc = check_grid(blocks, S::NT, "fra_linear_backward")) return rc;
    PJ_LAUNCH((pj_dx_kernel<T, S>), dim3((unsigned)blocks), S::NT, S::LDS, s, a);
    return FRA_OK;
}
// dx: its row tiles, or none; shares of dW, or none
template <typename T, typename S> static int launch_grads(GradArgs& a, bool dx, int shares, hipStream_t s) {
    int64_t blocks = 0;
    a.dx_blocks = a.dw_blocks = 0;
    if (dx) {
        a.dx.n_col_tiles = cdiv(a.dx.K, S::BJ);
        blocks = ((int64_t)a.dx.rows.n_tiles * a.dx.n_col_tiles + 7) / 8 * 8;
        if (int rc = check_grid(blocks, S::NT, "fra_linear_backward")) return rc;
        a.dx_blocks = (unsigned)blocks;
    }
    if (shares) {
        a.dw.n_ti = cdiv(a.dw.N, S::BI); a.dw.n_tj = cdiv(a.dw.K, S::BJ);
        const int64_t each = ((int64_t)a.dw.n_ti * a.dw.n_tj + 7) / 8 * 8;
        blocks += each * shares;
        if (int rc = check_grid(blocks, S::NT, "fra_linear_backward")) return rc;
        a.dw_blocks = (unsigned)each;
    }
    PJ_LAUNCH((pj_grads_kernel<T, S>), dim3((unsigned)blocks), S::NT, S::LDS, s, a);
    return FRA_OK;
}
template <typename T>
static int backward_t(const fra_linear_desc* d, const BackwardPlan& plan, const void* z, const void* dy, int64_t lddy, void* dx, void* dw,
                      void* db, void* ds, char* ws, hipStream_t s) {
    BackwardPlan p = plan;
    const fra_row_groups* g = d->groups;
    const int G = g ? g->n_groups : 1;
    // without groups or activation an aligned dy is dz
    if (!g && d->act == PJ_NONE && dma_ok<T>(dy, lddy, d->N)) p.need_dz = false;
    PrepArgs prep = {};
    int64_t prep_blocks = 0;
    if ((p.need_dz || p.need_sums) && d->M > 0) {
        DzArgs& a = prep.dz;
        a.rows = row_args(d, p.dz_rows);
        a.dy = dy; a.z = z; a.slope = d->slope;
        a.dz = p.need_dz ? ws + p.off_dz : nullptr;
        a.part_b = db ? (float*)(ws + p.off_b) : nullptr;
        a.part_s = ds ? (float*)(ws + p.off_s) : nullptr;
        a.lddy = lddy; a.N = d->N; a.Np = p.Np; a.act = d->act; a.slope_f32 = d->slope_dtype == FRA_F32;
        a.tile_rows = p.dz_rows;
        const int pieces = p.Np / Elem<T>::EPC;
        a.lpr_log2 = 0;
        while (a.lpr_log2 < 4 && (1 << a.lpr_log2) < pieces) ++a.lpr_log2;
        a.n_col_tiles = cdiv(pieces, 1 << a.lpr_log2);
        prep_blocks = (int64_t)a.rows.n_tiles * a.n_col_tiles;
        if (int rc = check_grid(prep_blocks, 256, "fra_linear_backward")) return rc;
        prep.dz_blocks = (unsigned)prep_blocks;
    }
    auto pack_blocks = [](int64_t rows, int cpr) { const int64_t b = (rows * cpr + 255) / 256; return (unsigned)(b < 2048 ? b : 2048); };
    if (p.pack_x && d->M > 0) {
        PackArgs& k = prep.x;
        k.src = d->x; k.dst = ws + p.off_x; k.order = g ? (const int*)g->order : nullptr; k.count = g ? g->offsets + G : nullptr;
        k.ld = d->ldx; k.rows = (int)d->M; k.cols = d->K; k.cpr = p.Kp / Elem<T>::EPC;
        k.blocks = pack_blocks(d->M, k.cpr);
        prep_blocks += k.blocks;
    }
    if (p.pack_w && d->M > 0) {
        PackArgs& k = prep.w;
        FRA_REQUIRE((int64_t)G * d->N <= 2147483647LL, FRA_ERR_ARG, "fra_linear_backward: %d matrices of %d rows", G, d->N);
        k.src = d->w; k.dst = ws + p.off_w; k.ld = d->ldw; k.gs = d->w_group_stride;
        k.rows = G * d->N; k.per_group = d->N; k.cols = d->K; k.cpr = p.Kp / Elem<T>::EPC;
        k.blocks = pack_blocks(k.rows, k.cpr);
        prep_blocks += k.blocks;
    }
    if (p.n_pieces) {
        PieceArgs& k = prep.pieces;
        k.offsets = g->offsets; k.pieces = (int4*)(ws + p.off_pieces); k.slots = (int*)(ws + p.off_slots);
        k.G = G; k.rows = p.piece_rows; k.n_pieces = p.n_pieces; k.blocks = 1;
        prep_blocks += 1;
    }
    if (prep_blocks > 0) {
        if (int rc = check_grid(prep_blocks, 256, "fra_linear_backward")) return rc;
        hipLaunchKernelGGL((pj_prep_kernel<T>), dim3((unsigned)prep_blocks), dim3(256), 0, s, prep);
        FRA_HIP(hipGetLastError());
    }
    const void* dz = p.need_dz ? ws + p.off_dz : dy;
    const int64_t lddz = p.need_dz ? p.Np : lddy;
    GradArgs a = {};
    const int dx_side = p.dx_side;
    if (dx_side) {
        a.dx.w = d->w; a.dx.ldw = d->ldw; a.dx.wg = d->w_group_stride;
        if (p.pack_w) {
            a.dx.w = ws + p.off_w; a.dx.ldw = p.Kp; a.dx.wg = (int64_t)d->N * p.Kp;
        }
        a.dx.rows = row_args(d, p.dx_side);
        a.dx.dz = dz; a.dx.dx = dx; a.dx.lddz = lddz; a.dx.K = d->K; a.dx.Kp = p.Kp; a.dx.N = d->N; a.dx.Np = p.Np;
    }
    const int shares = !dw ? 0 : g ? p.n_pieces : p.splits;
    if (dw) {
        a.dw.x = d->x; a.dw.ldx = d->ldx;
        if (p.pack_x) {
            a.dw.x = ws + p.off_x; a.dw.ldx = p.Kp;
        }
        a.dw.rows = row_args(d, 128);
        a.dw.dz = dz; a.dw.dw = dw; a.dw.part = (float*)(ws + p.off_part); a.dw.pieces = g ? (const int4*)(ws + p.off_pieces) : nullptr;
        a.dw.lddz = lddz; a.dw.K = d->K; a.dw.Kp = p.Kp; a.dw.N = d->N; a.dw.Np = p.Np; a.dw.splits = p.splits;
    }
    // dx by its own kernel where its tiles have a side that dW's never have, else with dW if the sides agree
    if constexpr (sizeof(T) == 2) {
        if (dx_side == 256)
            if (int rc = launch_dx<T, Huge>(a.dx, s)) return rc;
    }
    if (dx_side == 32)
        if (int rc = launch_dx<T, Tiny>(a.dx, s)) return rc;
    for (int side = 128; side >= 64; side /= 2) {
        const int sh = p.dw_side == side ? shares : 0;
        if (dx_side != side && !sh) continue;
        if (int rc = side == 128 ? launch_grads<T, Big>(a, dx_side == side, sh, s) : launch_grads<T, Small>(a, dx_side == side, sh, s)) return rc;
    }
    if (p.need_sums || p.n_parts) {
        FinishArgs a = {};
        int64_t blocks = 0;
        if (p.n_parts) {
            a.dw_part = (const float*)(ws + p.off_part); a.dw = dw; a.splits = p.splits;
            a.slots = g ? (const int*)(ws + p.off_slots) : nullptr;
            a.n_dw = (int64_t)d->N * d->K;
            const int64_t each = (a.n_dw + 4095) / 4096;
            blocks = each * G;
            if (int rc = check_grid(blocks, 1024, "fra_linear_backward")) return rc;
            a.join_each = (unsigned)each;
            a.n_join = (unsigned)blocks;
        }
        if (p.need_sums) {
            a.part[0] = (const float*)(ws + p.off_b); a.part[1] = (const float*)(ws + p.off_s);
            a.out[0] = db; a.out[1] = ds;
            a.out_f32[0] = d->bias_dtype == FRA_F32; a.out_f32[1] = d->slope_dtype == FRA_F32;
            a.tile_offsets = g ? (const int*)g->tile_offsets : nullptr;
            a.n_tiles = p.n_tiles; a.N = d->N; a.n_col_tiles = cdiv(d->N, 64); a.both = db && ds;
            blocks += (int64_t)a.n_col_tiles * G * (a.both ? 2 : 1);
            if (int rc = check_grid(blocks, 1024, "fra_linear_backward")) return rc;
        }
        hipLaunchKernelGGL((pj_finish_kernel<T>), dim3((unsigned)blocks), dim3(1024), 0, s, a);
        FRA_HIP(hipGetLastError());
    }
    return FRA_OK;
}

// sixteen waves where they make it one launch, too: 8192 rows of 16 groups 11.4 us, in two 10.1, but a launch costs the host 3
static int group_waves(int64_t M, int n_groups) {
    if (n_groups + 1 > GR_WIDE_KEYS) return 4;
    return M > GR_MANY_ROWS || (M > 4096 && M <= 8192) ? 16 : 8;
}
static int group_keys(int64_t M, int n_groups) {
    const int waves = group_waves(M, n_groups);
    return M > waves * 256 && M <= waves * 512 ? 8 : 4;
}
static int group_blocks(int64_t M, int n_groups) {
    const int per = group_waves(M, n_groups) * 64 * group_keys(M, n_groups);
    return M > per ? cdiv(M, per) : 1;
}
template <int NW, int KEYS> static int launch_groups(GroupArgs& a, hipStream_t s) {
    const int keys = a.G + 1, most = (NW > 4 ? GR_WIDE_KEYS : GR_MAX_GROUPS + 1) * 4, lds = (NW + 2) * keys * 4;
    static std::atomic<uint64_t> done_count{0}, done_place{0};
    if (int rc = raise_lds(pj_group_kernel<NW, KEYS, false>, (NW + 2) * most + GR_INLINE_SCAN * 4, done_place)) return rc;
    if constexpr (KEYS == 4) {
        if (a.nb > 1) {
            if (int rc = raise_lds(pj_group_kernel<NW, KEYS, true>, NW * most, done_count)) return rc;
            hipLaunchKernelGGL((pj_group_kernel<NW, KEYS, true>), dim3(a.nb), dim3(64 * NW), NW * keys * 4, s, a);
            FRA_HIP(hipGetLastError());
            a.scanned = (int64_t)a.nb * keys > GR_INLINE_SCAN;
            if (a.scanned) {
                hipLaunchKernelGGL(pj_group_scan_kernel, dim3(1), dim3(1024), 2 * keys * 4, s, a);
                FRA_HIP(hipGetLastError());
            }
        }
    }
    const int counts = a.nb > 1 && !a.scanned ? a.nb * keys * 4 : 0;
    hipLaunchKernelGGL((pj_group_kernel<NW, KEYS, false>), dim3(a.nb), dim3(64 * NW), lds + counts, s, a);
    FRA_HIP(hipGetLastError());
    return FRA_OK;
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
    FRA_REQUIRE(((uintptr_t)workspace & 15) == 0, FRA_ERR_ARG, "fra_linear_backward: workspace not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (d->dtype == FRA_F32) return backward_t<float>(d, p, preact, dy, lddy, dx, dw, dbias, dslope, ws, s);
    if (d->dtype == FRA_BF16) return backward_t<bf16>(d, p, preact, dy, lddy, dx, dw, dbias, dslope, ws, s);
    return backward_t<f16>(d, p, preact, dy, lddy, dx, dw, dbias, dslope, ws, s);
}

// rows of a tile, by the rows a group has on average: the kernel for few rows below 24, 64 x 64 tiles below 128
int fra_group_tile_rows(int64_t rows, int n_groups) {
    const int64_t average = n_groups >= 1 ? rows / n_groups : rows;
    return average >= 128 ? 128 : average >= 24 ? 64 : 16;
}
int fra_group_tiles(int64_t rows, int n_groups) {
    if (rows < 0 || n_groups < 1 || n_groups > GR_MAX_GROUPS) return 0;
    return (int)(rows / fra_group_tile_rows(rows, n_groups)) + n_groups + 1;
}
int fra_group_rows_workspace_bytes(int64_t rows, int n_groups, size_t* bytes) {
    FRA_REQUIRE(bytes, FRA_ERR_ARG, "fra_group_rows_workspace_bytes: null pointer");
    FRA_REQUIRE(rows >= 0 && rows <= 2147483647LL - 1024 && n_groups >= 1 && n_groups <= GR_MAX_GROUPS, FRA_ERR_ARG,
                "fra_group_rows_workspace_bytes: %lld rows, %d groups (1 to %d)", (long long)rows, n_groups, GR_MAX_GROUPS);
    const int nb = group_blocks(rows, n_groups);
    *bytes = nb > 1 ? (size_t)nb * (n_groups + 1) * 4 : 0;
    return FRA_OK;
}
int fra_group_rows(const void* ids, int ids_are_64bit, const fra_row_groups* g, void* workspace, size_t workspace_bytes, fra_stream stream) {
    FRA_REQUIRE(g, FRA_ERR_ARG, "fra_group_rows: null groups");
    size_t need = 0;
    if (int rc = fra_group_rows_workspace_bytes(g->rows, g->n_groups, &need)) return rc;
    FRA_REQUIRE((ids && g->order) || g->rows == 0, FRA_ERR_ARG, "fra_group_rows: null pointer");
    FRA_REQUIRE(g->offsets && g->tiles && g->tile_offsets, FRA_ERR_ARG, "fra_group_rows: null pointer");
    FRA_REQUIRE(((uintptr_t)g->tiles & 15) == 0 && ((uintptr_t)workspace & 15) == 0, FRA_ERR_ARG, "fra_group_rows: tiles or workspace not 16-byte aligned");
    FRA_REQUIRE(g->tile_rows == fra_group_tile_rows(g->rows, g->n_groups) && g->n_tiles == fra_group_tiles(g->rows, g->n_groups), FRA_ERR_ARG,
                "fra_group_rows: tile_rows / n_tiles are not those of fra_group_tile_rows / fra_group_tiles");
    FRA_REQUIRE(workspace_bytes >= need && (workspace || need == 0), FRA_ERR_WORKSPACE, "fra_group_rows: workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
    GroupArgs a;
    a.ids = ids; a.ids64 = ids_are_64bit != 0; a.M = (int)g->rows; a.G = g->n_groups; a.tile_rows = g->tile_rows; a.n_tiles = g->n_tiles;
    a.nb = group_blocks(a.M, a.G);
    a.counts = (int*)workspace;
    a.order = g->order; a.offsets = g->offsets; a.tile_offsets = g->tile_offsets; a.tiles = (int4*)g->tiles;
    a.scanned = 0;
    a.bits = 0;
    while ((1 << a.bits) < a.G + 1) ++a.bits;
    hipStream_t s = (hipStream_t)stream;
    const int waves = group_waves(a.M, a.G);
    if (group_keys(a.M, a.G) == 8) return waves == 16 ? launch_groups<16, 8>(a, s) : waves == 8 ? launch_groups<8, 8>(a, s) : launch_groups<4, 8>(a, s);
    return waves == 16 ? launch_groups<16, 4>(a, s) : waves == 8 ? launch_groups<8, 4>(a, s) : launch_groups<4, 4>(a, s);
}

}  // extern "C"
