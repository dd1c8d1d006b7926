// Orthogonalising a matrix by Newton-Schulz products: with X = G / |G|_F (transposed if taller than wide),
//     P = X X^T,   Q = b P + c P P,   X <- a X + Q X        `steps` times,
// an odd polynomial of every singular value, a s + b s^3 + c s^5, that drives them towards one.  No counterpart in the reference.
//
// The iteration multiplies small singular values by `a` each step (485 times in five steps of the usual coefficients) and a
// rounding error with them, so sixteen bits are too few between the products.  Every value is held as TWO f16, hi + lo, of
// 2^8 times itself: 22 significant bits down to 2^-10, an absolute step of 2^-32 below, range +-255.  A product is
// hi hi + hi lo + lo hi on the f16 matrix cores (lo lo is below 2^-22), accumulated in fp32: a third of their rate, which is
// over three times that of the fp32 matrix instructions.  Against 64 bits the results are as near as the same iteration with
// fp32 products (512 x 512: 1.4e-6 of the norm, fp32 2.1e-6).
//
// 17 launches for five steps.  Small matrices are bound by the launches' latency (512 x 512 fp32 108 us, 6 us each), large ones by
// the matrix cores: eight of 2048 x 1024 1.09 ms, one of 4096 x 4096 4.0 ms.  P and Q are symmetric: where that saves rounds of
// workgroups, only the tiles of the lower triangle are computed (1.27 and 4.9 ms with all of them).
#include "pj_tile.h"

namespace fra {

constexpr float OR_SCALE = 256.0f;

struct OrthDims {
    int m, n;                   // m <= n after the transposition
    int mp, np;                 // rounded up to 8: row pitches; columns past m / n hold zeros
    int batch, transposed;      // transposed: G and the result are [n][m]
};

// partial sums of squares in fp64 (no overflow, no underflow for any fp32 input): part[batch][gridDim.x]
template <typename T> __global__ __launch_bounds__(256) void orth_norm_kernel(const T* g, int64_t ldg, int64_t bs, int rows, int cols, double* part) {
    __shared__ double sums[4];
    const T* p = g + (int64_t)blockIdx.y * bs;
    double v = 0.0;
    const int64_t nv = (int64_t)rows * ((cols + 3) / 4), cpr = (cols + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nv; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cpr;
        const int c = (int)(i - r * cpr) * 4;
        float x[4];
        load_four<T>(p + r * ldg + c, cols - c, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) v += (double)x[e] * (double)x[e];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

__device__ __forceinline__ void split16(float v, f16& hi, f16& lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}

// G -> X hi / lo [m][np], normalised, transposed if need be, zeros in columns n .. np: 64 x 64 tiles through LDS, four neighbours
// at a time on both sides.  The tile's values are requested before the norm's partial sums are added.
template <typename T> __global__ __launch_bounds__(256) void orth_split_kernel(const T* g, int64_t ldg, int64_t bs, OrthDims d, const double* part,
                                                                              int n_part, f16* xh, f16* xl) {
    __shared__ float tile[64][65];
    __shared__ double factor;                                       // fp64: OR_SCALE / norm leaves fp32's range for a tiny matrix
    const int b = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    const T* p = g + (int64_t)b * bs;
    const int r0 = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4;
    // source rows: X's rows, or (transposed) X's columns
    const int sr0 = d.transposed ? j0 : i0, sc = (d.transposed ? i0 : j0) + c, nr = d.transposed ? d.n : d.m, nc = d.transposed ? d.m : d.n;
    float v[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int r = sr0 + r0 + 16 * q, left = r < nr ? nc - sc : 0;
        load_four<T>(p + (left > 0 ? (int64_t)r * ldg + sc : 0), left, v[q]);
    }
    if (threadIdx.x < 64) {
        double s = 0.0;
        for (int k = threadIdx.x; k < n_part; k += 64) s += part[(int64_t)b * n_part + k];
#pragma unroll
        for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k, 64);
        if (threadIdx.x == 0) factor = s == 0.0 ? 0.0 : (double)OR_SCALE / sqrt(s);        // a matrix of zeros stays one
    }
    __syncthreads();
    const double f = factor;
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = (float)((double)v[q][e] * f);
            if (d.transposed) tile[c + e][r0 + 16 * q] = x;
            else tile[r0 + 16 * q][c + e] = x;
        }
    __syncthreads();
    const int64_t base = (int64_t)b * d.m * d.np;
    if (j0 + c >= d.np) return;                                     // np is a multiple of 8: four neighbours are all in or all out
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int i = r0 + 16 * q;
        if (i0 + i >= d.m) continue;
        vec4<f16>::type hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f16 h, l;
            split16(tile[i][c + e], h, l);
            hi[e] = h;
            lo[e] = l;
        }
        const int64_t at = base + (int64_t)(i0 + i) * d.np + j0 + c;
        *reinterpret_cast<vec4<f16>::type*>(xh + at) = hi;
        *reinterpret_cast<vec4<f16>::type*>(xl + at) = lo;
    }
}

// C = alpha A B^T + beta E (or A B where B is k-major), everything hi / lo f16, a batch of matrices (a die works on one
// or on neighbours: spread over all dies, a matrix's panels went through every L2, 4.8 TB/s of misses)
struct OrthArgs {
    const f16 *ah, *al, *bh, *bl, *eh, *el;
    f16 *ch, *cl;               // nullptr: the last product, into out
    void* out;
    int64_t sa, sb, se, sc, so; // elements between the matrices of a batch
    int lda, ldb, lde, ldc;
    int64_t ldo;
    int I, J, Jp, K;            // C is [I][J], columns J .. Jp are written as zeros
    float alpha, beta;
    int n_row_tiles, n_col_tiles, batch, transposed;
};

// The product of pairs.  TOGETHER: a step brings the hi and lo tiles of both operands, four tiles for the three products (which
// one after the other need six); else the three products are one chain of steps, lo hi, hi lo, hi hi, with half the LDS per step,
// which makes room for tiles of twice the side.
template <bool BK, typename S, bool TOGETHER> struct PairProduct {
    typedef OperandA<f16, false, S> OA;
    typedef OperandB<f16, BK, S> OB;
    static constexpr int NB = S::NB, BUF = (TOGETHER ? 2 : 1) * S::STEP, NLD = (TOGETHER ? 2 : 1) * (OA::NLD + OB::NLD), LDS = NB * BUF;
    static_assert(NB >= 2 && S::KS == 2, "");
    OA A;
    OB B;
    int64_t a_lo, b_lo;         // elements from an operand's hi part to its lo part

    struct PairFrags {
        typename Elem<f16>::Frag ah[S::MI], al[S::MI], bh[S::MJ], bl[S::MJ];
        __device__ __forceinline__ void read(const char* step, int ks, int i0, int j0, int lane) {
#pragma unroll
            for (int mi = 0; mi < S::MI; ++mi) {
                ah[mi] = OA::frag(step, i0 + 16 * mi, ks, lane);
                al[mi] = OA::frag(step + OA::BYTES, i0 + 16 * mi, ks, lane);
            }
#pragma unroll
            for (int mj = 0; mj < S::MJ; ++mj) {
                bh[mj] = OB::frag(step + 2 * OA::BYTES, j0 + 16 * mj, ks, lane);
                bl[mj] = OB::frag(step + 2 * OA::BYTES + OB::BYTES, j0 + 16 * mj, ks, lane);
            }
        }
        __device__ __forceinline__ void mma(f32x4 (&acc)[S::MI][S::MJ]) const {
            // the small parts first
#pragma unroll
            for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
                for (int mj = 0; mj < S::MJ; ++mj) acc[mi][mj] = pj_mma<f16>(bh[mj], al[mi], acc[mi][mj]);
#pragma unroll
            for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
                for (int mj = 0; mj < S::MJ; ++mj) acc[mi][mj] = pj_mma<f16>(bl[mj], ah[mi], acc[mi][mj]);
#pragma unroll
            for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
                for (int mj = 0; mj < S::MJ; ++mj) acc[mi][mj] = pj_mma<f16>(bh[mj], ah[mi], acc[mi][mj]);
        }
    };
    __device__ __forceinline__ void run(int klen, char* lds, f32x4 (&acc)[S::MI][S::MJ]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int i0 = (wave % S::WI) * (S::BI / S::WI), j0 = (wave / S::WI) * (S::BJ / S::WJ);
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
            for (int mj = 0; mj < S::MJ; ++mj) acc[mi][mj] = zero;
        const int each = (klen + OA::KSTEP - 1) / OA::KSTEP, steps = TOGETHER ? each : 3 * each;
        typename OA::Src sa;
        typename OB::Src sb;
        A.init(sa, tid);
        B.init(sb, tid);
        const LdsPtr dst = (LdsPtr)lds + __builtin_amdgcn_readfirstlane(wave) * 1024;
        auto issue = [&](int t, LdsPtr to) {
            if constexpr (TOGETHER) {
                A.issue(sa, t, to, tid);
                A.issue(sa, t, to + OA::BYTES, tid, a_lo);
                B.issue(sb, t, to + 2 * OA::BYTES, tid);
                B.issue(sb, t, to + 2 * OA::BYTES + OB::BYTES, tid, b_lo);
            } else {
                const int part = t >= 2 * each ? 2 : t >= each ? 1 : 0, k = t - part * each;
                A.issue(sa, k, to, tid, part == 0 ? a_lo : 0);
                B.issue(sb, k, to + OA::BYTES, tid, part == 1 ? b_lo : 0);
            }
        };
#pragma unroll
        for (int t = 0; t < NB; ++t)
            if (t < steps) issue(t, dst + t * BUF);
        if constexpr (TOGETHER) run_steps<NB, NLD, BUF, PairFrags>(steps, lds, dst, issue, i0, j0, lane, acc);
        else run_steps<NB, NLD, BUF, Frags<f16, false, BK, S>>(steps, lds, dst, issue, i0, j0, lane, acc);
    }
};

// A piece is eight neighbours of a row (Jp is a multiple of 8: all in or all out).  T: the pairs' (f16) or the result's type
template <typename T> struct OrthEmit {
    static constexpr int V = 16 / sizeof(T);
    struct Pre {
        typename Elem<f16>::Frag h, l;
    };
    const OrthArgs& a;
    int64_t b;
    int i0, j0;
    __device__ __forceinline__ int row(int i) const { return i0 + i < a.I ? i0 + i : -1; }
    __device__ __forceinline__ Pre pre(int i, int j) const {
        Pre p = {};
        if (a.eh && i >= 0 && j0 + j < a.Jp) {
            const int64_t at = b * a.se + (int64_t)i * a.lde + ((j0 + j) & ~7);
            p.h = *reinterpret_cast<const typename Elem<f16>::Frag*>(a.eh + at);
            p.l = *reinterpret_cast<const typename Elem<f16>::Frag*>(a.el + at);
        }
        return p;
    }
    __device__ __forceinline__ void emit(int i, int jt, const Pre& p, float (&v)[V]) const {
        const int j = j0 + jt, from = V == 4 && (j & 4) ? 4 : 0;
        if (i < 0 || j >= a.Jp) return;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float pe = V == 8 ? (float)p.h[e] + (float)p.l[e] : from ? (float)p.h[(e + 4) & 7] + (float)p.l[(e + 4) & 7] : (float)p.h[e] + (float)p.l[e];
            v[e] = j + e < a.J ? a.alpha * v[e] + a.beta * pe : 0.0f;
        }
        if (a.ch) {
            if constexpr (V == 8) {
                typename Elem<f16>::Frag hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f16 h, l;
                    split16(v[e], h, l);
                    hi[e] = h;
                    lo[e] = l;
                }
                *reinterpret_cast<typename Elem<f16>::Frag*>(a.ch + b * a.sc + (int64_t)i * a.ldc + j) = hi;
                *reinterpret_cast<typename Elem<f16>::Frag*>(a.cl + b * a.sc + (int64_t)i * a.ldc + j) = lo;
            }
        } else {
            typename Elem<T>::Frag o;
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = (T)(v[e] * (1.0f / OR_SCALE));
            store_chunk<T>((T*)a.out + b * a.so + (int64_t)i * a.ldo + j, a.J - j, o);
        }
    }
};
// the last product of a transposed matrix: out[j][i], a wave's part turned through LDS, 32 rows at a time, so that a lane writes V
// neighbouring i
template <typename T, typename S, int LDS> __device__ __forceinline__ void orth_emit_transposed(const OrthArgs& a, int64_t b, int i0, int j0, const f32x4 (&acc)[S::MI][S::MJ], char* lds) {
    constexpr int MG = S::MI < 2 ? S::MI : 2, V = 16 / sizeof(T), ROWS = MG * 16, LPR = ROWS / V, RPP = 64 / LPR, PITCH = ROWS + 4;
    static_assert(S::WI * S::WJ * S::MJ * 16 * PITCH * 4 <= LDS && S::MI % MG == 0 && (S::MJ * 16) % RPP == 0, "the waves' parts fit");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = i0 + (wave % S::WI) * (S::BI / S::WI), wj = j0 + (wave / S::WI) * (S::BJ / S::WJ);
    float* strip = reinterpret_cast<float*>(lds) + wave * (S::MJ * 16 * PITCH);
#pragma unroll
    for (int m0 = 0; m0 < S::MI; m0 += MG) {
#pragma unroll
        for (int mi = 0; mi < MG; ++mi) {
            const int i = wi + 16 * (m0 + mi) + (lane & 15);
#pragma unroll
            for (int mj = 0; mj < S::MJ; ++mj) {
                const int jl = 16 * mj + 4 * (lane >> 4), j = wj + jl;
                float h[4] = {0, 0, 0, 0}, l[4] = {0, 0, 0, 0};
                if (i < a.I && j < a.Jp) {
                    load_four<f16>(a.eh + b * a.se + (int64_t)i * a.lde + j, 4, h);
                    load_four<f16>(a.el + b * a.se + (int64_t)i * a.lde + j, 4, l);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    strip[(jl + e) * PITCH + 16 * mi + (lane & 15)] = (a.alpha * acc[m0 + mi][mj][e] + a.beta * (h[e] + l[e])) * (1.0f / OR_SCALE);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int jl = 0; jl < S::MJ * 16; jl += RPP) {
            const int jr = jl + lane / LPR, j = wj + jr, il = (lane % LPR) * V, i = wi + 16 * m0 + il;
            typename Elem<T>::Frag o;
#pragma unroll
            for (int q = 0; q < V; q += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(strip + jr * PITCH + il + q);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[q + e] = (T)x[e];
            }
            if (j < a.J && i < a.I) store_chunk<T>((T*)a.out + b * a.so + (int64_t)j * a.ldo + i, a.I - i, o);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}
// LAST: the last product of the last step, into out (T)
template <typename T, bool BK, bool LAST, typename S, bool TOGETHER> __global__ __launch_bounds__(S::NT) void orth_product_kernel(OrthArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int rt, ct, mat;
    if (!tile_of_block(blockIdx.x, a.n_row_tiles, a.n_col_tiles, rt, ct, a.batch, mat)) return;
    const int i0 = rt * S::BI, j0 = ct * S::BJ;
    const int64_t b = mat;
    f32x4 acc[S::MI][S::MJ];
    PairProduct<BK, S, TOGETHER> p;
    p.A.order = nullptr; p.A.ld = a.lda; p.A.row0 = i0; p.A.rows = a.I - i0; p.A.klen = a.K; p.A.cols = 0; p.A.base = a.ah + b * a.sa;
    p.B.order = nullptr; p.B.ld = a.ldb; p.B.klen = a.K; p.B.base = a.bh + b * a.sb + (BK ? j0 : 0);
    p.B.row0 = BK ? 0 : j0; p.B.rows = BK ? 0 : a.J - j0; p.B.cols = BK ? a.Jp - j0 : 0;
    p.a_lo = a.al - a.ah; p.b_lo = a.bl - a.bh;
    p.run(a.K, lds, acc);
    if constexpr (!LAST) {
        tile_emit<f16, S>(acc, lds, OrthEmit<f16>{a, b, i0, j0});
    } else if (!a.transposed) {
        tile_emit<T, S>(acc, lds, OrthEmit<T>{a, b, i0, j0});
    } else {
        orth_emit_transposed<T, S, PairProduct<BK, S, TOGETHER>::LDS>(a, b, i0, j0, acc, lds);
    }
}

// ---- C = C^T (X X^T, and P P for a symmetric P): the lower triangle's tiles, each handed on to both sides of the diagonal

// hands the transposed results on: f as tile_emit's, whose rows are the tile's columns.  A wave's part, 32 of its rows at a time, goes
// through its own LDS as [column][row].
template <typename S, int LDS, typename F> __device__ __forceinline__ void mirror_emit(const f32x4 (&acc)[S::MI][S::MJ], char* lds, const F& f) {
    constexpr int MG = S::MI < 2 ? S::MI : 2, V = 8, ROWS = MG * 16, LPR = ROWS / V, RPP = 64 / LPR, PITCH = ROWS + 4;
    static_assert(S::WI * S::WJ * S::MJ * 16 * PITCH * 4 <= LDS && S::MI % MG == 0 && (S::MJ * 16) % RPP == 0, "the waves' parts fit");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = (wave % S::WI) * (S::BI / S::WI), wj = (wave / S::WI) * (S::BJ / S::WJ);
    float* strip = reinterpret_cast<float*>(lds) + wave * (S::MJ * 16 * PITCH);
#pragma unroll
    for (int m0 = 0; m0 < S::MI; m0 += MG) {
#pragma unroll
        for (int mi = 0; mi < MG; ++mi)
#pragma unroll
            for (int mj = 0; mj < S::MJ; ++mj)
#pragma unroll
                for (int e = 0; e < 4; ++e) strip[(16 * mj + 4 * (lane >> 4) + e) * PITCH + 16 * mi + (lane & 15)] = acc[m0 + mi][mj][e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int jl = 0; jl < S::MJ * 16; jl += RPP) {
            const int jr = jl + lane / LPR, il = (lane % LPR) * V, row = f.row(wj + jr), col = wi + 16 * m0 + il;
            const typename F::Pre pre = f.pre(row, col);
            float v[V];
#pragma unroll
            for (int q = 0; q < V; q += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(strip + jr * PITCH + il + q);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[q + e] = x[e];
            }
            f.emit(row, col, pre, v);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}
template <typename S, int LDS> __device__ __forceinline__ void symmetric_tile(const OrthArgs& a, int64_t b, int i0, int j0, char* lds) {
    f32x4 acc[S::MI][S::MJ];
    PairProduct<false, S, true> p;
    p.A.order = p.B.order = nullptr; p.A.ld = a.lda; p.B.ld = a.ldb; p.A.klen = p.B.klen = a.K; p.A.cols = p.B.cols = 0;
    p.A.row0 = i0; p.A.rows = a.I - i0; p.A.base = a.ah + b * a.sa;
    p.B.row0 = j0; p.B.rows = a.J - j0; p.B.base = a.bh + b * a.sb;
    p.a_lo = a.al - a.ah; p.b_lo = a.bl - a.bh;
    p.run(a.K, lds, acc);
    tile_emit<f16, S>(acc, lds, OrthEmit<f16>{a, b, i0, j0});
    if (i0 == j0) return;
    __syncthreads();                                                // another wave's part of LDS lies elsewhere now
    mirror_emit<S, LDS>(acc, lds, OrthEmit<f16>{a, b, j0, i0});
}
typedef Shape<128, 128, 4, 2, 2, 2> OrthBig;
typedef Shape<64, 64, 2, 2, 2, 2> OrthSmall;
typedef Shape<64, 64, 4, 2, 2, 2> OrthQuarter;      // of an OrthBig tile, by as many threads
// A die takes consecutive tiles (of one matrix, or of neighbours).  `whole` of them are W's, full rounds of one per compute unit; the
// rest would leave most units idle for a whole round and are cut into four (of 128 x 128 only).
template <typename W> __global__ __launch_bounds__(W::NT) void orth_symmetric_kernel(OrthArgs a, int side, int whole) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int LDS = PairProduct<false, W, true>::LDS;
    const int each = side * (side + 1) / 2, all = each * a.batch, x = blockIdx.x & 7, i = blockIdx.x >> 3;
    const int first = (int)((int64_t)all * x / 8), count = (int)((int64_t)all * (x + 1) / 8) - first;
    const int n_whole = count < whole ? count : whole, at = i < n_whole ? i : n_whole + ((i - n_whole) >> 2), quarter = (i - n_whole) & 3;
    if (at >= count) return;
    const int mat = (first + at) / each, t = first + at - mat * each;
    int r = (int)((__builtin_sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);       // the last r with r (r + 1) / 2 <= t
    while (r > 0 && r * (r + 1) / 2 > t) --r;
    while ((r + 1) * (r + 2) / 2 <= t) ++r;
    const int i0 = r * W::BI, j0 = (t - r * (r + 1) / 2) * W::BI;
    if (i < n_whole) {
        symmetric_tile<W, LDS>(a, mat, i0, j0, lds);
    } else if constexpr (W::BI == 128) {
        static_assert(PairProduct<false, OrthQuarter, true>::LDS <= LDS && OrthQuarter::NT == W::NT, "");
        const int qi = i0 + (quarter >> 1) * 64, qj = j0 + (quarter & 1) * 64;
        if (qi < qj || qi >= a.I) return;                           // above the diagonal, or past the last row (columns are no more)
        symmetric_tile<OrthQuarter, LDS>(a, mat, qi, qj, lds);
    }
}

typedef Shape<256, 256, 2, 4, 2, 2> OrthHuge;       // three products in a chain
typedef Shape<32, 32, 2, 1, 2, 3> OrthTiny;

template <typename T, bool BK, bool LAST, typename S, bool TOGETHER> static int launch_orth(OrthArgs& a, int batch, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    const int lds = PairProduct<BK, S, TOGETHER>::LDS;
    if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(orth_product_kernel<T, BK, LAST, S, TOGETHER>), lds, done)) return rc;
    a.n_row_tiles = (a.I + S::BI - 1) / S::BI;
    a.n_col_tiles = (a.Jp + S::BJ - 1) / S::BJ;
    a.batch = batch;
    const int64_t blocks = ((int64_t)a.n_row_tiles * a.n_col_tiles * batch + 7) / 8 * 8;
    FRA_REQUIRE(blocks <= 4294967295LL / S::NT, FRA_ERR_ARG, "fra_orthogonalize: %lld workgroups", (long long)blocks);    // threads of a launch: 32 bits
    hipLaunchKernelGGL((orth_product_kernel<T, BK, LAST, S, TOGETHER>), dim3((unsigned)blocks), dim3(S::NT), lds, s, a);
    FRA_HIP(hipGetLastError());
    return FRA_OK;
}
// rounds of one workgroup per compute unit that are at least nine tenths full.  Counted in tiles, whatever of them the matrices fill: many
// small ones take large tiles too (256 of 64 x 64 126 us, 250 of 100 x 100 231, 60 of 321 x 330 559)
static bool full_rounds(int64_t tiles) { return tiles >= 230 && tiles * 10 >= (tiles + 255) / 256 * 256 * 9; }
// Whether the lower triangle is worth it.  How long a product takes, in rounds of 128 x 128 tiles: a round of 256 x 256 is 3.3 of
// them; one of 64 x 64 on a unit 0.35, two 0.6 (eight of 1024 x 1024: P from X of 2048 columns 117 -> 81 us, Q 57 -> 47; a matrix
// of 1500 x 1500 665 -> 466 us for all steps; 24 of 512 x 512 456 -> 369).  Asked
// to be a sixth less, except against the same tiles (four of 700 x 700 220 -> 211).
struct SymPlan {
    int tile, side, whole, per_die;     // tile: 128 or 64, 0: not worth it; tiles along a side; whole tiles and workgroups of a die
};
static SymPlan symmetric_plan(int m, int64_t batch) {
    auto sides = [&](int tile) { return (int64_t)((m + tile - 1) / tile); };
    auto square = [&](int tile) { return sides(tile) * sides(tile) * batch; };
    auto lower = [&](int tile) { return sides(tile) * (sides(tile) + 1) / 2 * batch; };
    auto small = [](int64_t tiles) { return tiles <= 256 ? 0.35 : 0.6 * ((tiles + 511) / 512); };
    const bool now64 = !full_rounds(square(256)) && square(128) < 192;
    const double now = now64 ? small(square(64)) : full_rounds(square(256)) ? 3.3 * ((square(256) + 255) / 256) : (double)((square(128) + 255) / 256);
    const int64_t rounds = lower(128) / 256, rest = lower(128) % 256;
    const double by128 = rounds + (rest == 0 ? 0.0 : rest <= 64 ? 0.35 : rest <= 128 ? 0.7 : 1.0), by64 = small(lower(64));
    SymPlan p = {0, 0, 0, 0};
    if (lower(64) > 1 << 28 || (by128 > 0.85 * now && (now64 ? square(64) <= 256 : by64 > 0.85 * now))) return p;
    p.tile = by64 <= by128 ? 64 : 128;
    p.side = (int)sides(p.tile);
    const int most = (int)((lower(p.tile) + 7) / 8);                // a die's
    p.whole = p.tile == 64 || rest > 128 ? most : (int)rounds * 32;
    p.per_die = most <= p.whole ? most : p.whole + 4 * (most - p.whole);
    return p;
}
template <typename W> static int launch_symmetric(OrthArgs& a, const SymPlan& p, int batch, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    const int lds = PairProduct<false, W, true>::LDS;
    if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(orth_symmetric_kernel<W>), lds, done)) return rc;
    a.batch = batch;
    FRA_REQUIRE((int64_t)p.per_die * 8 <= 4294967295LL / W::NT, FRA_ERR_ARG, "fra_orthogonalize: %d workgroups of a die", p.per_die);
    hipLaunchKernelGGL((orth_symmetric_kernel<W>), dim3((unsigned)p.per_die * 8), dim3(W::NT), lds, s, a, p.side, p.whole);
    FRA_HIP(hipGetLastError());
    return FRA_OK;
}
template <typename T, bool BK, bool LAST> static int product(OrthArgs& a, int batch, hipStream_t s) {
    auto tiles = [&](int64_t bi, int64_t bj) { return (a.I + bi - 1) / bi * ((a.Jp + bj - 1) / bj) * batch; };
    if constexpr (!BK) {                                            // X X^T and P P
        const SymPlan p = symmetric_plan(a.I, batch);
        if (p.tile == 128) return launch_symmetric<OrthBig>(a, p, batch, s);
        if (p.tile == 64) return launch_symmetric<OrthSmall>(a, p, batch, s);
    }
    if (full_rounds(tiles(256, 256))) return launch_orth<T, BK, LAST, OrthHuge, false>(a, batch, s);
    if (tiles(128, 128) >= 192) return launch_orth<T, BK, LAST, OrthBig, true>(a, batch, s);
    if (tiles(64, 64) >= 192) return launch_orth<T, BK, LAST, OrthSmall, true>(a, batch, s);
    return launch_orth<T, BK, LAST, OrthTiny, true>(a, batch, s);
}

struct OrthPlan {
    OrthDims d;
    int n_part;
    size_t off_part, off_x[2], off_p, off_q, bytes;     // hi at the offset, lo behind it
};
static OrthPlan orth_plan(int64_t batch, int rows, int cols) {
    OrthPlan p;
    p.d.transposed = rows > cols;
    p.d.m = p.d.transposed ? cols : rows;
    p.d.n = p.d.transposed ? rows : cols;
    p.d.mp = (p.d.m + 7) / 8 * 8;
    p.d.np = (p.d.n + 7) / 8 * 8;
    p.d.batch = (int)batch;
    const int64_t quads = (int64_t)rows * ((cols + 3) / 4);
    p.n_part = (int)(quads / 1024 < 1 ? 1 : quads / 1024 > 256 ? 256 : quads / 1024);
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t x = up((size_t)batch * p.d.m * p.d.np * 4), q = up((size_t)batch * p.d.m * p.d.mp * 4);
    size_t at = 0;
    p.off_part = at; at += up((size_t)batch * p.n_part * 8);
    p.off_x[0] = at; at += x;
    p.off_x[1] = at; at += x;
    p.off_p = at; at += q;
    p.off_q = at; at += q;
    p.bytes = at;
    return p;
}

template <typename T>
static int orth_t(const OrthPlan& p, const T* g, int64_t ldg, int64_t bs, int steps, float ca, float cb, float cc, T* out, char* ws, hipStream_t s) {
    const OrthDims d = p.d;
    const int rows = d.transposed ? d.n : d.m, cols = d.transposed ? d.m : d.n;
    double* part = (double*)(ws + p.off_part);
    const int64_t xe = (int64_t)d.m * d.np, qe = (int64_t)d.m * d.mp;
    f16* xh[2] = {(f16*)(ws + p.off_x[0]), (f16*)(ws + p.off_x[1])};
    f16* ph = (f16*)(ws + p.off_p);
    f16* qh = (f16*)(ws + p.off_q);
    const int64_t xlo = xe * d.batch, qlo = qe * d.batch;            // lo parts follow the hi parts
    hipLaunchKernelGGL((orth_norm_kernel<T>), dim3(p.n_part, d.batch), dim3(256), 0, s, g, ldg, bs, rows, cols, part);
    FRA_HIP(hipGetLastError());
    hipLaunchKernelGGL((orth_split_kernel<T>), dim3((d.np + 63) / 64, (d.m + 63) / 64, d.batch), dim3(256), 0, s, g, ldg, bs, d, part, p.n_part,
                       xh[0], xh[0] + xlo);
    FRA_HIP(hipGetLastError());
    for (int t = 0; t < steps; ++t) {
        f16 *x = xh[t & 1], *y = xh[(t + 1) & 1];
        OrthArgs a;
        a.out = nullptr; a.so = 0; a.ldo = 0; a.transposed = 0;
        // P = X X^T
        a.ah = a.bh = x; a.al = a.bl = x + xlo; a.eh = a.el = nullptr; a.ch = ph; a.cl = ph + qlo;
        a.sa = a.sb = xe; a.se = 0; a.sc = qe; a.lda = a.ldb = d.np; a.lde = 0; a.ldc = d.mp;
        a.I = d.m; a.J = d.m; a.Jp = d.mp; a.K = d.np; a.alpha = 1.0f / OR_SCALE; a.beta = 0.0f;
        if (int rc = product<f16, false, false>(a, d.batch, s)) return rc;
        // Q = b P + c P P (P is symmetric)
        a.ah = a.bh = a.eh = ph; a.al = a.bl = a.el = ph + qlo; a.ch = qh; a.cl = qh + qlo;
        a.sa = a.sb = a.se = a.sc = qe; a.lda = a.ldb = a.lde = a.ldc = d.mp;
        a.K = d.mp; a.alpha = cc / OR_SCALE; a.beta = cb;
        if (int rc = product<f16, false, false>(a, d.batch, s)) return rc;
        // X <- a X + Q X
        a.ah = qh; a.al = qh + qlo; a.bh = a.eh = x; a.bl = a.el = x + xlo; a.ch = y; a.cl = y + xlo;
        a.sa = qe; a.sb = a.se = a.sc = xe; a.lda = d.mp; a.ldb = a.lde = a.ldc = d.np;
        a.I = d.m; a.J = d.n; a.Jp = d.np; a.K = d.m; a.alpha = 1.0f / OR_SCALE; a.beta = ca;
        if (t < steps - 1) {
            if (int rc = product<f16, true, false>(a, d.batch, s)) return rc;
        } else {
            a.ch = a.cl = nullptr;
            a.out = out; a.so = (int64_t)rows * cols; a.ldo = cols; a.transposed = d.transposed;
            if (int rc = product<T, true, true>(a, d.batch, s)) return rc;
        }
    }
    return FRA_OK;
}

static int check_orth(int64_t batch, int rows, int cols, const char* what) {
    FRA_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 1 && cols >= 1 && rows <= 32768 && cols <= 32768, FRA_ERR_ARG,
                "%s: %lld matrices of %d x %d (at most 65535, sides 1 to 32768)", what, (long long)batch, rows, cols);
    return FRA_OK;
}

}  // namespace fra

using namespace fra;

extern "C" {

int fra_orthogonalize_workspace_bytes(int64_t batch, int rows, int cols, size_t* bytes) {
    FRA_REQUIRE(bytes, FRA_ERR_ARG, "fra_orthogonalize_workspace_bytes: null pointer");
    if (int rc = check_orth(batch, rows, cols, "fra_orthogonalize_workspace_bytes")) return rc;
    *bytes = orth_plan(batch, rows, cols).bytes;
    return FRA_OK;
}

int fra_orthogonalize(int dtype, const void* g, int64_t ldg, int64_t batch_stride, int64_t batch, int rows, int cols, int steps, float a, float b,
                      float c, void* out, void* workspace, size_t workspace_bytes, fra_stream stream) {
    if (int rc = check_orth(batch, rows, cols, "fra_orthogonalize")) return rc;
    FRA_REQUIRE(dtype == FRA_F32 || dtype == FRA_BF16 || dtype == FRA_F16, FRA_ERR_ARG, "fra_orthogonalize: dtype %d unsupported", dtype);
    FRA_REQUIRE(steps >= 1 && steps <= 100, FRA_ERR_ARG, "fra_orthogonalize: %d steps (1 to 100)", steps);
    FRA_REQUIRE(a >= -16.0f && a <= 16.0f && b >= -16.0f && b <= 16.0f && c >= -16.0f && c <= 16.0f, FRA_ERR_ARG,
                "fra_orthogonalize: coefficients (%g, %g, %g) (each within +-16)", (double)a, (double)b, (double)c);
    FRA_REQUIRE(ldg >= cols && batch_stride >= 0, FRA_ERR_ARG, "fra_orthogonalize: pitch %lld below %d columns, or batch stride %lld", (long long)ldg, cols, (long long)batch_stride);
    if (batch == 0) return FRA_OK;
    FRA_REQUIRE(g && out, FRA_ERR_ARG, "fra_orthogonalize: null pointer");
    const OrthPlan p = orth_plan(batch, rows, cols);
    FRA_REQUIRE(workspace && workspace_bytes >= p.bytes, FRA_ERR_WORKSPACE, "fra_orthogonalize: workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
    FRA_REQUIRE(((uintptr_t)workspace & 15) == 0, FRA_ERR_ARG, "fra_orthogonalize: workspace not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (dtype == FRA_F32) return orth_t<float>(p, (const float*)g, ldg, batch_stride, steps, a, b, c, (float*)out, ws, s);
    if (dtype == FRA_BF16) return orth_t<bf16>(p, (const bf16*)g, ldg, batch_stride, steps, a, b, c, (bf16*)out, ws, s);
    return orth_t<f16>(p, (const f16*)g, ldg, batch_stride, steps, a, b, c, (f16*)out, ws, s);
}

}  // extern "C"
