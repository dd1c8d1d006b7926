// Orthogonalising a matrix by Newton-Schulz products: with X = G / |G|_F (transposed if taller than wide),
//     P = X X^T,   Q = b P + c P P,   X <- a X + Q X        `steps` times,
// an odd polynomial of every singular value, a s + b s^3 + c s^5, that drives them towards one.  No counterpart in the reference.
//
// The iteration multiplies small singular values by `a` each step (485 times in five steps of the usual coefficients) and a
// rounding error with them, so sixteen bits are too few between the products.  Every value is held as TWO f16, hi + lo, of
// 2^8 times itself: 22 significant bits down to 2^-10, an absolute step of 2^-32 below, range +-255.  A product is
// hi hi + hi lo + lo hi on the f16 matrix cores (lo lo is below 2^-22), accumulated in fp32: a third of their rate, which is
// over three times that of the fp32 matrix instructions.
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

// G -> X hi / lo [m][np], normalised, transposed if need be, zeros in columns n .. np: 64 x 64 tiles through LDS
template <typename T> __global__ __launch_bounds__(256) void orth_split_kernel(const T* g, int64_t ldg, int64_t bs, OrthDims d, const double* part,
                                                                              int n_part, f16* xh, f16* xl) {
    __shared__ float tile[64][65];
    __shared__ double factor;                                       // fp64: OR_SCALE / norm leaves fp32's range for a tiny matrix
    const int b = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    if (threadIdx.x < 64) {
        double v = 0.0;
        for (int p = threadIdx.x; p < n_part; p += 64) v += part[(int64_t)b * n_part + p];
#pragma unroll
        for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s, 64);
        if (threadIdx.x == 0) factor = v == 0.0 ? 0.0 : (double)OR_SCALE / sqrt(v);        // a matrix of zeros stays one
    }
    __syncthreads();
    const double f = factor;
    const T* p = g + (int64_t)b * bs;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave; r < 64; r += 4) {
        // source rows: X's rows, or (transposed) X's columns
        const int sr = (d.transposed ? j0 : i0) + r, sc = (d.transposed ? i0 : j0) + lane;
        const bool in = sr < (d.transposed ? d.n : d.m) && sc < (d.transposed ? d.m : d.n);
        const float v = in ? (float)((double)(float)p[(int64_t)sr * ldg + sc] * f) : 0.0f;
        if (d.transposed) tile[lane][r] = v;
        else tile[r][lane] = v;
    }
    __syncthreads();
    const int64_t base = (int64_t)b * d.m * d.np;
    for (int r = wave; r < 64; r += 4) {
        if (i0 + r >= d.m || j0 + lane >= d.np) continue;
        f16 hi, lo;
        split16(tile[r][lane], hi, lo);
        xh[base + (int64_t)(i0 + r) * d.np + j0 + lane] = hi;
        xl[base + (int64_t)(i0 + r) * d.np + j0 + lane] = lo;
    }
}

// C = alpha A B^T + beta E (or A B where B is contraction-major), everything hi / lo f16, batch in blockIdx.y
struct OrthArgs {
    const f16 *ah, *al, *bh, *bl, *eh, *el;
    f16 *ch, *cl;               // nullptr: the last product, into out
    void* out;
    int64_t sa, sb, se, sc, so; // elements between the matrices of a batch
    int lda, ldb, lde, ldc;
    int64_t ldo;
    int I, J, Jp, K;            // C is [I][J], columns J .. Jp are written as zeros
    float alpha, beta;
    int n_col_tiles, transposed;
};
template <typename T, bool BK, typename S> __global__ __launch_bounds__(S::NT) void orth_product_kernel(OrthArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int ct = blockIdx.x % a.n_col_tiles, rt = blockIdx.x / a.n_col_tiles;
    const int i0 = rt * S::BI, j0 = ct * S::BJ;
    const int64_t b = blockIdx.y;
    f32x4 acc[S::MI][S::MJ];
    Product<f16, false, BK, S, true> p;
    p.A.order = nullptr; p.A.ld = a.lda; p.A.row0 = i0; p.A.rows = a.I - i0; p.A.klen = a.K; p.A.cols = 0;
    p.B.order = nullptr; p.B.ld = a.ldb; p.B.klen = a.K;
    p.B.row0 = BK ? 0 : j0; p.B.rows = BK ? 0 : a.J - j0; p.B.cols = BK ? a.J - j0 : 0;
    const int64_t boff = b * a.sb + (BK ? j0 : 0);
    // the small parts first, so that they are added before the large ones
    p.A.base = a.al + b * a.sa; p.B.base = a.bh + boff;
    p.start(a.K, lds);
    p.run(lds, acc);
    p.A.base = a.ah + b * a.sa; p.B.base = a.bl + boff;
    p.start(a.K, lds);
    p.template run<true>(lds, acc);
    p.A.base = a.ah + b * a.sa; p.B.base = a.bh + boff;
    p.start(a.K, lds);
    p.template run<true>(lds, acc);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int li = (wave % S::WI) * (S::BI / S::WI) + (lane & 15), lj = (wave / S::WI) * (S::BJ / S::WJ) + 4 * (lane >> 4);
#pragma unroll
    for (int mi = 0; mi < S::MI; ++mi) {
        const int i = i0 + li + 16 * mi;
        if (i >= a.I) continue;
#pragma unroll
        for (int mj = 0; mj < S::MJ; ++mj) {
            const int j = j0 + lj + 16 * mj;
            if (j >= a.Jp) continue;
            float v[4], eh[4] = {0, 0, 0, 0}, el[4] = {0, 0, 0, 0};
            if (a.eh) {
                load_four<f16>(a.eh + b * a.se + (int64_t)i * a.lde + j, 4, eh);
                load_four<f16>(a.el + b * a.se + (int64_t)i * a.lde + j, 4, el);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = j + e < a.J ? a.alpha * acc[mi][mj][e] + a.beta * (eh[e] + el[e]) : 0.0f;
            if (a.ch) {
                float hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e] = (float)(f16)v[e];
                    lo[e] = v[e] - hi[e];
                }
                store_four<f16>(a.ch + b * a.sc + (int64_t)i * a.ldc + j, 4, hi);
                store_four<f16>(a.cl + b * a.sc + (int64_t)i * a.ldc + j, 4, lo);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= 1.0f / OR_SCALE;
                T* o = (T*)a.out + b * a.so;
                if (!a.transposed) {
                    if (a.J - j > 0) store_four<T>(o + (int64_t)i * a.ldo + j, a.J - j, v);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (j + e < a.J) o[(int64_t)(j + e) * a.ldo + i] = (T)v[e];
                }
            }
        }
    }
}

typedef Shape<64, 64, 2, 2, 2, 3> OrthTile;

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
    constexpr int LDS = OrthTile::LDS;
    static_assert(LDS <= 65536, "no raised limit needed");
    const int ti = (d.m + 63) / 64, tp = (d.mp + 63) / 64, tx = (d.np + 63) / 64;
    for (int t = 0; t < steps; ++t) {
        f16 *x = xh[t & 1], *y = xh[(t + 1) & 1];
        OrthArgs a;
        a.out = nullptr; a.so = 0; a.ldo = 0; a.transposed = 0;
        // P = X X^T
        a.ah = a.bh = x; a.al = a.bl = x + xlo; a.eh = a.el = nullptr; a.ch = ph; a.cl = ph + qlo;
        a.sa = a.sb = xe; a.se = 0; a.sc = qe; a.lda = a.ldb = d.np; a.lde = 0; a.ldc = d.mp;
        a.I = d.m; a.J = d.m; a.Jp = d.mp; a.K = d.n; a.alpha = 1.0f / OR_SCALE; a.beta = 0.0f; a.n_col_tiles = tp;
        hipLaunchKernelGGL((orth_product_kernel<T, false, OrthTile>), dim3(ti * tp, d.batch), dim3(OrthTile::NT), LDS, s, a);
        FRA_HIP(hipGetLastError());
        // Q = b P + c P P (P is symmetric)
        a.ah = a.bh = a.eh = ph; a.al = a.bl = a.el = ph + qlo; a.ch = qh; a.cl = qh + qlo;
        a.sa = a.sb = a.se = a.sc = qe; a.lda = a.ldb = a.lde = a.ldc = d.mp;
        a.K = d.m; a.alpha = cc / OR_SCALE; a.beta = cb;
        hipLaunchKernelGGL((orth_product_kernel<T, false, OrthTile>), dim3(ti * tp, d.batch), dim3(OrthTile::NT), LDS, s, a);
        FRA_HIP(hipGetLastError());
        // X <- a X + Q X
        a.ah = qh; a.al = qh + qlo; a.bh = a.eh = x; a.bl = a.el = x + xlo; a.ch = y; a.cl = y + xlo;
        a.sa = qe; a.sb = a.se = a.sc = xe; a.lda = d.mp; a.ldb = a.lde = a.ldc = d.np;
        a.I = d.m; a.J = d.n; a.Jp = d.np; a.K = d.m; a.alpha = 1.0f / OR_SCALE; a.beta = ca; a.n_col_tiles = tx;
        if (t == steps - 1) {
            a.ch = a.cl = nullptr;
            a.out = out; a.so = (int64_t)rows * cols; a.ldo = cols; a.transposed = d.transposed;
        }
        hipLaunchKernelGGL((orth_product_kernel<T, true, OrthTile>), dim3(ti * tx, d.batch), dim3(OrthTile::NT), LDS, s, a);
        FRA_HIP(hipGetLastError());
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
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (dtype == FRA_F32) return orth_t<float>(p, (const float*)g, ldg, batch_stride, steps, a, b, c, (float*)out, ws, s);
    if (dtype == FRA_BF16) return orth_t<bf16>(p, (const bf16*)g, ldg, batch_stride, steps, a, b, c, (bf16*)out, ws, s);
    return orth_t<f16>(p, (const f16*)g, ldg, batch_stride, steps, a, b, c, (f16*)out, ws, s);
}

}  // extern "C"
