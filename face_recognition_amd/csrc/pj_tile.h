// The tiled matrix product behind the projections: C[i][j] = sum_k A(i,k) B(j,k) on one workgroup, fp32 accumulation.
//
// Either operand may lie row by row ("row-major": k is the contiguous index) or contraction by contraction ("k-major": i or j
// is contiguous); the combinations are the forward product, the two gradients and the Gram products, with no transposed copy
// in memory.  A step covers KS groups of k: 32 sixteen-bit values (one 16x16x32 MFMA deep) or 16 floats (four 16x16x4) each.
//
// LDS images, in 16-byte chunks:
//   row-major  [DIM rows][4 KS chunks of k]; chunk c of row r at slot c ^ (r & 7) (KS = 2) or c ^ (r >> 1 & 3) (KS = 1): the eight
//              rows of a read's phase are on different banks;
//   k-major    [step's rows of k][DIM], 16 bit: chunk pair p of row k at p ^ ((k & 3) | (k >> 1 & 4)) (128 columns and more; with
//              64, two rows of k fill a row of banks: p ^ ((k >> 1 & 1) | (k >> 2 & 2)); with 32, four: p ^ (k >> 3 & 1)), so the
//              eight 32-byte pieces that half a wave's transposing read (ds_read_b64_tr_b16) takes are on different banks; float:
//              chunk c at c ^ 4 (k >> 2 & 3) (with 32 columns 4 (k >> 2 & 1), two lanes to a bank).
#pragma once

#include "common.h"

namespace fra {

template <typename T> struct Elem {                 // 16-bit element types
    static constexpr int EPC = 8;                   // elements per 16-byte chunk
    static constexpr int KG = 32;                   // contraction per group
    typedef typename vec8<T>::type Frag;            // one lane's operand of an MFMA group: 16 bytes
    typedef typename vec4<T>::type Quad;
};
template <> struct Elem<float> {
    static constexpr int EPC = 4;
    static constexpr int KG = 16;
    typedef f32x4 Frag;
    typedef f32x4 Quad;
};

template <typename T> __device__ __forceinline__ f32x4 pj_mma(typename Elem<T>::Frag a, typename Elem<T>::Frag b, f32x4 c) {
    if constexpr (sizeof(T) == 2) {
        return mfma16(a, b, c);
    } else {
        // a lane of k-group g holds k = 4 g + s in element s: step s multiplies the four k = 4 g + s of the groups
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
        return c;
    }
}

// 16 bytes from any address an element may have
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Chunk { typename Elem<T>::Frag v; };
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Four { typename Elem<T>::Quad v; };

// `n` valid elements (at most a chunk; none if n <= 0) from p, the rest zero
template <typename T> __device__ __forceinline__ typename Elem<T>::Frag load_chunk(const T* p, int n) {
    typename Elem<T>::Frag v;
    if (n >= Elem<T>::EPC) return reinterpret_cast<const Chunk<T>*>(p)->v;
#pragma unroll
    for (int e = 0; e < Elem<T>::EPC; ++e) v[e] = (T)0.0f;
    if (n > 0) {
#pragma unroll
        for (int e = 0; e < Elem<T>::EPC; ++e)
            if (e < n) v[e] = p[e];
    }
    return v;
}
template <typename T> __device__ __forceinline__ void store_chunk(T* p, int n, typename Elem<T>::Frag v) {
    if (n >= Elem<T>::EPC) {
        reinterpret_cast<Chunk<T>*>(p)->v = v;
    } else {
#pragma unroll
        for (int e = 0; e < Elem<T>::EPC; ++e)
            if (e < n) p[e] = v[e];
    }
}
template <typename T> __device__ __forceinline__ void load_four(const T* p, int n, float (&o)[4]) {
    if (n >= 4) {
        const typename Elem<T>::Quad v = reinterpret_cast<const Four<T>*>(p)->v;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (float)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = e < n ? (float)p[e] : 0.0f;
    }
}
template <typename T> __device__ __forceinline__ void store_four(T* p, int n, const float (&v)[4]) {
    if (n >= 4) {
        typename Elem<T>::Quad q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = (T)v[e];
        reinterpret_cast<Four<T>*>(p)->v = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = (T)v[e];
    }
}

template <int KS> __device__ __forceinline__ int swz_row_major(int row, int c) { return KS == 2 ? c ^ (row & 7) : c ^ ((row >> 1) & 3); }
template <typename T, int CPR> __device__ __forceinline__ int swz_k_major(int k, int c) {
    if constexpr (sizeof(T) == 4) return c ^ ((((k >> 2) & 3) << 2) & (CPR - 1));
    else if constexpr (CPR >= 16) return c ^ (((k & 3) | ((k >> 1) & 4)) << 1);
    else if constexpr (CPR == 8) return c ^ ((((k >> 1) & 1) | ((k >> 2) & 2)) << 1);       // two rows of k share a row of banks
    else return c ^ (((k >> 3) & 1) << 1);                                                  // four do
}

// 16 bytes per lane from global memory into LDS at `lds` + 16 lane, without passing through registers.  Written out (the
// instruction has no register result) so that the compiler does not put a wait for it in front of every LDS read; the loops
// that use it wait by count (dma_wait_barrier) before the barrier that publishes a tile.  m0 holds the LDS address (a clobber: the
// compiler sets m0 for its own uses, and keeps it across what does not name it); one wait state lies between its write and the load.
// The asm takes the LDS pointer itself: memory whose address never leaves the kernel's own loads counts as unwritten.
typedef __attribute__((address_space(3))) char* LdsPtr;
__device__ __forceinline__ void dma16(const void* g, LdsPtr lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(g) : "m0", "memory");
}
// at most N loads of this wave still on their way, all its LDS reads done; then the workgroup's barrier
template <int N> __device__ __forceinline__ void dma_wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// the oldest step on its way (NLD loads each) has arrived for every wave: at most Y younger ones are still out, fewer if fewer
// than that (`behind`) come after it
template <int Y, int NLD> __device__ __forceinline__ void step_arrived(int behind) {
    static_assert(Y * NLD < 64, "the counter's range");
    if (behind >= Y) dma_wait_barrier<Y * NLD>();
    else if constexpr (Y > 0) step_arrived<Y - 1, NLD>(behind);
}
// what a lane reads in place of a chunk outside its operand
static __device__ __attribute__((aligned(16))) const float pj_zeros[4] = {0.0f, 0.0f, 0.0f, 0.0f};

// One operand of a workgroup's tile: where its chunks come from and how a wave reads its fragments.
//   row-major: `rows` tile rows start at row0 of a row list (`order`, or the rows themselves), each `klen` long from k = 0;
//   k-major: columns 0 .. cols of `base`, whose rows row0 .. row0 + klen are summed over.
template <typename T, bool KMAJOR, int DIM, int NT, int KS> struct Operand {
    static constexpr int EPC = Elem<T>::EPC, KSTEP = KS * Elem<T>::KG;
    static constexpr int CPR = KMAJOR ? DIM / EPC : 4 * KS;         // chunks per LDS row
    static constexpr int CHUNKS = DIM * 4 * KS;                     // 16-byte chunks per tile
    static constexpr int BYTES = CHUNKS * 16;
    static constexpr int NLD = CHUNKS / NT;                         // per thread
    static constexpr int RPP = NT / CPR;                            // LDS rows per pass
    static_assert(CHUNKS % NT == 0 && NT % CPR == 0, "whole chunks per thread, whole rows per pass");
    typedef typename Elem<T>::Frag Frag;

    const T* base;
    const int* order;               // row-major only
    int64_t ld;
    int row0, rows, klen, cols;

    // this lane's chunk of every pass at step 0
    struct Src {
        const T* p[NLD];
    };
    // row-major: rows >= 1; tile row r stands for list entry row0 + min(r, rows - 1).  k-major: a chunk past `cols` stands for the
    // first one.  (Rows and columns past the end belong to results that are not stored; only k past `klen` has to be zero.)
    __device__ __forceinline__ void init(Src& d, int tid) const {
#pragma unroll
        for (int j = 0; j < NLD; ++j) {
            const int r = j * RPP + tid / CPR;
            if constexpr (!KMAJOR) {
                const int at = row0 + (r < rows ? r : rows - 1);
                d.p[j] = base + (int64_t)(order ? order[at] : at) * ld + swz_row_major<KS>(r, tid % CPR) * EPC;
            } else {
                const int col = swz_k_major<T, CPR>(r, tid % CPR) * EPC;
                d.p[j] = base + (int64_t)(row0 + r) * ld + (col < cols ? col : 0);
            }
        }
    }
    // elements of the lane's chunk of pass j that are inside at `step` (<= 0: none); k-major: of the chunk it stands for
    __device__ __forceinline__ int valid(int j, int step, int tid) const {
        const int r = j * RPP + tid / CPR;
        if constexpr (!KMAJOR) {
            return klen - step * KSTEP - swz_row_major<KS>(r, tid % CPR) * EPC;
        } else {
            const int col = swz_k_major<T, CPR>(r, tid % CPR) * EPC;
            return step * KSTEP + r < klen ? cols - (col < cols ? col : 0) : 0;
        }
    }
    __device__ __forceinline__ int64_t advance(int step) const {
        if constexpr (!KMAJOR) return (int64_t)step * KSTEP;
        else return (int64_t)step * KSTEP * ld;
    }

    // ---- staging through registers: any alignment, any number of valid elements
    __device__ __forceinline__ void load(const Src& d, Frag (&v)[NLD], int step, int tid) const {
#pragma unroll
        for (int j = 0; j < NLD; ++j) v[j] = load_chunk<T>(d.p[j] + advance(step), valid(j, step, tid));
    }
    static __device__ __forceinline__ void store(char* tile, const Frag (&v)[NLD], int tid) {
#pragma unroll
        for (int j = 0; j < NLD; ++j) *reinterpret_cast<Frag*>(tile + (j * NT + tid) * 16) = v[j];
    }
    // ---- staging by DMA: every chunk is wholly inside or outside (klen or cols, pitch and base multiples of 16 bytes)
    // `plus`: elements added to every address (a second operand of the same layout)
    __device__ __forceinline__ void issue(const Src& d, int step, LdsPtr lds, int tid, int64_t plus = 0) const {
        const int64_t at = advance(step) + plus;
        if ((step + 1) * KSTEP <= klen) {
#pragma unroll
            for (int j = 0; j < NLD; ++j) dma16(d.p[j] + at, lds + j * (NT * 16));
        } else {
#pragma unroll
            for (int j = 0; j < NLD; ++j)
                dma16(valid(j, step, tid) > 0 ? d.p[j] + at : reinterpret_cast<const T*>(pj_zeros), lds + j * (NT * 16));
        }
    }
    // fragment of the 16 rows / columns from `d0`, k group `ks` of the step
    static __device__ __forceinline__ Frag frag(const char* tile, int d0, int ks, int lane) {
        const int m = lane & 15, g = lane >> 4;
        if constexpr (!KMAJOR) {
            const int r = d0 + m;
            return *reinterpret_cast<const Frag*>(tile + (r * CPR + swz_row_major<KS>(r, ks * 4 + g)) * 16);
        } else if constexpr (sizeof(T) == 2) {
            // sixteen lanes take four rows of k x sixteen columns and receive one column of four k each
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) s16x4* LP;
            const int k = ks * 32 + g * 8 + (m >> 2);
            const int c0 = d0 / EPC + ((m >> 1) & 1);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (LP)(tile + (k * CPR + swz_k_major<T, CPR>(k, c0)) * 16 + (m & 1) * 8));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (LP)(tile + ((k + 4) * CPR + swz_k_major<T, CPR>(k + 4, c0)) * 16 + (m & 1) * 8));
            const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(Frag, v);
        } else {
            Frag v;
            const int col = d0 + m;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = ks * 16 + g * 4 + s;
                v[s] = *reinterpret_cast<const float*>(tile + (k * CPR + swz_k_major<T, CPR>(k, col >> 2)) * 16 + (col & 3) * 4);
            }
            return v;
        }
    }
};

// Workgroup shape: BI x BJ results on WI x WJ waves (a wave owns MI x MJ tiles of 16 x 16), KS groups of k per step, NB steps in
// LDS.
template <int BI_, int BJ_, int WI_, int WJ_, int KS_, int NB_> struct Shape {
    static constexpr int BI = BI_, BJ = BJ_, WI = WI_, WJ = WJ_, KS = KS_, NB = NB_, NT = 64 * WI * WJ;
    static constexpr int MI = BI / WI / 16, MJ = BJ / WJ / 16;
    static constexpr int STEP = (BI + BJ) * KS * 64, LDS = NB * STEP;
    static constexpr int STRIPS = BI * BJ / MI * 4;     // tile_emit's
    static constexpr int PER_CU = 163840 / LDS;         // workgroups that share a compute unit's LDS,
    static constexpr int WAVES = PER_CU * NT / 256;     // and their waves per SIMD, for which the registers have to do
    static_assert(STRIPS <= LDS, "");
};
template <typename T, bool KMAJOR, typename S> using OperandA = Operand<T, KMAJOR, S::BI, S::NT, S::KS>;
template <typename T, bool KMAJOR, typename S> using OperandB = Operand<T, KMAJOR, S::BJ, S::NT, S::KS>;

// Which tile of n_rt x n_ct a workgroup takes.  Workgroups are dealt out to the eight dies in turn, and each die has an L2 of its
// own, so die b % 8 gets one consecutive eighth of the tiles, walked in bands of eight row tiles, column by column: what runs on
// a die at a time is about square and reads each operand's panels once (with tiles dealt out row by row the dies together
// fetched 105 MB through their L2s for a 4096 x 2048 x 1024 product whose operands are 12 MB).  Launch 8 ceil(tiles / 8)
// workgroups at least; false: no tile left for this one.
// With several matrices of tiles the eighths run through them one after the other.
__device__ __forceinline__ bool tile_of_block(unsigned b, unsigned n_rt, unsigned n_ct, int& rt, int& ct, unsigned n_mat, int& mat) {
    const unsigned each = n_rt * n_ct, all = n_mat * each, x = b & 7, i = b >> 3, q = all >> 3, r = all & 7;   // below 2^31 (the launchers check)
    if (i >= q + (x < r)) return false;
    unsigned id = x * q + (x < r ? x : r) + i;
    mat = 0;
    if (n_mat > 1) {
        mat = (int)(id / each);
        id -= mat * each;
    }
    const unsigned band = 8 * n_ct, first = id / band * 8;
    const unsigned in = id - first * n_ct, rows = n_rt - first < 8 ? n_rt - first : 8;
    ct = (int)(in / rows);
    rt = (int)(first + in - ct * rows);
    return true;
}
__device__ __forceinline__ bool tile_of_block(unsigned b, unsigned n_rt, unsigned n_ct, int& rt, int& ct) {
    int mat;
    return tile_of_block(b, n_rt, n_ct, rt, ct, 1, mat);
}

// Hands a workgroup's results on as 16-byte pieces of rows: a wave turns its accumulators through its own part of LDS, 16 rows
// at a time (written as a lane's four neighbouring columns, chunk c of row r at c ^ r; read as V neighbouring columns, so that
// the lanes side by side cover a row's whole lines), and calls
//     row(i)              where row i of the tile goes, for the pieces of two strips first, then
//     pre(row, j)         for the same pieces, so that loads that the results wait for go out together, then
//     emit(row, j, state, v)  with the V = 16 / sizeof(T) values of columns j .. j + V of the tile.
// `strips`: S::STRIPS bytes that nobody else uses any more.
template <typename T, typename S, typename F> __device__ __forceinline__ void tile_emit(const f32x4 (&acc)[S::MI][S::MJ], char* strips, const F& f) {
    constexpr int COLS = S::MJ * 16, CH = COLS / 4, V = 16 / sizeof(T), LPR = COLS / V, RPP = 64 / LPR, NP = 16 / RPP;
    static_assert(16 % RPP == 0 && (CH & (CH - 1)) == 0, "whole passes per strip");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i0 = (wave % S::WI) * (S::BI / S::WI), j0 = (wave / S::WI) * (S::BJ / S::WJ);
    f32x4* strip = reinterpret_cast<f32x4*>(strips) + wave * (16 * CH);
    const int r = lane / LPR, c = (lane % LPR) * V;
    constexpr int MG = S::MI < 2 ? S::MI : 2;                       // strips whose loads go out together
    static_assert(S::MI % MG == 0, "");
#pragma unroll
    for (int m0 = 0; m0 < S::MI; m0 += MG) {
        int rows[MG * NP];
        typename F::Pre pre[MG * NP];
#pragma unroll
        for (int k = 0; k < MG * NP; ++k) rows[k] = f.row(i0 + 16 * m0 + k * RPP + r);
#pragma unroll
        for (int k = 0; k < MG * NP; ++k) pre[k] = f.pre(rows[k], j0 + c);
#pragma unroll
        for (int mi = 0; mi < MG; ++mi) {
#pragma unroll
            for (int mj = 0; mj < S::MJ; ++mj) strip[(lane & 15) * CH + ((4 * mj + (lane >> 4)) ^ (lane & (CH - 1) & 15))] = acc[m0 + mi][mj];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int row = p * RPP + r;
                float v[V];
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const f32x4 x = strip[row * CH + ((c / 4 + q) ^ (row & (CH - 1)))];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e];
                }
                f.emit(rows[mi * NP + p], j0 + c, pre[mi * NP + p], v);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// A wave's operands of one group of k, and the MFMAs on them.
template <typename T, bool AK, bool BK, typename S> struct Frags {
    typename Elem<T>::Frag a[S::MI], b[S::MJ];
    __device__ __forceinline__ void read(const char* step, int ks, int i0, int j0, int lane) {
        typedef OperandA<T, AK, S> OA;
        typedef OperandB<T, BK, S> OB;
#pragma unroll
        for (int mi = 0; mi < S::MI; ++mi) a[mi] = OA::frag(step, i0 + 16 * mi, ks, lane);
#pragma unroll
        for (int mj = 0; mj < S::MJ; ++mj) b[mj] = OB::frag(step + OA::BYTES, j0 + 16 * mj, ks, lane);
    }
    __device__ __forceinline__ void mma(f32x4 (&acc)[S::MI][S::MJ]) const {
#pragma unroll
        for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
            for (int mj = 0; mj < S::MJ; ++mj) acc[mi][mj] = pj_mma<T>(b[mj], a[mi], acc[mi][mj]);
    }
};

// `steps` steps through LDS, NB deep, the first NB already on their way.  issue(t, dst): sends for step t (NLD loads per wave).  A
// wave reads the second half of a step while the matrix cores work on the first, and the first half of the next step while they
// work on the second; between the two lies the one barrier of a step, which says that the next step has arrived for every wave and
// that every wave has read all of this one, whose buffer the load of step t + NB then takes.  On return every wave is past its last
// LDS read.
template <int NB, int NLD, int BUF, typename F, typename Issue, typename Acc>
__device__ __forceinline__ void run_steps(int steps, char* lds, LdsPtr dst, const Issue& issue, int i0, int j0, int lane, Acc& acc) {
    F f0, f1;
    step_arrived<NB - 1, NLD>(steps - 1);
    f0.read(lds, 0, i0, j0, lane);
    int cur = 0;
    for (int t = 0; t < steps; ++t) {
        f1.read(lds + cur, 1, i0, j0, lane);
        __builtin_amdgcn_sched_barrier(0);
        f0.mma(acc);
        __builtin_amdgcn_sched_barrier(0);
        const int nxt = cur + BUF == NB * BUF ? 0 : cur + BUF;
        if (t + 1 < steps) {
            step_arrived<NB - 2, NLD>(steps - 2 - t);
            if (t + NB < steps) issue(t + NB, dst + cur);
            f0.read(lds + nxt, 0, i0, j0, lane);
        }
        __builtin_amdgcn_sched_barrier(0);
        f1.mma(acc);
        __builtin_amdgcn_sched_barrier(0);
        cur = nxt;
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The product of a tile in two parts, between which a kernel sends for what it needs afterwards:
//   start   fetches the addresses and (DMA) issues the first NB steps; every wave is past its reads of those buffers;
//   run     acc[mi][mj][r] = C[i][j] with i = 16 mi + (lane & 15), j = 16 mj + 4 (lane >> 4) + r inside the wave's part: the j side
//           is the MFMA's row operand, so a lane holds four neighbouring j of one i.
//           On return every wave is past its last LDS read.
// klen: the longer of the operands' (an operand's chunks past its own are zeros).
// DMA: by run_steps; otherwise the next step waits in registers.
template <typename T, bool AK, bool BK, typename S, bool DMA> struct Product {
    typedef OperandA<T, AK, S> OA;
    typedef OperandB<T, BK, S> OB;
    static constexpr int NB = S::NB, BUF = S::STEP, NLD = OA::NLD + OB::NLD;
    static_assert(OA::BYTES + OB::BYTES == BUF && NB >= 2 && S::KS == 2, "");
    OA A;
    OB B;
    typename OA::Src sa;
    typename OB::Src sb;
    int steps;

    __device__ __forceinline__ static LdsPtr dma_base(char* lds) {
        return (LdsPtr)lds + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * 1024;
    }
    __device__ __forceinline__ void start(int klen, char* lds) {
        const int tid = threadIdx.x;
        steps = (klen + OA::KSTEP - 1) / OA::KSTEP;
        if (steps == 0) return;
        A.init(sa, tid);
        B.init(sb, tid);
        if constexpr (DMA) {
            const LdsPtr dst = dma_base(lds);
#pragma unroll
            for (int t = 0; t < NB; ++t)
                if (t < steps) {
                    A.issue(sa, t, dst + t * BUF, tid);
                    B.issue(sb, t, dst + t * BUF + OA::BYTES, tid);
                }
        }
    }
    __device__ __forceinline__ void run(char* lds, f32x4 (&acc)[S::MI][S::MJ]) const {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int i0 = (wave % S::WI) * (S::BI / S::WI), j0 = (wave / S::WI) * (S::BJ / S::WJ);
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int mi = 0; mi < S::MI; ++mi)
#pragma unroll
            for (int mj = 0; mj < S::MJ; ++mj) acc[mi][mj] = zero;
        if (steps == 0) return;
        if constexpr (DMA) {
            run_steps<NB, NLD, BUF, Frags<T, AK, BK, S>>(steps, lds, dma_base(lds), [&](int t, LdsPtr to) {
                A.issue(sa, t, to, tid);
                B.issue(sb, t, to + OA::BYTES, tid);
            }, i0, j0, lane, acc);
        } else {
            typename Elem<T>::Frag va[OA::NLD], vb[OB::NLD];
            A.load(sa, va, 0, tid);
            B.load(sb, vb, 0, tid);
            OA::store(lds, va, tid);
            OB::store(lds + OA::BYTES, vb, tid);
            __syncthreads();
            for (int t = 0; t < steps; ++t) {
                const char* ta = lds + (t & 1) * BUF;
                if (t + 1 < steps) {
                    A.load(sa, va, t + 1, tid);
                    B.load(sb, vb, t + 1, tid);
                }
                Frags<T, AK, BK, S> f;
#pragma unroll
                for (int ks = 0; ks < S::KS; ++ks) {
                    f.read(ta, ks, i0, j0, lane);
                    f.mma(acc);
                }
                if (t + 1 < steps) {
                    char* na = lds + ((t + 1) & 1) * BUF;
                    OA::store(na, va, tid);
                    OB::store(na + OA::BYTES, vb, tid);
                }
                __syncthreads();
            }
        }
    }
};

}  // namespace fra
