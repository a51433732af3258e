// Large f32 matrix products C[M,N] = op(A) . op(B) with both operands staged through LDS in 64-deep slabs, for the
// shapes where the generic implicit-GEMM tile (16-deep slabs, one dword load per element) tops out near 64 % of the
// MFMA peak.  Same product as launch_matmul of the reference (src/backend/cuda/kernels.rs:919-938, cpu.rs:967-1002).
//
// A block (4 waves) owns a BM x BN tile, BM = 32*WM, BN = 32*TN*(4/WM): the waves are laid out WM x (4/WM); a wave owns 32
// rows and 32*TN columns, i.e. TN accumulator blocks of 32x32 (v_mfma_f32_32x32x2_f32).  Large products take 128 x 128 or
// 128 x 64 tiles (WM = 4, TN = 4 or 2; gemm_pipe_kernel, 32-deep stages); products with too few of those to fill the chip (1024^3:
// 64 tiles) take 64 x 128 or 64 x 64 tiles (WM = 2, TN = 2 or 1; gemm_lds_kernel, 64-deep stages) instead of a K split with partial
// sums in memory; with one accumulator block per wave the even and the odd MFMA steps add into two accumulators (added once at the
// end), so that no MFMA waits for the one before it.
// In the 64-deep stages LDS holds both operand slabs in the form their memory layout gives for free:
//   k-contiguous operand (A as stored [M,K]; B given as [N,K]):  S[r][k], pitch 65  -> the 32 lanes of an MFMA operand
//                                                               read (r = lane % 32, k + lane / 32) hit 32 banks
//   row-contiguous operand (A given as [K,M]; B as stored [K,N]): S[k][r], pitch BM / BN -> lanes read 32 consecutive floats
// so staging is a straight copy of 16-byte global loads (four 4-byte LDS stores for the odd pitch, one 16-byte store
// otherwise) and the MFMA loop contains nothing but LDS reads with compile-time offsets.  The next stage's global
// loads are issued before the MFMA loop of the current stage and parked in registers.
// Workgroup ids are handed to the eight XCDs round-robin by the hardware; the id -> tile map gives each XCD a
// contiguous range of tiles so that the tiles resident on one XCD share operand panels in its L2.
#pragma once
#include "gemm_epilogue.hpp"

namespace glk {
using igemm::f32x16;
using igemm::ldg4;

constexpr int KC = 64, NT = 256;
constexpr int PK = KC + 1;  // pitch of a k-contiguous slab row
constexpr size_t LDS_BUDGET_MID = 104 * 1024;  // two stages of the 64-row tiles (one block per CU has to overlap by itself)

struct Params {
    const float* A;
    const float* B;
    float* C;
    const float* bias;  // optional, per column of C; with relu != 0 the sum is clamped at 0 afterwards
    int relu;
    int M, N, K;
    i64 lda, ldb;  // leading dimensions of the operands as stored
    int tiles_n, tiles, xcd_chunk;
    // a batch of independent products of one shape in one launch (blockIdx.y): element strides between them (0: shared operand)
    i64 sa = 0, sb = 0, sc = 0;
    int bias_per_row = 0;  // the bias belongs to the rows of C (a convolution's output channels) instead of its columns
    gep::Epilogue<float> ex;  // EP == EP_FULL
};
constexpr int EP_NONE = 0, EP_BIAS = 1, EP_FULL = 2;  // what the store does: nothing, bias (+ ReLU), the whole of gep::Epilogue

// The store of one wave's 32 x 32 TN block of the tile, rows from m0, columns from n0.  smem: the block's LDS, which nobody reads any more.
template <int TN, int EP, int NACC>
__device__ __forceinline__ void store_tile(const Params& p, float* Cb, float* smem, f32x16 (&acc)[NACC], int m0, int n0, int lane, int wave) {
    const int l32 = lane & 31;
    if constexpr (EP == EP_FULL) {
        // Each wave turns its 32 rows through LDS (its own piece; every wave has left the slabs through the barrier that ended the
        // last stage), 16-byte groups along a row then, so that bias, residual, pre and C move in 16-byte accesses and the
        // activation is compiled for four elements instead of 16 TN.
        constexpr int WC = 32 * TN, CG = WC / 4, RPI = 64 / CG;  // columns of the wave, groups per row, rows per pass
        float* const turn = smem + wave * (32 * WC);
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) turn[igemm::Mfma<float>::row(e, lane) * WC + j * 32 + l32] = acc[j][e];
        __syncthreads();
        const int n = n0 + 4 * (lane % CG), left = p.N - n;
        float bias[4] = {0.f, 0.f, 0.f, 0.f};
        if (p.ex.bias) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q < left) bias[q] = p.ex.bias[n + q];
        }
#pragma unroll 1
        for (int r = lane / CG; r < 32; r += RPI) {
            const int m = m0 + r;
            if (m >= p.M || left <= 0) continue;
            const i64 i = (i64)m * p.N + n;
            const float4 t4 = *reinterpret_cast<const float4*>(turn + r * WC + 4 * (lane % CG));
            float v[4] = {t4.x, t4.y, t4.z, t4.w}, res[4] = {0.f, 0.f, 0.f, 0.f};
            typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // a row of C starts at any element
            if (p.ex.residual) {
                if (left >= 4) {
                    const f4u q4 = *reinterpret_cast<const f4u*>(p.ex.residual + i);
                    res[0] = q4.x; res[1] = q4.y; res[2] = q4.z; res[3] = q4.w;
                } else {
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        if (q < left) res[q] = p.ex.residual[i + q];
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (p.ex.bias) v[q] = v[q] + bias[q];
            if (p.ex.pre) {
                if (left >= 4) {
                    *reinterpret_cast<f4u*>(p.ex.pre + i) = f4u{v[0], v[1], v[2], v[3]};
                } else {
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        if (q < left) p.ex.pre[i + q] = v[q];
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[q] = fxact::apply<float>(p.ex.act, v[q]);
                if (p.ex.residual) v[q] = v[q] + res[q];
            }
            if (left >= 4) {
                *reinterpret_cast<f4u*>(Cb + i) = f4u{v[0], v[1], v[2], v[3]};
            } else {
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    if (q < left) Cb[i + q] = v[q];
            }
        }
        return;
    }
    constexpr bool BIAS = EP == EP_BIAS;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = n0 + j * 32 + l32;
        const float bj = BIAS && !p.bias_per_row ? p.bias[n < p.N ? n : p.N - 1] : 0.f;
        if (n < p.N) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + igemm::Mfma<float>::row(e, lane);
                if (m < p.M) {
                    float v = acc[j][e];
                    if (BIAS) {
                        v = v + (p.bias_per_row ? p.bias[m] : bj);
                        if (p.relu) v = v > 0.f ? v : 0.f;
                    }
                    Cb[(i64)m * p.N + n] = v;
                }
            }
        }
    }
}

// TA: A is stored [K, M] (m contiguous); TB: B is stored [N, K] (k contiguous).
// KT (both operands k-contiguous only): K need not be a multiple of the stage depth -- the last stage loads what is left of the rows
// (K a multiple of 4: a 16-byte vector is inside a row or past it) and parks zeros behind it.
// The 64-row tiles (WM = 2).  They run where there is about one block per CU, so LDS keeps two stages: the next stage is parked while
// other waves still compute and a stage costs one barrier.
template <int TN, bool TA, bool TB, int EP, bool KT = false>
__global__ __launch_bounds__(NT, 2) void gemm_lds_kernel(const Params p) {
    static_assert(!KT || (!TA && TB), "the K tail is handled for k-contiguous operands");
    constexpr int WM = 2, WN = 4 / WM, BM = 32 * WM, BN = 32 * TN * WN;
    constexpr int NACC = TN == 1 ? 2 : TN;  // accumulator blocks of a wave (TN == 1: even and odd MFMA steps apart)
    constexpr int PA = TA ? BM : PK, PB = TB ? PK : BN;          // LDS pitches
    constexpr int ASZ = TA ? KC * BM : BM * PK, BSZ = TB ? BN * PK : KC * BN;
    constexpr int NA = BM * KC / 4 / NT, NB = BN * KC / 4 / NT;  // float4 per thread per stage
    static_assert(BN * KC % (4 * NT) == 0, "B slab must divide over the block");
    FX_DYNAMIC_SMEM(float, smem);
    float* As = smem;
    float* Bs = smem + ASZ;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
    const int wm = wave % WM, wn = wave / WM;
    const float* const Ab = p.A + (i64)blockIdx.y * p.sa;
    const float* const Bb = p.B + (i64)blockIdx.y * p.sb;
    float* const Cb = p.C + (i64)blockIdx.y * p.sc;

    // id -> tile: XCD x gets tiles [x * chunk, (x+1) * chunk) when the tile count divides by 8
    int tile = blockIdx.x;
    if (p.xcd_chunk) tile = (tile & 7) * p.xcd_chunk + (tile >> 3);
    const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
    const int m0 = tm * BM, n0 = tn * BN;

    f32x16 acc[NACC];
#pragma unroll
    for (int j = 0; j < NACC; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;

    // staging maps.  k-contiguous slab: thread t owns float4 column t % 16 (k = 4*(t%16)..+3) of rows t/16 + 16u.
    // row-contiguous slab of R floats per k: thread t owns float4 column t % (R/4) of k rows t/(R/4) + (NT/(R/4))u.
    uint32_t a_off[NA], b_off[NB];
    if (!TA) {
#pragma unroll
        for (int u = 0; u < NA; ++u) {
            const int r = min(m0 + (tid >> 4) + 16 * u, p.M - 1);  // rows past the matrix re-read its last row
            a_off[u] = (uint32_t)((i64)r * p.lda + 4 * (tid & 15)) * 4u;
        }
    } else {
        constexpr int Q = BM / 4, RS = NT / Q;  // float4 per k row, k rows per pass
        const int c4 = min(m0 + 4 * (tid % Q), p.M - 4);
#pragma unroll
        for (int u = 0; u < NA; ++u) a_off[u] = (uint32_t)((i64)(tid / Q + RS * u) * p.lda + c4) * 4u;
    }
    if (TB) {
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            const int r = min(n0 + (tid >> 4) + 16 * u, p.N - 1);
            b_off[u] = (uint32_t)((i64)r * p.ldb + 4 * (tid & 15)) * 4u;
        }
    } else {
        constexpr int Q = BN / 4, RS = NT / Q;  // float4 per k row, k rows per pass
        const int c4 = min(n0 + 4 * (tid % Q), p.N - 4);
#pragma unroll
        for (int u = 0; u < NB; ++u) b_off[u] = (uint32_t)((i64)(tid / Q + RS * u) * p.ldb + c4) * 4u;
    }
    float4 av[NA], bv[NB];
    bool dead = false;  // KT: this thread's four k of the stage in flight lie past K (its loads re-read the stage's first vector)
    auto prefetch = [&](int k0) {
        const float* a = TA ? Ab + (i64)k0 * p.lda : Ab + k0;
        const float* b = TB ? Bb + k0 : Bb + (i64)k0 * p.ldb;
        uint32_t back = 0;
        if constexpr (KT) {
            dead = k0 + 4 * (tid & 15) >= p.K;
            back = dead ? 16u * (tid & 15) : 0u;
        }
#pragma unroll
        for (int u = 0; u < NA; ++u) av[u] = ldg4(a, a_off[u] - back);
#pragma unroll
        for (int u = 0; u < NB; ++u) bv[u] = ldg4(b, b_off[u] - back);
    };
    auto park = [&](int buf) {
        int t = tid;
        FX_PIN_VGPR(t);  // recompute the LDS addresses here instead of keeping them alive over the MFMA loop
        float* const As = smem + buf * (ASZ + BSZ);
        float* const Bs = As + ASZ;
        if constexpr (KT) {
            if (dead) {
#pragma unroll
                for (int u = 0; u < NA; ++u) av[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int u = 0; u < NB; ++u) bv[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        if (!TA) {
#pragma unroll
            for (int u = 0; u < NA; ++u) {
                float* d = As + ((t >> 4) + 16 * u) * PK + 4 * (t & 15);
                d[0] = av[u].x; d[1] = av[u].y; d[2] = av[u].z; d[3] = av[u].w;
            }
        } else {
            constexpr int Q = BM / 4, RS = NT / Q;
#pragma unroll
            for (int u = 0; u < NA; ++u) *reinterpret_cast<float4*>(As + (t / Q + RS * u) * BM + 4 * (t % Q)) = av[u];
        }
        if (TB) {
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                float* d = Bs + ((t >> 4) + 16 * u) * PK + 4 * (t & 15);
                d[0] = bv[u].x; d[1] = bv[u].y; d[2] = bv[u].z; d[3] = bv[u].w;
            }
        } else {
            constexpr int Q = BN / 4, RS = NT / Q;
#pragma unroll
            for (int u = 0; u < NB; ++u) *reinterpret_cast<float4*>(Bs + (t / Q + RS * u) * BN + 4 * (t % Q)) = bv[u];
        }
    };

    // operand reads of MFMA step s (k = 2s, 2s+1; lane half h takes k = 2s + h)
    const float* const ar = TA ? As + half * PA + wm * 32 + l32 : As + (wm * 32 + l32) * PA + half;
    const float* const br = TB ? Bs + (wn * 32 * TN + l32) * PB + half : Bs + half * PB + wn * 32 * TN + l32;
    auto compute = [&](int buf) {
        float a0, b0[TN], a1, b1[TN];
        const float* const arb = ar + buf * (ASZ + BSZ);
        const float* const brb = br + buf * (ASZ + BSZ);
        auto rd = [&](float& a, float (&b)[TN], int s) {
            a = TA ? arb[2 * s * PA] : arb[2 * s];
#pragma unroll
            for (int j = 0; j < TN; ++j) b[j] = TB ? brb[j * 32 * PB + 2 * s] : brb[2 * s * PB + j * 32];
            __builtin_amdgcn_sched_barrier(0);
        };
        auto mma = [&](float a, const float (&b)[TN], int parity) {
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int q = TN == 1 ? parity : j;
                acc[q] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b[j], acc[q], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        // one block per CU, one wave per SIMD: the operand reads run two MFMA steps ahead (three register sets), which
        // covers the LDS latency that a second wave would otherwise hide
        float a2, b2[TN];
        rd(a0, b0, 0);
        rd(a1, b1, 1);
#pragma unroll
        for (int s = 0; s < KC / 2; s += 6) {
            if (s + 2 < KC / 2) rd(a2, b2, s + 2);
            mma(a0, b0, 0);
            if (s + 3 < KC / 2) rd(a0, b0, s + 3);
            mma(a1, b1, 1);
            if (s + 2 < KC / 2) {
                if (s + 4 < KC / 2) rd(a1, b1, s + 4);
                mma(a2, b2, 0);
            }
            if (s + 3 < KC / 2) {
                if (s + 5 < KC / 2) rd(a2, b2, s + 5);
                mma(a0, b0, 1);
            }
            if (s + 4 < KC / 2) {
                if (s + 6 < KC / 2) rd(a0, b0, s + 6);
                mma(a1, b1, 0);
            }
            if (s + 5 < KC / 2) {
                if (s + 7 < KC / 2) rd(a1, b1, s + 7);
                mma(a2, b2, 1);
            }
        }
    };

    prefetch(0);
    park(0);
    __syncthreads();
    int cur = 0;
    for (int k0 = 0; k0 < p.K; k0 += KC) {
        const bool more = k0 + KC < p.K;
        if (more) prefetch(k0 + KC);
        compute(cur);
        // the other buffer was last read in the stage before this one, which every wave has left through the barrier below
        if (more) park(cur ^ 1);
        __syncthreads();
        cur ^= 1;
    }

    if constexpr (TN == 1) {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[0][e] = acc[0][e] + acc[1][e];
    }
    store_tile<TN, EP>(p, Cb, smem, acc, m0 + wm * 32, n0 + wn * 32 * TN, lane, wave);
}

// The 128-row tiles (WM = 4), with two stages of 32 k in LDS and two more on their way in registers.  While a stage is computed, the
// next one goes from registers into the other buffer and the one three ahead is fetched, piece by piece between the MFMAs, so a
// stage costs one barrier and no wave ever waits for staging alone; k runs upwards in pairs as in gemm_lds_kernel.
//   k-contiguous operand: a row's even k, then its odd k (lane half h of an MFMA takes k = 2 s + h), pitch 36: one 16-byte LDS read
//                         feeds four MFMA steps; 16 rows of a read cover all banks.
//   row-contiguous operand: S[k][r] as above, one 4-byte read per step.
// Bound by the matrix pipe.  Measured (f32, NN / NT / TN / TT, TFLOP/s; in brackets one 64-deep stage per block, computing and staging in
// turns, as before): 4096 x 1024 x 4096 131 / 134 / 134 / 138 (117 / 123 / 125 / 121), 4096 x 4096 x 1024 132 / 133 / 133 / 134
// (124 / 125 / 127 / 126), 2048^3 128 / 134 / 131 / 134 (116 / 120 / 122 / 119); 4096^3 138 to 140 of 157.
// A . B^T in 128 x 64 tiles: B's rows without padding, their eight 16-byte groups permuted by the row (group q of row r lies at
// q ^ (r / 2 % 8): 16 rows of a read cover all banks as well), so that three blocks fit on a CU as in the other forms; with the padding
// two did, and products of several rounds of blocks lost by it (3000 x 3000 x 4096 735 us, so 622; 5000 x 5000 x 128 73.6, so 68.2).
constexpr int KP = 32, PP = KP + 4;
template <int TN, bool TA, bool TB> constexpr bool pipe_permuted() { return TN == 2 && !TA && TB; }
template <int TN, bool TA, bool TB> constexpr int pipe_b_pitch() { return TB ? (pipe_permuted<TN, TA, TB>() ? KP : PP) : 32 * TN; }
template <int TN, bool TA, bool TB> constexpr int pipe_stage_floats() {
    return (TA ? KP * 128 : 128 * PP) + (TB ? 32 * TN : KP) * pipe_b_pitch<TN, TA, TB>();
}
template <int TN, bool TA, bool TB, int EP, bool KT = false>
__global__ __launch_bounds__(NT, 2) void gemm_pipe_kernel(const Params p) {
    static_assert(!KT || (!TA && TB), "the K tail is handled for k-contiguous operands");
    constexpr int BM = 128, BN = 32 * TN;
    constexpr int ASZ = TA ? KP * BM : BM * PP, STAGE = pipe_stage_floats<TN, TA, TB>();
    constexpr bool PERM = pipe_permuted<TN, TA, TB>();
    constexpr int PB = pipe_b_pitch<TN, TA, TB>();
    constexpr int NA = BM * KP / 4 / NT, NB = BN * KP / 4 / NT;  // float4 per thread per stage
    FX_DYNAMIC_SMEM(float, smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
    const float* const Ab = p.A + (i64)blockIdx.y * p.sa;
    const float* const Bb = p.B + (i64)blockIdx.y * p.sb;
    float* const Cb = p.C + (i64)blockIdx.y * p.sc;
    int tile = blockIdx.x;
    if (p.xcd_chunk) tile = (tile & 7) * p.xcd_chunk + (tile >> 3);
    const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
    const int m0 = tm * BM, n0 = tn * BN;

    f32x16 acc[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;

    // staging maps.  k-contiguous: thread t owns float4 t % 8 (k = 4 (t % 8) ..) of rows t / 8 + 32 u; row-contiguous, R floats per k:
    // float4 t % (R / 4) of k rows t / (R / 4) + (NT / (R / 4)) u.  Rows past the matrix re-read its last row.
    uint32_t a_off[NA], b_off[NB];
    if (!TA) {
#pragma unroll
        for (int u = 0; u < NA; ++u) a_off[u] = (uint32_t)((i64)min(m0 + (tid >> 3) + 32 * u, p.M - 1) * p.lda + 4 * (tid & 7)) * 4u;
    } else {
        constexpr int Q = BM / 4, RS = NT / Q;
        const int c4 = min(m0 + 4 * (tid % Q), p.M - 4);
#pragma unroll
        for (int u = 0; u < NA; ++u) a_off[u] = (uint32_t)((i64)(tid / Q + RS * u) * p.lda + c4) * 4u;
    }
    if (TB) {
#pragma unroll
        for (int u = 0; u < NB; ++u) b_off[u] = (uint32_t)((i64)min(n0 + (tid >> 3) + 32 * u, p.N - 1) * p.ldb + 4 * (tid & 7)) * 4u;
    } else {
        constexpr int Q = BN / 4, RS = NT / Q;
        const int c4 = min(n0 + 4 * (tid % Q), p.N - 4);
#pragma unroll
        for (int u = 0; u < NB; ++u) b_off[u] = (uint32_t)((i64)(tid / Q + RS * u) * p.ldb + c4) * 4u;
    }
    typedef float f32x4 __attribute__((ext_vector_type(4)));  // one value for the compiler, not four: it stays in its four registers
    f32x4 v[2][NA + NB];            // two stages on their way
    bool past[2] = {false, false};  // KT: this thread's four k of the stage lie past K (its loads re-read the stage's first vector)
    // unit u of a stage's staging: one 16-byte load, and later its way into LDS
    auto fetch = [&](int set, int k0, int u) __attribute__((always_inline)) {
        uint32_t back = 0;
        if constexpr (KT) {
            past[set] = k0 + 4 * (tid & 7) >= p.K;
            back = past[set] ? 16u * (tid & 7) : 0u;
        }
        const float* const base = u < NA ? (TA ? Ab + (i64)k0 * p.lda : Ab + k0) : (TB ? Bb + k0 : Bb + (i64)k0 * p.ldb);
        const uint32_t off = u < NA ? a_off[u < NA ? u : 0] : b_off[u < NA ? 0 : u - NA];
        v[set][u] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(base) + (off - back));
    };
    auto park = [&](int set, int buf, int u) __attribute__((always_inline)) {
        f32x4& x = v[set][u];
        // the loaded values are first touched here: left alone, the compiler rearranges them for the write right behind the load and
        // waits for memory there
        FX_PIN_VGPR(x);
        if constexpr (KT) {
            if (past[set]) x = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const bool is_a = u < NA, kc = is_a ? !TA : TB;  // k-contiguous: even k, then odd k
        const int R = is_a ? BM : BN, Q = R / 4, w = is_a ? u : u - NA;
        float* const d = smem + buf * STAGE + (is_a ? 0 : ASZ);
        if (kc && !is_a && PERM) {
            const int row = (tid >> 3) + 32 * w, q = ((tid & 7) >> 1) ^ (row >> 1 & 7);
            float* const r = d + row * PB + 2 * (tid & 1);
            *reinterpret_cast<float2*>(r + 4 * q) = make_float2(x.x, x.z);
            *reinterpret_cast<float2*>(r + 4 * (q ^ 4)) = make_float2(x.y, x.w);
        } else if (kc) {
            float* const r = d + ((tid >> 3) + 32 * w) * PP + 2 * (tid & 7);
            *reinterpret_cast<float2*>(r) = make_float2(x.x, x.z);
            *reinterpret_cast<float2*>(r + KP / 2) = make_float2(x.y, x.w);
        } else {
            *reinterpret_cast<f32x4*>(d + (tid / Q + NT / Q * w) * R + 4 * (tid % Q)) = x;
        }
    };

    // operands of four MFMA steps (group g: steps 4 g .. 4 g + 3)
    const float* const ar = TA ? smem + half * BM + wave * 32 + l32 : smem + (wave * 32 + l32) * PP + half * (KP / 2);
    const float* const br = TB ? smem + ASZ + l32 * PB + (PERM ? 0 : half * (KP / 2)) : smem + ASZ + half * BN + l32;
    int group[4];  // PERM: where groups 0 .. 3 of this lane's half lie in its rows (l32 and l32 + 32 are permuted alike)
#pragma unroll
    for (int g = 0; g < 4; ++g) group[g] = PERM ? 4 * ((4 * half + g) ^ (l32 >> 1 & 7)) : 4 * g;
    auto read = [&](float (&a)[4], float (&b)[TN][4], int buf, int g) __attribute__((always_inline)) {
        const float* const x = ar + buf * STAGE;
        const float* const y = br + buf * STAGE;
        if (TA) {
#pragma unroll
            for (int q = 0; q < 4; ++q) a[q] = x[2 * (4 * g + q) * BM];
        } else {
            const float4 v = *reinterpret_cast<const float4*>(x + 4 * g);
            a[0] = v.x; a[1] = v.y; a[2] = v.z; a[3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            if (TB) {
                const float4 v = *reinterpret_cast<const float4*>(y + j * 32 * PB + group[g]);
                b[j][0] = v.x; b[j][1] = v.y; b[j][2] = v.z; b[j][3] = v.w;
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) b[j][q] = y[2 * (4 * g + q) * BN + j * 32];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // One step's MFMAs, then what `between` puts behind them: the matrix pipe works for 64 cycles per instruction, staging slips in.
    auto mma = [&](const float (&a)[4], const float (&b)[TN][4], auto&& between) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[q], b[j][q], acc[j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            between(q);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    float a0[4], b0[TN][4], a1[4], b1[TN][4];
    // One stage, in buffer `buf`, whose first group is in (a0, b0).  Set `set` holds the next stage, which goes into the other buffer
    // (last read in the stage before this one, which every wave has left through the barrier below), and takes the third one from here.
    // The barrier comes before the last group: its MFMAs cover the first reads of the next stage.  Nothing here is conditional -- past
    // the end the last stage is loaded once more, parked and never read -- since a branch around a load makes its result a copy of the
    // loaded registers, and the copy waits for memory on the spot.
    constexpr int UNITS = NA + NB, PER = (UNITS + 7) / 8;
    const int k_last = (p.K - 1) / KP * KP;
    auto stage = [&](int k0, int set, int buf) __attribute__((always_inline)) {
        const int k3 = min(k0 + 3 * KP, k_last);
        auto put = [&](int s) __attribute__((always_inline)) {
#pragma unroll
            for (int u = s * PER; u < (s + 1) * PER && u < UNITS; ++u) park(set, buf ^ 1, u);
        };
        read(a1, b1, buf, 1);
        mma(a0, b0, [&](int q) __attribute__((always_inline)) { put(q); });
        read(a0, b0, buf, 2);
        mma(a1, b1, [&](int q) __attribute__((always_inline)) { put(4 + q); });
        read(a1, b1, buf, 3);
        mma(a0, b0, [&](int q) __attribute__((always_inline)) {
#pragma unroll
            for (int u = q * 2 * PER; u < (q + 1) * 2 * PER && u < UNITS; ++u) fetch(set, k3, u);
        });
        __syncthreads();
        read(a0, b0, buf ^ 1, 0);
        mma(a1, b1, [](int) {});
    };
#pragma unroll
    for (int u = 0; u < UNITS; ++u) fetch(0, 0, u);
    __builtin_amdgcn_sched_barrier(0);  // the loads in the order in which the loop waits for them
#pragma unroll
    for (int u = 0; u < UNITS; ++u) fetch(1, min(KP, k_last), u);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) park(0, 0, u);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) fetch(0, min(2 * KP, k_last), u);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    read(a0, b0, 0, 0);
    int k0 = 0;
    for (; k0 + KP < p.K; k0 += 2 * KP) {
        stage(k0, 1, 0);
        stage(k0 + KP, 0, 1);
    }
    if constexpr (KT) {
        if (k0 < p.K) stage(k0, 1, 0);  // an odd number of stages (without a tail K is a multiple of two)
    }
    if constexpr (EP == EP_FULL) __syncthreads();  // the turn through LDS below: the last stage's readers are all through
    store_tile<TN, EP>(p, Cb, smem, acc, m0 + wave * 32, n0, lane, wave);
}

struct Plan {
    bool ok = false;
    int TN = 4, WM = 4, tiles_m = 0, tiles_n = 0;
    size_t smem = 0;
    int bm() const { return 32 * WM; }
    int bn() const { return 32 * TN * (4 / WM); }
};

// Taken for products that fill the chip without a K split: K a multiple of the 64-deep slab, 16-byte aligned rows,
// row-contiguous operands with a multiple of 4 rows, every byte offset inside a tile below 4 GiB.  batch: independent
// products of this shape that share the launch (their tiles count towards filling the chip).
inline Plan make_plan(int num_cus, bool ta, bool tb, i64 M, i64 N, i64 K, i64 lda, i64 ldb, i64 batch = 1) {
    Plan pl;
    // (a K that is no multiple of the stage depth: only with both operands k-contiguous, see KT in the kernel)
    if (K < 2 * KC || (K % KC != 0 && !(K % 4 == 0 && !ta && tb)) || lda % 4 != 0 || ldb % 4 != 0 || M < 64 || N < 64) return pl;
    if ((ta && M % 4 != 0) || (!tb && N % 4 != 0)) return pl;
    // tile shape: the one with the least (rounds of co-resident blocks) x (work of a block); a nearly empty last round
    // costs as much as a full one (3000 x 3000: 576 tiles of 128 x 128 take two rounds, 1128 of 128 x 64 take 2.2).  The
    // work of a block is its MFMA count weighted by what the tile reads per MFMA (narrower tiles re-read more).
    const i64 slots = 2 * (i64)std::max(1, num_cus);
    static const int shapes[4][3] = {{4, 4, 8}, {4, 2, 9}, {2, 2, 10}, {2, 1, 11}};  // WM, TN, cost per 32 x 32 block
    i64 best = -1, tiles = 0;
    for (const auto& sh : shapes) {
        const int wmv = sh[0], tn = sh[1], bm = 32 * wmv, bn = 32 * tn * (4 / wmv);
        if (M < bm) continue;
        const i64 t = fx::ceil_div(M, (i64)bm) * fx::ceil_div(N, (i64)bn) * batch;
        // fewer tiles than 3/4 of the block slots: a smaller tile, or (below half a block per CU even with the smallest)
        // the generic kernel's K split
        if (wmv == 4 ? t < slots * 3 / 4 : t < slots / 4) continue;
        const i64 cost = fx::ceil_div(t, slots) * (bm / 32) * (bn / 32) * sh[2];
        if (best < 0 || cost < best) {
            best = cost;
            pl.TN = tn;
            pl.WM = wmv;
            tiles = t;
        }
    }
    if (best < 0 || tiles > 0x7fffffff || batch > 65535) return pl;
    pl.tiles_m = (int)fx::ceil_div(M, (i64)pl.bm());
    pl.tiles_n = (int)fx::ceil_div(N, (i64)pl.bn());
    const i64 a_span = ta ? (i64)KC * lda + M : (i64)M * lda, b_span = tb ? (i64)N * ldb : (i64)KC * ldb + N;
    if (a_span * 4 >= (1ll << 32) || b_span * 4 >= (1ll << 32)) return pl;
    if (pl.WM == 2) {  // (the 128-row tiles' LDS goes by their template arguments)
        pl.smem = (size_t)((ta ? KC * pl.bm() : pl.bm() * PK) + (tb ? pl.bn() * PK : KC * pl.bn())) * sizeof(float) * 2;
        if (pl.smem > LDS_BUDGET_MID) return pl;
    }
    pl.ok = true;
    return pl;
}

template <int TN, bool TA, bool TB, int EP, bool KT> inline int launch_pipe_ep(fx_ctx* c, const Params& p, dim3 grid, dim3 blk) {
    constexpr size_t lds = 2 * sizeof(float) * pipe_stage_floats<TN, TA, TB>();
    static_assert(TN != 2 || 3 * lds <= 160 * 1024, "three blocks of the 128 x 64 tiles share a CU's LDS");
    static const hipError_t attr = hipFuncSetAttribute((const void*)gemm_pipe_kernel<TN, TA, TB, EP, KT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    FX_HIP_CHECK(attr);
    FX_LAUNCH(grid, blk, lds, c->stream, (p), gemm_pipe_kernel<TN, TA, TB, EP, KT>);
    FX_LAUNCH_CHECK();
    return FX_OK;
}
template <int TN, bool TA, bool TB, bool KT> inline int launch_pipe(fx_ctx* c, const Params& p, dim3 grid, dim3 blk) {
    if (p.ex.any()) return launch_pipe_ep<TN, TA, TB, EP_FULL, KT>(c, p, grid, blk);
    if (p.bias) return launch_pipe_ep<TN, TA, TB, EP_BIAS, KT>(c, p, grid, blk);
    return launch_pipe_ep<TN, TA, TB, EP_NONE, KT>(c, p, grid, blk);
}

template <int TN, int WM, bool TA, bool TB, bool KT = false>
inline int launch(fx_ctx* c, const Plan& pl, const Params& p, int batch) {
    const dim3 grid((unsigned)p.tiles, (unsigned)batch), blk(NT);
    if constexpr (!KT && !TA && TB) {
        if (p.K % KC != 0) return launch<TN, WM, TA, TB, true>(c, pl, p, batch);
    }
    if constexpr (WM == 4) {
        return launch_pipe<TN, TA, TB, KT>(c, p, grid, blk);
    } else {
        constexpr int budget = (int)LDS_BUDGET_MID;
        static const hipError_t attr0 = hipFuncSetAttribute((const void*)gemm_lds_kernel<TN, TA, TB, EP_NONE, KT>,
                                                            hipFuncAttributeMaxDynamicSharedMemorySize, budget);
        static const hipError_t attr1 = hipFuncSetAttribute((const void*)gemm_lds_kernel<TN, TA, TB, EP_BIAS, KT>,
                                                            hipFuncAttributeMaxDynamicSharedMemorySize, budget);
        FX_HIP_CHECK(attr0);
        FX_HIP_CHECK(attr1);
        if (p.ex.any()) {
            static const hipError_t attr2 = hipFuncSetAttribute((const void*)gemm_lds_kernel<TN, TA, TB, EP_FULL, KT>,
                                                                hipFuncAttributeMaxDynamicSharedMemorySize, budget);
            FX_HIP_CHECK(attr2);
            FX_LAUNCH(grid, blk, pl.smem, c->stream, (p), gemm_lds_kernel<TN, TA, TB, EP_FULL, KT>);
        } else if (p.bias) FX_LAUNCH(grid, blk, pl.smem, c->stream, (p), gemm_lds_kernel<TN, TA, TB, EP_BIAS, KT>);
        else FX_LAUNCH(grid, blk, pl.smem, c->stream, (p), gemm_lds_kernel<TN, TA, TB, EP_NONE, KT>);
        FX_LAUNCH_CHECK();
        return FX_OK;
    }
}
template <bool TA, bool TB>
inline int launch_tn(fx_ctx* c, const Plan& pl, const Params& p, int batch) {
    if (pl.WM == 4) return pl.TN == 4 ? launch<4, 4, TA, TB>(c, pl, p, batch) : launch<2, 4, TA, TB>(c, pl, p, batch);
    return pl.TN == 2 ? launch<2, 2, TA, TB>(c, pl, p, batch) : launch<1, 2, TA, TB>(c, pl, p, batch);
}

// A, B and C must be 16-byte aligned.  batch > 1: `batch` products in one launch, operand / result k of the batch sa / sb / sc
// elements after the first (a stride of 0 shares the operand); bias_per_row: the bias is indexed by the row of C.  ex: one product
// without bias / relu of its own, the epilogue ex in its store.
inline int run(fx_ctx* c, const Plan& pl, bool ta, bool tb, i64 M, i64 N, i64 K, const float* A, const float* B, float* C,
               const float* bias, int relu, i64 batch = 1, i64 sa = 0, i64 sb = 0, i64 sc = 0, int bias_per_row = 0,
               const gep::Epilogue<float>& ex = gep::Epilogue<float>()) {
    Params p;
    p.A = A; p.B = B; p.C = C; p.bias = bias; p.relu = relu;
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    p.lda = ta ? M : K;
    p.ldb = tb ? K : N;
    p.tiles_n = pl.tiles_n;
    p.tiles = pl.tiles_m * pl.tiles_n;
    p.xcd_chunk = p.tiles % 8 == 0 ? p.tiles / 8 : 0;
    p.sa = sa; p.sb = sb; p.sc = sc; p.bias_per_row = bias_per_row;
    p.ex = ex;
    if (!ta && !tb) return launch_tn<false, false>(c, pl, p, (int)batch);
    if (!ta && tb) return launch_tn<false, true>(c, pl, p, (int)batch);
    if (ta && !tb) return launch_tn<true, false>(c, pl, p, (int)batch);
    return launch_tn<true, true>(c, pl, p, (int)batch);
}

}  // namespace glk
