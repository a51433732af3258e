// Gated linear recurrence along the time axis of [B, T, D], one independent chain per (sequence, feature), and its backward pass:
//   f = sigmoid(z), k = 1 - f = sigmoid(-z);   h_t = f_t h_{t-1} + k_t x_t,  h_{-1} = h0 (or 0)
//   C_t = f_t (dh_t + C_{t+1}),  C_T = the gradient that arrives at the last state from the segment behind (or 0);
//   with S_t = dh_t + C_{t+1}:  dx_t = k_t S_t;  dz_t = S_t (h_{t-1} - x_t) f_t k_t;  dh0 = C_0
// The step h -> f h + u is an affine map and maps compose: (A, H) stands for h -> A h + H, and (A2, H2) after (A1, H1) is
// (A1 A2, A2 H1 + H2).  A block owns 64 chains; its waves take consecutive pieces of L time steps, compose each piece in registers,
// exchange the 64 maps through LDS, fold the pieces in front of their own onto the incoming state and then run their piece from the
// right state.  Every input is read once and every output written once.  Both passes are bound by memory (3 arrays forward, 6
// backward).  Products of gates only shrink (f <= 1): nothing is divided and no logarithm is taken.
// With few chains the time axis is split over blocks as well: a first launch composes the map of every piece of the axis, the
// second folds the maps in front of its piece and runs it (the gates and inputs are read twice then).
// The order of all operations depends on the sizes alone; there are no atomics and no waits between blocks.
#include <mutex>

#include "vecio.hpp"

namespace {
using namespace vio;

__device__ __forceinline__ float dev_exp(float x) { return expf(x); }
__device__ __forceinline__ double dev_exp(double x) { return exp(x); }

// f = sigmoid(z) and k = sigmoid(-z), both to full relative precision, from one exponential of -|z| (never overflows)
template <typename T> __device__ __forceinline__ void gate(T z, T& f, T& k) {
    const T e = dev_exp(z < T(0) ? z : -z);
    const T big = T(1) / (T(1) + e), small = e * big;
    f = z < T(0) ? small : big;
    k = z < T(0) ? big : small;
}

struct Shape {
    i64 chains, T, D;
    int pieces;   // of the time axis, one per block
    i64 piece;    // time steps of a piece (the last one may be shorter)
    unsigned tiles;  // blocks along the chains
};

// Where chain c starts in [B, T, D]: step t is D elements further on.
__device__ __forceinline__ i64 chain_base(const Shape& s, i64 c) { return (c / s.D) * (s.T * s.D) + c % s.D; }

// W waves, L steps per wave and round.  AGG: only the map of the piece, to aggA / aggH [piece][chain]; else the states.
template <typename T, int W, int L, bool AGG>
__global__ __launch_bounds__(64 * W) void recurrence_fwd_kernel(const T* __restrict__ z, const T* __restrict__ x, const T* __restrict__ h0,
                                                                T* __restrict__ h, T* __restrict__ aggA, T* __restrict__ aggH, const Shape s) {
    __shared__ T mapA[2][W][64], mapH[2][W][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles;
    const i64 chain = (i64)tile * 64 + lane;
    const bool live = chain < s.chains;
    const i64 base = chain_base(s, live ? chain : s.chains - 1);
    const i64 t0 = (i64)piece * s.piece, t1 = min(s.T, t0 + s.piece);
    T carry = T(0), total = T(1);
    if (!AGG) {
        if (h0) carry = h0[live ? chain : s.chains - 1];
        for (unsigned p = 0; p < piece; ++p) {
            const i64 i = (i64)p * s.chains + (live ? chain : s.chains - 1);
            carry = aggA[i] * carry + aggH[i];
        }
    }
    int buf = 0;
    for (i64 r = t0; r < t1; r += W * L, buf ^= 1) {
        const i64 ts = r + wave * L;
        T f[L], u[L];
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const i64 at = base + min(ts + l, s.T - 1) * s.D;
            f[l] = z[at];
            u[l] = x[at];
        }
        T A = T(1), H = T(0);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            T k;
            gate<T>(f[l], f[l], k);
            u[l] = k * u[l];
            if (ts + l >= t1) {  // past the piece: the identity
                f[l] = T(1);
                u[l] = T(0);
            }
            H = f[l] * H + u[l];
            A = A * f[l];
        }
        mapA[buf][wave][lane] = A;
        mapH[buf][wave][lane] = H;
        __syncthreads();  // one per round: the other buffer was last read before the barrier of the round before
        T v = carry;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w == wave) v = carry;
            carry = mapA[buf][w][lane] * carry + mapH[buf][w][lane];
            if (AGG) total = total * mapA[buf][w][lane];
        }
        if (!AGG) {
#pragma unroll
            for (int l = 0; l < L; ++l) {
                v = f[l] * v + u[l];
                if (live && ts + l < t1) h[base + (ts + l) * s.D] = v;
            }
        }
    }
    if (AGG && wave == 0 && live) {
        aggA[(i64)piece * s.chains + chain] = total;
        aggH[(i64)piece * s.chains + chain] = carry;
    }
}

// Backward: the same from the other end.  Piece 0 is the LAST steps; round and wave order run against time.
template <typename T, int W, int L, bool AGG>
__global__ __launch_bounds__(64 * W) void recurrence_bwd_kernel(const T* __restrict__ dh, const T* __restrict__ z, const T* __restrict__ x,
                                                                const T* __restrict__ h, const T* __restrict__ h0, const T* __restrict__ dnext,
                                                                T* __restrict__ dz, T* __restrict__ dx, T* __restrict__ dh0, T* __restrict__ aggA,
                                                                T* __restrict__ aggH, const Shape s) {
    __shared__ T mapA[2][W][64], mapH[2][W][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles;
    const i64 chain = (i64)tile * 64 + lane;
    const bool live = chain < s.chains;
    const i64 cc = live ? chain : s.chains - 1, base = chain_base(s, cc);
    const i64 q0 = (i64)piece * s.piece, q1 = min(s.T, q0 + s.piece);  // counted from the end: q = T - 1 - t
    T carry = T(0), total = T(1);
    if (!AGG) {
        if (dnext) carry = dnext[cc];
        for (unsigned p = 0; p < piece; ++p) carry = aggA[(i64)p * s.chains + cc] * carry + aggH[(i64)p * s.chains + cc];
    }
    int buf = 0;
    for (i64 r = q0; r < q1; r += W * L, buf ^= 1) {
        const i64 qs = r + wave * L;
        T f[L], k[L], g[L], e[L];
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const i64 t = s.T - 1 - min(qs + l, s.T - 1), at = base + t * s.D;
            f[l] = z[at];
            g[l] = dh[at];
            if (!AGG) {
                const T before = t > 0 ? h[at - s.D] : h0 ? h0[cc] : T(0);
                e[l] = before - x[at];
            }
        }
        T A = T(1), H = T(0);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            gate<T>(f[l], f[l], k[l]);
            if (qs + l < q1) {
                H = f[l] * (g[l] + H);
                A = A * f[l];
            }
        }
        mapA[buf][wave][lane] = A;
        mapH[buf][wave][lane] = H;
        __syncthreads();
        T v = carry;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w == wave) v = carry;
            carry = mapA[buf][w][lane] * carry + mapH[buf][w][lane];
            if (AGG) total = total * mapA[buf][w][lane];
        }
        if (!AGG) {
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const T S = g[l] + v;
                if (live && qs + l < q1) {
                    const i64 at = base + (s.T - 1 - (qs + l)) * s.D;
                    dx[at] = k[l] * S;
                    dz[at] = (S * e[l]) * (f[l] * k[l]);
                }
                v = f[l] * S;
            }
        }
    }
    if (AGG) {
        if (wave == 0 && live) {
            aggA[(i64)piece * s.chains + chain] = total;
            aggH[(i64)piece * s.chains + chain] = carry;
        }
    } else if (dh0 && q1 == s.T && wave == 0 && live) {
        dh0[chain] = carry;
    }
}

constexpr int W = 16, L = 8;

int make_shape(fx_ctx* c, Shape& s, i64 B, i64 T, i64 D) {
    s.chains = B * D;
    s.T = T;
    s.D = D;
    const i64 tiles = fx::ceil_div(s.chains, (i64)64);
    // the axis is split when the chains give less than one block to every CU; pieces of whole rounds, at least four of them
    i64 pieces = 1;
    if (tiles < (i64)c->num_cus) pieces = std::max<i64>(1, std::min<i64>(2 * (i64)c->num_cus / tiles, T / (4 * W * L)));
    s.piece = fx::ceil_div(fx::ceil_div(T, pieces), (i64)(W * L)) * (W * L);
    s.pieces = (int)fx::ceil_div(T, s.piece);
    s.tiles = (unsigned)tiles;
    FX_REQUIRE(tiles * s.pieces <= 0x7fffffff, "gated recurrence: too many chains");
    return FX_OK;
}

// the waves of a block: no more than the piece has work for
template <typename F> void with_waves(i64 steps, F&& f) {
    if (steps <= L) f(std::integral_constant<int, 1>());
    else if (steps <= 4 * L) f(std::integral_constant<int, 4>());
    else f(std::integral_constant<int, W>());
}

template <typename T> int check(fx_ctx* c, const char* what, i64 B, i64 steps, i64 D) {
    FX_CHECK_CTX(c);
    FX_REQUIRE(B >= 0 && steps >= 0 && D >= 0, "%s: bad shape [%lld, %lld, %lld]", what, (long long)B, (long long)steps, (long long)D);
    FX_REQUIRE(B < (1ll << 31) && steps < (1ll << 31) && D < (1ll << 31), "%s: dimension exceeds 2^31", what);
    // 64-bit offsets; the product of three dimensions below 2^31 could still pass them
    FX_REQUIRE(D == 0 || steps == 0 || B <= (1ll << 56) / D / steps, "%s: too many elements", what);
    return FX_OK;
}

template <typename T>
int recurrence_fwd(fx_ctx* c, const T* z, const T* x, const T* h0, T* h, i64 B, i64 steps, i64 D) {
    if (int rc = check<T>(c, "fx_gated_recurrence_fwd", B, steps, D)) return rc;
    const i64 n = B * steps * D;
    if (n == 0) return FX_OK;
    FX_REQUIRE(z && x && h, "fx_gated_recurrence_fwd: null pointer");
    FX_REQUIRE(!fx::overlap(h, n, z, n) && !fx::overlap(h, n, x, n) && !fx::overlap(h, n, h0, h0 ? B * D : 0), "fx_gated_recurrence_fwd: the output overlaps an input");
    std::lock_guard<std::mutex> lk(c->launch_mutex);
    Shape s;
    if (int rc = make_shape(c, s, B, steps, D)) return rc;
    T *aggA = nullptr, *aggH = nullptr;
    if (s.pieces > 1) {
        aggA = (T*)c->get_scratch(2 * (i64)s.pieces * s.chains * (i64)sizeof(T));
        if (!aggA) return FX_ERR_OOM;
        aggH = aggA + (i64)s.pieces * s.chains;
        FX_LAUNCH(dim3(s.tiles * (unsigned)(s.pieces - 1)), dim3(64 * W), 0, c->stream, (z, x, h0, h, aggA, aggH, s), recurrence_fwd_kernel<T, W, L, true>);
        FX_LAUNCH_CHECK();
    }
    with_waves(s.piece < steps ? s.piece : steps, [&](auto w) {
        constexpr int WV = decltype(w)::value;
        FX_LAUNCH(dim3(s.tiles * (unsigned)s.pieces), dim3(64 * WV), 0, c->stream, (z, x, h0, h, aggA, aggH, s), recurrence_fwd_kernel<T, WV, L, false>);
    });
    FX_LAUNCH_CHECK();
    return FX_OK;
}

template <typename T>
int recurrence_bwd(fx_ctx* c, const T* dh, const T* z, const T* x, const T* h, const T* h0, const T* dnext, T* dz, T* dx, T* dh0, i64 B, i64 steps, i64 D) {
    if (int rc = check<T>(c, "fx_gated_recurrence_bwd", B, steps, D)) return rc;
    const i64 n = B * steps * D, m = B * D;
    FX_REQUIRE(steps >= 1 || m == 0, "fx_gated_recurrence_bwd: no time steps");
    if (n == 0) return FX_OK;
    FX_REQUIRE(dh && z && x && h && dz && dx, "fx_gated_recurrence_bwd: null pointer");
    const T* ins[] = {dh, z, x, h, h0, dnext};
    T* outs[] = {dz, dx, dh0};
    for (int o = 0; o < 3; ++o) {
        for (int i = 0; i < 6; ++i)
            FX_REQUIRE(!fx::overlap<T>(outs[o], o < 2 ? n : m, ins[i], i < 4 ? n : m), "fx_gated_recurrence_bwd: an output overlaps an input");
        for (int p = 0; p < o; ++p)
            FX_REQUIRE(!fx::overlap<T>(outs[o], o < 2 ? n : m, outs[p], n), "fx_gated_recurrence_bwd: two outputs overlap");
    }
    std::lock_guard<std::mutex> lk(c->launch_mutex);
    Shape s;
    if (int rc = make_shape(c, s, B, steps, D)) return rc;
    T *aggA = nullptr, *aggH = nullptr;
    if (s.pieces > 1) {
        aggA = (T*)c->get_scratch(2 * (i64)s.pieces * s.chains * (i64)sizeof(T));
        if (!aggA) return FX_ERR_OOM;
        aggH = aggA + (i64)s.pieces * s.chains;
        FX_LAUNCH(dim3(s.tiles * (unsigned)(s.pieces - 1)), dim3(64 * W), 0, c->stream, (dh, z, x, h, h0, dnext, dz, dx, dh0, aggA, aggH, s),
                  recurrence_bwd_kernel<T, W, L, true>);
        FX_LAUNCH_CHECK();
    }
    with_waves(s.piece < steps ? s.piece : steps, [&](auto w) {
        constexpr int WV = decltype(w)::value;
        FX_LAUNCH(dim3(s.tiles * (unsigned)s.pieces), dim3(64 * WV), 0, c->stream, (dh, z, x, h, h0, dnext, dz, dx, dh0, aggA, aggH, s),
                  recurrence_bwd_kernel<T, WV, L, false>);
    });
    FX_LAUNCH_CHECK();
    return FX_OK;
}
}  // namespace

#define FX_DEFINE_RECURRENCE(T, S)                                                                                                     \
    extern "C" int fx_gated_recurrence_fwd_##S(fx_ctx* c, const T* z, const T* x, const T* h0, T* h, int64_t B, int64_t steps,          \
                                               int64_t D) {                                                                           \
        return recurrence_fwd<T>(c, z, x, h0, h, B, steps, D);                                                                        \
    }                                                                                                                                  \
    extern "C" int fx_gated_recurrence_bwd_##S(fx_ctx* c, const T* dh, const T* z, const T* x, const T* h, const T* h0,                \
                                               const T* dh_next, T* dz, T* dx, T* dh0, int64_t B, int64_t steps, int64_t D) {          \
        return recurrence_bwd<T>(c, dh, z, x, h, h0, dh_next, dz, dx, dh0, B, steps, D);                                               \
    }
FX_DEFINE_RECURRENCE(float, f32)
FX_DEFINE_RECURRENCE(double, f64)
