// Gated linear recurrence along the time axis of [B, T, D], one independent chain per (sequence, feature), and its backward pass:
//   f = sigmoid(z), k = 1 - f = sigmoid(-z);   h_t = f_t h_{t-1} + k_t x_t,  h_{-1} = h0 (or 0)
//   C_t = f_t (dh_t + C_{t+1}),  C_T = the gradient that arrives at the last state from the segment behind (or 0);
//   with S_t = dh_t + C_{t+1}:  dx_t = k_t S_t;  dz_t = S_t (h_{t-1} - x_t) f_t k_t;  dh0 = C_0
// The step h -> f h + u is an affine map and maps compose: (A, H) stands for h -> A h + H, and (A2, H2) after (A1, H1) is
// (A1 A2, A2 H1 + H2).  A block owns 64 chains and one piece of the time axis: W waves of L steps each, whose inputs it reads once into
// registers.  Every wave composes the map of its L steps, the waves exchange them through LDS, and each then runs its steps from the
// right state and writes once: both passes are bound by memory (3 arrays forward, 6 backward) and move each byte once.  Products of gates
// only shrink (f <= 1): nothing is divided and no logarithm is taken.
//
// A sequence of more than one piece is run by several blocks in ONE launch.  A block publishes its piece's map before it waits for
// anything, then collects the maps of the pieces in front of it (back to the last piece whose number is a multiple of GROUP, which
// also publishes the state it ended in, so that no block collects more than GROUP maps).
//   - Which piece of its 64 chains a block runs is its ticket from a counter that these chains have to themselves (one counter for all
//     served 80 blocks per microsecond and bounded the launch), so every piece it waits for has been taken by a block that is running
//     already and publishes after a bounded amount of work of its own: every wait ends.  (A wait that lasted for millions of polls all
//     the same would give up and yield NaN instead of hanging; by the order of the tickets none can.)
//   - A published value is whole in one 64-bit word (f32: A and H; f64: one word each), written and read by relaxed device-scope
//     atomics; no other memory is handed over, so no fence is needed.  Words start as all ones, a pattern that no published value has
//     (NaNs are replaced by the standard one first); a small kernel sets them and the counters before every launch.
//   - Maps are folded in the order of the pieces, whenever they arrive: the result does not depend on timing.
// Measured (MI355X): 2 x 8192 x 1024 f32 forward 50 us with the clearing, 201 MB at 4.0 TB/s (two launches, the first composing the maps of
// all pieces and reading the inputs once more: 75 us); 16 x 511 x 1000 f64 backward 90 us, 393 MB at 4.4 TB/s (one block per 64 chains
// that walks the axis: 106 us).
#include <mutex>
#include <type_traits>

#include "vecio.hpp"

namespace {
using namespace vio;

__device__ __forceinline__ float dev_exp(float x) { return expf(x); }
__device__ __forceinline__ double dev_exp(double x) { return exp(x); }

typedef unsigned long long u64;

// f = sigmoid(z) and k = sigmoid(-z), both to full relative precision, from one exponential of -|z| (never overflows)
template <typename T> __device__ __forceinline__ void gate(T z, T& f, T& k) {
    const T e = dev_exp(z < T(0) ? z : -z);
    const T big = T(1) / (T(1) + e), small = e * big;
    f = z < T(0) ? small : big;
    k = z < T(0) ? big : small;
}

// A product of gates that underflows though none of them is 0 is held as minus zero: an infinite state stays infinite under it, and
// becomes NaN under a product with a gate of 0.  Both products times infinity are NaN, so the maps are folded plainly, and once more by
// the functions below only where the result is NaN.
__device__ __forceinline__ bool is_minus_zero(float a) { return __float_as_uint(a) == 0x80000000u; }
__device__ __forceinline__ bool is_minus_zero(double a) { return (u64)__double_as_longlong(a) == 1ull << 63; }
// of gates, the smallest of them `least`
template <typename T> __device__ __forceinline__ T product_of(T A, T least) { return A == T(0) && least > T(0) ? -T(0) : A; }
// of two products
template <typename T> __device__ __forceinline__ T times(T a, T b) {
    const T p = a * b;
    if (p != T(0)) return p;  // NaN too
    return (a > T(0) || is_minus_zero(a)) && (b > T(0) || is_minus_zero(b)) ? -T(0) : T(0);
}
// the map (A, H) of the state v
template <typename T> __device__ __forceinline__ T mapped(T A, T H, T v) {
    const T r = A * v + H;
    return r != r && is_minus_zero(A) && v - v != T(0) ? v + H : r;
}

struct Shape {
    i64 chains, T, D;
    unsigned tiles, pieces;  // blocks along the chains, pieces of the time axis
};

// Where chain c starts in [B, T, D]: step t is D elements further on.
__device__ __forceinline__ i64 chain_base(const Shape& s, i64 c) { return (c / s.D) * (s.T * s.D) + c % s.D; }

// ---- what pieces hand to each other ---------------------------------------------------------------------------------------------
constexpr u64 EMPTY = ~0ull;
constexpr unsigned GROUP = 32;

__device__ __forceinline__ void put(u64* p, u64 v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ u64 get(const u64* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float plain_nan(float v) { return v == v ? v : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ double plain_nan(double v) { return v == v ? v : __longlong_as_double(0x7ff8000000000000ll); }

// polls until the word is there (wave-uniform exit: all lanes' words)
__device__ __forceinline__ u64 await(const u64* p) {
    u64 v = get(p);
    for (int spin = 0; __any(v == EMPTY); ++spin) {
        if (spin > (1 << 22)) return 0x7ff8000000000000ull | 0x7fc00000ull;  // NaN in either reading
        __builtin_amdgcn_s_sleep(1);
        if (v == EMPTY) v = get(p);
    }
    return v;
}

// words [pieces][chains] (f64: two planes), states [pieces / GROUP + 1][chains]
template <typename T> struct Board;
template <> struct Board<float> {
    u64* words;
    u64* states;
    i64 chains, plane;
    static constexpr int PLANES = 1;
    __device__ __forceinline__ void put_map(unsigned piece, i64 c, float A, float H) const {
        put(words + piece * chains + c, (u64)__float_as_uint(plain_nan(A)) | ((u64)__float_as_uint(plain_nan(H)) << 32));
    }
    __device__ __forceinline__ void get_map(unsigned piece, i64 c, float& A, float& H) const {
        const u64 v = await(words + piece * chains + c);
        A = __uint_as_float((uint32_t)v);
        H = __uint_as_float((uint32_t)(v >> 32));
    }
    __device__ __forceinline__ void peek_map(unsigned piece, i64 c, float& A, float& H) const {
        const u64 v = get(words + piece * chains + c);
        A = __uint_as_float((uint32_t)v);
        H = __uint_as_float((uint32_t)(v >> 32));
    }
    __device__ __forceinline__ void put_state(unsigned g, i64 c, float v) const { put(states + g * chains + c, (u64)__float_as_uint(plain_nan(v))); }
    __device__ __forceinline__ float get_state(unsigned g, i64 c) const { return __uint_as_float((uint32_t)await(states + g * chains + c)); }
};
template <> struct Board<double> {
    u64* words;
    u64* states;
    i64 chains, plane;
    static constexpr int PLANES = 2;
    __device__ __forceinline__ void put_map(unsigned piece, i64 c, double A, double H) const {
        put(words + piece * chains + c, (u64)__double_as_longlong(plain_nan(A)));
        put(words + plane + piece * chains + c, (u64)__double_as_longlong(plain_nan(H)));
    }
    __device__ __forceinline__ void get_map(unsigned piece, i64 c, double& A, double& H) const {
        A = __longlong_as_double((long long)await(words + piece * chains + c));
        H = __longlong_as_double((long long)await(words + plane + piece * chains + c));
    }
    __device__ __forceinline__ void peek_map(unsigned piece, i64 c, double& A, double& H) const {
        A = __longlong_as_double((long long)get(words + piece * chains + c));
        H = __longlong_as_double((long long)get(words + plane + piece * chains + c));
    }
    __device__ __forceinline__ void put_state(unsigned g, i64 c, double v) const { put(states + g * chains + c, (u64)__double_as_longlong(plain_nan(v))); }
    __device__ __forceinline__ double get_state(unsigned g, i64 c) const { return __longlong_as_double((long long)await(states + g * chains + c)); }
};

__global__ __launch_bounds__(256) void board_clear_kernel(u64* __restrict__ p, i64 n, unsigned* __restrict__ tickets, unsigned tiles) {
    const i64 i = (i64)blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (i + u * 256 < n) p[i + u * 256] = EMPTY;
    for (i64 t = (i64)blockIdx.x * 256 + threadIdx.x; t < tiles; t += (i64)gridDim.x * 256) tickets[t] = 0;
}

// The state in front of this wave's steps.  (A, H): the wave's own map; start: the state in front of piece 0.  All waves call it.
template <typename T, int W, bool CHAIN>
__device__ __forceinline__ T state_before(T A, T H, T start, unsigned piece, unsigned pieces, i64 chain, bool live, const Board<T>& board) {
    __shared__ T mapA[W][64], mapH[W][64], base[CHAIN ? 64 : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if constexpr (W > 1 || CHAIN) {
        mapA[wave][lane] = A;
        mapH[wave][lane] = H;
        __syncthreads();
    }
    T v = start;
    if constexpr (CHAIN) {
        __shared__ T preA[W][64], preH[W][64];
        if (wave == W - 1 && piece + 1 < pieces) {  // publish first
            T a = mapA[0][lane], h = mapH[0][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) {
                h = mapA[w][lane] * h + mapH[w][lane];
                a = a * mapA[w][lane];
            }
            if (a == T(0) || h != h) {
                a = mapA[0][lane], h = mapH[0][lane];
#pragma unroll 1
                for (int w = 1; w < W; ++w) {
                    h = mapped(mapA[w][lane], mapH[w][lane], h);
                    a = times(a, mapA[w][lane]);
                }
            }
            if (live) board.put_map(piece, chain, a, h);
        }
        // the maps of pieces g0 .. piece - 1, an equal share for every wave, in order
        const unsigned g0 = piece / GROUP * GROUP, per = (piece - g0 + W - 1) / W;
        T a = T(1), h = T(0);
        for (unsigned j = g0 + wave * per; j < g0 + (wave + 1) * per && j < piece; ++j) {
            T a1, h1;
            board.get_map(j, chain, a1, h1);
            h = a1 * h + h1;
            a = a * a1;
        }
        preA[wave][lane] = a;
        preH[wave][lane] = h;
        if (wave == 0) base[lane] = g0 ? board.get_state(g0 / GROUP - 1, chain) : start;
        __syncthreads();
        v = base[lane];
#pragma unroll
        for (int w = 0; w < W; ++w) v = preA[w][lane] * v + preH[w][lane];
    }
#pragma unroll
    for (int w = 0; w < W - 1; ++w)
        if (w < wave) v = mapA[w][lane] * v + mapH[w][lane];
    if (v != v) {  // once more, map by map
        v = start;
        if constexpr (CHAIN) {
            v = base[lane];
            for (unsigned j = piece / GROUP * GROUP; j < piece; ++j) {  // all published: some wave of this block has waited for each
                T a, h;
                board.peek_map(j, chain, a, h);
                v = mapped(a, h, v);
            }
        }
#pragma unroll 1
        for (int w = 0; w < wave; ++w) v = mapped(mapA[w][lane], mapH[w][lane], v);
    }
    return v;
}

// Which piece of its tile's chains this block runs: by ticket where pieces wait for one another.
template <bool CHAIN> __device__ __forceinline__ unsigned piece_of(unsigned tile, unsigned* tickets) {
    if constexpr (CHAIN) {
        __shared__ unsigned mine;
        if (threadIdx.x == 0) mine = atomicAdd(tickets + tile, 1u);
        __syncthreads();
        return mine;
    }
    return 0;
}

// W waves, L steps per wave.
template <typename T, int W, int L, bool CHAIN>
__global__ __launch_bounds__(64 * W) void recurrence_fwd_kernel(const T* __restrict__ z, const T* __restrict__ x, const T* __restrict__ h0,
                                                                T* __restrict__ h, const Shape s, const Board<T> board, unsigned* tickets) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned tile = blockIdx.x % s.tiles, piece = piece_of<CHAIN>(tile, tickets);
    const bool live = (i64)tile * 64 + lane < s.chains;
    const i64 chain = live ? (i64)tile * 64 + lane : s.chains - 1, base = chain_base(s, chain);
    const i64 ts = (i64)piece * (W * L) + wave * L;
    T f[L], u[L];
#pragma unroll
    for (int l = 0; l < L; ++l) {  // past the end: the last step again, without effect below
        const i64 at = base + min(ts + l, s.T - 1) * s.D;
        f[l] = z[at];
        u[l] = x[at];
    }
    const T start = h0 ? h0[chain] : T(0);
    T A = T(1), H = T(0), least = T(1);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        T k;
        gate<T>(f[l], f[l], k);
        u[l] = k * u[l];
        if (ts + l < s.T) {
            H = f[l] * H + u[l];
            A = A * f[l];
            least = min(least, f[l]);
        }
    }
    T v = state_before<T, W, CHAIN>(product_of(A, least), H, start, piece, s.pieces, chain, live, board);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        v = f[l] * v + u[l];
        if (live && ts + l < s.T) h[base + (ts + l) * s.D] = v;
    }
    if (CHAIN && wave == W - 1 && piece % GROUP == GROUP - 1 && piece + 1 < s.pieces && live) board.put_state(piece / GROUP, chain, v);
}

// Backward: the same from the other end; piece, round and step numbers q = T - 1 - t run against time.
template <typename T, int W, int L, bool CHAIN>
__global__ __launch_bounds__(64 * W) void recurrence_bwd_kernel(const T* __restrict__ dh, const T* __restrict__ z, const T* __restrict__ x,
                                                                const T* __restrict__ h, const T* __restrict__ h0, const T* __restrict__ dnext,
                                                                T* __restrict__ dz, T* __restrict__ dx, T* __restrict__ dh0, const Shape s,
                                                                const Board<T> board, unsigned* tickets) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned tile = blockIdx.x % s.tiles, piece = piece_of<CHAIN>(tile, tickets);
    const bool live = (i64)tile * 64 + lane < s.chains;
    const i64 chain = live ? (i64)tile * 64 + lane : s.chains - 1, base = chain_base(s, chain);
    const i64 qs = (i64)piece * (W * L) + wave * L;
    T f[L], k[L], g[L], e[L];
#pragma unroll
    for (int l = 0; l < L; ++l) {
        const i64 t = s.T - 1 - min(qs + l, s.T - 1), at = base + t * s.D;
        f[l] = z[at];
        g[l] = dh[at];
        k[l] = x[at];
        e[l] = *(t > 0 ? h + (at - s.D) : h0 ? h0 + chain : x + at);  // in front of step 0: h0, or what the next loop replaces by 0
    }
    const T start = dnext ? dnext[chain] : T(0);
    T A = T(1), H = T(0), least = T(1);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        if (qs + l >= s.T - 1 && !h0) e[l] = T(0);
        e[l] = e[l] - k[l];
        gate<T>(f[l], f[l], k[l]);
        e[l] = e[l] * (f[l] * k[l]);
        if (qs + l < s.T) {
            H = f[l] * (g[l] + H);
            A = A * f[l];
            least = min(least, f[l]);
        }
    }
    T v = state_before<T, W, CHAIN>(product_of(A, least), H, start, piece, s.pieces, chain, live, board);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        if (qs + l < s.T) {
            const T S = g[l] + v;
            if (live) {
                const i64 at = base + (s.T - 1 - (qs + l)) * s.D;
                dx[at] = k[l] * S;
                dz[at] = S * e[l];
            }
            v = f[l] * S;
        }
    }
    if (wave == W - 1 && live) {
        if (CHAIN && piece % GROUP == GROUP - 1 && piece + 1 < s.pieces) board.put_state(piece / GROUP, chain, v);
        if (dh0 && piece + 1 == s.pieces) dh0[chain] = v;
    }
}

template <int W_, int L_> struct Cut { static constexpr int W = W_, L = L_; };

// f(cut, chain): the block's waves and steps for `steps` steps, and whether more than one piece is needed.  Pieces of 8 waves with L
// steps each leave registers for two or more blocks per CU, whose loads cover each other's waits.  Measured with the board's clearing
// (us; f32 at 2 x 8192 x 1024, f64 at 16 x 511 x 1000), waves x steps:
//   f32 forward   16 x 16 51   16 x 8 51   8 x 16 49   8 x 8 57   4 x 16 56      f32 backward  16 x 16 166   16 x 8 92   8 x 16 93   8 x 8 91
//   f64 forward   16 x 8 53    8 x 16 55   8 x 8 46    8 x 4 50   4 x 8 51       f64 backward  16 x 8 149    8 x 16 106  8 x 8 95    8 x 4 88
template <int L, typename F> int with_cut(i64 steps, F&& f) {
    if (steps == 1) return f(Cut<1, 1>(), std::false_type());
    if (steps <= 8) return f(Cut<1, 8>(), std::false_type());
    if (steps <= 32) return f(Cut<4, 8>(), std::false_type());
    if constexpr (8 * L > 32) {
        if (steps <= 8 * L) return f(Cut<8, L>(), std::false_type());
    }
    return f(Cut<8, L>(), std::true_type());
}

// Sizes, and for a chain of pieces the board in the library's scratch, cleared.
template <typename T>
int launch_pieces(fx_ctx* c, Shape& s, Board<T>& board, unsigned*& tickets, i64 B, i64 steps, i64 D, i64 piece, int waves, bool chain) {
    s.chains = B * D;
    s.T = steps;
    s.D = D;
    const i64 tiles = fx::ceil_div(s.chains, (i64)64), pieces = fx::ceil_div(steps, piece);
    // a launch has fewer than 2^32 threads
    FX_REQUIRE(tiles <= 0x7fffffff && tiles * pieces < (1ll << 32) / (64 * waves), "gated recurrence: too many chains and steps");
    s.tiles = (unsigned)tiles;
    s.pieces = (unsigned)pieces;
    board = {nullptr, nullptr, s.chains, s.chains * pieces};
    tickets = nullptr;
    if (!chain) return FX_OK;
    const i64 words = Board<T>::PLANES * s.chains * pieces, all = words + s.chains * (pieces / GROUP + 1);
    const i64 head = fx::ceil_div(tiles, (i64)64) * 256;
    char* p = (char*)c->get_scratch(head + all * 8);
    if (!p) return FX_ERR_OOM;
    tickets = (unsigned*)p;
    board.words = (u64*)(p + head);
    board.states = board.words + words;
    FX_LAUNCH(dim3((unsigned)fx::ceil_div(all, (i64)1024)), dim3(256), 0, c->stream, (board.words, all, tickets, s.tiles), board_clear_kernel);
    FX_LAUNCH_CHECK();
    return FX_OK;
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
    return with_cut<(sizeof(T) == 4 ? 16 : 8)>(steps, [&](auto cut, auto chain) -> int {
        constexpr int W = decltype(cut)::W, L = decltype(cut)::L;
        constexpr bool CHAIN = decltype(chain)::value;
        Shape s;
        Board<T> board;
        unsigned* tickets;
        if (int rc = launch_pieces<T>(c, s, board, tickets, B, steps, D, W * L, W, CHAIN)) return rc;
        FX_LAUNCH(dim3(s.tiles * s.pieces), dim3(64 * W), 0, c->stream, (z, x, h0, h, s, board, tickets), recurrence_fwd_kernel<T, W, L, CHAIN>);
        FX_LAUNCH_CHECK();
        return FX_OK;
    });
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
    return with_cut<(sizeof(T) == 4 ? 16 : 4)>(steps, [&](auto cut, auto chain) -> int {
        constexpr int W = decltype(cut)::W, L = decltype(cut)::L;
        constexpr bool CHAIN = decltype(chain)::value;
        Shape s;
        Board<T> board;
        unsigned* tickets;
        if (int rc = launch_pieces<T>(c, s, board, tickets, B, steps, D, W * L, W, CHAIN)) return rc;
        FX_LAUNCH(dim3(s.tiles * s.pieces), dim3(64 * W), 0, c->stream, (dh, z, x, h, h0, dnext, dz, dx, dh0, s, board, tickets),
                  recurrence_bwd_kernel<T, W, L, CHAIN>);
        FX_LAUNCH_CHECK();
        return FX_OK;
    });
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
