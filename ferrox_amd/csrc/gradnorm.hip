// The global norm of a list of gradient tensors and their clipping by it, the step between the backward pass and the optimizer
// (fx_adam_step_multi / fx_sgd_step_multi take the same tables):
//   norm = sqrt(sum over all tensors and elements of g^2);   out_k = g_k * (norm > max_norm ? max_norm / norm : 1)
// Two passes over the gradients, bound by memory: the first leaves one partial sum of squares per block, the second adds the
// partials (every block for itself, in one fixed order, so that all blocks and all runs have the same factor) and scales.  Nothing
// returns to the host in between, so the pair can be recorded into a graph.
// The second pass goes from the end to the front: what the first one read last may still be in the Infinity Cache.  (Reading or
// writing past the caches, and keeping a chosen part of the gradients in them, made no difference: 302 to 304 us for 534 MB.)
// The tensor table travels in the kernel's arguments, which lie in host memory: every block copies it to LDS once, all entries in
// flight together, and finds a chunk's tensor by a ballot.
// Squares are added in f64 whatever the tensors' type: f32 gradients neither overflow nor lose small terms, and the extra work is
// hidden behind the loads.  Squares of f64 gradients can leave the range of f64 at either end: a thread adds a chunk's squares as they
// are and, where that sum is no good (it overflowed, or is so small that terms may have vanished), adds them again in three sums, of the
// large elements times 2^-600, of the small ones times 2^600 and of the rest.  A block whose two outer sums hold anything stores them
// and marks its partial by a negative sign; they are read only then (113 million f64 elements clipped: 502 us, with one sum alone 505).
// Everything is summed in a fixed order, no atomics.
// The norm is kept as root * 2^e until the factor max / norm is formed, which therefore has full precision wherever the norm lies.
// Elements that are infinite or NaN give such a norm, and nothing is scaled.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <new>
#include <vector>

#include "vecio.hpp"

namespace {
using namespace vio;

constexpr int NT = 256, CHUNK = 4096, TABLE = 96;  // elements of a chunk; tensors of one launch (the table travels in the arguments)
constexpr int MAX_PARTIALS = 2048;
// Elements above LARGE or below SMALL go to the outer sums: squares of the ones between lie in 2^-1022 .. 2^972, and 2^50 of them fit.
constexpr double LARGE = 0x1p486, SMALL = 0x1p-511, UP = 0x1p600, DOWN = 0x1p-600;

template <typename T> struct Tensors {
    const T* g[TABLE];
    T* out[TABLE];
    i64 n[TABLE];
    unsigned first[TABLE + 1];  // tensor t owns chunks first[t] .. first[t + 1]
    int count;
};

// The table in LDS, and the first chunks of the tensors in registers (lane l: tensors l and 64 + l).
template <typename T> struct Table {
    const T* g[TABLE];
    T* out[TABLE];
    i64 n[TABLE];
    unsigned first[TABLE];
};
struct Starts { unsigned a, b; };
template <typename T> __device__ __forceinline__ Starts stage_table(const Tensors<T>& tt, Table<T>& lds) {
    const int i = threadIdx.x, lane = i & 63;
    if (i < TABLE) {
        const int k = min(i, tt.count - 1);
        lds.g[i] = tt.g[k];
        lds.out[i] = tt.out[k];
        lds.n[i] = tt.n[k];
        lds.first[i] = tt.first[k];
    }
    __syncthreads();
    Starts s;
    s.a = lane < tt.count ? lds.first[lane] : 0xffffffffu;
    s.b = 64 + lane < tt.count ? lds.first[min(64 + lane, TABLE - 1)] : 0xffffffffu;
    return s;
}
static_assert(TABLE <= 128 && TABLE <= NT, "one wave holds the starts of all tensors");
__device__ __forceinline__ int tensor_of(const Starts& s, unsigned chunk) {  // the last tensor that starts at or before the chunk
    return __popcll(__ballot(s.a <= chunk)) + __popcll(__ballot(s.b <= chunk)) - 1;
}

// Sums of squares: of the elements between SMALL and LARGE, of the larger ones times DOWN, of the smaller ones times UP.
struct Squares {
    double mid = 0., large = 0., small = 0.;
    __device__ __forceinline__ void add(double v) {
        const double a = fabs(v);
        if (!(a <= LARGE)) large = fma(v * DOWN, v * DOWN, large);  // NaN too
        else if (a < SMALL) small = fma(v * UP, v * UP, small);
        else mid = fma(v, v, mid);
    }
};

// block_sum of v, and whether any thread is marked: one barrier for both.
__device__ __forceinline__ double block_sum_marked(double v, bool& marked, double* sm, int* marks) {
    const bool wave = __any(marked);
    if ((threadIdx.x & 63) == 0) marks[threadIdx.x >> 6] = wave;
    v = block_sum<NT>(v, sm);
    int all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) all |= marks[w];
    marked = all != 0;
    return v;
}

// part: 3 planes of `plane` partial sums (f32: the first one only)
template <typename T>
__global__ __launch_bounds__(NT) void sum_squares_kernel(const Tensors<T> tt, double* __restrict__ part, i64 plane) {
    constexpr int V = 16 / (int)sizeof(T), PER = CHUNK / NT / V;
    constexpr bool WIDE = sizeof(T) == 8;
    __shared__ double sm[3][NT / 64 + 1];
    __shared__ int marks[NT / 64];
    __shared__ Table<T> tab;
    const Starts starts = stage_table(tt, tab);
    Squares s;
    const unsigned chunks = tt.first[tt.count];
    for (unsigned q = blockIdx.x; q < chunks; q += gridDim.x) {
        const int t = tensor_of(starts, q);
        const i64 at = (i64)(q - tab.first[t]) * CHUNK;
        const T* g = tab.g[t] + at;
        const i64 left = tab.n[t] - at;
        if (left >= CHUNK) {
            T v[PER][V];
#pragma unroll
            for (int k = 0; k < PER; ++k) load<V>(g + (k * NT + threadIdx.x) * V, v[k]);
            double sum = s.mid;
#pragma unroll
            for (int k = 0; k < PER; ++k)
#pragma unroll
                for (int u = 0; u < V; ++u) sum = fma((double)v[k][u], (double)v[k][u], sum);
            // below 2^-900, terms that vanished could count; a sum of zeros comes here too and is added again for nothing
            if (!WIDE || (sum >= 0x1p-900 && sum <= 0x1p1000)) {
                s.mid = sum;
            } else {
#pragma unroll
                for (int k = 0; k < PER; ++k)
#pragma unroll
                    for (int u = 0; u < V; ++u) s.add((double)v[k][u]);
            }
        } else {
            for (int j = threadIdx.x; j < left; j += NT) {
                if constexpr (WIDE) s.add((double)g[j]);
                else s.mid = fma((double)g[j], (double)g[j], s.mid);
            }
        }
    }
    bool outer = WIDE && !(s.large == 0. && s.small == 0.);
    double mid = WIDE ? block_sum_marked(s.mid, outer, sm[0], marks) : block_sum<NT>(s.mid, sm[0]);
    if constexpr (WIDE) {
        if (outer) {
            mid = -mid;  // minus zero as well
            const double large = block_sum<NT>(s.large, sm[1]), small = block_sum<NT>(s.small, sm[2]);
            if (threadIdx.x == 0) {
                part[plane + blockIdx.x] = large;
                part[2 * plane + blockIdx.x] = small;
            }
        }
    }
    if (threadIdx.x == 0) part[blockIdx.x] = mid;
}

struct Norm {  // root * 2^e
    double root;
    int e;
    __device__ __forceinline__ double value() const { return ldexp(root, e); }
};
// The norm from all partials, the same bits in every block.
template <bool WIDE> __device__ __forceinline__ Norm norm_of(const double* __restrict__ part, i64 plane, int parts, double (*sm)[NT / 64 + 1]) {
    __shared__ int marks[NT / 64];
    double s = 0.;
    bool marked = false;
    for (int j = threadIdx.x; j < parts; j += NT) {
        const double p = part[j];
        marked |= __double2hiint(p) < 0;
        s = s + fabs(p);
    }
    s = WIDE ? block_sum_marked(s, marked, sm[0], marks) : block_sum<NT>(s, sm[0]);
    if constexpr (WIDE) {
        if (marked) {
            double large = 0., small = 0.;
            for (int j = threadIdx.x; j < parts; j += NT) {
                if (__double2hiint(part[j]) >= 0) continue;
                large = large + part[plane + j];
                small = small + part[2 * plane + j];
            }
            large = block_sum<NT>(large, sm[1]);
            small = block_sum<NT>(small, sm[2]);
            if (!(large == 0.)) return {sqrt(large + s * DOWN * DOWN), 600};
            if (s < 0x1p-400) return {sqrt(s * UP * UP + small), -600};
        }
    }
    return {sqrt(s), 0};
}

// max_norm / norm as c * 2^e; e is 0 unless the quotient is below the type's normal numbers (or max_norm is subnormal)
template <typename T> struct Factor {
    T c;
    int e;
    __device__ __forceinline__ T times(T g) const {
        const T v = g * c;
        return e ? ldexp(v, e) : v;
    }
};
template <typename T> __device__ __forceinline__ Factor<T> factor_of(const Norm& norm, double max_norm) {
    constexpr double LEAST = sizeof(T) == 4 ? 0x1p-126 : 0x1p-1022;  // the smallest normal number
    constexpr int LEAST_E = sizeof(T) == 4 ? -126 : -1022;
    const double most = ldexp(max_norm, -norm.e);
    if (!(norm.root > most) || !(norm.root <= 1.7976931348623157e308)) return {T(1), 0};  // nothing to scale, or infinite or NaN
    if (max_norm == 0.) return {T(0), 0};
    const double q = most / norm.root;
    if (most >= 0x1p-1022 && q >= LEAST) return {(T)q, 0};  // rounded once to the tensors' type
    int em, er;
    const double c = 0.5 * frexp(max_norm, &em) / frexp(norm.root, &er);  // in 1/4 .. 1
    const int e = em - er - norm.e + 1;
    if (e > LEAST_E + 2) return {(T)ldexp(c, e), 0};
    return {(T)c, e};
}

template <typename T>
__global__ __launch_bounds__(NT) void norm_kernel(const double* __restrict__ part, i64 plane, int parts, T* __restrict__ norm) {
    __shared__ double sm[3][NT / 64 + 1];
    const Norm v = norm_of<sizeof(T) == 8>(part, plane, parts, sm);
    if (threadIdx.x == 0) norm[0] = (T)v.value();
}

template <typename T>
__global__ __launch_bounds__(NT) void scale_kernel(const Tensors<T> tt, const double* __restrict__ part, i64 plane, int parts, double max_norm, T* norm) {
    constexpr int V = 16 / (int)sizeof(T), PER = CHUNK / NT / V;
    __shared__ double sm[3][NT / 64 + 1];
    __shared__ Table<T> tab;
    const Starts starts = stage_table(tt, tab);
    const Norm total = norm_of<sizeof(T) == 8>(part, plane, parts, sm);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (T)total.value();
    const Factor<T> factor = factor_of<T>(total, max_norm);
    const unsigned chunks = tt.first[tt.count];
    for (unsigned q0 = blockIdx.x; q0 < chunks; q0 += gridDim.x) {
        const unsigned q = chunks - 1 - q0;
        const int t = tensor_of(starts, q);
        const i64 at = (i64)(q - tab.first[t]) * CHUNK;
        const T* g = tab.g[t] + at;
        T* o = tab.out[t] + at;
        if (factor.c == T(1) && factor.e == 0 && g == o) continue;  // in place and nothing to scale
        const i64 left = tab.n[t] - at;
        if (left >= CHUNK) {
            T v[PER][V];
#pragma unroll
            for (int k = 0; k < PER; ++k) load<V>(g + (k * NT + threadIdx.x) * V, v[k]);
#pragma unroll
            for (int k = 0; k < PER; ++k) {
#pragma unroll
                for (int u = 0; u < V; ++u) v[k][u] = factor.times(v[k][u]);
                store<V>(o + (k * NT + threadIdx.x) * V, v[k]);
            }
        } else {
            for (int j = threadIdx.x; j < left; j += NT) o[j] = factor.times(g[j]);
        }
    }
}

// Fills the table of the tensors from `base` on (empty ones left out); returns the next tensor that did not fit.
template <typename T>
int fill_table(Tensors<T>& tt, int base, int count, const T* const* g, T* const* out, const int64_t* n) {
    tt.count = 0;
    i64 chunks = 0;
    int k = base;
    for (; k < count && tt.count < TABLE; ++k) {
        if (n[k] == 0) continue;
        const i64 more = fx::ceil_div(n[k], (i64)CHUNK);
        if (chunks + more > 0x7fffffff) break;
        const int t = tt.count++;
        tt.g[t] = g[k];
        tt.out[t] = out ? out[k] : nullptr;
        tt.n[t] = n[k];
        tt.first[t] = (unsigned)chunks;
        chunks += more;
    }
    tt.first[tt.count] = (unsigned)chunks;
    return k;
}

// No output (the norm is one) may share memory with another tensor of the call (its own gradient, exactly, excepted).
template <typename T>
int check_overlaps(int count, const T* const* g, T* const* out, const int64_t* n, const T* norm, const char* what) {
    struct Span { uintptr_t lo, hi; int k; bool out; };
    std::vector<Span> spans;
    try {
        spans.reserve(2 * (size_t)count + 1);
    } catch (const std::bad_alloc&) {
        fx::set_error("%s: no host memory for %d tensors", what, count);
        return FX_ERR_OOM;
    }
    for (int k = 0; k < count; ++k) {
        if (n[k] == 0) continue;
        const uintptr_t bytes = (uintptr_t)n[k] * sizeof(T);
        if (out) spans.push_back({(uintptr_t)out[k], (uintptr_t)out[k] + bytes, k, true});
        if (!out || g[k] != out[k]) spans.push_back({(uintptr_t)g[k], (uintptr_t)g[k] + bytes, k, false});
    }
    spans.push_back({(uintptr_t)norm, (uintptr_t)norm + sizeof(T), count, true});
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
    // walking up: the furthest end of the outputs so far, and of everything so far
    uintptr_t out_end = 0, any_end = 0;
    for (const Span& s : spans) {
        FX_REQUIRE(!(s.lo < out_end || (s.out && s.lo < any_end)), "%s: an output overlaps another tensor of the call (at tensor %d)", what, s.k);
        any_end = std::max(any_end, s.hi);
        if (s.out) out_end = std::max(out_end, s.hi);
    }
    return FX_OK;
}

// out == null: the norm alone
template <typename T>
int grad_norm(fx_ctx* c, int count, const T* const* g, T* const* out, const int64_t* n, double max_norm, T* norm, const char* what) {
    FX_CHECK_CTX(c);
    FX_REQUIRE(count >= 0, "%s: negative tensor count", what);
    FX_REQUIRE(norm != nullptr, "%s: null norm pointer", what);
    FX_REQUIRE(count == 0 || (g && n), "%s: null table", what);
    for (int k = 0; k < count; ++k) {
        FX_REQUIRE(n[k] >= 0, "%s: negative element count", what);
        FX_REQUIRE(n[k] <= (i64)0x7fffffff * CHUNK, "%s: too many elements in tensor %d", what, k);
        FX_REQUIRE(n[k] == 0 || (g[k] && (!out || out[k])), "%s: null pointer in tensor %d", what, k);
    }
    if (int rc = check_overlaps<T>(count, g, out, n, norm, what)) return rc;
    std::lock_guard<std::mutex> lk(c->launch_mutex);
    Tensors<T> tt;
    // launches of at most TABLE tensors each; together they leave at most about MAX_PARTIALS partial sums
    int launches = 0;
    for (int k = 0; k < count;) {
        k = fill_table<T>(tt, k, count, g, out, n);
        if (tt.count) ++launches;
    }
    const i64 per_launch = std::max<i64>(1, std::min<i64>(8 * (i64)c->num_cus, MAX_PARTIALS / std::max(1, launches)));
    const i64 plane = std::max<i64>(1, per_launch * launches);
    double* part = (double*)c->get_scratch((sizeof(T) == 8 ? 3 : 1) * plane * (i64)sizeof(double));
    if (!part) return FX_ERR_OOM;
    i64 parts = 0;
    for (int k = 0; k < count;) {
        k = fill_table<T>(tt, k, count, g, out, n);
        if (!tt.count) continue;
        const i64 blocks = std::min<i64>(per_launch, tt.first[tt.count]);
        FX_LAUNCH(dim3((unsigned)blocks), dim3(NT), 0, c->stream, (tt, part + parts, plane), sum_squares_kernel<T>);
        FX_LAUNCH_CHECK();
        parts += blocks;
    }
    FX_REQUIRE(parts <= 0x7fffffff, "%s: too many tensors", what);
    if (!out || parts == 0) {
        FX_LAUNCH(dim3(1), dim3(NT), 0, c->stream, (part, plane, (int)parts, norm), norm_kernel<T>);
        FX_LAUNCH_CHECK();
        return FX_OK;
    }
    T* norm_out = norm;
    for (int k = 0; k < count;) {
        k = fill_table<T>(tt, k, count, g, out, n);
        if (!tt.count) continue;
        const i64 blocks = std::min<i64>(8 * (i64)c->num_cus, tt.first[tt.count]);
        FX_LAUNCH(dim3((unsigned)blocks), dim3(NT), 0, c->stream, (tt, part, plane, (int)parts, max_norm, norm_out), scale_kernel<T>);
        FX_LAUNCH_CHECK();
        norm_out = nullptr;
    }
    return FX_OK;
}
}  // namespace

#define FX_DEFINE_GRADNORM(T, S)                                                                                                       \
    extern "C" int fx_grad_norm_multi_##S(fx_ctx* c, int count, const T* const* g, const int64_t* n, T* norm) {                         \
        return grad_norm<T>(c, count, g, nullptr, n, 0., norm, "fx_grad_norm_multi");                                                  \
    }                                                                                                                                  \
    extern "C" int fx_clip_grad_norm_multi_##S(fx_ctx* c, int count, const T* const* g, T* const* out, const int64_t* n,                \
                                               double max_norm, T* norm) {                                                            \
        FX_REQUIRE(count <= 0 || out, "fx_clip_grad_norm_multi: null table");                                                          \
        FX_REQUIRE(max_norm >= 0, "fx_clip_grad_norm_multi: max_norm must not be negative");                                          \
        return grad_norm<T>(c, count, g, out, n, max_norm, norm, "fx_clip_grad_norm_multi");                                           \
    }
FX_DEFINE_GRADNORM(float, f32)
FX_DEFINE_GRADNORM(double, f64)
