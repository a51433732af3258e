// Shared pieces of the language-model kernels: vectors of 16 bytes in registers, sums over a wave, a block and the rows of a matrix
// of partial results.
#pragma once
#include "common.hpp"

namespace vio {

// Element-aligned: the GPU's 16-byte global accesses may start at any element, so a row need not begin on a 16-byte border.
template <typename T, int V> struct VecOf { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename T, int V> using Vec = typename VecOf<T, V>::type;

template <int V, typename T> __device__ __forceinline__ void load(const T* p, T (&v)[V]) {
    const Vec<T, V> q = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int u = 0; u < V; ++u) v[u] = q[u];
}
template <int V, typename T> __device__ __forceinline__ void store(T* p, const T (&v)[V]) {
    Vec<T, V> q;
#pragma unroll
    for (int u = 0; u < V; ++u) q[u] = v[u];
    *reinterpret_cast<Vec<T, V>*>(p) = q;
}
// past the caches: large outputs that nothing reads soon
template <int V, typename T> __device__ __forceinline__ void store_stream(T* p, const T (&v)[V]) {
    Vec<T, V> q;
#pragma unroll
    for (int u = 0; u < V; ++u) q[u] = v[u];
    __builtin_nontemporal_store(q, reinterpret_cast<Vec<T, V>*>(p));
}

// The vector at column j < D of a row that ends at D: whole, or what is left of the row (the rest zero / not stored).  Compared
// unsigned, since j + V may pass 2^31 (by the difference D - j instead: f64 RMS norm of 4099 x 1001 34.7 us, so 27.7).
template <int V, typename T> __device__ __forceinline__ void load_part(const T* row, int j, int D, T (&v)[V]) {
    if ((unsigned)j + V <= (unsigned)D) {
        load<V>(row + j, v);
    } else {
#pragma unroll
        for (int u = 0; u < V; ++u) {
            v[u] = T(0);
            if ((unsigned)j + u < (unsigned)D) v[u] = row[j + u];
        }
    }
}
template <int V, typename T> __device__ __forceinline__ void store_part(T* row, int j, int D, const T (&v)[V]) {
    if ((unsigned)j + V <= (unsigned)D) {
        store<V>(row + j, v);
    } else {
#pragma unroll
        for (int u = 0; u < V; ++u)
            if ((unsigned)j + u < (unsigned)D) row[j + u] = v[u];
    }
}

template <typename T> __device__ __forceinline__ T wave_sum(T v) {  // every lane gets the sum, in one fixed tree
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = v + __shfl_xor(v, m, 64);
    return v;
}

// The sum over the NT threads of a block (NT a multiple of 64), in wave order; every thread gets it.  sm: NT / 64 + 1 values.
// Callers that use it twice put a barrier between the two.
template <int NT, typename T> __device__ __forceinline__ T block_sum(T v, T* sm) {
    v = wave_sum(v);
    if constexpr (NT == 64) return v;
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = sm[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s = s + sm[w];
    return s;
}

// out[c] = sum over r of part[r][c]: 16 waves of a block take rows w, w + 16, ... of 64 columns, then the 16 sums are added in wave
// order.  The second launch of a column sum (weight gradient of a norm, bias gradient); fixed order for a given number of rows.
template <typename T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const T* __restrict__ part, T* __restrict__ out, int rows, i64 cols) {
    __shared__ T sm[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const i64 c = (i64)blockIdx.x * 64 + lane;
    T s = T(0);
    if (c < cols) {
        int r = wave;
        for (; r + 7 * 16 < rows; r += 8 * 16) {
            T v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = part[(i64)(r + 16 * u) * cols + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) s = s + v[u];
        }
        for (; r < rows; r += 16) s = s + part[(i64)r * cols + c];
    }
    sm[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < cols) {
#pragma unroll
        for (int w = 1; w < 16; ++w) s = s + sm[w][lane];
        out[c] = s;
    }
}
template <typename T> inline int column_sum(fx_ctx* c, const T* part, T* out, int rows, i64 cols) {
    FX_LAUNCH(dim3((unsigned)fx::ceil_div(cols, (i64)64)), dim3(1024), 0, c->stream, (part, out, rows, cols), column_sum_kernel<T>);
    FX_LAUNCH_CHECK();
    return FX_OK;
}

}  // namespace vio
