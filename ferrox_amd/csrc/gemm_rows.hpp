// C[M,N] = act(A . B^T + bias) + residual for a few rows: A [M, K], B [N, K] as stored by a Linear layer, M <= 4 -- the layer as a
// program runs it that generates one token for each of a few streams.  Bound by reading B once (M products per element of B cost
// less than its load); the matrix pipes' tiles would be empty but for M of their 32 rows.
//   A block owns RN rows of B, its 4 waves take every fourth piece of K (256 f32 / 128 f64 elements, one 16-byte load per lane and
// row), M x RN sums per lane.  The sums go through a tree over the lanes and then over the waves, in one fixed order.
#pragma once
#include "gemm_epilogue.hpp"
#include "vecio.hpp"

namespace grows {
using vio::load_part;
using vio::wave_sum;

constexpr int NT = 256, WAVES = 4;

template <typename T, int M, int RN>
__global__ __launch_bounds__(NT) void rows_kernel(const T* __restrict__ A, const T* __restrict__ B, T* __restrict__ C, int rows, int N, int K,
                                                  const gep::Epilogue<T> ex) {
    constexpr int V = 16 / (int)sizeof(T), PIECE = 64 * V, U = 2;
    __shared__ T sm[WAVES][M * RN];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const i64 n0 = (i64)blockIdx.x * RN;
    T acc[M][RN];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < RN; ++r) acc[m][r] = T(0);
    const T *a[M], *b[RN];  // past the last row: the last row again, its sums unused
#pragma unroll
    for (int m = 0; m < M; ++m) a[m] = A + (i64)min(m, rows - 1) * K;
#pragma unroll
    for (int r = 0; r < RN; ++r) b[r] = B + min(n0 + r, (i64)N - 1) * K;
    int k = wave * PIECE + lane * V;
    // whole pieces, U of them in flight
    for (; k - lane * V + (U - 1) * WAVES * PIECE + PIECE <= K; k += U * WAVES * PIECE) {
        T x[U][M][V], y[U][RN][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int r = 0; r < RN; ++r) vio::load<V>(b[r] + k + u * WAVES * PIECE, y[u][r]);
#pragma unroll
            for (int m = 0; m < M; ++m) vio::load<V>(a[m] + k + u * WAVES * PIECE, x[u][m]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int r = 0; r < RN; ++r)
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[m][r] = fma(x[u][m][e], y[u][r][e], acc[m][r]);
    }
    for (; k - lane * V < K; k += WAVES * PIECE) {  // what is left: one piece at a time, the last one incomplete (zeros behind K)
        T x[M][V], y[RN][V];
#pragma unroll
        for (int r = 0; r < RN; ++r) load_part<V>(b[r], k, K, y[r]);
#pragma unroll
        for (int m = 0; m < M; ++m) load_part<V>(a[m], k, K, x[m]);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int r = 0; r < RN; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[m][r] = fma(x[m][e], y[r][e], acc[m][r]);
    }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < RN; ++r) {
            const T s = wave_sum(acc[m][r]);
            if (lane == 0) sm[wave][m * RN + r] = s;
        }
    __syncthreads();
    const int t = threadIdx.x;
    if (t < M * RN) {
        const int m = t / RN;
        const i64 n = n0 + t % RN;
        if (m < rows && n < N) {
            T v = sm[0][t];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) v = v + sm[w][t];
            C[(i64)m * N + n] = ex.finish(v, (i64)m * N + n, ex.bias ? ex.bias[n] : T(0));
        }
    }
}

// One row always; up to four where K is long enough to hide the M x RN sums' trees.  Measured at K = N = 4096 against the small-product
// kernel (us): f32 1 row 12.0 (67 MB at 5.6 TB/s) / 26.1, 2 rows 13.0 / 26.2, 4 rows 15.4 / 26.3, 8 rows 20.1 / 26.8; f64 23.8 / 43.6, 26.5 /
// 44.0, 29.9 / 45.2, 55.9 / 46.8.  4 rows at K = 128, N = 4096: 7.9 / 5.4, and 8 rows at K = 512, N = 256: 8.9 / 5.6.  Eight rows gain in
// f32 with long K and N alone; they would need a rule of their own and are left to the other kernels.
// A launch has fewer than 2^32 threads, 256 for four rows of B.
inline bool eligible(bool ta, bool tb, i64 M, i64 N, i64 K) {
    return !ta && tb && K >= 1 && K < (1ll << 30) && N <= (1ll << 26) - 4 && (M == 1 || (M <= 4 && K >= 512));
}

template <typename T, int M, int RN>
inline int launch(fx_ctx* c, i64 rows, i64 N, i64 K, const T* A, const T* B, T* C, const gep::Epilogue<T>& ex) {
    FX_LAUNCH(dim3((unsigned)fx::ceil_div(N, (i64)RN)), dim3(NT), 0, c->stream, (A, B, C, (int)rows, (int)N, (int)K, ex), rows_kernel<T, M, RN>);
    FX_LAUNCH_CHECK();
    return FX_OK;
}
template <typename T>
inline int run(fx_ctx* c, i64 M, i64 N, i64 K, const T* A, const T* B, T* C, const gep::Epilogue<T>& ex) {
    if (M == 1) return launch<T, 1, 4>(c, M, N, K, A, B, C, ex);
    if (M == 2) return launch<T, 2, 4>(c, M, N, K, A, B, C, ex);
    return launch<T, 4, 4>(c, M, N, K, A, B, C, ex);
}

}  // namespace grows
