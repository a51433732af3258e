// Root-mean-square norm over the rows of [rows, D] with the residual's addition in front of it, and its backward pass.
//   forward:   h = x + res;  rstd = (sum_j h_j^2 / D + eps)^(-1/2);  y_j = (h_j rstd) w_j
//   backward:  with n_j = h_j rstd, dx_j = dh_j + rstd (w_j dy_j - n_j (sum_k w_k dy_k n_k) / D);  dw_j = sum over rows of dy_j n_j
// Both are bound by memory: 2 reads and 2 writes of [rows, D] forward, 3 reads and 1 write backward.  A row stays in registers
// between its one read and its one write: up to 16 elements per thread, one wave per row up to 1024 elements, a block of 256 up to
// 4096 and of 1024 up to 16384.  All accesses to such rows are 16-byte vectors that start at any element (a row of an odd length moves the
// next one off the 16-byte grid); only the last, incomplete vector of a row goes element by element.  Sums are held in the tensors' own
// type (f32 or f64): of such a row a thread adds at most 16 terms before the tree of its block.  Longer rows are read twice, element by
// element, and a thread adds one term in 1024 of the row, one after the other.  Rows of a few elements leave most of their wave idle and
// are bound by its latency.
// Rows whose squares leave the type's range (their mean overflows, or is so small that squares may have vanished) are summed once more
// with their elements times a power of two; the branch is uniform over a row.
// The weight gradient is added up in registers over the rows that a block takes (thread t owns the same columns in every row), one
// partial row per block, and the partial rows are added by a second launch in a fixed order: no atomics.
#include <mutex>

#include "vecio.hpp"

namespace {
using namespace vio;

template <typename T> __device__ __forceinline__ T inv_sqrt(T v);
template <> __device__ __forceinline__ float inv_sqrt<float>(float v) { return 1.f / sqrtf(v); }
template <> __device__ __forceinline__ double inv_sqrt<double>(double v) { return 1. / sqrt(v); }

// Means of squares between these are taken as they are; below, the row counts UP-fold (an eps that matters there does not overflow by
// it), above and for NaN it counts DOWN-fold.
template <typename T> struct Range;
template <> struct Range<float> { static constexpr float LO = 0x1p-100f, HI = 0x1.fffffep127f, UP = 0x1p100f, DOWN = 0x1p-80f; };
template <> struct Range<double> { static constexpr double LO = 0x1p-900, HI = 0x1.fffffffffffffp1023, UP = 0x1p600, DOWN = 0x1p-600; };
template <typename T> __device__ __forceinline__ bool in_range(T mean) { return mean >= Range<T>::LO && mean <= Range<T>::HI; }
template <typename T> __device__ __forceinline__ T rescue(T mean) { return mean < Range<T>::LO ? Range<T>::UP : Range<T>::DOWN; }

constexpr int block_of(int nt) { return nt < 256 ? 256 : nt; }

// NT threads per row, E elements per thread, V per load.
template <typename T, int V, int NT, int E, bool RES>
__global__ __launch_bounds__(block_of(NT)) void rmsnorm_fwd_kernel(const T* x, const T* res, const T* __restrict__ w, T eps, T* h, T* y,
                                                                   T* __restrict__ rstd, i64 rows, int D) {
    constexpr int BT = block_of(NT), NV = E / V;
    __shared__ T sm[BT / 64 + 1];
    const int t = threadIdx.x % NT;
    const i64 row = (i64)blockIdx.x * (BT / NT) + threadIdx.x / NT;
    if (row >= rows) return;  // whole waves only: the variants with a barrier have one row per block
    const i64 base = row * D;
    T v[NV][V];
    T s = T(0);
#pragma unroll
    for (int k = 0; k < NV; ++k) load_part<V>(x + base, (k * NT + t) * V, D, v[k]);
    if constexpr (RES) {
        T r[NV][V];
#pragma unroll
        for (int k = 0; k < NV; ++k) load_part<V>(res + base, (k * NT + t) * V, D, r[k]);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int u = 0; u < V; ++u) v[k][u] = v[k][u] + r[k][u];
            store_part<V>(h + base, (k * NT + t) * V, D, v[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int u = 0; u < V; ++u) s = s + v[k][u] * v[k][u];
    s = block_sum<NT>(s, sm);
    const T mean = s / T(D) + eps;
    T r, f = T(1);
    if (in_range(mean)) {
        r = inv_sqrt<T>(mean);
    } else {
        f = rescue(mean);
        s = T(0);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int u = 0; u < V; ++u) {
                v[k][u] = v[k][u] * f;
                s = s + v[k][u] * v[k][u];
            }
        if (NT > 64) __syncthreads();  // the sums before have been read
        s = block_sum<NT>(s, sm);
        r = inv_sqrt<T>(s / T(D) + eps * f * f);
    }
    if (t == 0 && rstd) rstd[row] = r * f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        T g[V];
        load_part<V>(w, (k * NT + t) * V, D, g);
#pragma unroll
        for (int u = 0; u < V; ++u) g[u] = (v[k][u] * r) * g[u];
        store_part<V>(y + base, (k * NT + t) * V, D, g);
    }
}

constexpr i64 MOST_LONG = 0xffffffffll / 1024;  // rows of one launch of the long-row kernels

// Rows longer than a block's registers: the second pass reads the row again (the sum with the residual from h, where this thread put it).
template <typename T, bool RES>
__global__ __launch_bounds__(1024) void rmsnorm_fwd_long_kernel(const T* x, const T* res, const T* __restrict__ w, T eps, T* h, T* y,
                                                                T* __restrict__ rstd, i64 D) {
    __shared__ T sm[17];
    const i64 base = (i64)blockIdx.x * D;
    T s = T(0);
    for (i64 j = threadIdx.x; j < D; j += 1024) {
        T v = x[base + j];
        if constexpr (RES) {
            v = v + res[base + j];
            h[base + j] = v;
        }
        s = s + v * v;
    }
    s = block_sum<1024>(s, sm);
    const T* src = RES ? h : x;
    const T mean = s / T(D) + eps;
    T r, f = T(1);
    if (in_range(mean)) {
        r = inv_sqrt<T>(mean);
    } else {
        f = rescue(mean);
        s = T(0);
        for (i64 j = threadIdx.x; j < D; j += 1024) {
            const T v = src[base + j] * f;
            s = s + v * v;
        }
        __syncthreads();  // the sums before have been read
        s = block_sum<1024>(s, sm);
        r = inv_sqrt<T>(s / T(D) + eps * f * f);
    }
    if (threadIdx.x == 0 && rstd) rstd[blockIdx.x] = r * f;
    for (i64 j = threadIdx.x; j < D; j += 1024) y[base + j] = ((src[base + j] * f) * r) * w[j];
}

template <typename T, int V, int NT, int E>
int launch_fwd(fx_ctx* c, const T* x, const T* res, const T* w, T eps, T* h, T* y, T* rstd, i64 rows, i64 D) {
    constexpr int BT = block_of(NT);
    constexpr i64 MOST = 0xffffffffll / BT * (BT / NT);  // rows of one launch, which has fewer than 2^32 threads
    const dim3 blk(BT);
    for (i64 r = 0; r < rows; r += MOST) {
        const i64 n = std::min(rows - r, MOST), at = r * D;
        const dim3 grid((unsigned)fx::ceil_div(n, (i64)(BT / NT)));
        T* const rs = rstd ? rstd + r : nullptr;
        if (res) FX_LAUNCH(grid, blk, 0, c->stream, (x + at, res + at, w, eps, h + at, y + at, rs, n, (int)D), rmsnorm_fwd_kernel<T, V, NT, E, true>);
        else FX_LAUNCH(grid, blk, 0, c->stream, (x + at, nullptr, w, eps, nullptr, y + at, rs, n, (int)D), rmsnorm_fwd_kernel<T, V, NT, E, false>);
        FX_LAUNCH_CHECK();
    }
    return FX_OK;
}
template <typename T, int V>
int dispatch_fwd(fx_ctx* c, const T* x, const T* res, const T* w, T eps, T* h, T* y, T* rstd, i64 rows, i64 D) {
    if (D <= 64 * 4) return launch_fwd<T, V, 64, 4>(c, x, res, w, eps, h, y, rstd, rows, D);
    if (D <= 64 * 8) return launch_fwd<T, V, 64, 8>(c, x, res, w, eps, h, y, rstd, rows, D);
    if (D <= 64 * 16) return launch_fwd<T, V, 64, 16>(c, x, res, w, eps, h, y, rstd, rows, D);
    if (D <= 256 * 8) return launch_fwd<T, V, 256, 8>(c, x, res, w, eps, h, y, rstd, rows, D);
    if (D <= 256 * 16) return launch_fwd<T, V, 256, 16>(c, x, res, w, eps, h, y, rstd, rows, D);
    return launch_fwd<T, V, 1024, 16>(c, x, res, w, eps, h, y, rstd, rows, D);
}

template <typename T>
int rmsnorm_fwd(fx_ctx* c, const T* x, const T* res, const T* w, double eps, T* h, T* y, T* rstd, i64 rows, i64 D) {
    FX_CHECK_CTX(c);
    FX_REQUIRE(rows >= 0 && D >= 1, "fx_rmsnorm_fwd: bad shape [%lld, %lld]", (long long)rows, (long long)D);
    FX_REQUIRE(eps >= 0, "fx_rmsnorm_fwd: eps must not be negative");
    if (rows == 0) return FX_OK;
    FX_REQUIRE(x && w && y, "fx_rmsnorm_fwd: null pointer");
    FX_REQUIRE((res != nullptr) == (h != nullptr), "fx_rmsnorm_fwd: h is written exactly when a residual is given");
    FX_REQUIRE(D < (1ll << 31) && rows < (1ll << 31), "fx_rmsnorm_fwd: dimension exceeds 2^31");
    const i64 n = rows * D;
    // h and y may be x or res themselves (an element is read by the thread that writes it), nothing may overlap otherwise
    const T* ins[] = {x, res, w};
    T* outs[] = {h, y, rstd};
    for (int o = 0; o < 3; ++o) {
        const i64 on = o < 2 ? n : rows;
        for (int i = 0; i < 3; ++i)
            FX_REQUIRE((o < 2 && i < 2 && outs[o] == ins[i]) || !fx::overlap<T>(outs[o], on, ins[i], i < 2 ? n : D),
                       "fx_rmsnorm_fwd: an output overlaps an input that it is not");
        for (int p = 0; p < o; ++p) FX_REQUIRE(!fx::overlap<T>(outs[o], on, outs[p], n), "fx_rmsnorm_fwd: two outputs overlap");
    }
    constexpr int V = 16 / (int)sizeof(T);
    const T e = (T)eps;
    if (D > 1024 * 16) {
        for (i64 r = 0; r < rows; r += MOST_LONG) {
            const dim3 grid((unsigned)std::min(rows - r, MOST_LONG)), blk(1024);
            const i64 at = r * D;
            T* const rs = rstd ? rstd + r : nullptr;
            if (res) FX_LAUNCH(grid, blk, 0, c->stream, (x + at, res + at, w, e, h + at, y + at, rs, D), rmsnorm_fwd_long_kernel<T, true>);
            else FX_LAUNCH(grid, blk, 0, c->stream, (x + at, nullptr, w, e, nullptr, y + at, rs, D), rmsnorm_fwd_long_kernel<T, false>);
            FX_LAUNCH_CHECK();
        }
        return FX_OK;
    }
    return dispatch_fwd<T, V>(c, x, res, w, e, h, y, rstd, rows, D);
}

// ---- backward ------------------------------------------------------------------------------------------------------------------
// Row group g of block b takes rows b * groups + g, + gridDim * groups, ...; part (when the weight gradient is wanted) gets the
// block's row of partial sums.
template <typename T, int V, int NT, int E>
__global__ __launch_bounds__(block_of(NT)) void rmsnorm_bwd_kernel(const T* dy, const T* dh, const T* h, const T* __restrict__ w,
                                                                   const T* __restrict__ rstd, T* dx, T* __restrict__ part, i64 rows, int D) {
    constexpr int BT = block_of(NT), NV = E / V, GR = BT / NT;
    __shared__ T sm[GR > 1 ? GR * NT * E : BT / 64 + 1];
    const int t = threadIdx.x % NT, group = threadIdx.x / NT;
    T wv[NV][V], dw[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int u = 0; u < V; ++u) dw[k][u] = T(0);
        load_part<V>(w, (k * NT + t) * V, D, wv[k]);
    }
    for (i64 row = (i64)blockIdx.x * GR + group; row < rows; row += (i64)gridDim.x * GR) {
        const i64 base = row * D;
        const T r = rstd[row];
        T g[NV][V], hv[NV][V];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            load_part<V>(dy + base, (k * NT + t) * V, D, g[k]);
            load_part<V>(h + base, (k * NT + t) * V, D, hv[k]);
        }
        T s = T(0);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int u = 0; u < V; ++u) {
                hv[k][u] = hv[k][u] * r;
                dw[k][u] = dw[k][u] + g[k][u] * hv[k][u];
                g[k][u] = g[k][u] * wv[k][u];
                s = s + g[k][u] * hv[k][u];
            }
        if (GR == 1) __syncthreads();  // the sums of the row before have been read
        s = block_sum<NT>(s, sm);
        const T q = s / T(D);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            T d[V];
            if (dh) load_part<V>(dh + base, (k * NT + t) * V, D, d);
#pragma unroll
            for (int u = 0; u < V; ++u) {
                const T a = r * (g[k][u] - hv[k][u] * q);
                d[u] = dh ? a + d[u] : a;
            }
            store_part<V>(dx + base, (k * NT + t) * V, D, d);
        }
    }
    if (!part) return;
    if constexpr (GR > 1) {  // the groups' sums in group order
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int u = 0; u < V; ++u) sm[group * (NT * E) + (k * NT + t) * V + u] = dw[k][u];
        __syncthreads();
        for (int j = threadIdx.x; j < D; j += BT) {
            T s = sm[j];
#pragma unroll
            for (int q = 1; q < GR; ++q) s = s + sm[q * (NT * E) + j];
            part[(i64)blockIdx.x * D + j] = s;
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) store_part<V>(part + (i64)blockIdx.x * D, (k * NT + t) * V, D, dw[k]);
    }
}

// Long rows: dx row by row (the row read twice), the weight gradient by columns below.
template <typename T>
__global__ __launch_bounds__(1024) void rmsnorm_bwd_long_kernel(const T* dy, const T* dh, const T* h, const T* __restrict__ w,
                                                                const T* __restrict__ rstd, T* dx, i64 D) {
    __shared__ T sm[17];
    const i64 base = (i64)blockIdx.x * D;
    const T r = rstd[blockIdx.x];
    T s = T(0);
    for (i64 j = threadIdx.x; j < D; j += 1024) s = s + (dy[base + j] * w[j]) * (h[base + j] * r);
    s = block_sum<1024>(s, sm);
    const T q = s / T(D);
    for (i64 j = threadIdx.x; j < D; j += 1024) {
        const T a = r * (dy[base + j] * w[j] - (h[base + j] * r) * q);
        dx[base + j] = dh ? a + dh[base + j] : a;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void rmsnorm_dw_long_kernel(const T* __restrict__ dy, const T* __restrict__ h, const T* __restrict__ rstd,
                                                              T* __restrict__ part, i64 rows, i64 D) {
    const i64 j = (i64)blockIdx.x * 256 + threadIdx.x;
    if (j >= D) return;
    T s = T(0);
    for (i64 r = blockIdx.y; r < rows; r += gridDim.y) s = s + dy[r * D + j] * (h[r * D + j] * rstd[r]);
    part[(i64)blockIdx.y * D + j] = s;
}

template <typename T, int V, int NT, int E>
int launch_bwd(fx_ctx* c, const T* dy, const T* dh, const T* h, const T* w, const T* rstd, T* dx, T* dw, i64 rows, i64 D) {
    constexpr int BT = block_of(NT), GR = BT / NT;
    // enough blocks to fill the chip and no more: every block leaves a partial row of the weight gradient
    const i64 per_cu = BT >= 1024 ? 2 : 4;
    const i64 blocks = std::min<i64>(fx::ceil_div(rows, (i64)GR), per_cu * c->num_cus);
    T* part = nullptr;
    if (dw) {
        part = blocks == 1 ? dw : (T*)c->get_scratch(blocks * D * (i64)sizeof(T));
        if (!part) return FX_ERR_OOM;
    }
    FX_LAUNCH(dim3((unsigned)blocks), dim3(BT), 0, c->stream, (dy, dh, h, w, rstd, dx, part, rows, (int)D), rmsnorm_bwd_kernel<T, V, NT, E>);
    FX_LAUNCH_CHECK();
    return dw && blocks > 1 ? column_sum<T>(c, part, dw, (int)blocks, D) : FX_OK;
}
template <typename T, int V>
int dispatch_bwd(fx_ctx* c, const T* dy, const T* dh, const T* h, const T* w, const T* rstd, T* dx, T* dw, i64 rows, i64 D) {
    if (D <= 64 * 4) return launch_bwd<T, V, 64, 4>(c, dy, dh, h, w, rstd, dx, dw, rows, D);
    if (D <= 64 * 8) return launch_bwd<T, V, 64, 8>(c, dy, dh, h, w, rstd, dx, dw, rows, D);
    if (D <= 64 * 16) return launch_bwd<T, V, 64, 16>(c, dy, dh, h, w, rstd, dx, dw, rows, D);
    if (D <= 256 * 8) return launch_bwd<T, V, 256, 8>(c, dy, dh, h, w, rstd, dx, dw, rows, D);
    if (D <= 256 * 16) return launch_bwd<T, V, 256, 16>(c, dy, dh, h, w, rstd, dx, dw, rows, D);
    return launch_bwd<T, V, 1024, 16>(c, dy, dh, h, w, rstd, dx, dw, rows, D);
}

template <typename T>
int rmsnorm_bwd(fx_ctx* c, const T* dy, const T* dh, const T* h, const T* w, const T* rstd, T* dx, T* dw, i64 rows, i64 D) {
    FX_CHECK_CTX(c);
    FX_REQUIRE(rows >= 0 && D >= 1, "fx_rmsnorm_bwd: bad shape [%lld, %lld]", (long long)rows, (long long)D);
    FX_REQUIRE(D < (1ll << 31) && rows < (1ll << 31), "fx_rmsnorm_bwd: dimension exceeds 2^31");
    const i64 n = rows * D;
    if (rows == 0) {  // the sum over no rows
        if (!dw) return FX_OK;
        if constexpr (sizeof(T) == 4) return fx_fill_f32(c, dw, 0.f, D);
        else return fx_fill_f64(c, dw, 0., D);
    }
    FX_REQUIRE(dy && h && w && rstd && dx, "fx_rmsnorm_bwd: null pointer");
    const T* ins[] = {dy, dh, h, w, rstd};
    const i64 insz[] = {n, n, n, D, rows};
    for (int i = 0; i < 5; ++i)
        FX_REQUIRE(((i < 2 && dx == ins[i]) || !fx::overlap<T>(dx, n, ins[i], insz[i])) && !fx::overlap<T>(dw, D, ins[i], insz[i]),
                   "fx_rmsnorm_bwd: an output overlaps an input that it is not");
    FX_REQUIRE(!fx::overlap(dw, D, dx, n), "fx_rmsnorm_bwd: dx and dw overlap");
    constexpr int V = 16 / (int)sizeof(T);
    std::lock_guard<std::mutex> lk(c->launch_mutex);
    if (D > 1024 * 16) {
        if (dw) {  // first, since dx may be written over dy
            const i64 slices = std::min<i64>(rows, std::max<i64>(1, 8 * (i64)c->num_cus / fx::ceil_div(D, (i64)256)));
            T* part = slices == 1 ? dw : (T*)c->get_scratch(slices * D * (i64)sizeof(T));
            if (!part) return FX_ERR_OOM;
            FX_LAUNCH(dim3((unsigned)fx::ceil_div(D, (i64)256), (unsigned)slices), dim3(256), 0, c->stream, (dy, h, rstd, part, rows, D), rmsnorm_dw_long_kernel<T>);
            FX_LAUNCH_CHECK();
            if (slices > 1) {
                if (int rc = column_sum<T>(c, part, dw, (int)slices, D)) return rc;
            }
        }
        for (i64 r = 0; r < rows; r += MOST_LONG) {
            const i64 at = r * D;
            FX_LAUNCH(dim3((unsigned)std::min(rows - r, MOST_LONG)), dim3(1024), 0, c->stream,
                      (dy + at, dh ? dh + at : nullptr, h + at, w, rstd + r, dx + at, D), rmsnorm_bwd_long_kernel<T>);
            FX_LAUNCH_CHECK();
        }
        return FX_OK;
    }
    return dispatch_bwd<T, V>(c, dy, dh, h, w, rstd, dx, dw, rows, D);
}
}  // namespace

#define FX_DEFINE_RMSNORM(T, S)                                                                                                        \
    extern "C" int fx_rmsnorm_fwd_##S(fx_ctx* c, const T* x, const T* res, const T* w, double eps, T* h, T* y, T* rstd, int64_t rows,   \
                                      int64_t D) {                                                                                     \
        return rmsnorm_fwd<T>(c, x, res, w, eps, h, y, rstd, rows, D);                                                                 \
    }                                                                                                                                  \
    extern "C" int fx_rmsnorm_bwd_##S(fx_ctx* c, const T* dy, const T* dh, const T* h, const T* w, const T* rstd, T* dx, T* dw,         \
                                      int64_t rows, int64_t D) {                                                                       \
        return rmsnorm_bwd<T>(c, dy, dh, h, w, rstd, dx, dw, rows, D);                                                                 \
    }
FX_DEFINE_RMSNORM(float, f32)
FX_DEFINE_RMSNORM(double, f64)
