// A Linear layer with an activation and a residual, forward and backward:
//   forward   pre = op(A) . op(B) + bias[n];  C = act(pre) + residual       (pre is written too when the backward pass will need it)
//   backward  dpre = dY * act'(pre);  dX = dpre . W;  dW = dpre^T . X;  db[o] = sum over rows of dpre
// Activations: ReLU v > 0 ? v : 0;  GELU v Phi(v), Phi the normal distribution function (through erfc, which keeps its relative
// precision for negative v);  SiLU v sigmoid(v).
// The products run on the matrix pipes (gemm.hip) and bound both passes; dpre and its column sums are one pass over dY and pre,
// bound by memory.
#include <mutex>

#include "activation.hpp"
#include "vecio.hpp"

namespace {
using namespace vio;

// One thread per column vector, rows strided over blockIdx.y: block (x, y) leaves the column sums of rows y, y + gridDim.y, ... in part[y].
// G row groups of 64 threads share a block; their sums are added in group order.  first: where the launch's columns begin.
constexpr int GROUPS = 4;
template <typename T, int V, int ACT>
__global__ __launch_bounds__(64 * GROUPS) void act_bwd_kernel(const T* dy, const T* pre, T* dpre, T* __restrict__ part, i64 rows, i64 cols, i64 first) {
    __shared__ T sm[GROUPS][64 * V];
    const int lane = threadIdx.x & 63, group = threadIdx.x >> 6;
    const i64 c = first + ((i64)blockIdx.x * 64 + lane) * V;
    const bool live = c < cols;
    T s[V];
#pragma unroll
    for (int u = 0; u < V; ++u) s[u] = T(0);
    constexpr int U = 4;
    const i64 step = (i64)gridDim.y * GROUPS;
    if (live) {
        for (i64 r = (i64)blockIdx.y * GROUPS + group; r < rows; r += U * step) {
            T g[U][V], p[U][V];
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const i64 at = min(r + q * step, rows - 1) * cols;
                load_part<V>(dy + at, (int)c, (int)cols, g[q]);
                load_part<V>(pre + at, (int)c, (int)cols, p[q]);
            }
#pragma unroll
            for (int q = 0; q < U; ++q) {
                if (r + q * step < rows) {
#pragma unroll
                    for (int u = 0; u < V; ++u) {
                        g[q][u] = g[q][u] * fxact::grad<T, ACT>(p[q][u]);
                        s[u] = s[u] + g[q][u];
                    }
                    store_part<V>(dpre + (r + q * step) * cols, (int)c, (int)cols, g[q]);
                }
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int u = 0; u < V; ++u) sm[group][lane * V + u] = s[u];
    __syncthreads();
    if (group == 0 && live) {
#pragma unroll
        for (int u = 0; u < V; ++u)
            for (int w = 1; w < GROUPS; ++w) s[u] = s[u] + sm[w][lane * V + u];
        store_part<V>(part + (i64)blockIdx.y * cols, (int)c, (int)cols, s);
    }
}

template <typename T, int V>
int launch_act_bwd(fx_ctx* c, int act, const T* dy, const T* pre, T* dpre, T* db, i64 rows, i64 cols) {
    const i64 gx = fx::ceil_div(cols, (i64)64 * V);
    const i64 gy = std::min<i64>(fx::ceil_div(rows, (i64)GROUPS), std::max<i64>(1, 8 * (i64)c->num_cus / gx));
    T* part = nullptr;
    if (db) {
        part = gy == 1 ? db : (T*)c->get_scratch(gy * cols * (i64)sizeof(T));
        if (!part) return FX_ERR_OOM;
    }
    constexpr i64 MOST = 0xffffffffll / (64 * GROUPS);  // blocks along the columns of one launch, which has fewer than 2^32 threads
    for (i64 b = 0; b < gx; b += MOST) {
        const dim3 grid((unsigned)std::min(gx - b, MOST), (unsigned)gy), blk(64 * GROUPS);
        const i64 first = b * 64 * V;
        if (act == fxact::RELU) FX_LAUNCH(grid, blk, 0, c->stream, (dy, pre, dpre, part, rows, cols, first), act_bwd_kernel<T, V, fxact::RELU>);
        else if (act == fxact::GELU) FX_LAUNCH(grid, blk, 0, c->stream, (dy, pre, dpre, part, rows, cols, first), act_bwd_kernel<T, V, fxact::GELU>);
        else if (act == fxact::SILU) FX_LAUNCH(grid, blk, 0, c->stream, (dy, pre, dpre, part, rows, cols, first), act_bwd_kernel<T, V, fxact::SILU>);
        else FX_LAUNCH(grid, blk, 0, c->stream, (dy, pre, dpre, part, rows, cols, first), act_bwd_kernel<T, V, fxact::NONE>);
        FX_LAUNCH_CHECK();
    }
    return db && gy > 1 ? column_sum<T>(c, part, db, (int)gy, cols) : FX_OK;
}

template <typename T> struct Products;
template <> struct Products<float> {
    static int bwd(fx_ctx* c, i64 B, i64 in, i64 out, const float* g, const float* W, const float* X, float* dX, float* dW) {
        return fx_linear_bwd_f32(c, B, in, out, g, W, X, dX, dW, nullptr, 0);
    }
};
template <> struct Products<double> {
    static int bwd(fx_ctx* c, i64 B, i64 in, i64 out, const double* g, const double* W, const double* X, double* dX, double* dW) {
        return fx_linear_bwd_f64(c, B, in, out, g, W, X, dX, dW, nullptr, 0);
    }
};

template <typename T>
int linear_act_bwd(fx_ctx* c, i64 B, i64 in, i64 out, const T* dY, const T* W, const T* X, const T* pre, int act, T* dpre, T* dX, T* dW, T* db) {
    FX_CHECK_CTX(c);
    FX_REQUIRE(B >= 1 && in >= 1 && out >= 1 && B < (1ll << 31) && in < (1ll << 31) && out < (1ll << 31), "fx_linear_act_bwd: bad dimensions");
    FX_REQUIRE(act >= fxact::NONE && act <= fxact::SILU, "fx_linear_act_bwd: act must be 0 (none), 1 (relu), 2 (gelu) or 3 (silu)");
    FX_REQUIRE(dY && W && X && pre && dpre && dX && dW, "fx_linear_act_bwd: null pointer");
    const i64 n = B * out;
    FX_REQUIRE(dpre == dY || !fx::overlap<T>(dpre, n, dY, n), "fx_linear_act_bwd: dpre overlaps dY without being it");
    FX_REQUIRE(dpre == pre || !fx::overlap<T>(dpre, n, pre, n), "fx_linear_act_bwd: dpre overlaps pre without being it");
    const T* ins[] = {W, X, dY, pre};
    const i64 insz[] = {in * out, B * in, n, n};
    T* outs[] = {dpre, dX, dW, db};
    const i64 outsz[] = {n, B * in, in * out, db ? out : 0};
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < (o ? 4 : 2); ++i) FX_REQUIRE(!fx::overlap<T>(outs[o], outsz[o], ins[i], insz[i]), "fx_linear_act_bwd: an output overlaps an input");
        for (int p = 0; p < o; ++p) FX_REQUIRE(!fx::overlap<T>(outs[o], outsz[o], outs[p], outsz[p]), "fx_linear_act_bwd: two outputs overlap");
    }
    {
        std::lock_guard<std::mutex> lk(c->launch_mutex);
        constexpr int V = 16 / (int)sizeof(T);
        const int rc = launch_act_bwd<T, V>(c, act, dY, pre, dpre, db, B, out);
        if (rc) return rc;
    }
    return Products<T>::bwd(c, B, in, out, dpre, W, X, dX, dW);
}
}  // namespace

#define FX_DEFINE_LINEAR_ACT(T, S)                                                                                                     \
    extern "C" int fx_linear_act_bwd_##S(fx_ctx* c, int64_t B, int64_t in, int64_t out, const T* dY, const T* W, const T* X, const T* pre, \
                                         int act, T* dpre, T* dX, T* dW, T* db) {                                                     \
        return linear_act_bwd<T>(c, B, in, out, dY, W, X, pre, act, dpre, dX, dW, db);                                                 \
    }
FX_DEFINE_LINEAR_ACT(float, f32)
FX_DEFINE_LINEAR_ACT(double, f64)
