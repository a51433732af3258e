// What follows a matrix product before its result is stored:  pre = v + bias[n];  C = act(pre) + residual.
#pragma once
#include "activation.hpp"
#include "igemm_core.hpp"

namespace gep {

template <typename T> struct Epilogue {
    const T* bias = nullptr;      // per column of C
    const T* residual = nullptr;  // [M][N]
    T* pre = nullptr;             // [M][N], written
    int act = 0;
    bool any() const { return bias || residual || pre || act != fxact::NONE; }
    // element i = (m, n) of the product; bias_n: bias[n], which a kernel loads once per column; res: residual[i], which a kernel that
    // has only an element or two per thread loads up front
    __device__ __forceinline__ T finish(T v, i64 i, T bias_n, T res) const {
        if (bias) v = v + bias_n;
        if (pre) pre[i] = v;
        v = fxact::apply<T>(act, v);
        return residual ? v + res : v;
    }
    __device__ __forceinline__ T finish(T v, i64 i, T bias_n) const { return finish(v, i, bias_n, residual ? residual[i] : T(0)); }
};

// The general tiles' store (igemm::MatStore) with bias, ReLU, residual and pre.  A tile finishes up to 64 elements per thread in one
// unrolled sequence, so the activations of a hundred instructions are not inlined here (they go through the pass below).
template <typename T> struct TileStore {
    T* p;
    i64 ld;
    int M, N;
    Epilogue<T> ex;
    static bool takes(int act) { return act == fxact::NONE || act == fxact::RELU; }
    __device__ __forceinline__ int rows() const { return M; }
    __device__ __forceinline__ int cols() const { return N; }
    __device__ __forceinline__ i64 row_stride() const { return ld; }
    __device__ __forceinline__ T* col(int n, int) const { return p + n; }
    __device__ __forceinline__ T xform(int m, int n, T v) const {
        const i64 i = (i64)m * ld + n;
        if (ex.bias) v = v + ex.bias[n];
        if (ex.pre) ex.pre[i] = v;
        if (ex.act == fxact::RELU) v = v > T(0) ? v : T(0);
        return ex.residual ? v + ex.residual[i] : v;
    }
};

// The ordered sum of partial products with the epilogue in its store; outputs [rows][ncols], fewer than 2^31.
template <typename T> struct SumStore {
    Epilogue<T> ex;
    igemm::FastDiv div_cols;
    int ncols;
    __device__ __forceinline__ T apply(T s, i64 i) const {
        T b = T(0);
        if (ex.bias) b = ex.bias[(uint32_t)i - div_cols.div((uint32_t)i) * (uint32_t)ncols];
        return ex.finish(s, i, b);
    }
};
template <typename T> inline int launch_sum(fx_ctx* c, const T* part, T* out, i64 M, i64 N, int splits, const Epilogue<T>& ex) {
    SumStore<T> se;
    se.ex = ex;
    se.div_cols = igemm::FastDiv((uint32_t)N);
    se.ncols = (int)N;
    return igemm::launch_splitk_reduce_with<T>(c, part, out, M * N, splits, se);
}

// The epilogue as a pass of its own over the stored product.
template <typename T>
__global__ __launch_bounds__(256) void pass_kernel(T* C, i64 n, i64 N, const Epilogue<T> ep) {
    for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < n; i += (i64)gridDim.x * 256) C[i] = ep.finish(C[i], i, ep.bias ? ep.bias[i % N] : T(0));
}
template <typename T> inline int launch_pass(fx_ctx* c, T* C, i64 n, i64 N, const Epilogue<T>& ep) {
    const i64 blocks = std::min<i64>(fx::ceil_div(n, (i64)256), 1 << 23);  // a launch has fewer than 2^32 threads
    FX_LAUNCH(dim3((unsigned)blocks), dim3(256), 0, c->stream, (C, n, N, ep), pass_kernel<T>);
    FX_LAUNCH_CHECK();
    return FX_OK;
}

}  // namespace gep
