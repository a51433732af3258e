// What follows a matrix product before its result is stored:  pre = v + bias[n];  C = act(pre) + residual.
#pragma once
#include "activation.hpp"

namespace gep {

template <typename T> struct Epilogue {
    const T* bias = nullptr;      // per column of C
    const T* residual = nullptr;  // [M][N]
    T* pre = nullptr;             // [M][N], written
    int act = 0;
    bool any() const { return bias || residual || pre || act != fxact::NONE; }
    // element i = (m, n) of the product; bias_n: bias[n], which a kernel loads once per column
    __device__ __forceinline__ T finish(T v, i64 i, T bias_n) const {
        if (bias) v = v + bias_n;
        if (pre) pre[i] = v;
        v = fxact::apply<T>(act, v);
        return residual ? v + residual[i] : v;
    }
};

// The epilogue as a pass of its own over the stored product.
template <typename T>
__global__ __launch_bounds__(256) void pass_kernel(T* C, i64 n, i64 N, const Epilogue<T> ep) {
    const i64 i = (i64)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    C[i] = ep.finish(C[i], i, ep.bias ? ep.bias[i % N] : T(0));
}
template <typename T> inline int launch_pass(fx_ctx* c, T* C, i64 n, i64 N, const Epilogue<T>& ep) {
    const i64 blocks = fx::ceil_div(n, (i64)256);
    FX_REQUIRE(blocks <= 0x7fffffff, "matrix product epilogue: too many elements");
    FX_LAUNCH(dim3((unsigned)blocks), dim3(256), 0, c->stream, (C, n, N, ep), pass_kernel<T>);
    FX_LAUNCH_CHECK();
    return FX_OK;
}

}  // namespace gep
