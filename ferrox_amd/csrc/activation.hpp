// Activations of the matrix products' epilogue and their derivatives.
//   ReLU v > 0 ? v : 0      derivative at 0: 0, as ReLU::gradient of the reference (src/ops/unary.rs:358-375)
//   GELU v Phi(v), Phi(v) = erfc(-v / sqrt 2) / 2, which keeps its relative precision for negative v; derivative Phi(v) + v phi(v)
//   SiLU v s, s = 1 / (1 + exp(-v)); derivative s (1 + v (1 - s)), with 1 - s = 1 / (1 + exp(v)) from the same exponential of -|v|
#pragma once
#include "common.hpp"

namespace fxact {
constexpr int NONE = 0, RELU = 1, GELU = 2, SILU = 3;

__device__ __forceinline__ float dexp(float v) { return expf(v); }
__device__ __forceinline__ double dexp(double v) { return exp(v); }
__device__ __forceinline__ float derfc(float v) { return erfcf(v); }
__device__ __forceinline__ double derfc(double v) { return erfc(v); }

// s = sigmoid(v), c = sigmoid(-v)
template <typename T> __device__ __forceinline__ void sigmoid2(T v, T& s, T& c) {
    const T e = dexp(v < T(0) ? v : -v), big = T(1) / (T(1) + e), small = e * big;
    s = v < T(0) ? small : big;
    c = v < T(0) ? big : small;
}

template <typename T, int ACT> __device__ __forceinline__ T value(T v) {
    if constexpr (ACT == RELU) return v > T(0) ? v : T(0);
    if constexpr (ACT == GELU) {
        if (v < T(-40)) return T(0);  // Phi is 0 there in f32 and f64; also the limit at -inf, where the product has no value
        return v * (T(0.5) * derfc(v * T(-0.70710678118654752440)));
    }
    if constexpr (ACT == SILU) {
        T s, c;
        sigmoid2<T>(v, s, c);
        return s == T(0) ? T(0) : v * s;  // the limit at -inf
    }
    return v;
}

template <typename T, int ACT> __device__ __forceinline__ T grad(T v) {
    if constexpr (ACT == RELU) return v > T(0) ? T(1) : T(0);
    if constexpr (ACT == GELU) {
        const T Phi = T(0.5) * derfc(v * T(-0.70710678118654752440)), phi = T(0.39894228040143267794) * dexp(T(-0.5) * v * v);
        return phi > T(0) ? Phi + v * phi : Phi;
    }
    if constexpr (ACT == SILU) {
        T s, c;
        sigmoid2<T>(v, s, c);
        return c > T(0) && s > T(0) ? s * (T(1) + v * c) : s;
    }
    return T(1);
}

// act chosen at run time (wave-uniform): the epilogue of a product
template <typename T> __device__ __forceinline__ T apply(int act, T v) {
    if (act == RELU) return value<T, RELU>(v);
    if (act == GELU) return value<T, GELU>(v);
    if (act == SILU) return value<T, SILU>(v);
    return v;
}
}  // namespace fxact
