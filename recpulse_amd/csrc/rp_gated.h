// Gated linear layers, h = act(x . Wg + bg) * (x . Wu + bu) with W = [Wg | Wu] one [k, 2 n] matrix.
#pragma once
#include "rp_gemm.h"
#include "rp_teams.h"

namespace rp {

struct GatedArgs {
    void *h, *z;                   // z: [rows, 2 n] dense in the accumulate type, or null
    const void *x, *w, *bias;
    int rows, k, n, gate;
    long long x_rs, x_cs, w_rs, w_cs, h_rs;
};

template <typename A> __device__ __forceinline__ A logistic(A g) { return (A)1 / ((A)1 + natural_exp(-g)); }
__device__ __forceinline__ float error_function(float x) { return erff(x); }
__device__ __forceinline__ double error_function(double x) { return erf(x); }

// act(g) and, for the backward pass, its derivative
template <int GATE, typename A> __device__ __forceinline__ A gate_value(A g) {
    if constexpr (GATE == RP_GATE_SILU) return g * logistic(g);
    if constexpr (GATE == RP_GATE_GELU) return (A)0.5 * g * ((A)1 + error_function(g * (A)0.70710678118654752));
    if constexpr (GATE == RP_GATE_GELU_TANH) {
        // (1 + tanh v) / 2 is the logistic function of 2 v
        const A v = (A)0.79788456080286536 * (g + (A)0.044715 * g * g * g);
        return g * logistic((A)2 * v);
    }
    if constexpr (GATE == RP_GATE_RELU) return g > 0 ? g : g != g ? g : (A)0;
    return logistic(g);
}
template <int GATE, typename A> __device__ __forceinline__ A gate_slope(A g) {
    if constexpr (GATE == RP_GATE_SILU) { const A s = logistic(g); return s * ((A)1 + g * ((A)1 - s)); }
    if constexpr (GATE == RP_GATE_GELU) return (A)0.5 * ((A)1 + error_function(g * (A)0.70710678118654752)) + g * (A)0.39894228040143268 * natural_exp((A)-0.5 * g * g);
    if constexpr (GATE == RP_GATE_GELU_TANH) {
        const A v = (A)0.79788456080286536 * (g + (A)0.044715 * g * g * g), s = logistic((A)2 * v);
        const A c = g > (A)64 ? (A)64 : g < (A)-64 ? (A)-64 : g;      // (s is 0 or 1 there: what it multiplies stays finite)
        return s + c * (A)2 * s * ((A)1 - s) * (A)0.79788456080286536 * ((A)1 + (A)0.134145 * c * c);
    }
    if constexpr (GATE == RP_GATE_RELU) return g > 0 ? (A)1 : (A)0;
    const A s = logistic(g);
    return s * ((A)1 - s);
}

#define RP_DISPATCH_GATE(gate, ...)                                                          \
    switch (gate) {                                                                          \
        case RP_GATE_SILU:      { constexpr int GATE = RP_GATE_SILU;      __VA_ARGS__; break; } \
        case RP_GATE_GELU:      { constexpr int GATE = RP_GATE_GELU;      __VA_ARGS__; break; } \
        case RP_GATE_GELU_TANH: { constexpr int GATE = RP_GATE_GELU_TANH; __VA_ARGS__; break; } \
        case RP_GATE_RELU:      { constexpr int GATE = RP_GATE_RELU;      __VA_ARGS__; break; } \
        default:                { constexpr int GATE = RP_GATE_SIGMOID;   __VA_ARGS__; break; } \
    }

}  // namespace rp
