// Rows that a team of threads holds in registers (layer norm, distillation, the losses of a large vocabulary): a thread's 16-byte vectors of a row, and sums over
// a wave or a workgroup in a fixed order.
#pragma once
#include "rp_rows.h"

#include <type_traits>

namespace rp {

template <typename T> struct vec16 { static constexpr int N = 16 / sizeof(T); };
// (rows may start at any element)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) any16 { unsigned int v[4]; };

// A thread's vector number `e0` .. of a row of d >= N elements.  The last one of a row whose length is no whole number of vectors is loaded so that it ends with
// the row, and a thread behind the row's end loads the last one too (no load is out of range, none behind a branch): elements from `skip` on are the thread's own.
template <typename T> struct RowVector {
    static constexpr int N = vec16<T>::N;
    int at, skip;
    __device__ __forceinline__ RowVector() : at(0), skip(N) {}
    __device__ __forceinline__ RowVector(int e0, int d) {
        at = e0 < d - N ? e0 : d - N;
        skip = e0 - at < N ? e0 - at : N;
    }
    __device__ __forceinline__ void load(T (&x)[N], const T* row) const {
        const any16<T> v = *(const any16<T>*)(row + at);
        __builtin_memcpy(x, &v, 16);
    }
    __device__ __forceinline__ bool has(int u) const { return u >= skip; }
    // the thread's own elements, once each
    __device__ __forceinline__ void store(T* row, const T (&y)[N]) const {
        if (skip == 0) {
            any16<T> v;
            __builtin_memcpy(&v, y, 16);
            *(any16<T>*)(row + at) = v;
        } else {
#pragma unroll
            for (int u = 0; u < N; u++)
                if (has(u)) row[at + u] = y[u];
        }
    }
};

// Eight, four or two sums rounded to a 16-byte vector, 16-bit ones two to an instruction
template <typename T> __device__ __forceinline__ void round_vector(T (&out)[vec16<T>::N], const typename traits<T>::acc (&v)[vec16<T>::N]) {
    if constexpr (sizeof(T) == 2) {
        using half_t = std::conditional_t<std::is_same<T, bf16_t>::value, __bf16, _Float16>;
        typedef half_t __attribute__((ext_vector_type(2))) half2_t;
        typedef float __attribute__((ext_vector_type(2))) float2_t;
#pragma unroll
        for (int u = 0; u < vec16<T>::N; u += 2) {
            const half2_t pair = __builtin_convertvector((float2_t{v[u], v[u + 1]}), half2_t);
            __builtin_memcpy(&out[u], &pair, 4);
        }
    } else {
#pragma unroll
        for (int u = 0; u < vec16<T>::N; u++) out[u] = round_to<T>(v[u]);
    }
}

// The sum (largest) of a value over the wave, in every lane
template <typename A> __device__ __forceinline__ A wave_sum(A v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
    return v;
}
template <typename A> __device__ __forceinline__ A larger(A a, A b) { return a != a ? a : b != b ? b : a > b ? a : b; }      // NaN is above every number
template <typename A> __device__ __forceinline__ A wave_max(A v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v = larger(v, __shfl_xor(v, d));
    return v;
}
// ... and over the LANES threads of a team: a wave, or the whole workgroup, which meets twice.  `room`: LANES / 64 values of LDS for each of the N.
template <int LANES, int N, typename A> __device__ __forceinline__ void team_sums(A (&v)[N], A* room) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_sum(v[i]);
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        __syncthreads();                           // (the room's last readers are done)
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) room[i * WAVES + threadIdx.x / 64] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = room[i * WAVES];
#pragma unroll
            for (int w = 1; w < WAVES; w++) v[i] += room[i * WAVES + w];
        }
    }
}
// The same in a loop that uses two rooms in turn: the other one's barrier lies between a room's last readers and its next writers
template <int LANES, int N, typename A> __device__ __forceinline__ void team_sums_in_turn(A (&v)[N], A* room) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_sum(v[i]);
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) room[i * WAVES + threadIdx.x / 64] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = room[i * WAVES];
#pragma unroll
            for (int w = 1; w < WAVES; w++) v[i] += room[i * WAVES + w];
        }
    }
}
template <int LANES, int N, typename A> __device__ __forceinline__ void team_tops_in_turn(A (&v)[N], A* room) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_max(v[i]);
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) room[i * WAVES + threadIdx.x / 64] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = room[i * WAVES];
#pragma unroll
            for (int w = 1; w < WAVES; w++) v[i] = larger(v[i], room[i * WAVES + w]);
        }
    }
}
template <int LANES, typename A> __device__ __forceinline__ A team_max(A v, A* room) {
    v = wave_max(v);
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) room[threadIdx.x / 64] = v;
        __syncthreads();
        v = room[0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v = larger(v, room[w]);
    }
    return v;
}

__device__ __forceinline__ float natural_exp(float x) { return __expf(x); }
__device__ __forceinline__ double natural_exp(double x) { return exp(x); }
__device__ __forceinline__ float natural_log(float x) { return logf(x); }
__device__ __forceinline__ double natural_log(double x) { return log(x); }

// exp((x - top) scale) for many x of a row, as 2 to x s - b with s = scale log2 e and b = top s: in float32 one multiply-add and the hardware's exponential.  s and b are rounded, but the same for
// every x, and x s - b is rounded once: what two of them have in common, however far from zero the row lies, leaves their quotient, and `log`, which is of the same x s - b, a difference from another's.
template <typename A> struct ScaledExp;
template <> struct ScaledExp<float> {
    float scale, base;
    __device__ __forceinline__ ScaledExp(float s, float top) : scale(s * 1.44269504088896341f), base(top == -INFINITY ? 0.f : top * scale) {}
    __device__ __forceinline__ float operator()(float x) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, -base)); }
    __device__ __forceinline__ float log(float x) const { return __builtin_fmaf(x, scale, -base) * 0.693147180559945309f; }
    // what a sum of these is multiplied by to be one of `other`'s
    __device__ __forceinline__ float as(const ScaledExp& other) const { return __builtin_amdgcn_exp2f(base - other.base); }
};
template <> struct ScaledExp<double> {
    double scale, base;
    __device__ __forceinline__ ScaledExp(double s, double top) : scale(s), base(top == -(double)INFINITY ? 0.0 : top * s) {}
    __device__ __forceinline__ double operator()(double x) const { return exp(__builtin_fma(x, scale, -base)); }
    __device__ __forceinline__ double log(double x) const { return __builtin_fma(x, scale, -base); }
    __device__ __forceinline__ double as(const ScaledExp& other) const { return exp(base - other.base); }
};
__device__ __forceinline__ float plain_max(float a, float b) { return fmaxf(a, b); }       // (of a number and NaN the number)
__device__ __forceinline__ double plain_max(double a, double b) { return fmax(a, b); }

}  // namespace rp
