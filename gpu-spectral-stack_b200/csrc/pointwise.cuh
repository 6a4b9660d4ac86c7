#pragma once

// Shared pieces of the pointwise operators of an FNO block (group norm with an activation, 8-bit
// checkpoints, the gated feed-forward block): the three value types, vectors of them, and the
// activations with their slopes.

#include "../../include/spectral_b200.h"

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace spectral {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(f16 v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_float(float v)
{
    if constexpr (sizeof(T) == 4) {
        return v;
    } else if constexpr (std::is_same_v<T, bf16>) {
        return __float2bfloat16_rn(v);
    } else {
        return __float2half_rn(v);
    }
}

// V consecutive values moved by one access.
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

inline std::size_t dtype_size(int dtype) { return dtype == SPECTRAL_FLOAT32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype >= SPECTRAL_FLOAT32 && dtype <= SPECTRAL_FLOAT16; }
inline bool activation_known(int act) { return act >= SPECTRAL_ACT_NONE && act <= SPECTRAL_ACT_GELU; }
inline bool aligned_to(const void* p, std::size_t bytes) { return reinterpret_cast<std::uintptr_t>(p) % bytes == 0; }

// Calls f(T{}) with the value type of a SPECTRAL_* dtype code.
template <class F>
void with_dtype(int dtype, F&& f)
{
    switch (dtype) {
        case SPECTRAL_FLOAT32: f(float{}); return;
        case SPECTRAL_BFLOAT16: f(bf16{}); return;
        default: f(f16{}); return;
    }
}

// --- activations ---------------------------------------------------------------------------------

// 1 / (1 + exp(-z)) with the fast exponential and division (a few units in the last place; for
// z < -87 the exponential overflows to infinity and the quotient is 0, the limit).
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// The normal distribution function Phi(z), and exp(-z^2 / 2), which its density shares.
// Q(|z|) = 1 - Phi(|z|) = exp(-z^2 / 2) t P(t) with t = 1 / (1 + 0.28 |z|), the classical form of
// Hastings' approximations; P (degree 5) is a least-squares fit of this library's own, error
// below 1.5e-8. One exponential and one reciprocal give both the value and the slope of gelu,
// where erff and expf would cost about three times the instructions.
__device__ __forceinline__ float normal_cdf(float z, float& e)
{
    e = __expf(-0.5f * z * z);
    const float t = __fdividef(1.0f, fmaf(0.28f, fabsf(z), 1.0f));
    float p = -0.10655131936073303f;
    p = fmaf(p, t, 0.3929559588432312f);
    p = fmaf(p, t, -0.2420753836631775f);
    p = fmaf(p, t, 0.27307337522506714f);
    p = fmaf(p, t, 0.06580273061990738f);
    p = fmaf(p, t, 0.11679460108280182f);
    const float q = p * t * e;
    return z > 0.0f ? 1.0f - q : q;
}

template <int Act>
__device__ __forceinline__ float activate(float z)
{
    if constexpr (Act == SPECTRAL_ACT_SILU) {
        return z * sigmoid(z);
    } else if constexpr (Act == SPECTRAL_ACT_GELU) {
        float e;
        return z * normal_cdf(z, e);
    } else {
        return z;
    }
}

// The activation's value and slope at z.
template <int Act>
__device__ __forceinline__ float activate_slope(float z, float& slope)
{
    if constexpr (Act == SPECTRAL_ACT_SILU) {
        const float s = sigmoid(z);
        const float a = z * s;
        slope = fmaf(a, 1.0f - s, s);
        return a;
    } else if constexpr (Act == SPECTRAL_ACT_GELU) {
        float e;
        const float phi = normal_cdf(z, e);
        slope = fmaf(0.3989422804014327f * z, e, phi);
        return z * phi;
    } else {
        slope = 1.0f;
        return z;
    }
}

// Calls f(integral_constant<Act>) for an activation code.
template <class F>
void with_activation(int act, F&& f)
{
    switch (act) {
        case SPECTRAL_ACT_SILU: f(std::integral_constant<int, SPECTRAL_ACT_SILU>{}); return;
        case SPECTRAL_ACT_GELU: f(std::integral_constant<int, SPECTRAL_ACT_GELU>{}); return;
        default: f(std::integral_constant<int, SPECTRAL_ACT_NONE>{}); return;
    }
}

// --- 8-bit checkpoints -----------------------------------------------------------------------------

constexpr int kPackBlock = SPECTRAL_PACK8_BLOCK;     // values of a row that share one scale
constexpr float kPackTiny = 7.888609052210118e-31f;  // 2^-100: 127 / tiny is finite

// The value a code stands for, in the checkpoint's type. 127 scale can round past the largest float32;
// such a value is that largest one (the scale itself is never infinite).
template <class T>
__device__ __forceinline__ T restored(signed char code, float scale)
{
    float v = static_cast<float>(code) * scale;
    if (fabsf(v) > 3.4028234663852886e38f) {
        v = copysignf(3.4028234663852886e38f, v);
    }
    return from_float<T>(v);
}

// --- asynchronous copies -----------------------------------------------------------------------------

// One Bytes-sized copy from global to shared memory, asynchronous where the hardware has that
// size (4, 8, 16 bytes), else through a register. The copying thread waits with cp_async_wait.
template <int Bytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src)
{
    if constexpr (Bytes == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         static_cast<unsigned>(__cvta_generic_to_shared(dst))),
                     "l"(src)
                     : "memory");
    } else if constexpr (Bytes == 8 || Bytes == 4) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                         static_cast<unsigned>(__cvta_generic_to_shared(dst))),
                     "l"(src), "n"(Bytes)
                     : "memory");
    } else if constexpr (Bytes == 2) {
        *static_cast<unsigned short*>(dst) = *static_cast<const unsigned short*>(src);
    } else {
        *static_cast<unsigned char*>(dst) = *static_cast<const unsigned char*>(src);
    }
}

__device__ __forceinline__ void cp_async_wait_all()
{
    asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace spectral
