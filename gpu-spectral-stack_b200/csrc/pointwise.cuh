#pragma once

// Shared pieces of the pointwise operators of an FNO block (group norm with an activation, 8-bit
// checkpoints, the gated feed-forward block): the three value types, vectors of them, and the
// activations with their slopes.

#include "../../include/spectral_b200.h"

#include "common.cuh"

#include <cstdint>

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

// --- pairs of floats -------------------------------------------------------------------------------

// The pointwise kernels are close to bound by instruction issue, so they work on pairs: one packed
// FP32x2 instruction does both (the same IEEE rounding as the scalar form).
__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 operator+(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 operator*(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
// a - b: the product with -1 is exact, so there is one rounding.
__device__ __forceinline__ float2 operator-(float2 a, float2 b) { return __ffma2_rn(b, pair(-1.0f), a); }

// V values as pairs (an odd last one is paired with 0).
template <int V>
struct Floats {
    static constexpr int kPairs = (V + 1) / 2;
    float2 p[kPairs];

    __device__ __forceinline__ float at(int j) const { return j % 2 == 0 ? p[j / 2].x : p[j / 2].y; }
    __device__ __forceinline__ void set(int j, float v) { (j % 2 == 0 ? p[j / 2].x : p[j / 2].y) = v; }
    __device__ __forceinline__ void fill(float v)
    {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            p[i] = pair(v);
        }
    }
};

template <class T, int V>
__device__ __forceinline__ Floats<V> widen(const Vec<T, V>& v)
{
    Floats<V> f;
    if constexpr (V == 1) {
        f.p[0] = make_float2(to_float(v.v[0]), 0.0f);
    } else if constexpr (std::is_same_v<T, bf16>) {
        const auto* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {  // bf16 is the upper half of a float
            f.p[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
    } else if constexpr (std::is_same_v<T, f16>) {
        const auto* w = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            f.p[i] = __half22float2(w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            f.p[i] = make_float2(v.v[2 * i], v.v[2 * i + 1]);
        }
    }
    return f;
}

template <class T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const Floats<V>& f)
{
    Vec<T, V> v;
    if constexpr (V == 1) {
        v.v[0] = from_float<T>(f.p[0].x);
    } else if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            reinterpret_cast<__nv_bfloat162*>(&v)[i] = __float22bfloat162_rn(f.p[i]);
        }
    } else if constexpr (std::is_same_v<T, f16>) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            reinterpret_cast<__half2*>(&v)[i] = __float22half2_rn(f.p[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            v.v[2 * i] = f.p[i].x;
            v.v[2 * i + 1] = f.p[i].y;
        }
    }
    return v;
}

// --- activations ---------------------------------------------------------------------------------

// The hardware's 2^v and 1 / v (about one unit in the last place, subnormals as zero).
__device__ __forceinline__ float exp2_fast(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float reciprocal_fast(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// 1 / (1 + exp(-z)), of which T results are made. For float32 the rounding of z log2(e), which exp2 would turn into a
// relative error of up to |z| units of 2^-24, is carried along: exp2(e + r) = exp2(e) (1 + r log(2)). Past -87.5
// the result is 0, below float32's smallest normal number. (At z = -88 that error is 5e-6, far below a rounding to 16 bits.)
// It cost the float32 norm's backward pass from a checkpoint 10 us of 183 (64 x 128 x 128 x 64), the others nothing.
// `rest` is 1 - sigmoid, for float32 as exp(-z) sigmoid, which keeps its accuracy where the sigmoid is close to 1.
template <class T>
__device__ __forceinline__ float2 sigmoid2(float2 z, float2& rest)
{
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (sizeof(T) == 4) {
        constexpr float kLog2eRest = 1.9259630e-08f;  // log2(e) - kLog2e
        const float2 c = make_float2(fminf(fmaxf(z.x, -87.5f), 126.0f), fminf(fmaxf(z.y, -87.5f), 126.0f));
        const float2 e = c * pair(-kLog2e);
        const float2 off = fma2(c, pair(kLog2eRest), fma2(c, pair(kLog2e), e));  // -(e + c log2(e))
        const float2 q = make_float2(exp2_fast(e.x), exp2_fast(e.y));
        const float2 p = fma2(q * off, pair(-0.6931471805599453f), q);
        const float2 d = p + pair(1.0f);
        const float2 s = make_float2(reciprocal_fast(d.x), reciprocal_fast(d.y));
        rest = p * s;
        return s;
    } else {  // for z < -88 the power overflows to infinity and its reciprocal is 0, the limit
        const float2 e = z * pair(-kLog2e);
        const float2 d = make_float2(exp2_fast(e.x), exp2_fast(e.y)) + pair(1.0f);
        const float2 s = make_float2(reciprocal_fast(d.x), reciprocal_fast(d.y));
        rest = pair(1.0f) - s;
        return s;
    }
}

// u = Phi(z) for z >= 0 and -Phi(z) below, Phi the normal distribution function, so that |z| u = z Phi(z), with
// az = |z| and e = exp(-z^2 / 2), which the density shares. 1 - Phi(|z|) = e t P(t) with t = 1 / (1 + c |z|), the form of
// Hastings' approximations; below zero it is the value itself, so small values keep their relative accuracy.
// c and P are minimax fits of this library's own with P(1) = 1/2, of relative error: degree 7, 1.1e-7, and for
// results that are rounded to 16 bits degree 5, 2.2e-6 down to z = -6.2 and 5e-5 below (a rounding to bf16 or f16 is 2^-8,
// 2^-11). Evaluated in FP32 the first is off by 3.5e-7 of the value at z = -1/2, 8e-7 at -4: the exponent's rounding grows with z^2.
// Degrees 5 and 4 about Phi(|z|) - 1/2, with the value as z / 2 + |z| (Phi(|z|) - 1/2), were off by 3e-7 in absolute terms,
// 2e-4 of the value at z = -3.5, and 3 to 4 % faster in the norm (64 x 128 x 128 x 64 bf16: forward 77 us against 80, backward 140
// against 145).
template <class T>
__device__ __forceinline__ float2 normal2(float2 z, float2& az, float2& e)
{
    constexpr bool kShort = sizeof(T) == 2;
    const float2 x = (z * pair(-0.7213475204444817f)) * z;
    e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
    az = make_float2(fabsf(z.x), fabsf(z.y));
    const float2 d = fma2(az, pair(kShort ? 0.3f : 0.305f), pair(1.0f));
    const float2 t = make_float2(reciprocal_fast(d.x), reciprocal_fast(d.y));
    float2 p;  // -P
    if constexpr (kShort) {
        p = fma2(pair(0.0814674646f), t, pair(-0.229254112f));
        p = fma2(p, t, pair(0.0321748704f));
        p = fma2(p, t, pair(-0.152487561f));
        p = fma2(p, t, pair(-0.111625835f));
        p = fma2(p, t, pair(-0.120274834f));
    } else {
        p = fma2(pair(-0.0364528522f), t, pair(0.151998967f));
        p = fma2(p, t, pair(-0.184075385f));
        p = fma2(p, t, pair(0.0365235433f));
        p = fma2(p, t, pair(-0.120282948f));
        p = fma2(p, t, pair(-0.103635691f));
        p = fma2(p, t, pair(-0.122433834f));
        p = fma2(p, t, pair(-0.121641792f));
    }
    return fma2(p * t, e, make_float2(z.x >= 0.0f ? 1.0f : 0.0f, z.y >= 0.0f ? 1.0f : 0.0f));
}

// The activation of a value that is then rounded to T.
template <int Act, class T = float>
__device__ __forceinline__ float2 activate2(float2 z)
{
    if constexpr (Act == SPECTRAL_ACT_SILU) {
        float2 rest;
        return z * sigmoid2<T>(z, rest);
    } else if constexpr (Act == SPECTRAL_ACT_GELU) {
        float2 az, e;
        return normal2<T>(z, az, e) * az;
    } else {
        return z;
    }
}

// The activation's values and slopes at z, of which T results are made.
template <int Act, class T>
__device__ __forceinline__ float2 activate_slope2(float2 z, float2& slope)
{
    if constexpr (Act == SPECTRAL_ACT_SILU) {
        float2 rest;
        const float2 s = sigmoid2<T>(z, rest);
        const float2 a = z * s;
        slope = fma2(a, rest, s);
        return a;
    } else if constexpr (Act == SPECTRAL_ACT_GELU) {
        float2 az, e;
        const float2 u = normal2<T>(z, az, e);
        const float2 w = fma2(az * pair(0.3989422804014327f), e, u);  // Phi(z) + z phi(z), its sign turned below zero
        slope = make_float2(z.x >= 0.0f ? w.x : -w.x, z.y >= 0.0f ? w.y : -w.y);
        return u * az;
    } else {
        slope = pair(1.0f);
        return z;
    }
}

template <int Act>
__device__ __forceinline__ float activate(float z)
{
    return activate2<Act>(make_float2(z, 0.0f)).x;
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

// The values V codes stand for, in the checkpoint's type. A code's byte, offset by 128, becomes the low
// bits of 2^23 + byte, so one subtraction converts it. 127 scale can round past the largest float32;
// such a value is that largest one (the scale itself is never infinite; the 16-bit types are far
// from it).
template <class T, int V>
__device__ __forceinline__ Floats<V> restored(const Vec<signed char, V>& codes, float scale)
{
    Floats<V> f;
    if constexpr (V >= 4) {
        const auto* w = reinterpret_cast<const uint32_t*>(&codes);
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const uint32_t u = w[j] ^ 0x80808080u;
            f.p[2 * j] = make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)),
                                     __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441)));
            f.p[2 * j + 1] = make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)),
                                         __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443)));
        }
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            f.p[j] = (f.p[j] - pair(8388736.0f)) * pair(scale);
        }
    } else {
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            f.p[j].x = static_cast<float>(codes.v[2 * j]) * scale;
            f.p[j].y = 2 * j + 1 < V ? static_cast<float>(codes.v[2 * j + 1 < V ? 2 * j + 1 : 0]) * scale : 0.0f;
        }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float v = f.at(j);
            f.set(j, fabsf(v) > 3.4028234663852886e38f ? copysignf(3.4028234663852886e38f, v) : v);
        }
        return f;
    } else {
        return widen(narrow<T>(f));
    }
}

// The scale of a block whose largest magnitude has the bits `top` (a NaN's are above infinity's, and
// those above every number's), and the factor that turns its values into codes. A block with an
// infinity or NaN has the scale NaN and the codes 0.
struct PackScale {
    float scale;
    float per_unit;
};

__device__ __forceinline__ PackScale pack_scale(unsigned top)
{
    const bool finite = top < 0x7f800000u;
    const float m = finite ? fmaxf(__uint_as_float(top), kPackTiny) : 1.0f;
    return {finite ? __fdiv_rn(m, 127.0f) : __uint_as_float(0x7fc00000u), finite ? __fdiv_rn(127.0f, m) : 0.0f};
}

// The bits of the largest magnitude among the values: whole numbers order as the magnitudes do, in
// 16 bits as in 32.
template <class T, int V>
__device__ __forceinline__ unsigned top_bits(const Vec<T, V>& v)
{
    if constexpr (sizeof(T) == 4 || V == 1) {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            top = max(top, __float_as_uint(to_float(v.v[j])) & 0x7fffffffu);
        }
        return top;
    } else {
        const auto* w = reinterpret_cast<const unsigned*>(&v);
        unsigned two = w[0] & 0x7fff7fffu;
#pragma unroll
        for (int j = 1; j < V / 2; ++j) {
            two = __vmaxu2(two, w[j] & 0x7fff7fffu);
        }
        const unsigned short top = static_cast<unsigned short>(max(two & 0xffffu, two >> 16));
        return __float_as_uint(to_float(*reinterpret_cast<const T*>(&top)));
    }
}

// round(v * per_unit) as bytes. Adding 1.5 x 2^23 rounds to the nearest whole number, ties to even,
// and leaves it in the low bits (two's complement). A per_unit of 0 gives codes 0 whatever v is.
template <int V>
__device__ __forceinline__ Vec<signed char, V> pack_codes(const Floats<V>& f, float per_unit)
{
    Vec<signed char, V> c;
    uint32_t w[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        // The scalar intrinsics: the product is rounded before the sum (a packed multiply and add
        // may be contracted, which moved codes at ties).
        w[j] = __float_as_uint(__fadd_rn(__fmul_rn(f.at(j), per_unit), 12582912.0f));
    }
    const uint32_t keep = per_unit == 0.0f ? 0u : 0xffffffffu;
    if constexpr (V >= 4) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const uint32_t lo = __byte_perm(w[4 * j], w[4 * j + 1], 0x0040);
            const uint32_t hi = __byte_perm(w[4 * j + 2], w[4 * j + 3], 0x0040);
            reinterpret_cast<uint32_t*>(&c)[j] = __byte_perm(lo, hi, 0x5410) & keep;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            c.v[j] = static_cast<signed char>(w[j] & keep);
        }
    }
    return c;
}

// Packs K blocks at once. This lane holds one piece of each, v[k]; the kPackBlock / V lanes of a
// block sit side by side in the warp. Each lane computes the scale of one block (scale_at(k) is
// where it goes), the block's other lanes take it from there; put(k, codes) stores the codes.
template <class T, int V, int K, class ScaleAt, class Put>
__device__ __forceinline__ void pack_blocks(const Vec<T, V> (&v)[K], ScaleAt&& scale_at, Put&& put)
{
    constexpr int kLanes = kPackBlock / V;
    static_assert(K <= kLanes && kLanes <= 32, "a lane per block");
    const int lane = threadIdx.x & 31;
    const int sub = lane % kLanes;
    const unsigned mask = kLanes == 32 ? 0xffffffffu : ((1u << (kLanes % 32)) - 1u) << (lane / kLanes * kLanes);
    unsigned mine = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        unsigned top = top_bits(v[k]);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o /= 2) {
            top = max(top, __shfl_xor_sync(mask, top, o));
        }
        mine = k == 0 || sub == k ? top : mine;
    }
    const PackScale s = pack_scale(mine);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (sub == k) {
            float* at = scale_at(k);
            if (at != nullptr) {
                *at = s.scale;
            }
        }
        put(k, pack_codes<V>(widen(v[k]), __shfl_sync(mask, s.per_unit, k, kLanes)));
    }
}

// 32 bytes with one store; p is 32-byte aligned.
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
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

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Until at most N of this thread's committed groups are in flight.
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void cp_async_wait_all()
{
    asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace spectral
