#pragma once

// What the feed-forward block's kernels share: operand types and their splitting, the stores of
// their epilogues, and the host's view of a matrix.

#include "backend.hpp"
#include "launch.cuh"
#include "pointwise.cuh"
#include "umma.cuh"

namespace spectral::mlp {

constexpr int kTileM = 128;
constexpr int kChunk = umma::kAtom;  // K per stage
constexpr int kTileABytes = kTileM * umma::kRowBytes;
constexpr int kMaxSmem = 227 * 1024;

// The type matrix products run in, and the parts an operand of T is split into.
template <class T>
struct Operand {
    using Type = T;
    static constexpr int kPlanes = 1;
    static constexpr int kProducts = 1;
    static constexpr int kPassChunks = 1 << 24;  // one pass over all of K
};
template <>
struct Operand<float> {
    using Type = bf16;
    static constexpr int kPlanes = 3;
    static constexpr int kProducts = 6;
    static constexpr int kPassChunks = 2;
};

// Parts (a, b) of a float32 product's p-th MMA, the small ones first: (2,0) (0,2) (1,1) (1,0) (0,1)
// (0,0), two bits each. Other types have one part.
template <class T>
__device__ __forceinline__ int part_a(int p) { return sizeof(T) == 4 ? (0b00'00'01'01'00'10 >> (2 * p)) & 3 : 0; }
template <class T>
__device__ __forceinline__ int part_b(int p) { return sizeof(T) == 4 ? (0b00'01'00'01'10'00 >> (2 * p)) & 3 : 0; }

// v = hi + mid + lo in bf16 parts (exact but for parts below bf16's smallest). A hi that would round to
// infinity is cut instead, and an infinity or NaN has no further parts.
__device__ __forceinline__ void split3(float v, bf16& hi, bf16& mid, bf16& lo)
{
    hi = __float2bfloat16_rn(v);
    if (fabsf(v) > 3.3895313892515355e38f && fabsf(v) <= 3.4028234663852886e38f) {
        hi = __float2bfloat16_rz(v);
    }
    const float r = fabsf(v) <= 3.4028234663852886e38f ? v - __bfloat162float(hi) : 0.0f;
    mid = __float2bfloat16_rn(r);
    lo = __float2bfloat16_rn(r - __bfloat162float(mid));
}

// The tensor core cuts its FP32 accumulator once per MMA, which pulls a long sum towards zero: by 1.1e-7 of it per
// MMA (16 values of K) where the terms have one sign, 5.8e-4 at 87000 tokens, more than a rounding to f16. Sums
// over tokens therefore leave the accumulator after this many MMAs and add up in FP32 (rounded to
// nearest): 5.5e-5 at most, a fifth of that rounding. Sums over channels or hidden values stay in one accumulator:
// they would need 8192 to get there. (Backward passes past that, with and without: 262144 x 512 x 2048 bf16 4.75 and 4.57 ms,
// narrow at 4.2 M tokens 785 and 745 us; shorter sums are not touched.)
constexpr int kLongSum = 512;

// A run of N (16 or 32) values of one row; only the first `valid` exist.
template <class T, int N>
__device__ __forceinline__ void store_run(T* p, const T (&v)[N], int valid)
{
    constexpr int kPer = 32 / static_cast<int>(sizeof(T));  // values per 32 bytes
    if (valid >= N && (reinterpret_cast<std::uintptr_t>(p) & 31u) == 0) {
#pragma unroll
        for (int i = 0; i < N / kPer; ++i) {
            uint32_t w[8];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = __float_as_uint(v[i * kPer + j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    Vec<T, 2> two{{v[i * kPer + 2 * j], v[i * kPer + 2 * j + 1]}};
                    w[j] = *reinterpret_cast<uint32_t*>(&two);
                }
            }
            store32(p + i * kPer, w);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (j < valid) {
                p[j] = v[j];
            }
        }
    }
}

template <class T, int N>
__device__ __forceinline__ void store_values(T* p, const float (&v)[N], int valid)
{
    T out[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        out[j] = from_float<T>(v[j]);
    }
    store_run(p, out, valid);
}

// A warp's N columns (16 or 32) of 32 rows, lane l holding row l; p is the first row's first value, and `rows` rows and
// `cols` columns from there on exist. Where the rows' runs are whole sectors each lane stores its own. Else
// the values are transposed by shuffles and stored side by side (47519 x 895 bf16 results of 8 hidden
// values: 94 us, with single values of 32 rows at a time 440 us). `add` (FP32 results): to what an earlier
// call stored there; each lane meets only its own stores again.
template <class T, int N>
__device__ __forceinline__ void store_rows(T* p, long long pitch, float (&v)[N], long long rows, int cols, bool add = false)
{
    const int lane = threadIdx.x & 31;
    if (((reinterpret_cast<std::uintptr_t>(p) | static_cast<std::uintptr_t>(pitch * sizeof(T))) & 31u) == 0) {
        if (lane < rows && cols > 0) {
            if (add) {
                const T* before = p + lane * pitch;
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    if (j + 4 <= cols) {
                        const Vec<T, 4> b = *reinterpret_cast<const Vec<T, 4>*>(before + j);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[j + i] += to_float(b.v[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[j + i] += j + i < cols ? to_float(before[j + i]) : 0.0f;
                        }
                    }
                }
            }
            store_values<T>(p + lane * pitch, v, min(N, cols));
        }
        return;
    }
#pragma unroll
    for (int s = N / 2; s > 0; s >>= 1) {
        const bool upper = (lane & s) != 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if ((j & s) == 0) {
                const float other = __shfl_xor_sync(0xffffffffu, upper ? v[j] : v[j | s], s);
                v[j] = upper ? other : v[j];
                v[j | s] = upper ? v[j | s] : other;
            }
        }
    }
    const int row = lane & ~(N - 1);  // N lanes hold the columns of N rows
    const int col = lane & (N - 1);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (row + j < rows && col < cols) {
            T* at = p + (row + j) * pitch + col;
            *at = from_float<T>(add ? v[j] + to_float(*at) : v[j]);
        }
    }
}

// This warp has read the accumulator set that `bar` guards.
__device__ __forceinline__ void release(uint64_t* bar, int lane)
{
    umma::fence_before_sync();
    __syncwarp();
    if (lane == 0) {
        umma::arrive(bar);
    }
}

struct MlpShape {
    long long tokens;
    int channels;
    int hidden;
    int outputs;
    int act;
};

// A matrix as the product kernel reads it.
struct Matrix {
    const void* base = nullptr;
    long long rows = 0;
    long long cols = 0;
    long long pitch = 0;
    int planes = 1;
    bool is_bf16 = true;

    CUtensorMap map(int box_rows) const
    {
        return umma::matrix_map(base, is_bf16, rows, cols, pitch, planes, rows * pitch, box_rows);
    }
};

// The forward and backward passes with everything but x, y, dy, dx and the weights on chip
// (mlp_narrow.cu). The matrices are in the operand form, of type `dtype` (16 bits).
bool narrow_forward_fits(const MlpShape& n, int dtype);
void narrow_forward(const Matrix& x, const Matrix& wg, const Matrix& wu, const Matrix& wd, void* y, int dtype,
                    const MlpShape& n, cudaStream_t stream);
bool narrow_backward_fits(const MlpShape& n, int dtype);
// The CTAs of a backward call: each leaves its sums of the three weight gradients, back to back, in `partial`.
int narrow_backward_parts(const MlpShape& n);
void narrow_backward(const Matrix& dy, const Matrix& x, const Matrix& wg, const Matrix& wu, const Matrix& wd, void* dx,
                     float* partial, int dtype, const MlpShape& n, cudaStream_t stream);

}  // namespace spectral::mlp
