#pragma once

// What the attention kernels share: the call's arrays and sizes, which keys count, and the joining of
// results that were split over an axis.
//
// out = softmax(scale q k^T) v, with the rows of a key head's queries side by side: `group` = heads / kv_heads query
// heads read the same keys and values, and row r = token * group + (head in the group) of `rows` = queries * group.
// Scores are taken in base 2: p = 2^(c s - m), c = scale log2(e), m the row's largest c s (or an earlier one),
// out = sum p v / sum p. A row without keys has sum p = 0 and the result 0.

#include "../../include/spectral_b200.h"

#include "backend.hpp"
#include "launch.cuh"
#include "pointwise.cuh"
#include "workspace.hpp"

#include <cuda_fp8.h>

namespace spectral::attention {

constexpr float kLog2e = 1.4426950408889634f;

struct Strides {
    long long sample = 0;
    long long token = 0;
    long long head = 0;
};

struct Call {
    const void* q = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    Strides qs, ks, vs;
    const void* lengths = nullptr;
    int lengths64 = 0;
    const unsigned char* mask = nullptr;
    void* out = nullptr;       // (batch, queries, heads, dim)
    float2* stats = nullptr;   // (batch, kv_heads, rows): m and sum p; NULL: not kept
    unsigned char* rest = nullptr;  // 16-bit types: what out's rounding took, of out's shape; NULL: not kept
    // backward
    const void* dout = nullptr;  // (batch, queries, heads, dim)
    void* dq = nullptr;
    void* dk = nullptr;
    void* dv = nullptr;
    float* delta = nullptr;    // (batch, kv_heads, rows): sum over dim of dout out
    int dtype = 0;
    int batch = 0;
    int queries = 0;
    int keys = 0;
    int kv_heads = 0;
    int group = 1;
    int dim = 0;
    float scale = 1.0f;
    __host__ __device__ long long rows() const { return static_cast<long long>(queries) * group; }
    __host__ __device__ long long pairs() const { return static_cast<long long>(batch) * kv_heads; }
    // Values from the start of a (sample, key head)'s results to row r's.
    __host__ __device__ long long row_at(int b, int head, long long r) const
    {
        const long long t = r / group;
        return ((b * static_cast<long long>(queries) + t) * kv_heads + head) * group * dim + (r - t * group) * dim;
    }
};

// How many keys sample b has before its mask.
__device__ __forceinline__ int length_of(const Call& c, int b)
{
    if (c.lengths == nullptr) {
        return c.keys;
    }
    const long long n = c.lengths64 != 0 ? static_cast<const long long*>(c.lengths)[b] : static_cast<const int*>(c.lengths)[b];
    return static_cast<int>(max(0LL, min(n, static_cast<long long>(c.keys))));
}

// What rounding out to its type took from it, times 2^12, as e5m2 values (two mantissa bits; from 2^-28 up to 2^3). The backward
// pass needs sum over dim of dout out, the weighted mean of dout v, to subtract it from each dout v: with out as
// rounded, dq of 512 x 16384 keys in float16 was off by 5.5e-4 of its norm, with this byte by 3.1e-4 (one rounding to
// float16 is 2.1e-4, and the score gradients are rounded too).
constexpr float kRestScale = 4096.0f;

// The bytes of two values, the first the lower.
template <class T>
__device__ __forceinline__ unsigned short rest_of(float2 o)
{
    const Vec<T, 2> rounded = narrow<T>(Floats<2>{{o}});
    const float2 r = (o - widen(rounded).p[0]) * pair(kRestScale);
    return __nv_cvt_float2_to_fp8x2(r, __NV_SATFINITE, __NV_E5M2);
}

__device__ __forceinline__ float2 with_rest(float2 rounded, unsigned short bytes)
{
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(bytes, __NV_E5M2);
    return fma2(__half22float2(__half2(h)), pair(1.0f / kRestScale), rounded);
}

// Sums of `parts` float32 arrays of a result, in order, times `factor`, rounded once. Partial arrays are (part, pair, row,
// dim); the result's rows are those of Call::row_at (queries) or (sample, key, head) (keys).
struct Sum {
    const float* partial = nullptr;
    void* result = nullptr;
    int parts = 0;
    bool of_keys = false;
    float factor = 1.0f;
};
struct Sums {
    Sum job[3];
    int count = 0;
    void add(const float* partial, int parts, bool of_keys, void* result, float factor) { job[count++] = {partial, result, parts, of_keys, factor}; }
};
void add_parts(const Call& c, const Sums& sums, cudaStream_t stream);

// Joins the splits of a forward pass: partial (split, pair, row, dim) holds sum p v, stats (split, pair, row) m and
// sum p.
void join_splits(const Call& c, const float* partial, const float2* stats, int splits, cudaStream_t stream);

// The 16-bit kernels (attention_tc.cu, attention_tc_backward.cu).
std::size_t tensor_forward_workspace(const Call& c);
void tensor_forward(const Call& c, char* work, cudaStream_t stream);
std::size_t tensor_backward_workspace(const Call& c);
void tensor_backward(const Call& c, char* work, cudaStream_t stream);

// The float32 kernels on the tensor cores (attention_tc32.cu): at most 64 query heads to a key head.
std::size_t split_forward_workspace(const Call& c);
void split_forward(const Call& c, char* work, cudaStream_t stream);
std::size_t split_backward_workspace(const Call& c);
void split_backward(const Call& c, char* work, cudaStream_t stream);

// Forward passes of at most eight rows per key head (attention_few.cu).
bool few_rows(const Call& c);
std::size_t few_workspace(const Call& c);
void few_forward(const Call& c, char* work, cudaStream_t stream);

// (pair, tile of `tokens` tokens): -lse of the tile's rows in `width` places, then -delta (attention_tc_backward.cu).
void row_constants(const Call& c, float* out, int width, int tokens, int tiles, cudaStream_t stream);

inline int pieces(long long n, long long per) { return static_cast<int>((n + per - 1) / per); }

}  // namespace spectral::attention
