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

// What rounding out to its type took from it, as a byte: in steps of 2^-kRestBits of the last place of the rounded value, 64 at
// most, so that it is as accurate for small values of v as for large ones. (Places are counted from 2^-112 in bf16, so that a step is a
// normal number, and in float16 from 2^-14, below which they all are 2^-24.) The backward pass needs sum over dim of
// dout out, the weighted mean of dout v, to subtract it from each dout v: with out as
// rounded, dq of 512 x 16384 keys in float16 was off by 5.5e-4 of its norm, with this byte by 3.1e-4 (one rounding to
// float16 is 2.1e-4, and the score gradients are rounded too).
constexpr unsigned kRestBits = 7;
template <class T>
constexpr unsigned kPlaceBits = std::is_same_v<T, bf16> ? 7 : 10;  // behind the first

// The exponent bits of a rounded value, or those from which places are counted.
template <class T>
__device__ __forceinline__ unsigned rest_exponent(float rounded)
{
    constexpr unsigned kLeast = std::is_same_v<T, bf16> ? 15u << 23 : 113u << 23;
    return max(__float_as_uint(rounded) & 0x7f800000u, kLeast);
}

// The bytes of two values, the first the lower. Adding 1.5 x 2^23 leaves the whole number in the lowest bits; an infinite or NaN
// result leaves any.
template <class T>
__device__ __forceinline__ unsigned short rest_of(float2 o)
{
    const float2 rounded = widen(narrow<T>(Floats<2>{{o}})).p[0];
    const float2 r = o - rounded;
    // Steps to a value of one: 2^(kRestBits + kPlaceBits - exponent).
    const auto scale = [](float v) { return __uint_as_float(((127u + 127u + kRestBits + kPlaceBits<T>) << 23) - rest_exponent<T>(v)); };
    const float2 n = fma2(r, make_float2(scale(rounded.x), scale(rounded.y)), pair(12582912.0f));
    return static_cast<unsigned short>(__byte_perm(__float_as_uint(n.x), __float_as_uint(n.y), 0x0040));
}

template <class T>
__device__ __forceinline__ float2 with_rest(float2 rounded, unsigned short bytes)
{
    const auto step = [](float v) { return __uint_as_float(rest_exponent<T>(v) - ((kRestBits + kPlaceBits<T>) << 23)); };
    const float2 n = make_float2(static_cast<float>(static_cast<signed char>(bytes)), static_cast<float>(static_cast<signed char>(bytes >> 8)));
    return fma2(n, make_float2(step(rounded.x), step(rounded.y)), rounded);
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
