// Attention to states of another length: the C ABI (include/spectral_b200.h: spectral_cross_attention and
// its backward), the float32 kernels, and the kernels around the 16-bit ones.
//
// Float32 calls that the tensor-core kernels (attention_tc32.cu) do not take, those of 9 to 16 rows per key head and
// of more than 64 query heads to one, run on the CUDA cores: FP32 multiply-adds two to an instruction, tiles of rows x 64
// keys, operands staged through shared memory as float32 with what must not count as zeros. A pass over the keys keeps the
// running maximum and sum of each row. The backward pass recomputes the scores twice, once for the
// keys' gradients (a CTA per 64 keys, a loop over rows) and once for the queries' (a CTA per 64 rows, a loop over
// keys): every sum has one owner, so nothing is atomic and equal inputs give equal bits.

#include "attention.cuh"
#include "extent.hpp"

#include <algorithm>
#include <cmath>
#include <initializer_list>

namespace spectral::attention {
namespace {

constexpr int kThreads = 256;
constexpr int kKeys = 64;  // per tile

// A tile of `Rows` rows of float32 in shared memory; the pitch keeps reads of 16 rows apart.
template <int Dim>
constexpr int kPitch = Dim + 4;
constexpr int kScorePitch = kKeys + 4;

// A row of `dim` values into a tile's row, `Lanes` lanes side by side, zeros behind it; zeros throughout without a source.
// `vectors`: source rows are 16-byte aligned and dim is a multiple of 4.
template <int Dim, bool Vectors>
__device__ __forceinline__ void load_row(float* to, const float* from, int dim, int at)
{
    if constexpr (Vectors) {
        const int d = 4 * at;
        const float4 v = from != nullptr && d < dim ? *reinterpret_cast<const float4*>(from + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        *reinterpret_cast<float4*>(to + d) = v;
    } else {
        to[at] = from != nullptr && at < dim ? from[at] : 0.0f;
    }
}

// Rows [first, first + Rows) of queries (or of an array of their shape), zeros past the end.
template <int Dim, int Rows, bool Vectors>
__device__ __forceinline__ void fill_rows(float* tile, const Call& c, const float* base, const Strides& s, long long first)
{
    constexpr int kLanes = Vectors ? Dim / 4 : Dim;  // per row
    constexpr int kAtOnce = kThreads / kLanes;
    const int at = threadIdx.x % kLanes;
#pragma unroll 8
    for (int row = threadIdx.x / kLanes; row < Rows; row += kAtOnce) {
        const unsigned r = static_cast<unsigned>(first) + row;  // rows stay below 2^31
        const unsigned t = r / static_cast<unsigned>(c.group);
        const float* from = base + t * s.token + static_cast<int>(r - t * c.group) * s.head;
        load_row<Dim, Vectors>(tile + row * kPitch<Dim>, r < c.rows() ? from : nullptr, c.dim, at);
    }
}

template <int Dim, int Rows>
__device__ __forceinline__ void load_rows(float* tile, const Call& c, const void* p, const Strides& s, bool vectors, int b, int head, long long first)
{
    const float* base = static_cast<const float*>(p) + b * s.sample + head * c.group * s.head;
    if (vectors) {
        fill_rows<Dim, Rows, true>(tile, c, base, s, first);
    } else {
        fill_rows<Dim, Rows, false>(tile, c, base, s, first);
    }
}

// Keys [first, first + kKeys) of k or v, zeros where `valid` is not set.
template <int Dim, bool Vectors>
__device__ __forceinline__ void fill_keys(float* tile, const Call& c, const float* base, const Strides& s, unsigned long long valid)
{
    constexpr int kLanes = Vectors ? Dim / 4 : Dim;
    constexpr int kAtOnce = kThreads / kLanes;
    const int at = threadIdx.x % kLanes;
#pragma unroll 8
    for (int key = threadIdx.x / kLanes; key < kKeys; key += kAtOnce) {
        load_row<Dim, Vectors>(tile + key * kPitch<Dim>, (valid >> key & 1) != 0 ? base + key * s.token : nullptr, c.dim, at);
    }
}

template <int Dim>
__device__ __forceinline__ void load_keys(float* tile, const Call& c, const void* p, const Strides& s, bool vectors, int b, int head, long long first,
                                          unsigned long long valid)
{
    const float* base = static_cast<const float*>(p) + b * s.sample + head * s.head + first * s.token;
    if (vectors) {
        fill_keys<Dim, true>(tile, c, base, s, valid);
    } else {
        fill_keys<Dim, false>(tile, c, base, s, valid);
    }
}

// One bit per key of the tile at `first` that counts (the same in every thread). `votes`: two words.
__device__ __forceinline__ unsigned long long valid_keys(const Call& c, int b, int length, long long first, unsigned* votes)
{
    const int key = threadIdx.x;
    __syncthreads();
    if (key < kKeys) {
        bool ok = first + key < length;
        if (ok && c.mask != nullptr) {
            ok = c.mask[static_cast<long long>(b) * c.keys + first + key] != 0;
        }
        const unsigned word = __ballot_sync(0xffffffffu, ok);
        if ((key & 31) == 0) {
            votes[key >> 5] = word;
        }
    }
    __syncthreads();
    return votes[0] | static_cast<unsigned long long>(votes[1]) << 32;
}

// R x 4 dot products over dim: rows row0 .. of a, rows col + 16 j of b.
template <int Dim, int R>
__device__ __forceinline__ void products(const float* a, const float* b, int dim, int row0, int col, float (&out)[R][4])
{
    float2 acc[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[i][j] = pair(0.0f);
        }
    }
#pragma unroll 2
    for (int d = 0; d < dim; d += 4) {  // what lies between dim and the next 4 is zero
        float4 x[R], y[4];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            x[i] = *reinterpret_cast<const float4*>(a + (row0 + i) * kPitch<Dim> + d);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            y[j] = *reinterpret_cast<const float4*>(b + (col + 16 * j) * kPitch<Dim> + d);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[i][j] = fma2(make_float2(x[i].x, x[i].y), make_float2(y[j].x, y[j].y), acc[i][j]);
                acc[i][j] = fma2(make_float2(x[i].z, x[i].w), make_float2(y[j].z, y[j].w), acc[i][j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            out[i][j] = acc[i][j].x + acc[i][j].y;
        }
    }
}

// The pairs of values a thread holds of a row of Dim: p * 32 + 2 col and the next.
template <int Dim>
constexpr int kPairs = Dim / 32;

// acc[i] += sum over keys of s[row0 + i][key] * m[key][its values].
template <int Dim, int R>
__device__ __forceinline__ void weigh_rows(const float* s, const float* m, int row0, int col, float2 (&acc)[R][kPairs<Dim>])
{
#pragma unroll 2
    for (int key = 0; key < kKeys; key += 4) {
        float4 w[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            w[i] = *reinterpret_cast<const float4*>(s + (row0 + i) * kScorePitch + key);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 v[kPairs<Dim>];
#pragma unroll
            for (int p = 0; p < kPairs<Dim>; ++p) {
                v[p] = *reinterpret_cast<const float2*>(m + (key + j) * kPitch<Dim> + p * 32 + 2 * col);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float f = j == 0 ? w[i].x : j == 1 ? w[i].y : j == 2 ? w[i].z : w[i].w;
#pragma unroll
                for (int p = 0; p < kPairs<Dim>; ++p) {
                    acc[i][p] = fma2(pair(f), v[p], acc[i][p]);
                }
            }
        }
    }
}

// acc[i] += sum over rows of s[row][key0 + i] * m[row][its values], eight keys.
template <int Dim, int Rows>
__device__ __forceinline__ void weigh_keys(const float* s, const float* m, int key0, int col, float2 (&acc)[8][kPairs<Dim>])
{
#pragma unroll 4
    for (int row = 0; row < Rows; ++row) {
        const float4 a = *reinterpret_cast<const float4*>(s + row * kScorePitch + key0);
        const float4 b = *reinterpret_cast<const float4*>(s + row * kScorePitch + key0 + 4);
#pragma unroll
        for (int p = 0; p < kPairs<Dim>; ++p) {
            const float2 v = *reinterpret_cast<const float2*>(m + row * kPitch<Dim> + p * 32 + 2 * col);
            acc[0][p] = fma2(pair(a.x), v, acc[0][p]);
            acc[1][p] = fma2(pair(a.y), v, acc[1][p]);
            acc[2][p] = fma2(pair(a.z), v, acc[2][p]);
            acc[3][p] = fma2(pair(a.w), v, acc[3][p]);
            acc[4][p] = fma2(pair(b.x), v, acc[4][p]);
            acc[5][p] = fma2(pair(b.y), v, acc[5][p]);
            acc[6][p] = fma2(pair(b.z), v, acc[6][p]);
            acc[7][p] = fma2(pair(b.w), v, acc[7][p]);
        }
    }
}

template <int Dim>
__device__ __forceinline__ void store_pairs(float* p, int dim, int col, const float2 (&v)[kPairs<Dim>], float factor)
{
#pragma unroll
    for (int j = 0; j < kPairs<Dim>; ++j) {
        const int d = j * 32 + 2 * col;
        if (d < dim) {
            p[d] = v[j].x * factor;
        }
        if (d + 1 < dim) {
            p[d + 1] = v[j].y * factor;
        }
    }
}

__device__ __forceinline__ float lanes16_max(float v)
{
#pragma unroll
    for (int o = 8; o > 0; o /= 2) {
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}
__device__ __forceinline__ float lanes16_sum(float v)
{
#pragma unroll
    for (int o = 8; o > 0; o /= 2) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// Where a kernel's results go: the call's arrays, or float32 parts of them.
struct Parts {
    bool vectors = false;     // every array's rows are 16-byte aligned
    int count = 1;
    long long span = 0;       // keys (forward, dq) or rows (dk, dv) of a part
    float* first = nullptr;   // sum p v, dq or dk: (part, pair, row, dim)
    float* second = nullptr;  // dv
    float2* stats = nullptr;  // forward: (part, pair, row)
};

// Forward: 16 R rows per CTA, thread (row group, column) of a 16 x 16 grid.
template <int Dim, int R>
__global__ void __launch_bounds__(kThreads, Dim == 128 ? 1 : 2) forward_kernel(const Call c, const Parts parts)
{
    constexpr int kRows = 16 * R;
    extern __shared__ __align__(16) float shared[];
    float* sq = shared;
    float* sk = sq + kRows * kPitch<Dim>;
    float* sv = sk + kKeys * kPitch<Dim>;
    float* sp = sv + kKeys * kPitch<Dim>;
    __shared__ unsigned votes[2];
    const int col = threadIdx.x & 15;
    const int row0 = (threadIdx.x >> 4) * R;
    const long long at = blockIdx.y;
    const int b = static_cast<int>(at / c.kv_heads), head = static_cast<int>(at - static_cast<long long>(b) * c.kv_heads);
    const long long first = static_cast<long long>(blockIdx.x) * kRows;
    const int part = blockIdx.z;
    allow_next_grid();
    wait_for_previous_grid();
    const int length = length_of(c, b);
    const long long begin = part * parts.span;
    const long long end = min(static_cast<long long>(length), begin + parts.span);
    load_rows<Dim, kRows>(sq, c, c.q, c.qs, parts.vectors, b, head, first);
    const float scale = c.scale * kLog2e;
    float most[R], total[R];
    float2 acc[R][kPairs<Dim>];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        most[i] = -INFINITY;
        total[i] = 0.0f;
#pragma unroll
        for (int p = 0; p < kPairs<Dim>; ++p) {
            acc[i][p] = pair(0.0f);
        }
    }
    for (long long key0 = begin; key0 < end; key0 += kKeys) {
        const unsigned long long valid = valid_keys(c, b, static_cast<int>(end), key0, votes);
        if (valid == 0) {
            continue;
        }
        load_keys<Dim>(sk, c, c.k, c.ks, parts.vectors, b, head, key0, valid);
        load_keys<Dim>(sv, c, c.v, c.vs, parts.vectors, b, head, key0, valid);
        __syncthreads();
        float s[R][4];
        products<Dim, R>(sq, sk, c.dim, row0, col, s);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float m = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = (valid >> (col + 16 * j) & 1) != 0 ? s[i][j] * scale : -INFINITY;
                m = fmaxf(m, s[i][j]);
            }
            m = fmaxf(most[i], lanes16_max(m));
            const float base = m == -INFINITY ? 0.0f : m;
            const float keep = exp2f(most[i] - base);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(s[i][j] - base);
                sum += p;
                sp[(row0 + i) * kScorePitch + col + 16 * j] = p;
            }
            most[i] = m;
            total[i] = total[i] * keep + lanes16_sum(sum);
#pragma unroll
            for (int p = 0; p < kPairs<Dim>; ++p) {
                acc[i][p] = acc[i][p] * pair(keep);
            }
        }
        __syncwarp();  // a row's scores are written and read by one warp
        weigh_rows<Dim, R>(sp, sv, row0, col, acc);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const long long r = first + row0 + i;
        if (r >= c.rows()) {
            continue;
        }
        const float base = most[i] == -INFINITY ? 0.0f : most[i];
        if (parts.count == 1) {
            store_pairs<Dim>(static_cast<float*>(c.out) + c.row_at(b, head, r), c.dim, col, acc[i], total[i] == 0.0f ? 0.0f : 1.0f / total[i]);
            if (c.stats != nullptr && col == 0) {
                c.stats[at * c.rows() + r] = make_float2(base, total[i]);
            }
        } else {
            const long long to = (part * c.pairs() + at) * c.rows() + r;
            store_pairs<Dim>(parts.first + to * c.dim, c.dim, col, acc[i], 1.0f);
            if (col == 0) {
                parts.stats[to] = make_float2(most[i], total[i]);
            }
        }
    }
}

// Scores of a tile, turned into p and p (dp - delta): what both backward kernels need.
template <int Dim>
__device__ __forceinline__ void score_gradients(const float* sq, const float* sk, const float* sv, const float* sdo, int dim, int row0, int col,
                                                float scale, unsigned long long valid, const float2 (&stats)[4], const float (&delta)[4],
                                                float (&p)[4][4], float (&ds)[4][4])
{
    products<Dim, 4>(sq, sk, dim, row0, col, p);
    products<Dim, 4>(sdo, sv, dim, row0, col, ds);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool ok = (valid >> (col + 16 * j) & 1) != 0;
            p[i][j] = ok ? exp2f(p[i][j] * scale - stats[i].x) * stats[i].y : 0.0f;
            ds[i][j] = ok ? p[i][j] * (ds[i][j] - delta[i]) : 0.0f;
        }
    }
}

// m and 1 / sum p, and delta, of rows row0 .. of the tile at `first`; zeros past the end and for empty rows.
__device__ __forceinline__ void row_constants(const Call& c, long long at, long long first, int row0, float2 (&stats)[4], float (&delta)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long r = first + row0 + i;
        stats[i] = make_float2(0.0f, 0.0f);
        delta[i] = 0.0f;
        if (r < c.rows()) {
            const float2 s = c.stats[at * c.rows() + r];
            stats[i] = make_float2(s.x, s.y == 0.0f ? 0.0f : 1.0f / s.y);
            delta[i] = c.delta[at * c.rows() + r];
        }
    }
}

template <int Dim>
__global__ void __launch_bounds__(kThreads, Dim == 128 ? 1 : 2) keys_backward_kernel(const Call c, const Parts parts)
{
    extern __shared__ __align__(16) float shared[];
    float* sk = shared;
    float* sv = sk + kKeys * kPitch<Dim>;
    float* sq = sv + kKeys * kPitch<Dim>;
    float* sdo = sq + 64 * kPitch<Dim>;
    float* sp = sdo + 64 * kPitch<Dim>;
    float* sds = sp + 64 * kScorePitch;
    __shared__ unsigned votes[2];
    const int col = threadIdx.x & 15;
    const int row0 = (threadIdx.x >> 4) * 4;
    const long long at = blockIdx.y;
    const int b = static_cast<int>(at / c.kv_heads), head = static_cast<int>(at - static_cast<long long>(b) * c.kv_heads);
    const long long key0 = static_cast<long long>(blockIdx.x) * kKeys;
    const int part = blockIdx.z;
    allow_next_grid();
    wait_for_previous_grid();
    const unsigned long long valid = valid_keys(c, b, length_of(c, b), key0, votes);
    load_keys<Dim>(sk, c, c.k, c.ks, parts.vectors, b, head, key0, valid);
    load_keys<Dim>(sv, c, c.v, c.vs, parts.vectors, b, head, key0, valid);
    const Strides dense{static_cast<long long>(c.queries) * c.kv_heads * c.group * c.dim, static_cast<long long>(c.kv_heads) * c.group * c.dim,
                        c.dim};
    // Half of the threads sum dv, the others dk: eight keys each.
    const bool of_v = threadIdx.x < kThreads / 2;
    const int keys0 = (threadIdx.x % (kThreads / 2) >> 4) * 8;
    float2 acc[8][kPairs<Dim>];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int p = 0; p < kPairs<Dim>; ++p) {
            acc[i][p] = pair(0.0f);
        }
    }
    const long long end = min(c.rows(), (part + 1) * parts.span);
    for (long long first = part * parts.span; first < end && valid != 0; first += 64) {
        __syncthreads();
        load_rows<Dim, 64>(sq, c, c.q, c.qs, parts.vectors, b, head, first);
        load_rows<Dim, 64>(sdo, c, c.dout, dense, parts.vectors, b, head, first);
        float2 stats[4];
        float delta[4], p[4][4], ds[4][4];
        row_constants(c, at, first, row0, stats, delta);
        __syncthreads();
        score_gradients<Dim>(sq, sk, sv, sdo, c.dim, row0, col, c.scale * kLog2e, valid, stats, delta, p, ds);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sp[(row0 + i) * kScorePitch + col + 16 * j] = p[i][j];
                sds[(row0 + i) * kScorePitch + col + 16 * j] = ds[i][j];
            }
        }
        __syncthreads();
        weigh_keys<Dim, 64>(of_v ? sp : sds, of_v ? sdo : sq, keys0, col, acc);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long key = key0 + keys0 + i;
        if (key >= c.keys) {
            continue;
        }
        if (parts.count == 1) {
            const long long to = ((static_cast<long long>(b) * c.keys + key) * c.kv_heads + head) * c.dim;
            store_pairs<Dim>(static_cast<float*>(of_v ? c.dv : c.dk) + to, c.dim, col, acc[i], of_v ? 1.0f : c.scale);
        } else {
            const long long to = ((part * c.pairs() + at) * c.keys + key) * c.dim;
            store_pairs<Dim>((of_v ? parts.second : parts.first) + to, c.dim, col, acc[i], 1.0f);
        }
    }
}

template <int Dim>
__global__ void __launch_bounds__(kThreads, Dim == 128 ? 1 : 2) rows_backward_kernel(const Call c, const Parts parts)
{
    extern __shared__ __align__(16) float shared[];
    float* sk = shared;
    float* sv = sk + kKeys * kPitch<Dim>;
    float* sq = sv + kKeys * kPitch<Dim>;
    float* sdo = sq + 64 * kPitch<Dim>;
    float* sds = sdo + 64 * kPitch<Dim>;
    __shared__ unsigned votes[2];
    const int col = threadIdx.x & 15;
    const int row0 = (threadIdx.x >> 4) * 4;
    const long long at = blockIdx.y;
    const int b = static_cast<int>(at / c.kv_heads), head = static_cast<int>(at - static_cast<long long>(b) * c.kv_heads);
    const long long first = static_cast<long long>(blockIdx.x) * 64;
    const int part = blockIdx.z;
    allow_next_grid();
    wait_for_previous_grid();
    const Strides dense{static_cast<long long>(c.queries) * c.kv_heads * c.group * c.dim, static_cast<long long>(c.kv_heads) * c.group * c.dim,
                        c.dim};
    load_rows<Dim, 64>(sq, c, c.q, c.qs, parts.vectors, b, head, first);
    load_rows<Dim, 64>(sdo, c, c.dout, dense, parts.vectors, b, head, first);
    float2 stats[4];
    float delta[4];
    row_constants(c, at, first, row0, stats, delta);
    float2 dq[4][kPairs<Dim>];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int p = 0; p < kPairs<Dim>; ++p) {
            dq[i][p] = pair(0.0f);
        }
    }
    const long long begin = part * parts.span;
    const long long end = min(static_cast<long long>(length_of(c, b)), begin + parts.span);
    for (long long key0 = begin; key0 < end; key0 += kKeys) {
        const unsigned long long valid = valid_keys(c, b, static_cast<int>(end), key0, votes);
        if (valid == 0) {
            continue;
        }
        load_keys<Dim>(sk, c, c.k, c.ks, parts.vectors, b, head, key0, valid);
        load_keys<Dim>(sv, c, c.v, c.vs, parts.vectors, b, head, key0, valid);
        __syncthreads();
        float p[4][4], ds[4][4];
        score_gradients<Dim>(sq, sk, sv, sdo, c.dim, row0, col, c.scale * kLog2e, valid, stats, delta, p, ds);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sds[(row0 + i) * kScorePitch + col + 16 * j] = ds[i][j];
            }
        }
        __syncwarp();
        weigh_rows<Dim, 4>(sds, sk, row0, col, dq);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long r = first + row0 + i;
        if (r >= c.rows()) {
            continue;
        }
        if (parts.count == 1) {
            store_pairs<Dim>(static_cast<float*>(c.dq) + c.row_at(b, head, r), c.dim, col, dq[i], c.scale);
        } else {
            const long long to = ((part * c.pairs() + at) * c.rows() + r) * c.dim;
            store_pairs<Dim>(parts.first + to, c.dim, col, dq[i], 1.0f);
        }
    }
}

// --- around them -------------------------------------------------------------------------------------

// A warp per row.
__global__ void __launch_bounds__(kThreads) row_products_kernel(const Call c)
{
    allow_next_grid();
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31;
    const long long all = static_cast<long long>(c.batch) * c.queries * c.kv_heads * c.group;
    const float* __restrict__ o = static_cast<const float*>(c.out);
    const float* __restrict__ g = static_cast<const float*>(c.dout);
    for (long long i = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); i < all;
         i += static_cast<long long>(gridDim.x) * (kThreads / 32)) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < SPECTRAL_HEAD_DIM_MAX / 32; ++k) {
            const int d = lane + 32 * k;
            if (d < c.dim) {
                sum = fmaf(o[i * c.dim + d], g[i * c.dim + d], sum);
            }
        }
#pragma unroll
        for (int s = 16; s > 0; s /= 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, s);
        }
        if (lane == 0) {
            // (sample, token, head) to (sample, key head, row).
            const int heads = c.kv_heads * c.group;
            const long long token = i / heads;  // of all samples
            const int h = static_cast<int>(i - token * heads);
            const long long b = token / c.queries;
            const int kv = h / c.group;
            c.delta[(b * c.kv_heads + kv) * c.rows() + (token - b * c.queries) * c.group + (h - kv * c.group)] = sum;
        }
    }
}

// V values of a row per thread.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) add_parts_kernel(const Call c, const __grid_constant__ Sums sums)
{
    allow_next_grid();
    wait_for_previous_grid();
    const Sum& job = sums.job[blockIdx.y];
    const float* __restrict__ partial = job.partial;
    T* __restrict__ result = static_cast<T*>(job.result);
    const bool of_keys = job.of_keys;
    const int parts = job.parts;
    const float factor = job.factor;
    const unsigned per_row = static_cast<unsigned>(c.dim / V);
    const unsigned count = of_keys ? c.keys : static_cast<unsigned>(c.rows());
    const long long rows = c.pairs() * count;
    const long long all = rows * c.dim;
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < rows * per_row; i += static_cast<long long>(gridDim.x) * kThreads) {
        Floats<V> sum;
        sum.fill(0.0f);
        for (int p = 0; p < parts; ++p) {
            const Floats<V> v = widen(*reinterpret_cast<const Vec<float, V>*>(partial + p * all + i * V));
#pragma unroll
            for (int j = 0; j < Floats<V>::kPairs; ++j) {
                sum.p[j] = sum.p[j] + v.p[j];
            }
        }
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            sum.p[j] = sum.p[j] * pair(factor);
        }
        long long row, at;
        if (rows * per_row < (1LL << 32)) {
            row = static_cast<unsigned>(i) / per_row;
            at = static_cast<unsigned>(row) / count;
        } else {
            row = i / per_row;
            at = row / count;
        }
        const int d = static_cast<int>(i - row * per_row) * V;
        const int r = static_cast<int>(row - at * count);
        const int b = static_cast<int>(at) / c.kv_heads, head = static_cast<int>(at) - b * c.kv_heads;
        const int token = of_keys ? r : r / c.group;
        const long long to = of_keys ? ((static_cast<long long>(b) * c.keys + r) * c.kv_heads + head) * c.dim
                                     : ((static_cast<long long>(b) * c.queries + token) * c.kv_heads + head) * c.group * c.dim + (r - token * c.group) * c.dim;
        *reinterpret_cast<Vec<T, V>*>(result + to + d) = narrow<T>(sum);
    }
}

// A warp per row.
template <class T>
__global__ void __launch_bounds__(kThreads) join_kernel(const Call c, const float* __restrict__ partial, const float2* __restrict__ stats,
                                                        int splits)
{
    allow_next_grid();
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31;
    const long long all = c.pairs() * c.rows();
    for (long long i = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); i < all;
         i += static_cast<long long>(gridDim.x) * (kThreads / 32)) {
        float most = -INFINITY;
        for (int s = lane; s < splits; s += 32) {
            most = fmaxf(most, stats[s * all + i].x);
        }
#pragma unroll
        for (int o = 16; o > 0; o /= 2) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        const float base = most == -INFINITY ? 0.0f : most;
        float total = 0.0f;
        float acc[SPECTRAL_HEAD_DIM_MAX / 32] = {};
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            const float2 st = stats[s * all + i];
            const float w = exp2f(st.x - base);
            total = fmaf(st.y, w, total);
#pragma unroll
            for (int k = 0; k < SPECTRAL_HEAD_DIM_MAX / 32; ++k) {
                const int d = lane + 32 * k;
                if (d < c.dim) {
                    acc[k] = fmaf(partial[(s * all + i) * c.dim + d], w, acc[k]);
                }
            }
        }
        const long long at = i / c.rows();
        const long long r = i - at * c.rows();
        const int b = static_cast<int>(at / c.kv_heads), head = static_cast<int>(at - static_cast<long long>(b) * c.kv_heads);
        const float f = total == 0.0f ? 0.0f : 1.0f / total;
        const long long to = c.row_at(b, head, r);
        T* out = static_cast<T*>(c.out) + to;
#pragma unroll
        for (int k = 0; k < SPECTRAL_HEAD_DIM_MAX / 32; ++k) {
            const int d = lane + 32 * k;
            if (d < c.dim) {
                out[d] = from_float<T>(acc[k] * f);
                if constexpr (sizeof(T) == 2) {
                    if (c.rest != nullptr) {
                        c.rest[to + d] = static_cast<unsigned char>(rest_of<T>(make_float2(acc[k] * f, 0.0f)));
                    }
                }
            }
        }
        if (c.stats != nullptr && lane == 0) {
            c.stats[i] = make_float2(base, total);
        }
    }
}

}  // namespace

void add_parts(const Call& c, const Sums& sums, cudaStream_t stream)
{
    if (sums.count == 0) {
        return;
    }
    bool fours = c.dim % 4 == 0;
    for (int i = 0; i < sums.count; ++i) {
        fours = fours && aligned_to(sums.job[i].result, 4 * dtype_size(c.dtype));
    }
    const long long all = c.pairs() * std::max<long long>(c.keys, c.rows()) * c.dim / (fours ? 4 : 1);
    const dim3 grid(static_cast<unsigned>(std::min<long long>((all + kThreads - 1) / kThreads, 148 * 16)), sums.count);
    with_dtype(c.dtype, [&](auto t) {
        using T = decltype(t);
        launch_pdl(fours ? add_parts_kernel<T, 4> : add_parts_kernel<T, 1>, grid, dim3(kThreads), 0, stream, c, sums);
    });
}

void join_splits(const Call& c, const float* partial, const float2* stats, int splits, cudaStream_t stream)
{
    const auto grid = static_cast<unsigned>(std::min<long long>((c.pairs() * c.rows() + 7) / 8, 148 * 16));
    with_dtype(c.dtype, [&](auto t) {
        launch_pdl(join_kernel<decltype(t)>, dim3(grid), dim3(kThreads), 0, stream, c, partial, stats, splits);
    });
}

namespace {

// delta = sum over dim of dout out.
void row_products(const Call& c, cudaStream_t stream)
{
    const auto grid = static_cast<unsigned>(std::min<long long>((c.pairs() * c.rows() + 7) / 8, 148 * 16));
    launch_pdl(row_products_kernel, dim3(grid), dim3(kThreads), 0, stream, c);
}

constexpr int kSms = 148;

// Calls f(integral_constant<Dim>) with the padded head size.
template <class F>
void with_dim(int dim, F&& f)
{
    if (dim <= 32) {
        f(std::integral_constant<int, 32>{});
    } else if (dim <= 64) {
        f(std::integral_constant<int, 64>{});
    } else {
        f(std::integral_constant<int, 128>{});
    }
}

// Rows per forward CTA: 64, or 16 where there are no more.
int forward_rows(const Call& c) { return c.rows() <= 16 ? 16 : 64; }

// Parts of an axis of `length` in tiles of 64, so that `tiles` CTAs per part fill the GPU about twice; a part's
// span is a whole number of tiles.
Parts split(long long tiles, long long length)
{
    Parts p;
    const long long all = pieces(length, 64);
    const long long wanted = std::max(1LL, std::min({all, (2LL * kSms + tiles - 1) / tiles, 256LL}));
    p.span = (all + wanted - 1) / wanted * 64;
    p.count = static_cast<int>(std::max(1LL, (length + p.span - 1) / std::max(1LL, p.span)));
    return p;
}

struct ForwardPlan {
    Parts parts;
    Arena arena;
    std::size_t partial = 0, stats = 0;

    explicit ForwardPlan(const Call& c)
    {
        parts = split(c.pairs() * pieces(c.rows(), forward_rows(c)), c.keys);
        if (parts.count > 1) {
            const std::size_t rows = static_cast<std::size_t>(c.pairs()) * c.rows() * parts.count;
            partial = arena.take(rows * c.dim * sizeof(float));
            stats = arena.take(rows * sizeof(float2));
        }
    }
};

// Float32 calls that run on the tensor cores: those whose tiles hold a token's heads, forward with more rows than a few (12
// rows over 8192 keys, 2 x 8 heads of 64: 96 us on them, 67 on the CUDA cores; backward 176 and 399).
bool on_tensor_cores(const Call& c, bool back) { return c.group <= 64 && c.keys > 0 && (back || c.rows() > 16); }

std::size_t forward_workspace(const Call& c)
{
    return few_rows(c)                       ? few_workspace(c)
           : c.dtype != SPECTRAL_FLOAT32 ? tensor_forward_workspace(c) : on_tensor_cores(c, false) ? split_forward_workspace(c) : ForwardPlan(c).arena.size();
}

struct BackwardPlan {
    Parts of_rows, of_keys;
    Arena arena;
    std::size_t delta = 0, dq = 0, dk = 0, dv = 0;

    explicit BackwardPlan(const Call& c)
    {
        const std::size_t rows = static_cast<std::size_t>(c.pairs()) * c.rows();
        const std::size_t keys = static_cast<std::size_t>(c.pairs()) * c.keys;
        delta = arena.take(rows * sizeof(float));
        of_keys = split(c.pairs() * pieces(c.rows(), 64), c.keys);
        of_rows = split(c.pairs() * pieces(c.keys, 64), c.rows());
        if (of_keys.count > 1) {
            dq = arena.take(rows * c.dim * of_keys.count * sizeof(float));
        }
        if (of_rows.count > 1) {
            dk = arena.take(keys * c.dim * of_rows.count * sizeof(float));
            dv = arena.take(keys * c.dim * of_rows.count * sizeof(float));
        }
    }
};

std::size_t backward_workspace(const Call& c)
{
    return c.dtype != SPECTRAL_FLOAT32 ? tensor_backward_workspace(c)
           : on_tensor_cores(c, true)  ? split_backward_workspace(c) : BackwardPlan(c).arena.size();
}

bool in_vectors(const Call& c, std::initializer_list<const void*> arrays, std::initializer_list<const Strides*> strides)
{
    bool ok = c.dim % 4 == 0;
    for (const void* p : arrays) {
        ok = ok && aligned_to(p, 16);
    }
    for (const Strides* s : strides) {
        ok = ok && s->sample % 4 == 0 && s->token % 4 == 0 && s->head % 4 == 0;
    }
    return ok;
}

template <class K, class... A>
void launch(K kernel, dim3 grid, std::size_t smem, cudaStream_t stream, const A&... args)
{
    const auto* f = reinterpret_cast<const void*>(kernel);
    SPECTRAL_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    SPECTRAL_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    launch_pdl(kernel, grid, dim3(kThreads), smem, stream, args...);
}

void forward(const Call& c, char* work, cudaStream_t stream)
{
    ForwardPlan plan(c);
    plan.parts.first = reinterpret_cast<float*>(work + plan.partial);
    plan.parts.stats = reinterpret_cast<float2*>(work + plan.stats);
    plan.parts.vectors = in_vectors(c, {c.q, c.k, c.v}, {&c.qs, &c.ks, &c.vs});
    const int rows = forward_rows(c);
    const dim3 grid(pieces(c.rows(), rows), static_cast<unsigned>(c.pairs()), plan.parts.count);
    with_dim(c.dim, [&](auto d) {
        constexpr int Dim = decltype(d)::value;
        const std::size_t smem = ((rows + 2 * kKeys) * kPitch<Dim> + rows * kScorePitch) * sizeof(float);
        if (rows == 16) {
            launch(forward_kernel<Dim, 1>, grid, smem, stream, c, plan.parts);
        } else {
            launch(forward_kernel<Dim, 4>, grid, smem, stream, c, plan.parts);
        }
    });
    if (plan.parts.count > 1) {
        join_splits(c, plan.parts.first, plan.parts.stats, plan.parts.count, stream);
    }
}

void backward(Call c, char* work, cudaStream_t stream)
{
    BackwardPlan plan(c);
    c.delta = reinterpret_cast<float*>(work + plan.delta);
    plan.of_keys.first = reinterpret_cast<float*>(work + plan.dq);
    plan.of_rows.first = reinterpret_cast<float*>(work + plan.dk);
    plan.of_rows.second = reinterpret_cast<float*>(work + plan.dv);
    plan.of_keys.vectors = plan.of_rows.vectors = in_vectors(c, {c.q, c.k, c.v, c.dout}, {&c.qs, &c.ks, &c.vs});
    row_products(c, stream);
    with_dim(c.dim, [&](auto d) {
        constexpr int Dim = decltype(d)::value;
        const std::size_t tiles = 4 * 64 * kPitch<Dim> * sizeof(float);
        constexpr std::size_t kScores = 64 * kScorePitch * sizeof(float);
        launch(keys_backward_kernel<Dim>, dim3(pieces(c.keys, 64), static_cast<unsigned>(c.pairs()), plan.of_rows.count), tiles + 2 * kScores, stream,
               c, plan.of_rows);
        launch(rows_backward_kernel<Dim>, dim3(pieces(c.rows(), 64), static_cast<unsigned>(c.pairs()), plan.of_keys.count), tiles + kScores, stream, c,
               plan.of_keys);
    });
    Sums sums;
    if (plan.of_rows.count > 1) {
        sums.add(plan.of_rows.first, plan.of_rows.count, true, c.dk, c.scale);
        sums.add(plan.of_rows.second, plan.of_rows.count, true, c.dv, 1.0f);
    }
    if (plan.of_keys.count > 1) {
        sums.add(plan.of_keys.first, plan.of_keys.count, false, c.dq, c.scale);
    }
    add_parts(c, sums, stream);
}

int invalid(const std::string& message)
{
    set_last_error(message);
    return SPECTRAL_INVALID_ARGUMENT;
}

// Sizes into `c`; strides may be NULL (contiguous arrays).
int sizes(const char* op, Call& c, const long long* strides, int dtype, long long batch, long long queries, long long keys, int heads,
          int kv_heads, int dim)
{
    const std::string name(op);
    if (!dtype_known(dtype)) {
        return invalid(name + ": dtype must be SPECTRAL_FLOAT32, SPECTRAL_BFLOAT16 or SPECTRAL_FLOAT16");
    }
    if (dim < 1 || dim > SPECTRAL_HEAD_DIM_MAX) {
        return invalid(name + ": need 1 <= dim <= " + std::to_string(SPECTRAL_HEAD_DIM_MAX));
    }
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0) {
        return invalid(name + ": heads must be a multiple of kv_heads, both at least 1");
    }
    if (heads / kv_heads > 128) {
        return invalid(name + ": at most 128 query heads may share a head of k and v");
    }
    constexpr long long kMost = (1LL << 31) - 256;
    if (batch < 0 || queries < 0 || keys < 0 || keys > kMost || queries > kMost / (heads / kv_heads) || batch > 65535 / kv_heads) {
        return invalid(name + ": need batch * kv_heads <= 65535, and keys and queries * heads / kv_heads below 2^31 - 256");
    }
    c.dtype = dtype;
    c.batch = static_cast<int>(batch);
    c.queries = static_cast<int>(queries);
    c.keys = static_cast<int>(keys);
    c.kv_heads = kv_heads;
    c.group = heads / kv_heads;
    c.dim = dim;
    const long long d = dim;
    c.qs = {queries * heads * d, heads * d, d};
    c.ks = {keys * kv_heads * d, kv_heads * d, d};
    c.vs = c.ks;
    if (strides != nullptr) {
        c.qs = {strides[0], strides[1], strides[2]};
        c.ks = {strides[3], strides[4], strides[5]};
        c.vs = {strides[6], strides[7], strides[8]};
    }
    return SPECTRAL_OK;
}

// What the arrays of a call can touch.
struct Extents {
    Extent q, k, v, rest, stats, lengths, mask;

    Extents(const Call& c, const void* lengths_at, int lengths64, const void* mask_at, const void* rest_at, const void* stats_at)
    {
        const std::size_t size = dtype_size(c.dtype);
        const long long heads = static_cast<long long>(c.kv_heads) * c.group;
        const long long q_count[3] = {c.batch, c.queries, heads}, k_count[3] = {c.batch, c.keys, c.kv_heads};
        const long long q_step[3] = {c.qs.sample, c.qs.token, c.qs.head}, k_step[3] = {c.ks.sample, c.ks.token, c.ks.head};
        const long long v_step[3] = {c.vs.sample, c.vs.token, c.vs.head};
        q = Extent(c.q, q_step, q_count, c.dim, size);
        k = Extent(c.k, k_step, k_count, c.dim, size);
        v = Extent(c.v, v_step, k_count, c.dim, size);
        const unsigned long long values = static_cast<unsigned long long>(c.batch) * c.queries * heads * c.dim;
        rest = Extent(rest_at, c.dtype == SPECTRAL_FLOAT32 ? 0 : values);
        stats = Extent(stats_at, values / c.dim * sizeof(float2));
        lengths = Extent(lengths_at, static_cast<unsigned long long>(c.batch) * (lengths64 != 0 ? 8 : 4));
        mask = Extent(mask_at, static_cast<unsigned long long>(c.batch) * c.keys);
    }
};

}  // namespace
}  // namespace spectral::attention

extern "C" int spectral_cross_attention_workspace(const void* q, const void* k, const void* v, const long long* strides, int dtype,
                                                  long long batch, long long queries, long long keys, int heads, int kv_heads, int dim,
                                                  size_t* count)
{
    using namespace spectral;
    using namespace spectral::attention;
    Call c;
    const int status = sizes("cross_attention_workspace", c, strides, dtype, batch, queries, keys, heads, kv_heads, dim);
    if (status != SPECTRAL_OK || count == nullptr) {
        return status != SPECTRAL_OK ? status : invalid("cross_attention_workspace: null count");
    }
    c.q = q;
    c.k = k;
    c.v = v;
    *count = 0;
    if (c.pairs() * c.rows() > 0) {
        try {
            *count = work_bytes(forward_workspace(c)) / 8;
        } catch (const std::exception& e) {
            set_last_error(e.what());
            return SPECTRAL_CUDA_ERROR;
        }
    }
    return SPECTRAL_OK;
}

extern "C" int spectral_cross_attention(const void* q, const void* k, const void* v, const long long* strides, const void* lengths,
                                        int lengths64, const void* mask, void* out, void* rest, float* stats, int dtype, long long batch,
                                        long long queries, long long keys, int heads, int kv_heads, int dim, float scale, void* work,
                                        void* stream)
{
    using namespace spectral;
    using namespace spectral::attention;
    Call c;
    const int status = sizes("cross_attention", c, strides, dtype, batch, queries, keys, heads, kv_heads, dim);
    if (status != SPECTRAL_OK) {
        return status;
    }
    if (c.pairs() * c.rows() == 0) {
        return SPECTRAL_OK;
    }
    const std::size_t size = dtype_size(dtype);
    if (q == nullptr || out == nullptr || (keys > 0 && (k == nullptr || v == nullptr))) {
        return invalid("cross_attention: null array");
    }
    for (const void* p : {q, k, v, static_cast<const void*>(out)}) {
        if (!aligned_to(p, size)) {
            return invalid("cross_attention: arrays must be aligned to their element size");
        }
    }
    if (!aligned_to(stats, 8) || !aligned_to(lengths, lengths64 != 0 ? 8 : 4) || !aligned_to(work, 8)) {
        return invalid("cross_attention: stats and work must be 8-byte aligned, lengths to their element size");
    }
    c.q = q;
    c.k = k;
    c.v = v;
    c.lengths = lengths;
    c.lengths64 = lengths64;
    c.mask = static_cast<const unsigned char*>(mask);
    c.out = out;
    c.rest = static_cast<unsigned char*>(rest);
    c.stats = reinterpret_cast<float2*>(stats);
    c.scale = scale;
    const Extents e(c, lengths, lengths64, mask, rest, stats);
    const Extent result(out, static_cast<unsigned long long>(batch) * queries * heads * dim * size);
    if (any_overlap({result, e.rest, e.stats}, {e.q, e.k, e.v, e.lengths, e.mask})) {
        return invalid("cross_attention: out, rest and stats must not overlap each other or the arguments");
    }
    try {
        const std::size_t needed = work_bytes(forward_workspace(c));
        if (work == nullptr && needed > 0) {
            return invalid("cross_attention: needs a workspace");
        }
        if (any_overlap({Extent(work, needed)}, {result, e.rest, e.stats, e.q, e.k, e.v, e.lengths, e.mask})) {
            return invalid("cross_attention: work must not overlap the arrays");
        }
        if (few_rows(c)) {
            few_forward(c, work_base(work), static_cast<cudaStream_t>(stream));
        } else if (dtype == SPECTRAL_FLOAT32 && on_tensor_cores(c, false)) {
            split_forward(c, work_base(work), static_cast<cudaStream_t>(stream));
        } else if (dtype == SPECTRAL_FLOAT32) {
            forward(c, work_base(work), static_cast<cudaStream_t>(stream));
        } else {
            tensor_forward(c, work_base(work), static_cast<cudaStream_t>(stream));
        }
        return SPECTRAL_OK;
    } catch (const InvalidArgument& e) {
        return invalid(e.what());
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}

extern "C" int spectral_cross_attention_backward_workspace(const void* dout, const void* q, const void* k, const void* v, const long long* strides, int dtype,
                                                           long long batch, long long queries, long long keys, int heads, int kv_heads,
                                                           int dim, size_t* count)
{
    using namespace spectral;
    using namespace spectral::attention;
    Call c;
    const int status = sizes("cross_attention_backward_workspace", c, strides, dtype, batch, queries, keys, heads, kv_heads, dim);
    if (status != SPECTRAL_OK || count == nullptr) {
        return status != SPECTRAL_OK ? status : invalid("cross_attention_backward_workspace: null count");
    }
    c.dout = dout;
    c.q = q;
    c.k = k;
    c.v = v;
    *count = 0;
    if (c.pairs() * c.rows() > 0 && keys > 0) {
        try {
            *count = work_bytes(backward_workspace(c)) / 8;
        } catch (const std::exception& e) {
            set_last_error(e.what());
            return SPECTRAL_CUDA_ERROR;
        }
    }
    return SPECTRAL_OK;
}

extern "C" int spectral_cross_attention_backward(const void* dout, const void* q, const void* k, const void* v, const long long* strides,
                                                 const void* out, const void* rest, const float* stats, const void* lengths, int lengths64, const void* mask,
                                                 void* dq, void* dk, void* dv, int dtype, long long batch, long long queries, long long keys,
                                                 int heads, int kv_heads, int dim, float scale, void* work, void* stream)
{
    using namespace spectral;
    using namespace spectral::attention;
    Call c;
    const int status = sizes("cross_attention_backward", c, strides, dtype, batch, queries, keys, heads, kv_heads, dim);
    if (status != SPECTRAL_OK) {
        return status;
    }
    const std::size_t size = dtype_size(dtype);
    const unsigned long long q_bytes = static_cast<unsigned long long>(batch) * queries * heads * dim * size;
    const unsigned long long k_bytes = static_cast<unsigned long long>(batch) * keys * kv_heads * dim * size;
    if ((q_bytes > 0 && dq == nullptr) || (k_bytes > 0 && (dk == nullptr || dv == nullptr))) {
        return invalid("cross_attention_backward: null array");
    }
    const auto s = static_cast<cudaStream_t>(stream);
    try {
        if (q_bytes == 0 || k_bytes == 0) {  // nothing attends, or to nothing
            for (const auto& z : {std::pair<void*, unsigned long long>{dq, q_bytes}, {dk, k_bytes}, {dv, k_bytes}}) {
                if (z.second > 0) {
                    SPECTRAL_CUDA(cudaMemsetAsync(z.first, 0, z.second, s));
                }
            }
            return SPECTRAL_OK;
        }
        if (dout == nullptr || q == nullptr || k == nullptr || v == nullptr || out == nullptr || stats == nullptr || work == nullptr) {
            return invalid("cross_attention_backward: null array");
        }
        for (const void* p : {dout, q, k, v, out, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)}) {
            if (!aligned_to(p, size)) {
                return invalid("cross_attention_backward: arrays must be aligned to their element size");
            }
        }
        if (!aligned_to(stats, 8) || !aligned_to(lengths, lengths64 != 0 ? 8 : 4) || !aligned_to(work, 8)) {
            return invalid("cross_attention_backward: stats and work must be 8-byte aligned, lengths to their element size");
        }
        c.q = q;
        c.k = k;
        c.v = v;
        c.lengths = lengths;
        c.lengths64 = lengths64;
        c.mask = static_cast<const unsigned char*>(mask);
        c.out = const_cast<void*>(out);
        c.rest = const_cast<unsigned char*>(static_cast<const unsigned char*>(rest));
        c.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
        c.dout = dout;
        c.dq = dq;
        c.dk = dk;
        c.dv = dv;
        c.scale = scale;
        const Extents e(c, lengths, lengths64, mask, rest, stats);
        const Extent of_dq(dq, q_bytes), of_dk(dk, k_bytes), of_dv(dv, k_bytes), of_dout(dout, q_bytes), of_out(out, q_bytes);
        if (any_overlap({of_dq, of_dk, of_dv}, {e.q, e.k, e.v, of_dout, of_out, e.rest, e.stats, e.lengths, e.mask})
            || any_overlap({Extent(work, work_bytes(backward_workspace(c)))},
                           {of_dq, of_dk, of_dv, e.q, e.k, e.v, of_dout, of_out, e.rest, e.stats, e.lengths, e.mask})) {
            return invalid("cross_attention_backward: gradients and work must not overlap each other or the arguments");
        }
        if (dtype == SPECTRAL_FLOAT32 && on_tensor_cores(c, true)) {
            split_backward(c, work_base(work), s);
        } else if (dtype == SPECTRAL_FLOAT32) {
            backward(c, work_base(work), s);
        } else {
            tensor_backward(c, work_base(work), s);
        }
        return SPECTRAL_OK;
    } catch (const InvalidArgument& e) {
        return invalid(e.what());
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}
