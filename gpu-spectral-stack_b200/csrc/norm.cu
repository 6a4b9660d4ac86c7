// Group norm with an activation over channels-last fields, forward and backward:
//     y = act(xhat w_c + b_c),  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),
// mean and var over the n = points x (channels / groups) values of one sample's group.
// Backward, with z = xhat w + b, dz = dy act'(z) and t = w dz:
//     dbias = sum dz, dweight = sum dz xhat  (over samples and points),
//     dx = rstd (t - mean(t) - xhat mean(t xhat))  (means over the group).
//
// HBM-bound: forward reads x and writes y, backward reads x (or its 8-bit checkpoint) and dy and
// writes dx; everything else is per channel. Both need all of a group before the first output: the
// values either stay on chip in between or are read twice. gelu and its slope keep the issue slots
// about as busy as the memory (pointwise.cuh).
//
// Resident form, for small arrays and small units: a unit is one sample's slice of whole groups. A
// cluster of 1 to 16 CTAs holds it in shared memory: each thread copies 16-byte pieces of its rows
// with cp.async and later reads only its own pieces, so the copies need no barrier. The CTAs reduce
// their part (mean first, then the centred squares, both from shared memory), exchange the
// partial results through distributed shared memory in rank order (the same bits every time), and
// write the outputs: one launch, each value read once. On large arrays its barriers cost more than
// the second read (64 x 16384 x 64 bf16: 119 us forward, 329 us backward).
//
// Two-pass form: chunks of a sample's rows give partial results (means and squares about them, joined
// block by block, so that neither a large mean nor an outlier cancels), a small kernel joins them, and
// the outputs are computed from a second read, which runs backwards to meet what is still in L2.
// Same array with gelu, calls in a graph: 77 us forward (402 MB in three passes: 5.2 TB/s; 67 us with no activation),
// 138 us backward (671 MB: 4.9 TB/s; 111 us), from an 8-bit checkpoint 169 us (100 us); float32 132 us (6.1 TB/s) and
// 209 us (6.4 TB/s), from a checkpoint 201 us. What bounds the 16-bit types with gelu are its instructions, computed
// twice in the backward pass: their kernels fill 61 to 71 % of the issue slots with a third of the warps.
// Cutting the batch so that a part's second read stays in L2 measured slower at every cut (2 to 16
// parts: 105 to 330 us forward, 180 to 470 us backward): each part pays its launches' ends.
// Keeping the second read in L2, with persistent CTAs that take sum and apply tasks a few samples
// apart, measured 97 us and 207 us: a sample's statistics take some 10 us from its last sum to its
// first output (fences, atomics, flags), and at this bandwidth 65 MB pass in that time.
//
// Samples of a few values each are the weak side of both: a CTA each, whatever they hold (65536 x 16 x 64: 850 us).
//
// All sums are FP32; 16-bit types are widened when read and rounded once when written.

#include "../../include/spectral_b200.h"

#include "backend.hpp"
#include "launch.cuh"
#include "pointwise.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace spectral {

void pack8(const void* x, int dtype, signed char* codes, float* scales, long long rows, int width, cudaStream_t stream);

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kCtaBytes = 200 * 1024;    // the most of a unit one CTA holds
constexpr int kGoodBytes = 64 * 1024;    // of a CTA's part: three share an SM
constexpr int kChunkBytes = 128 * 1024;  // two-pass form: of a CTA's chunk (64 KiB measured 5 % slower)
constexpr long long kResidentBytes = 8LL << 20;  // the resident form's largest array
constexpr long long kSmallSample = 32 * 1024;    // and the largest samples of larger arrays

// What the kernels need of one call. x holds values of T, or codes8 / scales their checkpoint.
struct NormShape {
    long long batch;
    long long points;
    int channels;
    int groups;
    int per_group;   // channels / groups
    int act;
    float eps;
};

// How the resident form cuts the work: slices of `width` channels (whole groups), clusters of
// `cluster` CTAs with `rows` points each, `lanes` threads across a row.
struct Slicing {
    int width = 0;
    int slices = 0;
    int lanes = 0;
    int rows_per_pass = 0;
    int cluster = 0;
    long long rows = 0;
    int passes = 0;
    std::size_t smem = 0;
};

// --- block-wide sums by channel -------------------------------------------------------------------

// Adds up part[0 .. V) over the threads that share a channel offset; on return sums[c] holds
// the total of channel c of the slice (c < width), visible to all threads. `scratch` holds
// kThreads * V floats. Threads past the last whole row pass zeros.
template <int V>
__device__ __forceinline__ void channel_sums(const Floats<V>& part, float* scratch, float* sums, int lanes, int width)
{
    const int tid = threadIdx.x;
    float p[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        p[j] = part.at(j);
    }
    __syncthreads();  // scratch and sums may still be read from the previous use
    int rows;
    if (lanes <= 32 && (lanes & (lanes - 1)) == 0) {
        // The lanes of a warp `lanes` apart hold the same channels.
        for (int o = 16; o >= lanes; o >>= 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                p[j] += __shfl_xor_sync(0xffffffffu, p[j], o);
            }
        }
        if ((tid & 31) < lanes) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                scratch[(tid >> 5) * width + (tid & 31) * V + j] = p[j];
            }
        }
        rows = kWarps;
    } else {
        rows = kThreads / lanes;
        if (tid < rows * lanes) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                scratch[(tid / lanes) * width + (tid % lanes) * V + j] = p[j];
            }
        }
    }
    __syncthreads();
    for (int c = tid; c < width; c += kThreads) {
        float s = 0.0f;
        for (int r = 0; r < rows; ++r) {
            s += scratch[r * width + c];
        }
        sums[c] = s;
    }
    __syncthreads();
}

// out[g] = the sum over group g's channels of sums[c] (times weight[c] where given), over `divisor`.
__device__ __forceinline__ void group_sums(const float* sums, const float* weight, float divisor, float* out, int groups,
                                           int per_group)
{
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    for (int g = warp; g < groups; g += kWarps) {
        float s = 0.0f;
        for (int c = lane; c < per_group; c += 32) {
            const float v = sums[g * per_group + c];
            s = weight != nullptr ? fmaf(v, weight[g * per_group + c], s) : s + v;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        if (lane == 0) {
            out[g] = __fdiv_rn(s, divisor);  // a constant group's mean is exact
        }
    }
    __syncthreads();
}

// --- resident form -----------------------------------------------------------------------------------

template <class T, int V, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_resident_kernel(const T* __restrict__ x, const float* __restrict__ weight, const float* __restrict__ bias,
                         T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, NormShape n,
                         Slicing s)
{
    using Piece = Vec<T, V>;
    allow_next_grid();
    extern __shared__ __align__(16) unsigned char smem[];
    auto* data = reinterpret_cast<Piece*>(smem);  // [pass][thread]
    float* scratch = reinterpret_cast<float*>(smem + static_cast<std::size_t>(s.passes) * kThreads * sizeof(Piece));
    float* sums = scratch + kThreads * V;
    float* mine = sums + s.width;        // this CTA's (mean, centred squares) per group: read by the cluster
    const int groups = s.width / n.per_group;
    float* mean = mine + 2 * groups;
    float* rstd = mean + groups;

    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
    const long long unit = blockIdx.x / s.cluster;
    const long long sample = unit / s.slices;
    const int c0 = static_cast<int>(unit % s.slices) * s.width;
    const int tid = threadIdx.x;
    const int lane_c = (tid % s.lanes) * V;
    const int row0 = tid / s.lanes;
    const bool active = row0 < s.rows_per_pass;
    const long long begin = rank * s.rows < n.points ? rank * s.rows : n.points;
    const long long count = (begin + s.rows < n.points ? begin + s.rows : n.points) - begin;
    const long long base = (sample * n.points + begin) * n.channels + c0 + lane_c;
    wait_for_previous_grid();

    int held = 0;  // passes this thread has a row for
    if (active) {
        for (int i = 0; i < s.passes; ++i) {
            const long long r = row0 + static_cast<long long>(i) * s.rows_per_pass;
            if (r >= count) {
                break;
            }
            copy_async<sizeof(Piece)>(&data[i * kThreads + tid], x + base + r * n.channels);
            held = i + 1;
        }
    }
    Floats<V> w, b;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w.set(j, weight != nullptr && active ? weight[c0 + lane_c + j] : 1.0f);
        b.set(j, bias != nullptr && active ? bias[c0 + lane_c + j] : 0.0f);
    }
    cp_async_wait_all();

    const Piece* own = data + tid;
    Floats<V> part;
    part.fill(0.0f);
#pragma unroll 4
    for (int i = 0; i < held; ++i) {
        const Floats<V> f = widen(own[i * kThreads]);
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            part.p[j] = part.p[j] + f.p[j];
        }
    }
    const float here = static_cast<float>(count) * static_cast<float>(n.per_group);
    channel_sums<V>(part, scratch, sums, s.lanes, s.width);
    group_sums(sums, nullptr, fmaxf(here, 1.0f), mean, groups, n.per_group);
    Floats<V> m;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        m.set(j, active ? mean[(lane_c + j) / n.per_group] : 0.0f);
    }
    part.fill(0.0f);
#pragma unroll 4
    for (int i = 0; i < held; ++i) {
        const Floats<V> f = widen(own[i * kThreads]);
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            const float2 d = f.p[j] - m.p[j];
            part.p[j] = fma2(d, d, part.p[j]);
        }
    }
    channel_sums<V>(part, scratch, sums, s.lanes, s.width);
    group_sums(sums, nullptr, 1.0f, rstd, groups, n.per_group);  // the centred squares for now
    for (int g = tid; g < groups; g += kThreads) {
        mine[2 * g] = mean[g];
        mine[2 * g + 1] = rstd[g];
    }
    cluster.sync();
    // The CTAs' means and squares join by the parallel form: squares about the joint mean are the
    // own squares plus count x (own mean - joint mean)^2.
    const float total = static_cast<float>(n.points) * static_cast<float>(n.per_group);
    for (int g = tid; g < groups; g += kThreads) {
        // The joint mean as a correction to the first CTA's (which always has rows).
        const float first = cluster.map_shared_rank(mine, 0)[2 * g];
        float joint = 0.0f, square = 0.0f;
        for (int k = 1; k < s.cluster; ++k) {
            const long long left = n.points - k * s.rows;
            const float share = static_cast<float>(left < 0 ? 0 : left < s.rows ? left : s.rows)
                                * static_cast<float>(n.per_group);
            joint += share > 0.0f ? (cluster.map_shared_rank(mine, k)[2 * g] - first) * (share / total) : 0.0f;
        }
        joint += first;
        for (int k = 0; k < s.cluster; ++k) {
            const long long left = n.points - k * s.rows;
            const float share = static_cast<float>(left < 0 ? 0 : left < s.rows ? left : s.rows)
                                * static_cast<float>(n.per_group);
            const float* theirs = cluster.map_shared_rank(mine, k) + 2 * g;
            const float d = theirs[0] - joint;
            square += share > 0.0f ? fmaf(share * d, d, theirs[1]) : 0.0f;
        }
        const float r = rsqrtf(square / total + n.eps);
        mean[g] = joint;
        rstd[g] = r;
        if (rank == 0 && mean_out != nullptr) {
            const long long at = sample * n.groups + c0 / n.per_group + g;
            mean_out[at] = joint;
            rstd_out[at] = r;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = active ? (lane_c + j) / n.per_group : 0;
        m.set(j, mean[g]);
        w.set(j, w.at(j) * rstd[g]);
    }
    T* out = y + base + row0 * static_cast<long long>(n.channels);
    const long long step = static_cast<long long>(s.rows_per_pass) * n.channels;
#pragma unroll 2
    for (int i = 0; i < held; ++i) {
        Floats<V> f = widen(own[i * kThreads]);
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            f.p[j] = activate2<Act, T>(fma2(f.p[j] - m.p[j], w.p[j], b.p[j]));
        }
        *reinterpret_cast<Piece*>(out) = narrow<T>(f);
        out += step;
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
}

// The x operand of the backward kernels: values of T, or the codes and scales of a checkpoint.
template <class T, int V, bool Packed>
struct Input {
    using Value = std::conditional_t<Packed, signed char, T>;
    using Raw = Vec<Value, V>;
    const T* x;
    const signed char* codes;
    const float* scales;  // one per row and block of 64 channels

    __device__ __forceinline__ const void* at(long long index) const
    {
        if constexpr (Packed) {
            return codes + index;
        } else {
            return x + index;
        }
    }
    // V > 1 divides both the block and the piece's first channel, so a piece lies in one block.
    __device__ __forceinline__ const float* scale_at(long long row, int channel, int channels) const
    {
        return scales + row * ((channels + kPackBlock - 1) / kPackBlock) + channel / kPackBlock;
    }
    __device__ static __forceinline__ Floats<V> values(const Raw& raw, float scale)
    {
        if constexpr (Packed) {
            return restored<T, V>(raw, scale);
        } else {
            return widen(raw);
        }
    }
};

// What a thread of the backward kernels needs of its V channels.
template <int V>
struct Channels {
    Floats<V> mean, rstd, weight, bias;

    __device__ __forceinline__ void load(const float* mean_in, const float* rstd_in, const float* w, const float* b,
                                         const NormShape& n, long long sample, int c0, bool active)
    {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = active ? c0 + j : 0;
            const long long g = sample * n.groups + c / n.per_group;
            mean.set(j, mean_in[g]);
            rstd.set(j, rstd_in[g]);
            weight.set(j, w != nullptr ? w[c] : 1.0f);
            bias.set(j, b != nullptr ? b[c] : 0.0f);
        }
        if constexpr (V == 1) {
            mean.p[0].y = 0.0f;
            rstd.p[0].y = 0.0f;
            weight.p[0].y = 0.0f;
            bias.p[0].y = 0.0f;
        }
    }
    // xhat and dz = dy act'(z) of pair j.
    template <int Act, class T>
    __device__ __forceinline__ float2 slope(float2 x, float2 dy, int j, float2& xhat) const
    {
        xhat = (x - mean.p[j]) * rstd.p[j];
        float2 s;
        activate_slope2<Act, T>(fma2(xhat, weight.p[j], bias.p[j]), s);
        return dy * s;
    }
};

template <class T, int V, bool Packed, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_backward_resident_kernel(const T* __restrict__ dy, Input<T, V, Packed> in, const float* __restrict__ weight,
                                  const float* __restrict__ bias, const float* __restrict__ mean,
                                  const float* __restrict__ rstd, T* __restrict__ dx, float* __restrict__ sample_sums,
                                  NormShape n, Slicing s)
{
    using Piece = Vec<T, V>;
    using Raw = typename Input<T, V, Packed>::Raw;
    allow_next_grid();
    extern __shared__ __align__(16) unsigned char smem[];
    const std::size_t pieces = static_cast<std::size_t>(s.passes) * kThreads;
    auto* data_dy = reinterpret_cast<Piece*>(smem);
    auto* data_x = reinterpret_cast<Raw*>(smem + pieces * sizeof(Piece));
    // pieces is a multiple of kThreads, so every array starts aligned.
    auto* data_scale = reinterpret_cast<float*>(smem + pieces * (sizeof(Piece) + sizeof(Raw)));
    float* scratch = data_scale + (Packed ? pieces : 0);
    float* sum_dz = scratch + kThreads * V;   // per channel: this CTA's, read by the cluster
    float* sum_dzx = sum_dz + s.width;
    float* all_dz = sum_dzx + s.width;        // per channel: the whole unit's
    float* all_dzx = all_dz + s.width;
    float* w_smem = all_dzx + s.width;
    const int groups = s.width / n.per_group;
    float* mean_t = w_smem + s.width;         // per group: mean(t) and mean(t xhat)
    float* mean_tx = mean_t + groups;

    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
    const long long unit = blockIdx.x / s.cluster;
    const long long sample = unit / s.slices;
    const int c0 = static_cast<int>(unit % s.slices) * s.width;
    const int tid = threadIdx.x;
    const int lane_c = (tid % s.lanes) * V;
    const int row0 = tid / s.lanes;
    const bool active = row0 < s.rows_per_pass;
    const long long begin = rank * s.rows < n.points ? rank * s.rows : n.points;
    const long long count = (begin + s.rows < n.points ? begin + s.rows : n.points) - begin;
    const long long base = (sample * n.points + begin) * n.channels + c0 + lane_c;
    wait_for_previous_grid();

    int held = 0;
    if (active) {
        for (int i = 0; i < s.passes; ++i) {
            const long long r = row0 + static_cast<long long>(i) * s.rows_per_pass;
            if (r >= count) {
                break;
            }
            copy_async<sizeof(Piece)>(&data_dy[i * kThreads + tid], dy + base + r * n.channels);
            copy_async<sizeof(Raw)>(&data_x[i * kThreads + tid], in.at(base + r * n.channels));
            if constexpr (Packed) {
                copy_async<4>(&data_scale[i * kThreads + tid],
                              in.scale_at(sample * n.points + begin + r, c0 + lane_c, n.channels));
            }
            held = i + 1;
        }
    }
    Channels<V> ch;
    ch.load(mean, rstd, weight, bias, n, sample, c0 + lane_c, active);
    for (int c = tid; c < s.width; c += kThreads) {
        w_smem[c] = weight != nullptr ? weight[c0 + c] : 1.0f;
    }
    cp_async_wait_all();

    Floats<V> part_dz, part_dzx;
    part_dz.fill(0.0f);
    part_dzx.fill(0.0f);
#pragma unroll 2
    for (int i = 0; i < held; ++i) {
        const Floats<V> g = widen(data_dy[i * kThreads + tid]);
        const Floats<V> f = Input<T, V, Packed>::values(data_x[i * kThreads + tid], Packed ? data_scale[i * kThreads + tid] : 1.0f);
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            float2 xhat;
            const float2 dz = ch.template slope<Act, T>(f.p[j], g.p[j], j, xhat);
            part_dz.p[j] = part_dz.p[j] + dz;
            part_dzx.p[j] = fma2(dz, xhat, part_dzx.p[j]);
        }
    }
    channel_sums<V>(part_dz, scratch, sum_dz, s.lanes, s.width);
    channel_sums<V>(part_dzx, scratch, sum_dzx, s.lanes, s.width);
    cluster.sync();
    for (int c = tid; c < s.width; c += kThreads) {
        float a = 0.0f, ax = 0.0f;
        for (int k = 0; k < s.cluster; ++k) {
            a += cluster.map_shared_rank(sum_dz, k)[c];
            ax += cluster.map_shared_rank(sum_dzx, k)[c];
        }
        all_dz[c] = a;
        all_dzx[c] = ax;
        if (rank == 0 && sample_sums != nullptr) {  // [2][sample][channel]: dbias, dweight of the sample
            sample_sums[sample * n.channels + c0 + c] = a;
            sample_sums[(n.batch + sample) * n.channels + c0 + c] = ax;
        }
    }
    __syncthreads();
    const float values = static_cast<float>(n.points) * static_cast<float>(n.per_group);
    group_sums(all_dz, w_smem, values, mean_t, groups, n.per_group);
    group_sums(all_dzx, w_smem, values, mean_tx, groups, n.per_group);
    Floats<V> mt, mtx;
    mt.fill(0.0f);
    mtx.fill(0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = active ? (lane_c + j) / n.per_group : 0;
        mt.set(j, mean_t[g]);
        mtx.set(j, mean_tx[g]);
    }
    T* out = dx + base + row0 * static_cast<long long>(n.channels);
    const long long step = static_cast<long long>(s.rows_per_pass) * n.channels;
#pragma unroll 2
    for (int i = 0; i < held; ++i) {
        const Floats<V> g = widen(data_dy[i * kThreads + tid]);
        Floats<V> f = Input<T, V, Packed>::values(data_x[i * kThreads + tid], Packed ? data_scale[i * kThreads + tid] : 1.0f);
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            float2 xhat;
            const float2 dz = ch.template slope<Act, T>(f.p[j], g.p[j], j, xhat);
            const float2 t = fma2(dz, ch.weight.p[j], pair(0.0f) - mt.p[j]);
            f.p[j] = ch.rstd.p[j] * (t - xhat * mtx.p[j]);
        }
        *reinterpret_cast<Piece*>(out) = narrow<T>(f);
        out += step;
    }
    cluster.sync();
}

// --- two-pass form -----------------------------------------------------------------------------------------

constexpr int kTileLanes = 64;   // threads across the channels of a tile, at most

// How the two-pass form cuts the work: tiles of `lanes` (a power of two) pieces across the channels,
// chunks of `rows` points; a CTA takes one chunk of one tile.
struct Chunking {
    int width = 0;
    int lanes = 0;
    int tiles = 0;
    int chunks = 0;
    long long rows = 0;
    // Statistics per chunk: one result per group where tiles hold whole groups, else per channel.
    int columns = 0;
    int merge = 0;    // channels that share one
};

struct Task {
    long long sample;
    int chunk;
    int c0;
    int count;  // rows
};

__device__ __forceinline__ long long chunk_count(const Chunking& s, long long points, int chunk)
{
    const long long left = points - chunk * s.rows;
    return left < 0 ? 0 : left < s.rows ? left : s.rows;
}

// The CTA's task. The second pass goes backwards: what the first read last is still in L2.
__device__ __forceinline__ Task task_of(const Chunking& s, const NormShape& n, bool second)
{
    const unsigned per = static_cast<unsigned>(s.chunks) * static_cast<unsigned>(s.tiles);
    const unsigned i = second ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    Task t;
    t.sample = i / per;
    t.chunk = static_cast<int>(i % per / static_cast<unsigned>(s.tiles));
    t.c0 = static_cast<int>(i % static_cast<unsigned>(s.tiles)) * s.width;
    t.count = static_cast<int>(chunk_count(s, n.points, t.chunk));
    return t;
}

// The warps' sums of a CTA: two values for each of a warp's channels.
template <int V>
struct Sums {
    float a[kWarps][32 * V];
    float b[kWarps][32 * V];
    float count[kWarps][32];  // rows behind them, per piece
};

// Mean and centred squares of K values per channel joined to the running ones of `have` values,
// by the parallel form; the block's own are taken about its own mean.
template <int V, int K>
__device__ __forceinline__ void join_block(const Floats<V> (&f)[K], float have, Floats<V>& mean, Floats<V>& square)
{
    const float all = have + static_cast<float>(K);
    const float2 share = pair(__fdividef(static_cast<float>(K), all));
    const float2 cross = pair(have * share.x);
#pragma unroll
    for (int j = 0; j < Floats<V>::kPairs; ++j) {
        float2 sum = f[0].p[j];
#pragma unroll
        for (int k = 1; k < K; ++k) {
            sum = sum + f[k].p[j];
        }
        const float2 m = sum * pair(1.0f / static_cast<float>(K));
        float2 q = square.p[j];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float2 d = f[k].p[j] - m;
            q = fma2(d, d, q);
        }
        const float2 d = m - mean.p[j];
        mean.p[j] = fma2(d, share, mean.p[j]);
        square.p[j] = fma2(d * d, cross, q);
    }
}

// Which warps of the CTA hold channel c of a tile: those with lane groups over it (lanes <= 32: all
// eight; 64: every second one, from c's half on); and c's index among a warp's channels.
__device__ __forceinline__ int in_warp(const Chunking& s, int vec, int c) { return s.lanes > 32 ? c % (32 * vec) : c; }
__device__ __forceinline__ int first_warp(const Chunking& s, int vec, int c) { return s.lanes > 32 ? c / (32 * vec) : 0; }
__device__ __forceinline__ int warp_step(const Chunking& s) { return s.lanes > 32 ? 2 : 1; }

__device__ __forceinline__ float block_sum(float v, float* scratch)
{
    const int tid = threadIdx.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    __syncthreads();
    if ((tid & 31) == 0) {
        scratch[tid >> 5] = v;
    }
    __syncthreads();
    float s = 0.0f;
    for (int k = 0; k < kWarps; ++k) {
        s += scratch[k];
    }
    return s;
}

// One CTA per sample and group: the chunks' results joined to the group's mean and rstd.
__global__ void __launch_bounds__(kThreads)
    norm_join_kernel(const float2* __restrict__ partial, float* __restrict__ mean, float* __restrict__ rstd, NormShape n,
                     Chunking s)
{
    __shared__ float scratch[kWarps];
    allow_next_grid();
    const long long sample = blockIdx.x / static_cast<unsigned>(n.groups);
    const int each = s.columns / n.groups;  // results per chunk and group
    const float2* src = partial + sample * s.chunks * s.columns + static_cast<int>(blockIdx.x % static_cast<unsigned>(n.groups)) * each;
    const float total = static_cast<float>(n.points) * static_cast<float>(n.per_group);
    wait_for_previous_grid();
    const float first = src[0].x;  // the joint mean is a correction to it
    float m = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x; i < each * s.chunks; i += kThreads) {
        const int chunk = i / each;
        const float2 p = src[static_cast<long long>(chunk) * s.columns + i % each];
        m = fmaf(p.x - first, static_cast<float>(chunk_count(s, n.points, chunk)) * static_cast<float>(s.merge), m);
    }
    const float joint = first + __fdiv_rn(block_sum(m, scratch), total);
    float q = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x; i < each * s.chunks; i += kThreads) {
        const int chunk = i / each;
        const float2 p = src[static_cast<long long>(chunk) * s.columns + i % each];
        const float d = p.x - joint;
        q += fmaf(static_cast<float>(chunk_count(s, n.points, chunk)) * static_cast<float>(s.merge) * d, d, p.y);
    }
    q = block_sum(q, scratch);
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = joint;
        rstd[blockIdx.x] = rsqrtf(__fdiv_rn(q, total) + n.eps);
    }
}

// One CTA per sample and group: the chunks added up per channel (every so many threads one channel,
// joined in a fixed order), and the group's mean(t) and mean(t xhat).
__global__ void __launch_bounds__(kThreads)
    norm_backward_join_kernel(const float2* __restrict__ partial, const float* __restrict__ weight,
                              float* __restrict__ sample_sums, float2* __restrict__ group_means, NormShape n, Chunking s)
{
    __shared__ float scratch[2 * kThreads];
    allow_next_grid();
    const int tid = threadIdx.x;
    const long long sample = blockIdx.x / static_cast<unsigned>(n.groups);
    const int first = static_cast<int>(blockIdx.x % static_cast<unsigned>(n.groups)) * n.per_group;
    const int across = min(n.per_group, kThreads);
    const int parts = kThreads / across;
    const int part = tid / across;
    wait_for_previous_grid();
    float t = 0.0f, tx = 0.0f;
    for (int c0 = 0; c0 < n.per_group; c0 += across) {
        const int c = c0 + tid % across;
        float a = 0.0f, ax = 0.0f;
        if (part < parts && c < n.per_group) {
            const float2* src = partial + sample * s.chunks * n.channels + first + c;
#pragma unroll 4
            for (int k = part; k < s.chunks; k += parts) {
                const float2 p = src[static_cast<long long>(k) * n.channels];
                a += p.x;
                ax += p.y;
            }
        }
        __syncthreads();
        scratch[tid] = a;
        scratch[kThreads + tid] = ax;
        __syncthreads();
        if (part == 0 && c < n.per_group) {
            for (int k = 1; k < parts; ++k) {
                a += scratch[k * across + tid];
                ax += scratch[kThreads + k * across + tid];
            }
            sample_sums[sample * n.channels + first + c] = a;
            sample_sums[(n.batch + sample) * n.channels + first + c] = ax;
            const float w = weight != nullptr ? weight[first + c] : 1.0f;
            t = fmaf(w, a, t);
            tx = fmaf(w, ax, tx);
        }
    }
    t = block_sum(t, scratch);
    tx = block_sum(tx, scratch);
    if (tid == 0) {
        const float values = static_cast<float>(n.points) * static_cast<float>(n.per_group);
        group_means[blockIdx.x] = make_float2(__fdiv_rn(t, values), __fdiv_rn(tx, values));
    }
}

// A working thread's rows of a task.
struct Place {
    int mine;        // passes it has a row for
    long long row;   // its first row, over the whole batch
    long long base;  // its first piece, in values
};

__device__ __forceinline__ Place place_of(const Task& t, const Chunking& s, const NormShape& n, int lane_c, int row0)
{
    Place p;
    const int rows_per_pass = kThreads / s.lanes;
    const bool active = lane_c < s.width && t.c0 + lane_c < n.channels;
    p.mine = active && row0 < t.count ? (t.count - row0 + rows_per_pass - 1) / rows_per_pass : 0;
    p.row = t.sample * n.points + t.chunk * s.rows + row0;
    p.base = p.row * n.channels + t.c0 + lane_c;
    return p;
}

template <int V>
__device__ __forceinline__ void to_shared(float* p, const Floats<V>& f)
{
#pragma unroll
    for (int j = 0; j < V; ++j) {
        p[j] = f.at(j);
    }
}

// Rows of x on their way to a thread of the forward kernels: blocks of kRun rows, two in flight while one is
// used. As in Ring, a thread reads only what it has copied.
constexpr int kRun = 4;
template <class T, int V>
struct RowRing {
    Vec<T, V> x[3 * kRun][kThreads];
};

// Calls f(pieces, i) for the thread's passes i ..: kRun rows at a time, then row by row.
template <class T, int V, class F>
__device__ __forceinline__ void for_rows(RowRing<T, V>& ring, const T* src, long long step, int mine, F&& f)
{
    using Piece = Vec<T, V>;
    const int tid = threadIdx.x;
    const int blocks = mine / kRun;
    int ahead = 0;  // blocks issued
    const auto issue = [&](int slot) {
        if (ahead < blocks) {
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                copy_async<sizeof(Piece)>(&ring.x[slot * kRun + k][tid], src);
                src += step;
            }
            ++ahead;
        }
        cp_async_commit();
    };
    issue(0);
    issue(1);
    int slot = 0;
    for (int b = 0; b < blocks; ++b) {
        cp_async_wait<1>();
        Piece raw[kRun];
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            raw[k] = ring.x[slot * kRun + k][tid];
        }
        issue(slot == 0 ? 2 : slot - 1);  // the slot of the block before, which has been used
        slot = slot == 2 ? 0 : slot + 1;
        f(raw, b * kRun);
    }
    for (int i = blocks * kRun; i < mine; ++i) {
        const Piece raw[1] = {*reinterpret_cast<const Piece*>(src)};
        f(raw, i);
        src += step;
    }
}

// Forward, first pass: the mean and centred squares of a chunk into `partial` ([sample][chunk][column]),
// and on the way, where asked, the 8-bit checkpoint.
template <class T, int V, bool Keep8>
__global__ void __launch_bounds__(kThreads)
    norm_sum_kernel(const T* __restrict__ x, signed char* __restrict__ codes, float* __restrict__ scales, float2* __restrict__ partial, NormShape n,
                    Chunking s)
{
    using Piece = Vec<T, V>;
    allow_next_grid();
    __shared__ union {
        RowRing<T, V> ring;
        Sums<V> sums;
    } shared;
    Sums<V>& sums = shared.sums;
    const int tid = threadIdx.x;
    const int lane = tid & 31;
    const int warp = tid >> 5;
    const Task t = task_of(s, n, false);
    const int lane_c = (tid % s.lanes) * V;
    const int rows_per_pass = kThreads / s.lanes;
    const Place at = place_of(t, s, n, lane_c, tid / s.lanes);
    const long long step = static_cast<long long>(rows_per_pass) * n.channels;
    const int blocks_per_row = (n.channels + kPackBlock - 1) / kPackBlock;
    wait_for_previous_grid();
    Floats<V> m, q;
    m.fill(0.0f);
    q.fill(0.0f);
    for_rows<T, V>(shared.ring, x + at.base, step, at.mine, [&](const auto& raw, int i) {
        constexpr int K = sizeof(raw) / sizeof(Piece);
        Floats<V> f[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            f[k] = widen(raw[k]);
        }
        join_block<V, K>(f, static_cast<float>(i), m, q);
        if constexpr (Keep8) {
            pack_blocks(
                raw,
                [&](int k) {
                    return scales + (at.row + static_cast<long long>(i + k) * rows_per_pass) * blocks_per_row
                           + (t.c0 + lane_c) / kPackBlock;
                },
                [&](int k, const Vec<signed char, V>& c) {
                    *reinterpret_cast<Vec<signed char, V>*>(codes + at.base + (i + k) * step) = c;
                });
        }
    });
    // The warp's rows of each channel joined about one of them: means and squares are then plain
    // sums (a reference this close costs at most a bit or two).
    __syncthreads();  // the sums lie where the rows did
    float count = static_cast<float>(at.mine);
    if (s.lanes < 32) {
        float total = count;
        for (int o = 16; o >= s.lanes; o >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, o);
        }
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            const float2 ref = make_float2(__shfl_sync(0xffffffffu, m.p[j].x, lane % s.lanes),
                                           __shfl_sync(0xffffffffu, m.p[j].y, lane % s.lanes));
            float2 d = at.mine > 0 ? m.p[j] - ref : pair(0.0f);
            float2 sq = fma2(pair(count) * d, d, q.p[j]);
            d = pair(count) * d;
            for (int o = 16; o >= s.lanes; o >>= 1) {
                d.x += __shfl_xor_sync(0xffffffffu, d.x, o);
                d.y += __shfl_xor_sync(0xffffffffu, d.y, o);
                sq.x += __shfl_xor_sync(0xffffffffu, sq.x, o);
                sq.y += __shfl_xor_sync(0xffffffffu, sq.y, o);
            }
            const float2 off = d * pair(__fdividef(1.0f, fmaxf(total, 1.0f)));
            m.p[j] = ref + off;
            q.p[j] = sq - d * off;
        }
        count = total;
    }
    if (lane < s.lanes && lane_c < s.width) {
        const int i = tid % s.lanes % 32;
        to_shared(&sums.a[warp][i * V], m);
        to_shared(&sums.b[warp][i * V], q);
        sums.count[warp][i] = count;
    }
    __syncthreads();
    // The warps', then the channels of a group's.
    float2* out = partial + (t.sample * s.chunks + t.chunk) * s.columns;
    const int width = min(s.width, n.channels - t.c0);
    const float total = static_cast<float>(t.count);
    for (int c = tid; c < width; c += kThreads) {
        const int w0 = first_warp(s, V, c), each = warp_step(s), i = in_warp(s, V, c);
        float cm = 0.0f, cq = 0.0f;
        for (int w = w0; w < kWarps; w += each) {
            cm = fmaf(sums.a[w][i], sums.count[w][i / V], cm);
        }
        cm = __fdiv_rn(cm, total);
        for (int w = w0; w < kWarps; w += each) {
            const float d = sums.a[w][i] - cm;
            cq += fmaf(sums.count[w][i / V] * d, d, sums.b[w][i]);
        }
        if (s.merge == 1) {
            out[t.c0 + c] = make_float2(cm, cq);
        } else {  // only this thread reads column i of these warps
            sums.a[w0][i] = cm;
            sums.b[w0][i] = cq;
        }
    }
    if (s.merge > 1) {
        __syncthreads();
        for (int g = tid; g < width / s.merge; g += kThreads) {
            float gm = 0.0f, gq = 0.0f;
            for (int c = g * s.merge; c < (g + 1) * s.merge; ++c) {
                gm += sums.a[first_warp(s, V, c)][in_warp(s, V, c)];
            }
            gm = __fdiv_rn(gm, static_cast<float>(s.merge));
            for (int c = g * s.merge; c < (g + 1) * s.merge; ++c) {
                const int w = first_warp(s, V, c), i = in_warp(s, V, c);
                const float d = sums.a[w][i] - gm;
                gq += fmaf(total * d, d, sums.b[w][i]);
            }
            out[t.c0 / s.merge + g] = make_float2(gm, gq);
        }
    }
}

// Forward, second pass.
template <class T, int V, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_apply_kernel(const T* __restrict__ x, const float* __restrict__ weight, const float* __restrict__ bias,
                      const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ y, NormShape n,
                      Chunking s)
{
    using Piece = Vec<T, V>;
    allow_next_grid();
    __shared__ RowRing<T, V> ring;
    const int tid = threadIdx.x;
    const Task t = task_of(s, n, true);
    const int lane_c = (tid % s.lanes) * V;
    const int rows_per_pass = kThreads / s.lanes;
    const Place at = place_of(t, s, n, lane_c, tid / s.lanes);
    const long long step = static_cast<long long>(rows_per_pass) * n.channels;
    wait_for_previous_grid();
    if (at.mine == 0) {
        return;
    }
    Channels<V> ch;
    ch.load(mean, rstd, weight, bias, n, t.sample, t.c0 + lane_c, true);
#pragma unroll
    for (int j = 0; j < Floats<V>::kPairs; ++j) {
        ch.weight.p[j] = ch.weight.p[j] * ch.rstd.p[j];
    }
    T* dst = y + at.base;
    for_rows<T, V>(ring, x + at.base, step, at.mine, [&](const auto& raw, int) {
        constexpr int K = sizeof(raw) / sizeof(Piece);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Floats<V> f = widen(raw[k]);
#pragma unroll
            for (int j = 0; j < Floats<V>::kPairs; ++j) {
                f.p[j] = activate2<Act, T>(fma2(f.p[j] - ch.mean.p[j], ch.weight.p[j], ch.bias.p[j]));
            }
            *reinterpret_cast<Piece*>(dst) = narrow<T>(f);
            dst += step;
        }
    });
}

// Rows of dy and x on their way to a thread of the backward kernels, kAhead of them in flight. Each thread
// copies its own pieces and reads only those, so nothing but its own wait is needed. In registers, two
// rows ahead, they left two CTAs of 120 registers a thread on an SM and half the bandwidth unused.
constexpr int kAhead = 4;
template <class T, int V, bool Packed>
struct Ring {
    Vec<T, V> g[kAhead + 1][kThreads];
    typename Input<T, V, Packed>::Raw v[kAhead + 1][kThreads];
    float scale[Packed ? kAhead + 1 : 1][kThreads];
};

// Backward: calls f(dy, x) for the thread's rows.
template <class T, int V, bool Packed, class F>
__device__ __forceinline__ void for_gradient_rows(Ring<T, V, Packed>& ring, const T* dy, const Input<T, V, Packed>& in,
                                                  const Place& at, int channel, const NormShape& n, int rows_per_pass, F&& f)
{
    using Piece = Vec<T, V>;
    using Raw = typename Input<T, V, Packed>::Raw;
    const int tid = threadIdx.x;
    // One pointer per array, moved by a constant: the addresses were a third of the instructions.
    const int step = rows_per_pass * n.channels;
    const int scale_step = rows_per_pass * ((n.channels + kPackBlock - 1) / kPackBlock);
    const T* g = dy + at.base;
    const auto* v = static_cast<const typename Input<T, V, Packed>::Value*>(in.at(at.base));
    const float* scale = Packed ? in.scale_at(at.row, channel, n.channels) : nullptr;
    int left = at.mine;
    const auto issue = [&](int slot) {
        if (left > 0) {
            copy_async<sizeof(Piece)>(&ring.g[slot][tid], g);
            copy_async<sizeof(Raw)>(&ring.v[slot][tid], v);
            if constexpr (Packed) {
                copy_async<4>(&ring.scale[slot][tid], scale);
            }
        }
        --left;
        g += step;
        v += step;
        scale += Packed ? scale_step : 0;
        cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        issue(k);
    }
    int slot = 0;
    for (int i = 0; i < at.mine; ++i) {
        cp_async_wait<kAhead - 1>();
        const Piece dyv = ring.g[slot][tid];
        const Raw raw = ring.v[slot][tid];
        const float s = Packed ? ring.scale[slot][tid] : 1.0f;
        issue(slot == 0 ? kAhead : slot - 1);  // the slot of the row before, which has been used
        slot = slot == kAhead ? 0 : slot + 1;
        f(widen(dyv), Input<T, V, Packed>::values(raw, s));
    }
}

// What the backward kernels need of a thread's channels: dz = dy act'(z) with z = d w rstd + b, d = x - mean.
template <int V>
struct Folded {
    Floats<V> mean, scale, bias;

    __device__ __forceinline__ explicit Folded(const Channels<V>& c) : mean(c.mean), bias(c.bias)
    {
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            scale.p[j] = c.weight.p[j] * c.rstd.p[j];
        }
    }
    template <int Act, class T>
    __device__ __forceinline__ float2 slope(float2 x, float2 dy, int j, float2& d) const
    {
        d = x - mean.p[j];
        float2 s;
        activate_slope2<Act, T>(fma2(d, scale.p[j], bias.p[j]), s);
        return dy * s;
    }
};

// Backward, first pass: sum dz and sum dz xhat of a chunk per channel.
template <class T, int V, bool Packed, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_backward_sum_kernel(const T* __restrict__ dy, Input<T, V, Packed> in, const float* __restrict__ weight,
                             const float* __restrict__ bias, const float* __restrict__ mean,
                             const float* __restrict__ rstd, float2* __restrict__ partial, NormShape n, Chunking s)
{
    allow_next_grid();
    __shared__ union {
        Ring<T, V, Packed> ring;
        Sums<V> sums;
    } shared;
    Sums<V>& sums = shared.sums;
    const int tid = threadIdx.x;
    const int lane = tid & 31;
    const int warp = tid >> 5;
    const Task t = task_of(s, n, false);
    const int lane_c = (tid % s.lanes) * V;
    const int rows_per_pass = kThreads / s.lanes;
    const Place at = place_of(t, s, n, lane_c, tid / s.lanes);
    wait_for_previous_grid();
    Floats<V> a, b;
    a.fill(0.0f);
    b.fill(0.0f);
    {
        Channels<V> all;
        all.load(mean, rstd, weight, bias, n, t.sample, t.c0 + lane_c, at.mine > 0);
        const Folded<V> ch(all);
        for_gradient_rows<T, V, Packed>(shared.ring, dy, in, at, t.c0 + lane_c, n, rows_per_pass,
                                        [&](const Floats<V>& g, const Floats<V>& x) {
#pragma unroll
            for (int j = 0; j < Floats<V>::kPairs; ++j) {
                float2 d;
                const float2 dz = ch.template slope<Act, T>(x.p[j], g.p[j], j, d);
                a.p[j] = a.p[j] + dz;
                b.p[j] = fma2(dz, d, b.p[j]);
            }
        });
    }
    if (at.mine > 0) {  // sum dz xhat = rstd sum dz (x - mean)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            b.set(j, b.at(j) * rstd[t.sample * n.groups + (t.c0 + lane_c + j) / n.per_group]);
        }
    }
    __syncthreads();  // the sums lie where the rows did
    for (int o = 16; o >= s.lanes; o >>= 1) {
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            a.p[j].x += __shfl_xor_sync(0xffffffffu, a.p[j].x, o);
            a.p[j].y += __shfl_xor_sync(0xffffffffu, a.p[j].y, o);
            b.p[j].x += __shfl_xor_sync(0xffffffffu, b.p[j].x, o);
            b.p[j].y += __shfl_xor_sync(0xffffffffu, b.p[j].y, o);
        }
    }
    if (lane < s.lanes && lane_c < s.width) {
        const int i = tid % s.lanes % 32;
        to_shared(&sums.a[warp][i * V], a);
        to_shared(&sums.b[warp][i * V], b);
    }
    __syncthreads();
    float2* out = partial + (t.sample * s.chunks + t.chunk) * n.channels + t.c0;
    const int width = min(s.width, n.channels - t.c0);
    for (int c = tid; c < width; c += kThreads) {
        float ca = 0.0f, cb = 0.0f;
        const int i = in_warp(s, V, c);
        for (int w = first_warp(s, V, c); w < kWarps; w += warp_step(s)) {
            ca += sums.a[w][i];
            cb += sums.b[w][i];
        }
        out[c] = make_float2(ca, cb);
    }
}

// Backward, second pass.
template <class T, int V, bool Packed, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_backward_apply_kernel(const T* __restrict__ dy, Input<T, V, Packed> in, const float* __restrict__ weight,
                               const float* __restrict__ bias, const float* __restrict__ mean,
                               const float* __restrict__ rstd, const float2* __restrict__ group_means,
                               T* __restrict__ dx, NormShape n, Chunking s)
{
    allow_next_grid();
    __shared__ Ring<T, V, Packed> ring;
    const int tid = threadIdx.x;
    const Task t = task_of(s, n, true);
    const int lane_c = (tid % s.lanes) * V;
    const int rows_per_pass = kThreads / s.lanes;
    const Place at = place_of(t, s, n, lane_c, tid / s.lanes);
    wait_for_previous_grid();
    if (at.mine == 0) {
        return;
    }
    Channels<V> all;
    all.load(mean, rstd, weight, bias, n, t.sample, t.c0 + lane_c, true);
    const Folded<V> ch(all);
    // dx = rstd (w dz - mean(t) - xhat mean(t xhat)) = scale dz - c0 - d c1
    Floats<V> c0, c1;
    c0.fill(0.0f);
    c1.fill(0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 gm = group_means[t.sample * n.groups + (t.c0 + lane_c + j) / n.per_group];
        const float r = all.rstd.at(j);
        c0.set(j, -r * gm.x);
        c1.set(j, -r * (r * gm.y));
    }
    T* dst = dx + at.base;
    const long long step = static_cast<long long>(rows_per_pass) * n.channels;
    for_gradient_rows<T, V, Packed>(ring, dy, in, at, t.c0 + lane_c, n, rows_per_pass, [&](const Floats<V>& g, const Floats<V>& x) {
        Floats<V> f;
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            float2 d;
            const float2 dz = ch.template slope<Act, T>(x.p[j], g.p[j], j, d);
            f.p[j] = fma2(ch.scale.p[j], dz, fma2(d, c1.p[j], c0.p[j]));
        }
        *reinterpret_cast<Vec<T, V>*>(dst) = narrow<T>(f);
        dst += step;
    });
}

// --- inputs with the channels first in memory --------------------------------------------------------------

// A spectral convolution leaves (batch, channels, points); the forward pass reads that as it lies, which
// saves a transposing copy's read and write.

// First pass: one warp per channel over a chunk of its points, into the same partial results (one per
// channel and chunk).
template <class T>
__global__ void __launch_bounds__(kThreads)
    norm_first_sum_kernel(const T* __restrict__ x, float2* __restrict__ partial, NormShape n, Chunking s)
{
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    allow_next_grid();
    __shared__ RowRing<T, V> ring;
    const int lane = threadIdx.x & 31;
    const int c = static_cast<int>(blockIdx.x % static_cast<unsigned>(s.tiles)) * kWarps + static_cast<int>(threadIdx.x >> 5);
    const long long i = blockIdx.x / static_cast<unsigned>(s.tiles);
    const int chunk = static_cast<int>(i % s.chunks);
    const long long sample = i / s.chunks;
    if (c >= n.channels) {
        return;
    }
    const int count = static_cast<int>(chunk_count(s, n.points, chunk)) / V;  // pieces
    const int mine = lane < count ? (count - lane + 31) / 32 : 0;
    wait_for_previous_grid();
    Floats<V> m, q;
    m.fill(0.0f);
    q.fill(0.0f);
    for_rows<T, V>(ring, x + (sample * n.channels + c) * n.points + chunk * s.rows + lane * V, 32 * V, mine,
                                     [&](const auto& raw, int k0) {
                                         constexpr int K = sizeof(raw) / sizeof(Vec<T, V>);
                                         Floats<V> f[K];
#pragma unroll
                                         for (int k = 0; k < K; ++k) {
                                             f[k] = widen(raw[k]);
                                         }
                                         join_block<V, K>(f, static_cast<float>(k0), m, q);
                                     });
    // The thread's V means and squares, of as many values each; then the warp's, about the first lane's.
    const float held = static_cast<float>(mine);
    float tm = 0.0f, tq = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        tm += m.at(j);
    }
    tm *= 1.0f / V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float d = m.at(j) - tm;
        tq += fmaf(held * d, d, q.at(j));
    }
    const float ref = __shfl_sync(0xffffffffu, tm, 0);
    float d = mine > 0 ? tm - ref : 0.0f;
    float sq = fmaf(held * V * d, d, tq);
    d *= held * V;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        d += __shfl_xor_sync(0xffffffffu, d, o);
        sq += __shfl_xor_sync(0xffffffffu, sq, o);
    }
    if (lane == 0) {
        const float off = __fdiv_rn(d, static_cast<float>(count) * V);
        partial[(sample * s.chunks + chunk) * n.channels + c] = make_float2(ref + off, fmaxf(fmaf(-d, off, sq), 0.0f));
    }
}

// Second pass, and the transposing copy alone (Copy). A thread reads V consecutive points of eight
// channels (16 bytes each, a warp's reads of a channel 512 contiguous bytes) and writes each
// point's eight channels (whole 32-byte sectors in float32); the CTA's warps take channels side by
// side.
template <class T, int Act, bool Copy>
__global__ void __launch_bounds__(kThreads)
    norm_first_apply_kernel(const T* __restrict__ x, const float* __restrict__ weight, const float* __restrict__ bias,
                            const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ y, NormShape n,
                            Chunking s)
{
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    constexpr int kChannels = 8;
    allow_next_grid();
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const unsigned b = gridDim.x - 1 - blockIdx.x;
    const int across = min(n.channels / kChannels, kWarps);  // warps side by side
    const int c0 = (static_cast<int>(b % static_cast<unsigned>(s.tiles)) * across + warp % across) * kChannels;
    const long long i = b / static_cast<unsigned>(s.tiles);
    const int chunk = static_cast<int>(i % s.chunks);
    const long long sample = i / s.chunks;
    const int along = kWarps / across;
    if (warp / across >= along || c0 >= n.channels) {
        return;
    }
    const int count = static_cast<int>(chunk_count(s, n.points, chunk));
    wait_for_previous_grid();
    float2 m[kChannels], w[kChannels], o[kChannels];
    if constexpr (!Copy) {
#pragma unroll
        for (int c = 0; c < kChannels; ++c) {
            const long long g = sample * n.groups + (c0 + c) / n.per_group;
            m[c] = pair(mean[g]);
            w[c] = pair(rstd[g] * (weight != nullptr ? weight[c0 + c] : 1.0f));
            o[c] = pair(bias != nullptr ? bias[c0 + c] : 0.0f);
        }
    }
    const T* src = x + (sample * n.channels + c0) * n.points + chunk * s.rows;
    T* dst = y + (sample * n.points + chunk * s.rows) * n.channels + c0;
    const bool whole = (reinterpret_cast<std::uintptr_t>(dst) & 31u) == 0;  // then every point's eight values are a sector
    // float32 loads the next points before it works on these: 16 warps an SM are too few to cover one with the other (gelu,
    // 64 x 128 x 128 x 64: 156 us, without 191). The 16-bit types would be left with eight warps (142 registers).
    const int step = along * 32 * V;
    constexpr bool kAheadOne = sizeof(T) == 4 && !Copy;
    Vec<T, V> in[kChannels];
    const auto load = [&](int r) {
#pragma unroll
        for (int c = 0; c < kChannels; ++c) {
            in[c] = *reinterpret_cast<const Vec<T, V>*>(src + c * n.points + r);
        }
    };
    int r = (warp / across * 32 + lane) * V;
    if (kAheadOne && r < count) {
        load(r);
    }
    for (; r < count; r += step) {
        Vec<T, V> now[kChannels];
        if constexpr (!kAheadOne) {
            load(r);
        }
#pragma unroll
        for (int c = 0; c < kChannels; ++c) {
            now[c] = in[c];
        }
        if (kAheadOne && r + step < count) {
            load(r + step);
        }
        Vec<T, kChannels> out[V];
#pragma unroll
        for (int c = 0; c < kChannels; ++c) {
            Vec<T, V> v = now[c];
            if constexpr (!Copy) {
                Floats<V> f = widen(v);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    f.p[j] = activate2<Act, T>(fma2(f.p[j] - m[c], w[c], o[c]));
                }
                v = narrow<T>(f);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                out[j].v[c] = v.v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            T* at = dst + static_cast<long long>(r + j) * n.channels;
            if (sizeof(T) == 4 && whole) {
                store32(at, *reinterpret_cast<const uint32_t(*)[8]>(&out[j]));
            } else if constexpr (sizeof(T) == 4) {
                reinterpret_cast<Vec<T, 4>*>(at)[0] = *reinterpret_cast<const Vec<T, 4>*>(&out[j].v[0]);
                reinterpret_cast<Vec<T, 4>*>(at)[1] = *reinterpret_cast<const Vec<T, 4>*>(&out[j].v[4]);
            } else {
                *reinterpret_cast<Vec<T, kChannels>*>(at) = out[j];
            }
        }
    }
}

// dbias[c] and dweight[c]: the samples' sums added up. 32 row lanes per channel, joined in a fixed order
// (4096 samples: eight took 150 us of a backward pass).
constexpr int kSumLanes = 32;
__global__ void __launch_bounds__(32 * kSumLanes)
    norm_parameter_kernel(const float* __restrict__ sample_sums, float* __restrict__ dweight, float* __restrict__ dbias,
                          long long batch, int channels)
{
    __shared__ float sb[kSumLanes][33], sw[kSumLanes][33];
    allow_next_grid();
    wait_for_previous_grid();
    const int c = static_cast<int>(blockIdx.x) * 32 + static_cast<int>(threadIdx.x & 31);
    const int part = static_cast<int>(threadIdx.x >> 5);
    float b = 0.0f, w = 0.0f;
    if (c < channels) {
#pragma unroll 4
        for (long long k = part; k < batch; k += kSumLanes) {
            b += sample_sums[k * channels + c];
            w += sample_sums[(batch + k) * channels + c];
        }
    }
    sb[part][threadIdx.x & 31] = b;
    sw[part][threadIdx.x & 31] = w;
    __syncthreads();
    if (part == 0 && c < channels) {
        for (int k = 1; k < kSumLanes; ++k) {
            b += sb[k][threadIdx.x & 31];
            w += sw[k][threadIdx.x & 31];
        }
        if (dbias != nullptr) {
            dbias[c] = b;
        }
        if (dweight != nullptr) {
            dweight[c] = w;
        }
    }
}

// --- host side -----------------------------------------------------------------------------------------

// The resident form's slicing, or false where the two-pass form serves better. `held` is the bytes of
// shared memory per channel of a row (x; x and dy in the backward pass), `arrays` the floats per
// channel and `group_arrays` per group next to the data.
//
// The rule, from both forms measured over 16 KB to 270 MB (forward, silu and gelu): arrays up to 8 MiB are
// resident if a unit fits a cluster (one launch instead of three: 12 against 17 us at 2 MB, 15 against
// 17 us at 8 MB, where 17 MB are 31 against 19 us), and larger ones only where the
// samples are small (4096 x 64 x 64 bf16: 65 against 121 us, backward 152 against 220 us; 2048 x 256 x 64, at
// the limit: 78 and 81 us, 163 and 162 us; 64 x 1000 x 512: 59 against 51 us, backward 113 against 86 us).
bool slice(const NormShape& n, int vec, int elem, int held, int arrays, int group_arrays, Slicing& s)
{
    s.width = 0;
    for (int k = 1; k <= n.groups; ++k) {
        // Whole groups, whole pieces, whole sectors, and not less than 16 KiB a unit.
        const long long width = static_cast<long long>(k) * n.per_group;
        if (n.groups % k == 0 && width % vec == 0
            && ((width * elem >= 32 && width * elem * n.points >= 16 * 1024) || k == n.groups || width / vec > kThreads / 2)) {
            s.width = width / vec <= kThreads ? static_cast<int>(width) : 0;
            break;
        }
    }
    if (s.width == 0) {
        return false;
    }
    s.slices = n.channels / s.width;
    s.lanes = s.width / vec;
    s.rows_per_pass = kThreads / s.lanes;
    const long long units = n.batch * s.slices;
    for (s.cluster = 1; s.cluster <= kMaxCluster; s.cluster *= 2) {
        s.rows = (n.points + s.cluster - 1) / s.cluster;
        s.passes = static_cast<int>(std::min<long long>((s.rows + s.rows_per_pass - 1) / s.rows_per_pass, 1 << 20));
        const long long bytes = static_cast<long long>(s.passes) * kThreads * vec * held;
        s.smem = static_cast<std::size_t>(bytes) + 4ull * kThreads * vec + 4ull * arrays * s.width
                 + 4ull * group_arrays * (s.width / n.per_group);
        // Small parts keep several CTAs on an SM; few units are spread further, down to four
        // passes, so that the GPU is full.
        const bool small = bytes <= kGoodBytes || (s.cluster >= 8 && s.smem <= kCtaBytes);
        const bool spread = units * s.cluster >= 2 * 148 || s.passes <= 4;
        if ((small && spread) || (s.cluster == kMaxCluster && s.smem <= kCtaBytes)) {
            const long long sample = n.points * n.channels * elem;
            const bool worth = (s.cluster == 1 && sample <= kSmallSample) || n.batch * sample <= kResidentBytes;
            return worth && units * s.cluster <= 0x7fffffffLL;
        }
    }
    return false;
}

// Chunks of about 128 KiB; smaller ones where there would be too few CTAs to fill the GPU.
Chunking chunking_of(const NormShape& n, int vec, int elem)
{
    Chunking s;
    // Lanes across a row: a power of two; a row of more than 32 pieces in tiles of 32 or 64 lanes,
    // whichever leaves fewer of them idle.
    const int pieces = n.channels / vec;
    s.lanes = 1;
    while (s.lanes < pieces && s.lanes < 32) {
        s.lanes *= 2;
    }
    if (pieces > 32 && (pieces + 63) / 64 * 2 <= (pieces + 31) / 32) {
        s.lanes = kTileLanes;
    }
    s.tiles = (pieces + s.lanes - 1) / s.lanes;
    s.width = s.tiles == 1 ? n.channels : s.lanes * vec;
    const long long rows_per_pass = kThreads / s.lanes;
    const long long fill = n.batch * n.points * s.tiles / (148LL * 6);
    const long long good = kChunkBytes / (static_cast<long long>(s.lanes) * vec * elem);
    s.rows = std::max(std::min<long long>(good, fill), 4 * rows_per_pass);
    s.rows = (s.rows + rows_per_pass * 8 - 1) / (rows_per_pass * 8) * (rows_per_pass * 8);
    s.rows = std::max(s.rows, (n.points + 1023) / 1024);  // keeps the join of a sample's chunks short
    // One CTA per chunk and tile in a grid of at most 2^31 - 1 of them.
    while (n.batch * ((n.points + s.rows - 1) / s.rows) * s.tiles > 0x7fffffffLL && s.rows < n.points) {
        s.rows *= 2;
    }
    s.rows = std::min(s.rows, 1LL << 30);
    s.chunks = static_cast<int>((n.points + s.rows - 1) / s.rows);
    s.merge = s.width % n.per_group == 0 ? n.per_group : 1;
    s.columns = n.channels / s.merge;
    return s;
}

// Workspace of the two-pass form, in 8-byte values: the chunks' results.
std::size_t chunk_work(const NormShape& n, const Chunking& s)
{
    return static_cast<std::size_t>(n.batch) * s.chunks * n.channels;
}

template <auto Kernel, class... Args>
void launch_cluster(long long units, const Slicing& s, cudaStream_t stream, Args&&... args)
{
    static std::atomic<bool> opted[kMaxDevices];
    const int device = current_device();
    if (!opted[device].load(std::memory_order_relaxed)) {
        SPECTRAL_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        SPECTRAL_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        opted[device].store(true, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {static_cast<unsigned>(s.cluster), 1, 1};
    cfg.gridDim = dim3(static_cast<unsigned>(units * s.cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = s.smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SPECTRAL_CUDA(cudaLaunchKernelEx(&cfg, Kernel, static_cast<Args&&>(args)...));
}

dim3 chunk_grid(const NormShape& n, const Chunking& s)
{
    return dim3(static_cast<unsigned>(n.batch * s.chunks * s.tiles));
}

// Calls f with the values per piece: 16 bytes where the rows are whole such pieces and every array is
// aligned to them, else pairs of values, else single ones.
template <class T, class F>
void with_pieces(int channels, std::initializer_list<const void*> arrays, const void* codes, F&& f)
{
    constexpr int kWide = 16 / static_cast<int>(sizeof(T));
    const auto fits = [&](int values) {
        bool ok = channels % values == 0 && aligned_to(codes, static_cast<std::size_t>(values));
        for (const void* p : arrays) {
            ok = ok && aligned_to(p, values * sizeof(T));
        }
        return ok;
    };
    if (fits(kWide)) {
        f(std::integral_constant<int, kWide>{});
    } else if (fits(2)) {
        f(std::integral_constant<int, 2>{});
    } else {
        f(std::integral_constant<int, 1>{});
    }
}

void norm_forward(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                  signed char* codes, float* scales, int dtype, const NormShape& n, void* work, cudaStream_t stream)
{
    bool packed = false;  // the checkpoint has been written on the way
    with_dtype(dtype, [&](auto type) {
        using T = decltype(type);
        with_pieces<T>(n.channels, {x, y}, nullptr, [&](auto pieces) {
            constexpr int V = decltype(pieces)::value;
            with_activation(n.act, [&](auto act) {
                constexpr int Act = decltype(act)::value;
                Slicing s;
                if (slice(n, V, sizeof(T), sizeof(T), 1, 4, s)) {
                    launch_cluster<norm_resident_kernel<T, V, Act>>(n.batch * s.slices, s, stream,
                                   static_cast<const T*>(x), weight, bias, static_cast<T*>(y), mean, rstd, n, s);
                    return;
                }
                const Chunking st = chunking_of(n, V, sizeof(T));
                auto* partial = static_cast<float2*>(work);
                float* m = mean;
                float* r = rstd;
                if (m == nullptr) {  // inference: the statistics live behind the partial results
                    m = reinterpret_cast<float*>(partial + chunk_work(n, st));
                    r = m + n.batch * n.groups;
                }
                const auto sum = [&](auto keep) {
                    constexpr bool kKeep = decltype(keep)::value;
                    launch_pdl(norm_sum_kernel<T, V, kKeep>, chunk_grid(n, st), dim3(kThreads), 0, stream,
                               static_cast<const T*>(x), kKeep ? codes : nullptr, kKeep ? scales : nullptr, partial, n, st);
                };
                // The checkpoint on the way where whole blocks sit side by side in a warp.
                if constexpr (V >= 4) {
                    packed = codes != nullptr && n.channels % kPackBlock == 0 && aligned_to(codes, V);
                    if (packed) {
                        sum(std::true_type{});
                    }
                }
                if (!packed) {
                    sum(std::false_type{});
                }
                launch_pdl(norm_join_kernel, dim3(static_cast<unsigned>(n.batch * n.groups)), dim3(kThreads), 0, stream,
                           static_cast<const float2*>(partial), m, r, n, st);
                launch_pdl(norm_apply_kernel<T, V, Act>, chunk_grid(n, st), dim3(kThreads), 0, stream,
                           static_cast<const T*>(x), weight, bias, static_cast<const float*>(m),
                           static_cast<const float*>(r), static_cast<T*>(y), n, st);
            });
        });
    });
    if (codes != nullptr && !packed) {
        pack8(x, dtype, codes, scales, n.batch * n.points, n.channels, stream);
    }
}

// Whether the kernels for inputs with the channels first take these arrays.
bool first_fits(const void* x, const void* y, int dtype, long long points, int channels)
{
    const int values = 16 / static_cast<int>(dtype_size(dtype));
    return channels % 8 == 0 && points % values == 0 && aligned_to(x, 16) && aligned_to(y, 16);
}

// Chunks of 4096 points, fewer where there would be too few CTAs; tiles of 8 channels for the sums, of up to
// 64 for the outputs.
Chunking first_chunking(const NormShape& n, int tiles)
{
    Chunking s;
    s.tiles = tiles;
    const long long fill = n.batch * n.points * tiles / (148LL * 6);
    s.rows = std::max<long long>(512, std::min<long long>(4096, fill / 256 * 256));
    s.rows = std::max(s.rows, (n.points + 1023) / 1024 * 8);
    while (n.batch * ((n.points + s.rows - 1) / s.rows) * s.tiles > 0x7fffffffLL && s.rows < n.points) {
        s.rows *= 2;
    }
    s.chunks = static_cast<int>((n.points + s.rows - 1) / s.rows);
    s.merge = 1;
    s.columns = n.channels;
    return s;
}

int first_sum_tiles(const NormShape& n) { return (n.channels + kWarps - 1) / kWarps; }
int first_apply_tiles(const NormShape& n)
{
    const int eights = n.channels / 8;
    return (eights + kWarps - 1) / kWarps;
}

void channels_last(const void* x, void* y, int dtype, const NormShape& n, cudaStream_t stream)
{
    with_dtype(dtype, [&](auto type) {
        using T = decltype(type);
        const Chunking s = first_chunking(n, first_apply_tiles(n));
        launch_pdl(norm_first_apply_kernel<T, SPECTRAL_ACT_NONE, true>, chunk_grid(n, s), dim3(kThreads), 0, stream,
                   static_cast<const T*>(x), static_cast<const float*>(nullptr), static_cast<const float*>(nullptr),
                   static_cast<const float*>(nullptr), static_cast<const float*>(nullptr), static_cast<T*>(y), n, s);
    });
}

void norm_first_forward(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd, int dtype,
                        const NormShape& n, void* work, cudaStream_t stream)
{
    with_dtype(dtype, [&](auto type) {
        using T = decltype(type);
        with_activation(n.act, [&](auto act) {
            constexpr int Act = decltype(act)::value;
            const Chunking sum = first_chunking(n, first_sum_tiles(n));
            const Chunking apply = first_chunking(n, first_apply_tiles(n));
            auto* partial = static_cast<float2*>(work);
            float* m = mean;
            float* r = rstd;
            if (m == nullptr) {
                m = reinterpret_cast<float*>(partial + chunk_work(n, sum));
                r = m + n.batch * n.groups;
            }
            launch_pdl(norm_first_sum_kernel<T>, chunk_grid(n, sum), dim3(kThreads), 0, stream, static_cast<const T*>(x),
                       partial, n, sum);
            launch_pdl(norm_join_kernel, dim3(static_cast<unsigned>(n.batch * n.groups)), dim3(kThreads), 0, stream,
                       static_cast<const float2*>(partial), m, r, n, sum);
            launch_pdl(norm_first_apply_kernel<T, Act, false>, chunk_grid(n, apply), dim3(kThreads), 0, stream,
                       static_cast<const T*>(x), weight, bias, static_cast<const float*>(m), static_cast<const float*>(r),
                       static_cast<T*>(y), n, apply);
        });
    });
}

template <class T, int V, bool Packed, int Act>
void norm_backward_typed(const T* dy, const Input<T, V, Packed>& in, const float* weight, const float* bias,
                         const float* mean, const float* rstd, T* dx, float* dweight, float* dbias, const NormShape& n,
                         float* work, cudaStream_t stream)
{
    float* sample_sums = work;
    Slicing s;
    constexpr int kHeld = sizeof(T) + (Packed ? 1 + (4 + V - 1) / V : sizeof(T));
    if (slice(n, V, sizeof(T), kHeld, 5, 2, s)) {
        launch_cluster<norm_backward_resident_kernel<T, V, Packed, Act>>(n.batch * s.slices, s, stream, dy, in, weight,
                       bias, mean, rstd, dx, sample_sums, n, s);
    } else {
        const Chunking st = chunking_of(n, V, sizeof(T));
        auto* group_means = reinterpret_cast<float2*>(sample_sums + 2 * n.batch * n.channels);
        float2* partial = group_means + n.batch * n.groups;
        launch_pdl(norm_backward_sum_kernel<T, V, Packed, Act>, chunk_grid(n, st), dim3(kThreads), 0, stream, dy, in, weight,
                   bias, mean, rstd, partial, n, st);
        launch_pdl(norm_backward_join_kernel, dim3(static_cast<unsigned>(n.batch * n.groups)), dim3(kThreads), 0, stream,
                   static_cast<const float2*>(partial), weight, sample_sums, group_means, n, st);
        launch_pdl(norm_backward_apply_kernel<T, V, Packed, Act>, chunk_grid(n, st), dim3(kThreads), 0, stream, dy, in,
                   weight, bias, mean, rstd, static_cast<const float2*>(group_means), dx, n, st);
    }
    if (dweight != nullptr || dbias != nullptr) {
        launch_pdl(norm_parameter_kernel, dim3(static_cast<unsigned>((n.channels + 31) / 32)), dim3(32 * kSumLanes), 0, stream,
                   static_cast<const float*>(sample_sums), dweight, dbias, n.batch, n.channels);
    }
}

void norm_backward(const void* dy, const void* x, const signed char* codes, const float* scales, const float* weight,
                   const float* bias, const float* mean, const float* rstd, void* dx, float* dweight, float* dbias,
                   int dtype, const NormShape& n, float* work, cudaStream_t stream)
{
    with_dtype(dtype, [&](auto type) {
        using T = decltype(type);
        with_pieces<T>(n.channels, {dy, dx, x}, codes, [&](auto pieces) {
            constexpr int V = decltype(pieces)::value;
            with_activation(n.act, [&](auto act) {
                constexpr int Act = decltype(act)::value;
                if (codes != nullptr) {
                    const Input<T, V, true> in{nullptr, codes, scales};
                    norm_backward_typed<T, V, true, Act>(static_cast<const T*>(dy), in, weight, bias, mean, rstd,
                                                         static_cast<T*>(dx), dweight, dbias, n, work, stream);
                } else {
                    const Input<T, V, false> in{static_cast<const T*>(x), nullptr, nullptr};
                    norm_backward_typed<T, V, false, Act>(static_cast<const T*>(dy), in, weight, bias, mean, rstd,
                                                          static_cast<T*>(dx), dweight, dbias, n, work, stream);
                }
            });
        });
    });
}

int invalid(const std::string& message)
{
    set_last_error(message);
    return SPECTRAL_INVALID_ARGUMENT;
}

int check(const char* op, int dtype, long long batch, long long points, int channels, int groups, int act)
{
    const std::string name(op);
    if (!dtype_known(dtype)) {
        return invalid(name + ": dtype must be SPECTRAL_FLOAT32, SPECTRAL_BFLOAT16 or SPECTRAL_FLOAT16");
    }
    if (!activation_known(act)) {
        return invalid(name + ": activation must be SPECTRAL_ACT_NONE, _SILU or _GELU");
    }
    if (batch < 0 || points < 0 || channels < 1 || groups < 1 || channels % groups != 0) {
        return invalid(name + ": need batch >= 0, points >= 0 and groups dividing channels, got " + std::to_string(channels)
                       + " channels in " + std::to_string(groups) + " groups");
    }
    if (batch > (1LL << 30) || batch * groups > 0x7fffffffLL || channels > (1 << 20)
        || (batch > 0 && points > (1LL << 46) / channels / batch)) {
        return invalid(name + ": at most 2^30 samples, 2^31 - 1 groups over all samples, 2^20 channels and 2^46 values");
    }
    return SPECTRAL_OK;
}

bool overlap(const void* a, unsigned long long a_bytes, const void* b, unsigned long long b_bytes)
{
    const auto p = reinterpret_cast<unsigned long long>(a);
    const auto q = reinterpret_cast<unsigned long long>(b);
    return p < q + b_bytes && q < p + a_bytes;
}

bool overlap(const void* a, const void* b, unsigned long long bytes) { return overlap(a, bytes, b, bytes); }

// The float arrays beside the values: parameters, statistics, scales (null ones are not given).
bool floats_aligned(std::initializer_list<const void*> arrays)
{
    for (const void* p : arrays) {
        if (!aligned_to(p, sizeof(float))) {
            return false;
        }
    }
    return true;
}

}  // namespace
}  // namespace spectral

namespace spectral {
namespace {

// The two-pass form's most chunks, over the piece sizes, decide the workspace.
std::size_t most_chunk_words(const NormShape& n, int dtype)
{
    const int elem = static_cast<int>(dtype_size(dtype));
    std::size_t most = 0;
    for (const int vec : {1, 2, 16 / elem}) {
        if (n.channels % vec == 0) {
            most = std::max(most, chunk_work(n, chunking_of(n, vec, elem)));
        }
    }
    return std::max(most, chunk_work(n, first_chunking(n, first_sum_tiles(n))));
}

}  // namespace
}  // namespace spectral

extern "C" int spectral_group_norm_act_workspace(int dtype, long long batch, long long points, int channels, int groups,
                                                 size_t* count)
{
    using namespace spectral;
    const int status = check("group_norm_act_workspace", dtype, batch, points, channels, groups, SPECTRAL_ACT_NONE);
    if (status != SPECTRAL_OK || count == nullptr) {
        return status != SPECTRAL_OK ? status : invalid("group_norm_act_workspace: null count");
    }
    // The two-pass form's, and statistics the caller does not keep.
    const NormShape n{batch, points, channels, groups, channels / groups, 0, 0.0f};
    *count = batch == 0 || points == 0 ? 0 : most_chunk_words(n, dtype) + static_cast<size_t>(batch) * groups;
    return SPECTRAL_OK;
}

extern "C" int spectral_group_norm_act_backward_workspace(int dtype, long long batch, long long points, int channels,
                                                          int groups, size_t* count)
{
    using namespace spectral;
    const int status = check("group_norm_act_backward_workspace", dtype, batch, points, channels, groups, SPECTRAL_ACT_NONE);
    if (status != SPECTRAL_OK || count == nullptr) {
        return status != SPECTRAL_OK ? status : invalid("group_norm_act_backward_workspace: null count");
    }
    // The samples' parameter sums, the groups' means, and the two-pass form's.
    const NormShape n{batch, points, channels, groups, channels / groups, 0, 0.0f};
    *count = batch == 0 || points == 0
                 ? 0
                 : most_chunk_words(n, dtype) + static_cast<size_t>(batch) * (static_cast<size_t>(channels) + groups);
    return SPECTRAL_OK;
}

extern "C" int spectral_group_norm_act(const void* x, const float* weight, const float* bias, void* y, float* mean,
                                       float* rstd, void* codes, float* scales, int dtype, int channels_first,
                                       long long batch, long long points, int channels, int groups, float eps,
                                       int activation, void* work, void* stream)
{
    using namespace spectral;
    const int status = check("group_norm_act", dtype, batch, points, channels, groups, activation);
    if (status != SPECTRAL_OK || batch == 0 || points == 0) {
        return status;
    }
    if (!(eps >= 0.0f)) {
        return invalid("group_norm_act: eps must be at least 0");
    }
    if (x == nullptr || y == nullptr || work == nullptr || (mean == nullptr) != (rstd == nullptr)
        || (codes == nullptr) != (scales == nullptr)) {
        return invalid("group_norm_act: x, y and work must be given, mean with rstd, and codes with scales");
    }
    if (!aligned_to(x, dtype_size(dtype)) || !aligned_to(y, dtype_size(dtype)) || !aligned_to(work, 8)
        || !floats_aligned({weight, bias, mean, rstd, scales})) {
        return invalid("group_norm_act: arrays must be aligned to their element size, work to 8 bytes");
    }
    if (overlap(x, y, static_cast<unsigned long long>(batch * points) * channels * dtype_size(dtype))) {
        return invalid("group_norm_act: x and y must not overlap");
    }
    if (channels_first != 0 && (codes != nullptr || !first_fits(x, y, dtype, points, channels))) {
        return invalid("group_norm_act: x with the channels first needs channels a multiple of 8, points of 16 bytes, 16-byte "
                       "aligned arrays and no checkpoint; see spectral_channels_last");
    }
    try {
        const NormShape n{batch, points, channels, groups, channels / groups, activation, eps};
        if (channels_first != 0) {
            norm_first_forward(x, weight, bias, y, mean, rstd, dtype, n, work, static_cast<cudaStream_t>(stream));
            return SPECTRAL_OK;
        }
        norm_forward(x, weight, bias, y, mean, rstd, static_cast<signed char*>(codes), scales, dtype, n, work,
                     static_cast<cudaStream_t>(stream));
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}

extern "C" int spectral_group_norm_act_backward(const void* dy, const void* x, const void* codes, const float* scales,
                                                const float* weight, const float* bias, const float* mean,
                                                const float* rstd, void* dx, float* dweight, float* dbias, int dtype,
                                                long long batch, long long points, int channels, int groups,
                                                int activation, void* work, void* stream)
{
    using namespace spectral;
    const int status = check("group_norm_act_backward", dtype, batch, points, channels, groups, activation);
    if (status != SPECTRAL_OK) {
        return status;
    }
    const auto s = static_cast<cudaStream_t>(stream);
    try {
        if (batch == 0 || points == 0) {  // sums over nothing
            if (!floats_aligned({dweight, dbias})) {
                return invalid("group_norm_act_backward: arrays must be aligned to their element size");
            }
            if (dweight != nullptr) {
                SPECTRAL_CUDA(cudaMemsetAsync(dweight, 0, sizeof(float) * channels, s));
            }
            if (dbias != nullptr) {
                SPECTRAL_CUDA(cudaMemsetAsync(dbias, 0, sizeof(float) * channels, s));
            }
            return SPECTRAL_OK;
        }
        if (dy == nullptr || dx == nullptr || work == nullptr || mean == nullptr || rstd == nullptr
            || (codes == nullptr) == (x == nullptr) || (codes == nullptr) != (scales == nullptr)) {
            return invalid("group_norm_act_backward: dy, dx, mean, rstd and work must be given, and either x or codes with scales");
        }
        const std::size_t size = dtype_size(dtype);
        if (!aligned_to(dy, size) || !aligned_to(dx, size) || !aligned_to(x, size) || !aligned_to(work, 8)
            || !floats_aligned({scales, weight, bias, mean, rstd, dweight, dbias})) {
            return invalid("group_norm_act_backward: arrays must be aligned to their element size, work to 8 bytes");
        }
        const unsigned long long bytes = static_cast<unsigned long long>(batch * points) * channels * size;
        if (overlap(dx, dy, bytes) || (x != nullptr && overlap(dx, x, bytes))) {
            return invalid("group_norm_act_backward: dx must not overlap dy or x");
        }
        const unsigned long long rows = static_cast<unsigned long long>(batch * points);
        if (codes != nullptr
            && (overlap(dx, bytes, codes, rows * channels)
                || overlap(dx, bytes, scales, rows * ((channels + kPackBlock - 1) / kPackBlock) * sizeof(float)))) {
            return invalid("group_norm_act_backward: dx must not overlap the checkpoint");
        }
        const NormShape n{batch, points, channels, groups, channels / groups, activation, 0.0f};
        norm_backward(dy, x, static_cast<const signed char*>(codes), scales, weight, bias, mean, rstd, dx, dweight, dbias,
                      dtype, n, static_cast<float*>(work), s);
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}

extern "C" int spectral_channels_last(const void* x, void* y, int dtype, long long batch, long long points, int channels,
                                      void* stream)
{
    using namespace spectral;
    const int status = check("channels_last", dtype, batch, points, channels, 1, SPECTRAL_ACT_NONE);
    if (status != SPECTRAL_OK || batch == 0 || points == 0) {
        return status;
    }
    if (x == nullptr || y == nullptr || !first_fits(x, y, dtype, points, channels)) {
        return invalid("channels_last: needs channels a multiple of 8, points of 16 bytes and 16-byte aligned arrays");
    }
    if (overlap(x, y, static_cast<unsigned long long>(batch * points) * channels * dtype_size(dtype))) {
        return invalid("channels_last: x and y must not overlap");
    }
    try {
        const NormShape n{batch, points, channels, 1, channels, SPECTRAL_ACT_NONE, 0.0f};
        channels_last(x, y, dtype, n, static_cast<cudaStream_t>(stream));
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}
