// Group norm with an activation over channels-last fields, forward and backward:
//     y = act(xhat w_c + b_c),  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),
// mean and var over the n = points x (channels / groups) values of one sample's group.
// Backward, with z = xhat w + b, dz = dy act'(z) and t = w dz:
//     dbias = sum dz, dweight = sum dz xhat  (over samples and points),
//     dx = rstd (t - mean(t) - xhat mean(t xhat))  (means over the group).
//
// HBM-bound: forward reads x and writes y, backward reads x (or its 8-bit checkpoint) and dy and
// writes dx; everything else is per channel. Both need all of a group before the first output,
// so the group has to stay on chip between the sums and the outputs.
//
// Resident form: a unit is one sample's slice of whole groups (at least 32 bytes wide). A cluster
// of 1 to 16 CTAs holds it in shared memory: each thread copies 16-byte pieces of its rows with
// cp.async and later reads only its own pieces, so the copies need no barrier. The CTAs reduce
// their part (mean first, then the centred squares, both from shared memory), exchange the
// partial results through distributed shared memory in rank order (the same bits every time), and
// write the outputs: one read and one write of HBM per value.
//
// Two-pass form: a unit too large for a cluster. Chunks of a sample's rows give per-channel
// partial sums (shifted by the chunk's first value, so that a large mean does not cancel), a small
// kernel joins them, and an elementwise kernel re-reads the inputs.
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
constexpr int kGoodBytes = 64 * 1024;    // three such CTAs share an SM, so loads, sums and stores overlap

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
__device__ __forceinline__ void channel_sums(const float (&part)[V], float* scratch, float* sums, int lanes, int width)
{
    const int tid = threadIdx.x;
    float p[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        p[j] = part[j];
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
    float w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w[j] = weight != nullptr && active ? weight[c0 + lane_c + j] : 1.0f;
        b[j] = bias != nullptr && active ? bias[c0 + lane_c + j] : 0.0f;
    }
    cp_async_wait_all();

    float part[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        part[j] = 0.0f;
    }
    for (int i = 0; i < held; ++i) {
        const Piece p = data[i * kThreads + tid];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            part[j] += to_float(p.v[j]);
        }
    }
    const float here = static_cast<float>(count) * static_cast<float>(n.per_group);
    channel_sums<V>(part, scratch, sums, s.lanes, s.width);
    group_sums(sums, nullptr, fmaxf(here, 1.0f), mean, groups, n.per_group);
    float m[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        m[j] = active ? mean[(lane_c + j) / n.per_group] : 0.0f;
        part[j] = 0.0f;
    }
    for (int i = 0; i < held; ++i) {
        const Piece p = data[i * kThreads + tid];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = to_float(p.v[j]) - m[j];
            part[j] = fmaf(d, d, part[j]);
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
        m[j] = mean[g];
        w[j] *= rstd[g];
    }
    for (int i = 0; i < held; ++i) {
        const Piece p = data[i * kThreads + tid];
        Piece out;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            out.v[j] = from_float<T>(activate<Act>(fmaf(to_float(p.v[j]) - m[j], w[j], b[j])));
        }
        const long long r = row0 + static_cast<long long>(i) * s.rows_per_pass;
        *reinterpret_cast<Piece*>(y + base + r * n.channels) = out;
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
}

// The x operand of the backward kernels: values of T, or the codes and scales of a checkpoint.
template <class T, int V, bool Packed>
struct Input {
    using Raw = std::conditional_t<Packed, Vec<signed char, V>, Vec<T, V>>;
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
    __device__ static __forceinline__ float value(const Raw& raw, int j, float scale)
    {
        if constexpr (Packed) {
            return to_float(restored<T>(raw.v[j], scale));
        } else {
            return to_float(raw.v[j]);
        }
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
    float m[V], r[V], w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = c0 + lane_c + j;
        const long long g = sample * n.groups + (active ? c / n.per_group : 0);
        m[j] = mean[g];
        r[j] = rstd[g];
        w[j] = weight != nullptr && active ? weight[c] : 1.0f;
        b[j] = bias != nullptr && active ? bias[c] : 0.0f;
    }
    for (int c = tid; c < s.width; c += kThreads) {
        w_smem[c] = weight != nullptr ? weight[c0 + c] : 1.0f;
    }
    cp_async_wait_all();

    float part_dz[V], part_dzx[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        part_dz[j] = 0.0f;
        part_dzx[j] = 0.0f;
    }
    for (int i = 0; i < held; ++i) {
        const Piece p = data_dy[i * kThreads + tid];
        const Raw q = data_x[i * kThreads + tid];
        const float scale = Packed ? data_scale[i * kThreads + tid] : 1.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float xhat = (Input<T, V, Packed>::value(q, j, scale) - m[j]) * r[j];
            float slope;
            activate_slope<Act>(fmaf(xhat, w[j], b[j]), slope);
            const float dz = to_float(p.v[j]) * slope;
            part_dz[j] += dz;
            part_dzx[j] = fmaf(dz, xhat, part_dzx[j]);
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
    float mt[V], mtx[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = active ? (lane_c + j) / n.per_group : 0;
        mt[j] = mean_t[g];
        mtx[j] = mean_tx[g];
    }
    for (int i = 0; i < held; ++i) {
        const Piece p = data_dy[i * kThreads + tid];
        const Raw q = data_x[i * kThreads + tid];
        const float scale = Packed ? data_scale[i * kThreads + tid] : 1.0f;
        Piece out;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float xhat = (Input<T, V, Packed>::value(q, j, scale) - m[j]) * r[j];
            float slope;
            activate_slope<Act>(fmaf(xhat, w[j], b[j]), slope);
            const float t = to_float(p.v[j]) * slope * w[j];
            out.v[j] = from_float<T>(r[j] * (t - mt[j] - xhat * mtx[j]));
        }
        const long long row = row0 + static_cast<long long>(i) * s.rows_per_pass;
        *reinterpret_cast<Piece*>(dx + base + row * n.channels) = out;
    }
    cluster.sync();
}

// --- two-pass form -------------------------------------------------------------------------------------

// Rows of a channel tile: lanes threads across, kThreads / lanes rows per pass, chunks of rows.
struct Tiling {
    int width;    // channels per CTA
    int lanes;
    int tiles;
    int chunks;
    long long rows;  // per chunk
};

__host__ __device__ __forceinline__ long long chunk_count(const Tiling& t, long long points, int chunk)
{
    const long long left = points - chunk * t.rows;
    return left < 0 ? 0 : left < t.rows ? left : t.rows;
}

// Per (sample, chunk, channel): mean and centred squares of the chunk's values -> partial
// [sample][chunk][channel] float2.
template <class T, int V>
__global__ void __launch_bounds__(kThreads)
    norm_partial_kernel(const T* __restrict__ x, float2* __restrict__ partial, NormShape n, Tiling t)
{
    using Piece = Vec<T, V>;
    allow_next_grid();
    extern __shared__ __align__(16) float fsmem[];
    float* scratch = fsmem;
    float* s1 = scratch + kThreads * V;
    float* s2 = s1 + t.width;
    float* first = s2 + t.width;
    const int tid = threadIdx.x;
    const long long sample = blockIdx.y;
    const int chunk = blockIdx.x;
    const int c0 = static_cast<int>(blockIdx.z) * t.width;
    const int rows_per_pass = kThreads / t.lanes;
    const int lane_c = (tid % t.lanes) * V;
    const int row0 = tid / t.lanes;
    const bool active = row0 < rows_per_pass && c0 + lane_c < n.channels;
    const long long count = chunk_count(t, n.points, chunk);
    const T* src = x + (sample * n.points + chunk * t.rows) * n.channels + c0 + lane_c;
    wait_for_previous_grid();
    float shift[V], p1[V], p2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        shift[j] = active && count > 0 ? to_float(src[j]) : 0.0f;
        p1[j] = 0.0f;
        p2[j] = 0.0f;
    }
    if (active) {
#pragma unroll 4
        for (long long r = row0; r < count; r += rows_per_pass) {
            const Piece p = *reinterpret_cast<const Piece*>(src + r * n.channels);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = to_float(p.v[j]) - shift[j];
                p1[j] += d;
                p2[j] = fmaf(d, d, p2[j]);
            }
        }
        if (row0 == 0) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                first[lane_c + j] = shift[j];
            }
        }
    }
    channel_sums<V>(p1, scratch, s1, t.lanes, t.width);
    channel_sums<V>(p2, scratch, s2, t.lanes, t.width);
    const float inv = count > 0 ? 1.0f / static_cast<float>(count) : 0.0f;
    for (int c = tid; c < t.width && c0 + c < n.channels; c += kThreads) {
        const float d = s1[c] * inv;
        partial[(sample * t.chunks + chunk) * n.channels + c0 + c] =
            make_float2(first[c] + d, fmaxf(fmaf(-s1[c], d, s2[c]), 0.0f));
    }
}

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

// One CTA per (sample, group): joins the chunks' and channels' partial results.
__global__ void __launch_bounds__(kThreads)
    norm_join_kernel(const float2* __restrict__ partial, float* __restrict__ mean, float* __restrict__ rstd, NormShape n,
                     Tiling t)
{
    __shared__ float scratch[kWarps];
    allow_next_grid();
    wait_for_previous_grid();
    const long long sample = blockIdx.x / n.groups;
    const int c0 = static_cast<int>(blockIdx.x % n.groups) * n.per_group;
    const float2* src = partial + sample * t.chunks * n.channels + c0;
    const float total = static_cast<float>(n.points) * static_cast<float>(n.per_group);
    const long long items = static_cast<long long>(t.chunks) * n.per_group;
    const float first = src[0].x;  // the joint mean is a correction to it
    float s = 0.0f;
    for (long long i = threadIdx.x; i < items; i += kThreads) {
        const int chunk = static_cast<int>(i / n.per_group);
        const float2 p = src[static_cast<long long>(chunk) * n.channels + i % n.per_group];
        s = fmaf(p.x - first, static_cast<float>(chunk_count(t, n.points, chunk)) / total, s);
    }
    const float joint = first + block_sum(s, scratch);
    float q = 0.0f;
    for (long long i = threadIdx.x; i < items; i += kThreads) {
        const int chunk = static_cast<int>(i / n.per_group);
        const float2 p = src[static_cast<long long>(chunk) * n.channels + i % n.per_group];
        const float d = p.x - joint;
        const float count = static_cast<float>(chunk_count(t, n.points, chunk));
        q += count > 0.0f ? fmaf(count * d, d, p.y) : 0.0f;
    }
    q = block_sum(q, scratch);
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = joint;
        rstd[blockIdx.x] = rsqrtf(q / total + n.eps);
    }
}

template <class T, int V, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_apply_kernel(const T* __restrict__ x, const float* __restrict__ weight, const float* __restrict__ bias,
                      const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ y, NormShape n,
                      Tiling t)
{
    using Piece = Vec<T, V>;
    allow_next_grid();
    const int tid = threadIdx.x;
    // Last chunk first: what the statistics read last is still in L2.
    const long long sample = gridDim.y - 1 - blockIdx.y;
    const int chunk = static_cast<int>(gridDim.x - 1 - blockIdx.x);
    const int c0 = static_cast<int>(blockIdx.z) * t.width;
    const int rows_per_pass = kThreads / t.lanes;
    const int lane_c = (tid % t.lanes) * V;
    const int row0 = tid / t.lanes;
    wait_for_previous_grid();
    if (row0 >= rows_per_pass || c0 + lane_c >= n.channels) {
        return;
    }
    const long long count = chunk_count(t, n.points, chunk);
    const long long base = (sample * n.points + chunk * t.rows) * n.channels + c0 + lane_c;
    float m[V], w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = c0 + lane_c + j;
        const long long g = sample * n.groups + c / n.per_group;
        m[j] = mean[g];
        w[j] = (weight != nullptr ? weight[c] : 1.0f) * rstd[g];
        b[j] = bias != nullptr ? bias[c] : 0.0f;
    }
#pragma unroll 2
    for (long long r = row0; r < count; r += rows_per_pass) {
        const Piece p = *reinterpret_cast<const Piece*>(x + base + r * n.channels);
        Piece out;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            out.v[j] = from_float<T>(activate<Act>(fmaf(to_float(p.v[j]) - m[j], w[j], b[j])));
        }
        *reinterpret_cast<Piece*>(y + base + r * n.channels) = out;
    }
}

// Per (sample, chunk, channel): sum dz and sum dz xhat -> partial [sample][chunk][channel].
template <class T, int V, bool Packed, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_backward_partial_kernel(const T* __restrict__ dy, Input<T, V, Packed> in, const float* __restrict__ weight,
                                 const float* __restrict__ bias, const float* __restrict__ mean,
                                 const float* __restrict__ rstd, float2* __restrict__ partial, NormShape n, Tiling t)
{
    using Piece = Vec<T, V>;
    using Raw = typename Input<T, V, Packed>::Raw;
    allow_next_grid();
    extern __shared__ __align__(16) float fsmem[];
    float* scratch = fsmem;
    float* s1 = scratch + kThreads * V;
    float* s2 = s1 + t.width;
    const int tid = threadIdx.x;
    const long long sample = blockIdx.y;
    const int chunk = blockIdx.x;
    const int c0 = static_cast<int>(blockIdx.z) * t.width;
    const int rows_per_pass = kThreads / t.lanes;
    const int lane_c = (tid % t.lanes) * V;
    const int row0 = tid / t.lanes;
    const bool active = row0 < rows_per_pass && c0 + lane_c < n.channels;
    const long long count = chunk_count(t, n.points, chunk);
    const long long first_row = sample * n.points + chunk * t.rows;
    const long long base = first_row * n.channels + c0 + lane_c;
    wait_for_previous_grid();
    float p1[V], p2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        p1[j] = 0.0f;
        p2[j] = 0.0f;
    }
    if (active) {
        float m[V], r[V], w[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = c0 + lane_c + j;
            const long long g = sample * n.groups + c / n.per_group;
            m[j] = mean[g];
            r[j] = rstd[g];
            w[j] = weight != nullptr ? weight[c] : 1.0f;
            b[j] = bias != nullptr ? bias[c] : 0.0f;
        }
#pragma unroll 2
        for (long long row = row0; row < count; row += rows_per_pass) {
            const Piece p = *reinterpret_cast<const Piece*>(dy + base + row * n.channels);
            const Raw q = *static_cast<const Raw*>(in.at(base + row * n.channels));
            const float scale = Packed ? *in.scale_at(first_row + row, c0 + lane_c, n.channels) : 1.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xhat = (Input<T, V, Packed>::value(q, j, scale) - m[j]) * r[j];
                float slope;
                activate_slope<Act>(fmaf(xhat, w[j], b[j]), slope);
                const float dz = to_float(p.v[j]) * slope;
                p1[j] += dz;
                p2[j] = fmaf(dz, xhat, p2[j]);
            }
        }
    }
    channel_sums<V>(p1, scratch, s1, t.lanes, t.width);
    channel_sums<V>(p2, scratch, s2, t.lanes, t.width);
    for (int c = tid; c < t.width && c0 + c < n.channels; c += kThreads) {
        partial[(sample * t.chunks + chunk) * n.channels + c0 + c] = make_float2(s1[c], s2[c]);
    }
}

// One CTA per (sample, group): the sample's channel sums and the group's mean(t), mean(t xhat).
__global__ void __launch_bounds__(kThreads)
    norm_backward_join_kernel(const float2* __restrict__ partial, const float* __restrict__ weight,
                              float* __restrict__ sample_sums, float2* __restrict__ group_means, NormShape n, Tiling t)
{
    __shared__ float scratch[kWarps];
    allow_next_grid();
    wait_for_previous_grid();
    const long long sample = blockIdx.x / n.groups;
    const int c0 = static_cast<int>(blockIdx.x % n.groups) * n.per_group;
    float mt = 0.0f, mtx = 0.0f;
    for (int c = threadIdx.x; c < n.per_group; c += kThreads) {
        float a = 0.0f, ax = 0.0f;
        for (int k = 0; k < t.chunks; ++k) {
            const float2 p = partial[(sample * t.chunks + k) * n.channels + c0 + c];
            a += p.x;
            ax += p.y;
        }
        sample_sums[sample * n.channels + c0 + c] = a;
        sample_sums[(n.batch + sample) * n.channels + c0 + c] = ax;
        const float w = weight != nullptr ? weight[c0 + c] : 1.0f;
        mt = fmaf(w, a, mt);
        mtx = fmaf(w, ax, mtx);
    }
    mt = block_sum(mt, scratch);
    mtx = block_sum(mtx, scratch);
    if (threadIdx.x == 0) {
        const float share = 1.0f / (static_cast<float>(n.points) * static_cast<float>(n.per_group));
        group_means[blockIdx.x] = make_float2(mt * share, mtx * share);
    }
}

template <class T, int V, bool Packed, int Act>
__global__ void __launch_bounds__(kThreads)
    norm_backward_apply_kernel(const T* __restrict__ dy, Input<T, V, Packed> in, const float* __restrict__ weight,
                               const float* __restrict__ bias, const float* __restrict__ mean,
                               const float* __restrict__ rstd, const float2* __restrict__ group_means,
                               T* __restrict__ dx, NormShape n, Tiling t)
{
    using Piece = Vec<T, V>;
    using Raw = typename Input<T, V, Packed>::Raw;
    allow_next_grid();
    const int tid = threadIdx.x;
    const long long sample = gridDim.y - 1 - blockIdx.y;
    const int chunk = static_cast<int>(gridDim.x - 1 - blockIdx.x);
    const int c0 = static_cast<int>(blockIdx.z) * t.width;
    const int rows_per_pass = kThreads / t.lanes;
    const int lane_c = (tid % t.lanes) * V;
    const int row0 = tid / t.lanes;
    wait_for_previous_grid();
    if (row0 >= rows_per_pass || c0 + lane_c >= n.channels) {
        return;
    }
    const long long count = chunk_count(t, n.points, chunk);
    const long long first_row = sample * n.points + chunk * t.rows;
    const long long base = first_row * n.channels + c0 + lane_c;
    float m[V], r[V], w[V], b[V], mt[V], mtx[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = c0 + lane_c + j;
        const long long g = sample * n.groups + c / n.per_group;
        m[j] = mean[g];
        r[j] = rstd[g];
        w[j] = weight != nullptr ? weight[c] : 1.0f;
        b[j] = bias != nullptr ? bias[c] : 0.0f;
        const float2 gm = group_means[g];
        mt[j] = gm.x;
        mtx[j] = gm.y;
    }
#pragma unroll 2
    for (long long row = row0; row < count; row += rows_per_pass) {
        const Piece p = *reinterpret_cast<const Piece*>(dy + base + row * n.channels);
        const Raw q = *static_cast<const Raw*>(in.at(base + row * n.channels));
        const float scale = Packed ? *in.scale_at(first_row + row, c0 + lane_c, n.channels) : 1.0f;
        Piece out;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float xhat = (Input<T, V, Packed>::value(q, j, scale) - m[j]) * r[j];
            float slope;
            activate_slope<Act>(fmaf(xhat, w[j], b[j]), slope);
            const float tv = to_float(p.v[j]) * slope * w[j];
            out.v[j] = from_float<T>(r[j] * (tv - mt[j] - xhat * mtx[j]));
        }
        *reinterpret_cast<Piece*>(dx + base + row * n.channels) = out;
    }
}

// dbias[c] and dweight[c]: the samples' sums added up. Eight row lanes per channel, joined in
// a fixed order.
__global__ void __launch_bounds__(kThreads)
    norm_parameter_kernel(const float* __restrict__ sample_sums, float* __restrict__ dweight, float* __restrict__ dbias,
                          long long batch, int channels)
{
    __shared__ float sb[8][33], sw[8][33];
    allow_next_grid();
    wait_for_previous_grid();
    const int c = static_cast<int>(blockIdx.x) * 32 + static_cast<int>(threadIdx.x & 31);
    const int part = static_cast<int>(threadIdx.x >> 5);
    float b = 0.0f, w = 0.0f;
    if (c < channels) {
        for (long long k = part; k < batch; k += 8) {
            b += sample_sums[k * channels + c];
            w += sample_sums[(batch + k) * channels + c];
        }
    }
    sb[part][threadIdx.x & 31] = b;
    sw[part][threadIdx.x & 31] = w;
    __syncthreads();
    if (part == 0 && c < channels) {
        for (int k = 1; k < 8; ++k) {
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

// The resident form's slicing, or false where a unit does not fit. `held` is the bytes of shared
// memory per channel of a row (x; x and dy in the backward pass), `arrays` the floats per channel
// and `group_arrays` per group next to the data.
bool slice(const NormShape& n, int vec, int elem, int held, int arrays, int group_arrays, Slicing& s)
{
    s.width = 0;
    for (int k = 1; k <= n.groups; ++k) {
        const long long width = static_cast<long long>(k) * n.per_group;
        if (n.groups % k == 0 && width % vec == 0 && (width * elem >= 32 || k == n.groups)) {
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
            return units * s.cluster <= 0x7fffffffLL;
        }
    }
    return false;
}

// The two-pass form's parts of a sample: about four CTAs an SM over the whole call.
long long max_chunks(long long batch) { return std::max<long long>(1, 4LL * 148 / std::max<long long>(1, batch)); }

Tiling tiling(const NormShape& n, int vec)
{
    Tiling t{};
    t.lanes = std::min(n.channels / vec, 64);
    t.width = t.lanes * vec;
    t.tiles = (n.channels + t.width - 1) / t.width;
    const int rows_per_pass = kThreads / t.lanes;
    const long long want = max_chunks(n.batch * t.tiles);
    const long long most = std::max<long long>(1, n.points / (4 * rows_per_pass));  // four passes each, or more
    t.chunks = static_cast<int>(std::min(want, most));
    t.rows = (n.points + t.chunks - 1) / t.chunks;
    return t;
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

// 16-byte pieces where the rows are whole pieces and every array is aligned, else single values.
template <class T, class F>
void with_pieces(bool wide, F&& f)
{
    if (wide) {
        f(std::integral_constant<int, 16 / static_cast<int>(sizeof(T))>{});
    } else {
        f(std::integral_constant<int, 1>{});
    }
}

void norm_forward(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd, int dtype,
                  const NormShape& n, void* work, cudaStream_t stream)
{
    with_dtype(dtype, [&](auto type) {
        using T = decltype(type);
        const bool wide = n.channels % (16 / static_cast<int>(sizeof(T))) == 0 && aligned_to(x, 16) && aligned_to(y, 16);
        with_pieces<T>(wide, [&](auto pieces) {
            constexpr int V = decltype(pieces)::value;
            with_activation(n.act, [&](auto act) {
                constexpr int Act = decltype(act)::value;
                Slicing s;
                if (slice(n, V, sizeof(T), sizeof(T), 1, 4, s)) {
                    launch_cluster<norm_resident_kernel<T, V, Act>>(n.batch * s.slices, s, stream,
                                   static_cast<const T*>(x), weight, bias, static_cast<T*>(y), mean, rstd, n, s);
                    return;
                }
                const Tiling t = tiling(n, V);
                auto* partial = static_cast<float2*>(work);
                if (mean == nullptr) {  // inference: the statistics live behind the partial results
                    mean = reinterpret_cast<float*>(partial + n.batch * max_chunks(n.batch) * n.channels);
                    rstd = mean + n.batch * n.groups;
                }
                const dim3 grid(static_cast<unsigned>(t.chunks), static_cast<unsigned>(n.batch), static_cast<unsigned>(t.tiles));
                launch_pdl(norm_partial_kernel<T, V>, grid, dim3(kThreads), 4u * (kThreads * V + 3 * t.width), stream,
                           static_cast<const T*>(x), partial, n, t);
                launch_pdl(norm_join_kernel, dim3(static_cast<unsigned>(n.batch * n.groups)), dim3(kThreads), 0, stream,
                           static_cast<const float2*>(partial), mean, rstd, n, t);
                launch_pdl(norm_apply_kernel<T, V, Act>, grid, dim3(kThreads), 0, stream, static_cast<const T*>(x), weight,
                           bias, static_cast<const float*>(mean), static_cast<const float*>(rstd), static_cast<T*>(y), n, t);
            });
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
        const Tiling t = tiling(n, V);
        auto* group_means = reinterpret_cast<float2*>(sample_sums + 2 * n.batch * n.channels);
        float2* partial = group_means + n.batch * n.groups;
        const dim3 grid(static_cast<unsigned>(t.chunks), static_cast<unsigned>(n.batch), static_cast<unsigned>(t.tiles));
        launch_pdl(norm_backward_partial_kernel<T, V, Packed, Act>, grid, dim3(kThreads), 4u * (kThreads * V + 2 * t.width),
                   stream, dy, in, weight, bias, mean, rstd, partial, n, t);
        launch_pdl(norm_backward_join_kernel, dim3(static_cast<unsigned>(n.batch * n.groups)), dim3(kThreads), 0, stream,
                   static_cast<const float2*>(partial), weight, sample_sums, group_means, n, t);
        launch_pdl(norm_backward_apply_kernel<T, V, Packed, Act>, grid, dim3(kThreads), 0, stream, dy, in, weight, bias,
                   mean, rstd, static_cast<const float2*>(group_means), dx, n, t);
    }
    if (dweight != nullptr || dbias != nullptr) {
        launch_pdl(norm_parameter_kernel, dim3(static_cast<unsigned>((n.channels + 31) / 32)), dim3(kThreads), 0, stream,
                   static_cast<const float*>(sample_sums), dweight, dbias, n.batch, n.channels);
    }
}

void norm_backward(const void* dy, const void* x, const signed char* codes, const float* scales, const float* weight,
                   const float* bias, const float* mean, const float* rstd, void* dx, float* dweight, float* dbias,
                   int dtype, const NormShape& n, float* work, cudaStream_t stream)
{
    with_dtype(dtype, [&](auto type) {
        using T = decltype(type);
        constexpr int kWide = 16 / static_cast<int>(sizeof(T));
        const bool wide = n.channels % kWide == 0 && aligned_to(dy, 16) && aligned_to(dx, 16)
                          && (codes != nullptr ? aligned_to(codes, kWide) : aligned_to(x, 16));
        with_pieces<T>(wide, [&](auto pieces) {
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
    if (batch > 65535 || channels > (1 << 20) || static_cast<long long>(batch) * groups > 0x7fffffffLL
        || (batch > 0 && points > (1LL << 46) / (batch * channels))) {
        return invalid(name + ": at most 65535 samples, 2^20 channels and 2^46 values");
    }
    return SPECTRAL_OK;
}

bool overlap(const void* a, const void* b, unsigned long long bytes)
{
    const auto p = reinterpret_cast<unsigned long long>(a);
    const auto q = reinterpret_cast<unsigned long long>(b);
    return p < q + bytes && q < p + bytes;
}

}  // namespace
}  // namespace spectral

extern "C" int spectral_group_norm_act_workspace(long long batch, int channels, int groups, size_t* count)
{
    using namespace spectral;
    if (batch < 0 || channels < 1 || groups < 1 || count == nullptr) {
        return invalid("group_norm_act_workspace: need batch >= 0, channels >= 1, groups >= 1");
    }
    // Per-channel partial results of the two-pass form, and statistics the caller does not keep.
    *count = static_cast<size_t>(batch) * (static_cast<size_t>(max_chunks(batch)) * channels + groups);
    return SPECTRAL_OK;
}

extern "C" int spectral_group_norm_act_backward_workspace(long long batch, int channels, int groups, size_t* count)
{
    using namespace spectral;
    if (batch < 0 || channels < 1 || groups < 1 || count == nullptr) {
        return invalid("group_norm_act_backward_workspace: need batch >= 0, channels >= 1, groups >= 1");
    }
    // The samples' parameter sums, the groups' means, the two-pass form's partial results.
    *count = static_cast<size_t>(batch) * (static_cast<size_t>(max_chunks(batch) + 1) * channels + groups);
    return SPECTRAL_OK;
}

extern "C" int spectral_group_norm_act(const void* x, const float* weight, const float* bias, void* y, float* mean,
                                       float* rstd, void* codes, float* scales, int dtype, long long batch,
                                       long long points, int channels, int groups, float eps, int activation, void* work,
                                       void* stream)
{
    using namespace spectral;
    const int status = check("group_norm_act", dtype, batch, points, channels, groups, activation);
    if (status != SPECTRAL_OK || batch == 0 || points == 0) {
        return status;
    }
    if (x == nullptr || y == nullptr || work == nullptr || (mean == nullptr) != (rstd == nullptr)
        || (codes == nullptr) != (scales == nullptr)) {
        return invalid("group_norm_act: x, y and work must be given, mean with rstd, and codes with scales");
    }
    if (!aligned_to(x, dtype_size(dtype)) || !aligned_to(y, dtype_size(dtype)) || !aligned_to(work, 8)) {
        return invalid("group_norm_act: arrays must be aligned to their element size, work to 8 bytes");
    }
    if (overlap(x, y, static_cast<unsigned long long>(batch * points) * channels * dtype_size(dtype))) {
        return invalid("group_norm_act: x and y must not overlap");
    }
    try {
        const NormShape n{batch, points, channels, groups, channels / groups, activation, eps};
        norm_forward(x, weight, bias, y, mean, rstd, dtype, n, work, static_cast<cudaStream_t>(stream));
        if (codes != nullptr) {
            pack8(x, dtype, static_cast<signed char*>(codes), scales, batch * points, channels,
                  static_cast<cudaStream_t>(stream));
        }
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
        if (!aligned_to(dy, size) || !aligned_to(dx, size) || !aligned_to(x, size) || !aligned_to(work, 8)) {
            return invalid("group_norm_act_backward: arrays must be aligned to their element size, work to 8 bytes");
        }
        const unsigned long long bytes = static_cast<unsigned long long>(batch * points) * channels * size;
        if (overlap(dx, dy, bytes) || (x != nullptr && overlap(dx, x, bytes))) {
            return invalid("group_norm_act_backward: dx must not overlap dy or x");
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
