// Queries and keys before an attention: the norm of each head and the rotation by position, in one
// pass over both (include/spectral_b200.h: spectral_qk_norm_rotary and its backward).
//
// Over one head x of `dim` values, with r = 1 / sqrt(mean(x^2) + eps):
//   u = x r w,  and of each pair (u1, u2) turned by its angle a: (u1 cos a - u2 sin a, u1 sin a + u2 cos a)
// Backward, with g the upstream gradient turned back by -a:
//   dw = sum over rows of g x r,  dx = r (g w - x r^2 mean(g w x))
//
// Memory would bound it: a value is read and written once (backward: two reads, one write), some ten operations
// each. A lane holds one 16-byte piece of a head (8 bytes or 4 where rows are aligned to no more), a head's
// lanes sit side by side, so its sums are a few shuffles and so is the exchange of the pairs that lie half
// an axis apart. The angles of a token serve all of its heads: a CTA takes as many tokens as its shared memory
// holds tables for, asks for the first pieces, fills the table of cosines and sines while they arrive, then works
// through the heads. An angle is position * frequency in turns, in two floats or in 64 bits until whole turns
// are taken off (a position of 2^20 leaves an angle of 2^-4 in 32 bits), then float32: see turn_of.
// Sums over dim, and those of the weights' gradients over rows, are float32 in a fixed order.
// What bounds it is the number of instructions, 31 a value at two heads a token: 64 x 16384 tokens of 2 x 32 bf16 values and
// 256 keys a sample take 102 us (2.8 TB/s; the bytes alone 43 us), forward and backward 239 us.

#include "../../include/spectral_b200.h"

#include "backend.hpp"
#include "extent.hpp"
#include "launch.cuh"
#include "pointwise.cuh"

#include <algorithm>
#include <cmath>

namespace spectral {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = SPECTRAL_HEAD_DIM_MAX;
constexpr double kNearTurns = 65536.0;  // see turn_of
constexpr int kTableBytes = 40 * 1024;  // places, positions and tables, at most

// Heads a lane works on at a time, while it waits for as many more.
// (64 x 16384 x 2 x 32 bf16, measured side by side: four CTAs an SM and fewer heads a lane 105 us, backward 268; two CTAs 124 and
// 288; this form 102 and 245, and 102 and 239 with the steps that followed.)
__host__ __device__ constexpr int rows_in_flight(int units, bool back) { return units > 1 ? (back ? 1 : 2) : back ? 2 : 4; }

struct Side {
    const void* x = nullptr;
    const void* dy = nullptr;
    void* out = nullptr;  // y, or dx
    const float* weight = nullptr;
    const void* positions = nullptr;
    float* partial = nullptr;  // backward: a row of dim sums per CTA
    long long stride[3] = {0, 0, 0};
    long long position_stride[3] = {0, 0, 0};
    int position_type = 0;
    int heads = 0;
    long long tokens = 0;  // of a sample
    long long total = 0;   // of all samples
    int tile_tokens = 1;
    int ctas = 0;
};

struct Plan {
    Side side[2];
    int dim = 0;
    int rotated = 0;
    int axes = 1;
    int per_axis = 0;  // pairs
    int table_pitch = 0;    // pairs of a token in the table, a multiple of 4
    int table_columns = 1;  // the power of two from there on
    int token_bytes = 8;    // of a token's place and positions
    bool neighbours = false;
    float eps = 0.0f;
    float near = 0.0f;  // float positions up to here make less than kNearTurns
    double turns[kMaxDim / 2];  // angle per position, in turns, of an axis's pairs
};

// (cos, sin) of a fraction of a turn between -1/2 and 1/2 (or just past it). For results rounded to 16 bits the hardware's functions on
// [-pi, pi], off by 2^-20 at most, do.
template <class T>
__device__ __forceinline__ float2 unit(float turn)
{
    float2 cs;
    if constexpr (sizeof(T) == 4) {
        sincospif(2.0f * turn, &cs.y, &cs.x);
    } else {
        __sincosf(6.283185307179586f * turn, &cs.y, &cs.x);
    }
    return cs;
}

// A pair's frequency in turns per position: in 64 bits, and as the sum of two floats.
struct Frequency {
    double turns;
    float high;
    float low;
};

// What is left of position * frequency without its whole turns. A float's product with the two floats is exact but for
// 2^-48 of it, and as long as it makes less than kNearTurns the rounded product's error, which is not reduced again, is below 2^-7
// of a turn. Whole numbers, and floats that make more, go through 64 bits: off by 2^-53 of all turns for the
// product, and by (4 + |ln frequency|) times that for the frequency.
template <class P>
__device__ __forceinline__ float turn_of(P position, const Frequency& f)
{
    if constexpr (std::is_same_v<P, float>) {
        const float a = position * f.high;
        return (a - rintf(a)) + fmaf(position, f.low, fmaf(position, f.high, -a));
    } else {
        const double a = position * f.turns;
        return static_cast<float>(a - rint(a));
    }
}

template <class W>
__device__ __forceinline__ W shuffle_words(const W& v, int src)
{
    static_assert(sizeof(W) % 4 == 0, "whole words");
    W out;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(W) / 4); ++i) {
        reinterpret_cast<uint32_t*>(&out)[i] = __shfl_sync(0xffffffffu, reinterpret_cast<const uint32_t*>(&v)[i], src);
    }
    return out;
}

__device__ __forceinline__ float sum_lanes(float v, int lanes)
{
    for (int o = lanes / 2; o > 0; o /= 2) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// V values of a head per piece, `lanes` (a power of two) lanes a head with U pieces each, piece k of lane l the
// (l + k lanes)th; V = 1: any dim and alignment. Forward needs x, backward also dy.
template <class T, int V, int U, bool Back>
__global__ void __launch_bounds__(kThreads, 3) rotary_kernel(const __grid_constant__ Plan plan, int lanes)
{
    constexpr int kRows = rows_in_flight(U, Back);
    using Piece = Vec<T, V>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) float exchange[U > 1 ? kThreads / 32 : 1][U > 1 ? kMaxDim : 4];
    const bool second_side = static_cast<int>(blockIdx.x) >= plan.side[0].ctas;
    const Side& s = plan.side[second_side ? 1 : 0];
    const int cta = blockIdx.x - (second_side ? plan.side[0].ctas : 0);
    const int dim = plan.dim;
    const int rotated = s.positions != nullptr ? plan.rotated : 0;
    const int n = plan.per_axis;
    const int pitch = plan.table_pitch;
    const int span = s.tile_tokens;
    // Of each token of a tile: where it starts, its positions (floats, or whole numbers in 64 bits), the cosines of its
    // pairs, the sines.
    auto* const places = reinterpret_cast<long long*>(smem);
    auto* const whole_positions = reinterpret_cast<double*>(places + span);
    auto* const float_positions = reinterpret_cast<float*>(places + span);
    // (on 16 bytes: the tables are read in vectors)
    auto* const cosines = reinterpret_cast<float*>(smem + (static_cast<size_t>(span) * plan.token_bytes + 15) / 16 * 16);
    const bool floats = s.position_type == SPECTRAL_POSITIONS_FLOAT32;

    const int lane = threadIdx.x & 31;
    const int sub = lane & (lanes - 1);
    const int group = threadIdx.x / lanes;
    const int groups = kThreads / lanes;
    // This lane's pieces: where in the head, which pairs of the table, where the partners are (halves) and the sign of
    // their sines.
    int d[U], pair_at[U], partner[U];
    bool live[U], turned[U];
    float sign[U];
    Floats<V> w[U], wp[U], dw[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
        d[k] = (sub + k * lanes) * V;
        live[k] = d[k] < dim;
        turned[k] = live[k] && d[k] < rotated;
        bool first = true;
        partner[k] = d[k];
        pair_at[k] = d[k] / 2;
        if (plan.neighbours) {
            if (V == 1) {
                first = d[k] % 2 == 0;
                partner[k] = d[k] ^ 1;
            }
        } else if (turned[k]) {
            const int axis = d[k] / (2 * n);
            const int off = d[k] - axis * 2 * n;
            first = off < n;
            partner[k] = first ? d[k] + n : d[k] - n;
            pair_at[k] = axis * n + (first ? off : off - n);
        }
        sign[k] = first != Back ? -1.0f : 1.0f;
        w[k].fill(1.0f);
        wp[k].fill(1.0f);
        dw[k].fill(0.0f);
    }
    // This thread's column of the table: one pair, every `table_rows`-th token.
    const int column = threadIdx.x % plan.table_columns;
    const int table_rows = kThreads / plan.table_columns;
    const int column_axis = column < rotated / 2 ? column / n : 0;
    Frequency frequency{column < rotated / 2 ? plan.turns[column - column_axis * n] : 0.0, 0.0f, 0.0f};
    frequency.high = static_cast<float>(frequency.turns);
    frequency.low = static_cast<float>(frequency.turns - frequency.high);
    allow_next_grid();
    wait_for_previous_grid();
    if (s.weight != nullptr) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (live[k]) {
                    w[k].set(j, s.weight[d[k] + j]);
                    wp[k].set(j, turned[k] ? s.weight[partner[k] + j] : 0.0f);
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {  // what a partner's value meets: weight and sign (backward: the sign)
#pragma unroll
        for (int j = 0; j < Floats<V>::kPairs; ++j) {
            wp[k].p[j] = Back ? pair(sign[k]) : wp[k].p[j] * pair(sign[k]);
        }
    }
    const int heads = s.heads;
    const int step_tokens = groups / heads;
    const int step_heads = groups - step_tokens * heads;
    const float per_dim = 1.0f / static_cast<float>(dim);
    float* const sines = cosines + span * pitch;

    for (long long start = static_cast<long long>(cta) * span; start < s.total; start += static_cast<long long>(s.ctas) * span) {
        const int tokens = static_cast<int>(min(static_cast<long long>(span), s.total - start));
        int close = 1;
        for (int t = threadIdx.x; t < tokens; t += kThreads) {
            const long long token = start + t;
            const long long b = s.total < (1LL << 31) ? static_cast<unsigned>(token) / static_cast<unsigned>(s.tokens) : token / s.tokens;
            const long long in = token - b * s.tokens;
            places[t] = b * s.stride[0] + in * s.stride[1];
            if (rotated > 0) {
                const long long at = b * s.position_stride[0] + in * s.position_stride[1];
                for (int axis = 0; axis < plan.axes; ++axis) {
                    const long long from = at + axis * s.position_stride[2];
                    if (floats) {
                        const float position = static_cast<const float*>(s.positions)[from];
                        float_positions[axis * span + t] = position;
                        close &= fabsf(position) <= plan.near ? 1 : 0;
                    } else {
                        whole_positions[axis * span + t] = s.position_type == SPECTRAL_POSITIONS_INT32
                                                               ? static_cast<double>(static_cast<const int*>(s.positions)[from])
                                                               : static_cast<double>(static_cast<const long long*>(s.positions)[from]);
                    }
                }
            }
        }
        const bool near = __syncthreads_and(close) != 0;
        const T* __restrict__ x = static_cast<const T*>(s.x);
        const T* __restrict__ dy = static_cast<const T*>(s.dy) + start * heads * dim;
        T* __restrict__ out = static_cast<T*>(s.out) + start * heads * dim;
        const int rows = tokens * heads;  // a tile is at most a CTA's share of the call: its values stay below 2^31
        int next_token = group / heads;
        int next_head = group - next_token * heads;
        for (int base = 0; base < rows; base += kRows * groups) {
            Piece px[kRows][U], pg[kRows][U];
            int token_of[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int row = base + group + r * groups;
                token_of[r] = min(next_token, tokens - 1);
                const T* from = x + places[token_of[r]] + next_head * s.stride[2];
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    px[r][k] = Piece{};
                    pg[r][k] = Piece{};
                    if (row < rows && live[k]) {
                        px[r][k] = *reinterpret_cast<const Piece*>(from + d[k]);
                        if constexpr (Back) {
                            pg[r][k] = *reinterpret_cast<const Piece*>(dy + row * dim + d[k]);
                        }
                    }
                }
                next_token += step_tokens;
                next_head += step_heads;
                if (next_head >= heads) {
                    next_head -= heads;
                    ++next_token;
                }
            }
            if (base == 0) {  // the first pieces are on their way
                if (rotated > 0 && column < pitch) {
                    const auto fill = [&](const auto* from, auto turn) {
                        from += column_axis * span;
                        int t = threadIdx.x / plan.table_columns;
                        float* to = cosines + t * pitch + column;
                        const int step = table_rows * pitch, across = span * pitch;
#pragma unroll 4
                        for (; t < tokens; t += table_rows, to += step) {
                            const float2 cs = unit<T>(turn(from[t]));
                            to[0] = cs.x;
                            to[across] = cs.y;
                        }
                    };
                    if (column >= rotated / 2) {  // of a piece that reaches past `rotated`: whatever the position, not turned
                        for (int t = threadIdx.x / plan.table_columns; t < tokens; t += table_rows) {
                            cosines[t * pitch + column] = 1.0f;
                            sines[t * pitch + column] = 0.0f;
                        }
                    } else if (!floats) {
                        fill(whole_positions, [&](double p) { return turn_of(p, frequency); });
                    } else if (near) {
                        fill(float_positions, [&](float p) { return turn_of(p, frequency); });
                    } else {  // each by its own size: a token's bits do not depend on its neighbours
                        fill(float_positions,
                             [&](float p) { return fabsf(p) <= plan.near ? turn_of(p, frequency) : turn_of(static_cast<double>(p), frequency); });
                    }
                }
                __syncthreads();
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int row = base + group + r * groups;
                if (base + r * groups >= rows) {  // none in the whole CTA
                    break;
                }
                Floats<V> xs[U], f[U];
                float2 square = pair(0.0f);
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    xs[k] = widen(px[r][k]);
#pragma unroll
                    for (int j = 0; j < Floats<V>::kPairs; ++j) {
                        square = fma2(xs[k].p[j], xs[k].p[j], square);
                    }
                }
                // (A row behind the tile's last holds zeros: with eps = 0 its root's inverse would be infinite, and 0 times that a NaN
                // in the weights' sums.)
                const float norm = rsqrtf(fmaf(sum_lanes(square.x + square.y, lanes), per_dim, plan.eps));
                const float inv = !Back || row < rows ? norm : 0.0f;
                // What is turned: x w forward (inv comes at the end), the upstream gradient (the other way) backward.
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    f[k] = Back ? widen(pg[r][k]) : xs[k];
                }
                if (rotated > 0) {
                    const float* c = cosines + token_of[r] * pitch;
                    const float* e = sines + token_of[r] * pitch;
                    if constexpr (U > 1) {
                        float* buf = exchange[threadIdx.x >> 5];
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < U; ++k) {
                            if (live[k]) {
#pragma unroll
                                for (int j = 0; j < V; ++j) {
                                    buf[d[k] + j] = f[k].at(j);
                                }
                            }
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (int k = 0; k < U; ++k) {
                        if (V > 1 && plan.neighbours) {
                            if constexpr (!Back) {
#pragma unroll
                                for (int j = 0; j < Floats<V>::kPairs; ++j) {
                                    f[k].p[j] = f[k].p[j] * w[k].p[j];
                                }
                            }
                            if (turned[k]) {
                                const auto cs = *reinterpret_cast<const Vec<float, V / 2 + (V == 1)>*>(c + pair_at[k]);
                                const auto sn = *reinterpret_cast<const Vec<float, V / 2 + (V == 1)>*>(e + pair_at[k]);
#pragma unroll
                                for (int j = 0; j < V / 2; ++j) {
                                    const float sine = Back ? -sn.v[j] : sn.v[j];
                                    const float2 v = f[k].p[j];
                                    f[k].p[j] = fma2(v, pair(cs.v[j]), make_float2(-v.y * sine, v.x * sine));
                                }
                            }
                        } else {
                            Floats<V> other;
                            if constexpr (U > 1) {
#pragma unroll
                                for (int j = 0; j < V; ++j) {
                                    other.set(j, exchange[threadIdx.x >> 5][live[k] ? partner[k] + j : 0]);
                                }
                            } else {
                                other = widen(shuffle_words(Back ? pg[r][k] : px[r][k], lane - sub + partner[k] / V));
                            }
                            if (turned[k]) {
                                const auto cs = *reinterpret_cast<const Vec<float, V>*>(c + pair_at[k]);
                                const auto sn = *reinterpret_cast<const Vec<float, V>*>(e + pair_at[k]);
                                const Floats<V> c2 = widen(cs), s2 = widen(sn);
#pragma unroll
                                for (int j = 0; j < Floats<V>::kPairs; ++j) {
                                    const float2 a = Back ? c2.p[j] : c2.p[j] * w[k].p[j];
                                    f[k].p[j] = fma2(f[k].p[j], a, other.p[j] * (s2.p[j] * wp[k].p[j]));
                                }
                            } else if constexpr (!Back) {
#pragma unroll
                                for (int j = 0; j < Floats<V>::kPairs; ++j) {
                                    f[k].p[j] = f[k].p[j] * w[k].p[j];
                                }
                            }
                        }
                    }
                } else if constexpr (!Back) {
#pragma unroll
                    for (int k = 0; k < U; ++k) {
#pragma unroll
                        for (int j = 0; j < Floats<V>::kPairs; ++j) {
                            f[k].p[j] = f[k].p[j] * w[k].p[j];
                        }
                    }
                }
                if constexpr (Back) {
                    float2 dot = pair(0.0f);
#pragma unroll
                    for (int k = 0; k < U; ++k) {
#pragma unroll
                        for (int j = 0; j < Floats<V>::kPairs; ++j) {
                            const float2 gx = f[k].p[j] * xs[k].p[j];
                            dw[k].p[j] = fma2(gx, pair(inv), dw[k].p[j]);
                            dot = fma2(gx, w[k].p[j], dot);
                        }
                    }
                    const float c = -sum_lanes(dot.x + dot.y, lanes) * per_dim * inv * inv;
#pragma unroll
                    for (int k = 0; k < U; ++k) {
#pragma unroll
                        for (int j = 0; j < Floats<V>::kPairs; ++j) {
                            f[k].p[j] = fma2(xs[k].p[j], pair(c), f[k].p[j] * w[k].p[j]);
                        }
                    }
                }
                if (row < rows) {
#pragma unroll
                    for (int k = 0; k < U; ++k) {
                        if (live[k]) {
#pragma unroll
                            for (int j = 0; j < Floats<V>::kPairs; ++j) {
                                f[k].p[j] = f[k].p[j] * pair(inv);
                            }
                            *reinterpret_cast<Piece*>(out + row * dim + d[k]) = narrow<T>(f[k]);
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
    if constexpr (Back) {
        if (s.partial == nullptr) {
            return;
        }
        // The groups' sums of each value, in order: through shared memory, a value a thread.
        auto* sums = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int k = 0; k < U; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (live[k]) {
                    sums[group * dim + d[k] + j] = dw[k].at(j);
                }
            }
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < dim) {
            float total = 0.0f;
            for (int g = 0; g < groups; ++g) {
                total += sums[g * dim + threadIdx.x];
            }
            s.partial[static_cast<long long>(cta) * dim + threadIdx.x] = total;
        }
    }
}

// dweight = the sum of the CTAs' rows; a CTA per side and 32 values, eight warps side by side over the rows.
struct Sums {
    const float* partial[2];
    float* out[2];
    int rows[2];
    int dim;
};

__global__ void __launch_bounds__(256) weight_sum_kernel(const Sums g)
{
    __shared__ float part[8][32];
    wait_for_previous_grid();
    const int side = blockIdx.y;
    const int d = blockIdx.x * 32 + (threadIdx.x & 31);
    const int warp = threadIdx.x >> 5;
    if (g.out[side] == nullptr) {
        return;
    }
    float total = 0.0f;
    if (d < g.dim) {
#pragma unroll 4
        for (int r = warp; r < g.rows[side]; r += 8) {
            total += g.partial[side][static_cast<long long>(r) * g.dim + d];
        }
    }
    part[warp][threadIdx.x & 31] = total;
    __syncthreads();
    if (warp == 0 && d < g.dim) {
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            total += part[i][threadIdx.x];
        }
        g.out[side][d] = total;
    }
}

// --- host ------------------------------------------------------------------------------------------

int invalid(const std::string& message)
{
    set_last_error(message);
    return SPECTRAL_INVALID_ARGUMENT;
}

// Values per access that every row of the call allows: whole pieces in a head (and in half an axis's values, where
// partners lie that far apart), at most a warp's worth, aligned.
int vector_width(const spectral_heads* const (&sides)[2], int dtype, long long batch, int dim, int rotated, int axes, int pairs)
{
    const int size = static_cast<int>(dtype_size(dtype));
    const int n = static_cast<int>(rotated / (2LL * axes));
    for (int v = 16 / size; v >= 2; v /= 2) {
        bool ok = dim % v == 0 && dim / v <= (v == 2 ? 64 : 32) && (rotated == 0 || pairs == SPECTRAL_PAIRS_NEIGHBOURS || n % v == 0);
        for (const spectral_heads* s : sides) {
            if (s == nullptr) {
                continue;
            }
            ok = ok && aligned_to(s->x, v * size) && aligned_to(s->out, v * size) && aligned_to(s->dy, v * size)
                 && (batch <= 1 || s->stride[0] % v == 0) && (s->tokens <= 1 || s->stride[1] % v == 0)
                 && (s->heads <= 1 || s->stride[2] % v == 0);
        }
        if (ok) {
            return v;
        }
    }
    return 1;
}

int lanes_for(int dim, int v)
{
    int lanes = 1;
    while (lanes < 32 && lanes * v < dim) {
        lanes *= 2;
    }
    return lanes;
}

constexpr int kMostResident = 4;  // CTAs of an SM, by the tables
int most_ctas() { return device_sm_count(current_device()) * kMostResident; }

// Calls f(kernel, cache of its residency) for the variant of a call.
template <class F>
void with_kernel(int dtype, int v, int units, bool back, F&& f)
{
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const auto pick = [&](auto width, auto pieces) {
            constexpr int V = decltype(width)::value;
            constexpr int U = decltype(pieces)::value;
            static std::atomic<int> cache[2][kMaxDevices];
            if (back) {
                f(rotary_kernel<T, V, U, true>, cache[1]);
            } else {
                f(rotary_kernel<T, V, U, false>, cache[0]);
            }
        };
        constexpr std::integral_constant<int, 1> one;
        constexpr std::integral_constant<int, 2> two;
        constexpr std::integral_constant<int, 4> four;
        switch (v) {
            case 8:
                if constexpr (sizeof(T) == 2) {
                    pick(std::integral_constant<int, 8>{}, one);
                }
                break;
            case 4: pick(four, one); break;
            case 2:
                if (units == 2) {
                    pick(two, two);
                } else {
                    pick(two, one);
                }
                break;
            default: pick(one, four); break;
        }
    });
}

int check(const char* op, const spectral_heads* const (&sides)[2], bool back, int dtype, long long batch, int dim, int rotated,
          int axes, int pairs, float eps, float theta)
{
    const std::string name(op);
    if (!dtype_known(dtype)) {
        return invalid(name + ": dtype must be SPECTRAL_FLOAT32, SPECTRAL_BFLOAT16 or SPECTRAL_FLOAT16");
    }
    if (dim < 1 || dim > kMaxDim) {
        return invalid(name + ": need 1 <= dim <= " + std::to_string(kMaxDim));
    }
    if (axes < 1 || rotated < 0 || rotated > dim || rotated % (2LL * axes) != 0) {
        return invalid(name + ": rotated must be a multiple of 2 * axes from 0 to dim");
    }
    if (pairs != SPECTRAL_PAIRS_HALVES && pairs != SPECTRAL_PAIRS_NEIGHBOURS) {
        return invalid(name + ": pairs must be SPECTRAL_PAIRS_HALVES or SPECTRAL_PAIRS_NEIGHBOURS");
    }
    if (!(eps >= 0.0f) || !(theta > 0.0f) || std::isinf(theta)) {
        return invalid(name + ": need eps >= 0 and a finite theta > 0");
    }
    if (sides[0] == nullptr && sides[1] == nullptr) {
        return invalid(name + ": needs q or k");
    }
    for (const spectral_heads* s : sides) {
        if (s == nullptr) {
            continue;
        }
        if (batch < 0 || s->tokens < 0 || s->heads < 1 || s->heads > (1 << 20) || batch >= (1LL << 31) || s->tokens >= (1LL << 31)
            || (s->tokens > 0 && batch > (1LL << 40) / s->tokens)) {
            return invalid(name + ": need 0 <= batch, tokens < 2^31, batch * tokens <= 2^40 and heads from 1 to 2^20");
        }
        if (batch * s->tokens == 0) {
            continue;
        }
        const std::size_t size = dtype_size(dtype);
        if (s->x == nullptr || s->out == nullptr || (back && s->dy == nullptr)) {
            return invalid(name + ": null array");
        }
        if (!aligned_to(s->x, size) || !aligned_to(s->out, size) || !aligned_to(s->dy, size) || !aligned_to(s->weight, 4)
            || !aligned_to(s->dweight, 4)) {
            return invalid(name + ": arrays must be aligned to their element size");
        }
        if (s->positions != nullptr && rotated > 0) {
            if (s->position_type < SPECTRAL_POSITIONS_FLOAT32 || s->position_type > SPECTRAL_POSITIONS_INT64) {
                return invalid(name + ": position_type must be SPECTRAL_POSITIONS_FLOAT32, _INT32 or _INT64");
            }
            if (!aligned_to(s->positions, s->position_type == SPECTRAL_POSITIONS_INT64 ? 8 : 4)) {
                return invalid(name + ": positions must be aligned to their element size");
            }
        }
    }
    // The results are contiguous; an input may be a strided view, whose extent bounds what it can touch. A CTA works on one
    // side while others work on the other, so neither side's results may lie in an array of either.
    Extent x[2], weight[2], positions[2], out[2], dy[2], dweight[2];
    for (int i = 0; i < 2; ++i) {
        const spectral_heads* s = sides[i];
        if (s == nullptr || batch * s->tokens == 0) {
            continue;
        }
        const long long count[3] = {batch, s->tokens, s->heads};
        const std::size_t size = dtype_size(dtype);
        const unsigned long long bytes = static_cast<unsigned long long>(batch) * s->tokens * s->heads * dim * size;
        x[i] = Extent(s->x, s->stride, count, dim, size);
        out[i] = Extent(s->out, bytes);
        weight[i] = Extent(s->weight, dim * sizeof(float));
        if (rotated > 0) {
            const long long places[3] = {batch, s->tokens, axes};
            positions[i] = Extent(s->positions, s->position_stride, places, 1, s->position_type == SPECTRAL_POSITIONS_INT64 ? 8 : 4);
        }
        if (back) {
            dy[i] = Extent(s->dy, bytes);
            dweight[i] = Extent(s->dweight, dim * sizeof(float));
        }
    }
    if (any_overlap({out[0], out[1], dweight[0], dweight[1]},
                    {x[0], x[1], dy[0], dy[1], weight[0], weight[1], positions[0], positions[1]})) {
        return invalid(name + ": the results must not overlap each other or the arguments");
    }
    return SPECTRAL_OK;
}

void run(const spectral_heads* const (&sides)[2], bool back, int dtype, long long batch, int dim, int rotated, int axes,
         int pairs, float eps, float theta, float* work, cudaStream_t stream)
{
    Plan plan;
    plan.dim = dim;
    plan.axes = axes;
    plan.neighbours = pairs == SPECTRAL_PAIRS_NEIGHBOURS;
    plan.eps = eps;
    bool any = false;
    for (const spectral_heads* s : sides) {
        any = any || (s != nullptr && s->positions != nullptr);
    }
    plan.rotated = any ? rotated : 0;
    plan.per_axis = static_cast<int>(std::max(1LL, plan.rotated / (2LL * axes)));
    // A piece that reaches past `rotated` (neighbours only) finds cosines of 1 and sines of 0 there.
    plan.table_pitch = plan.rotated == 0 ? 0 : ((plan.neighbours ? (dim + 1) / 2 : plan.rotated / 2) + 3) / 4 * 4;
    while (plan.table_columns < plan.table_pitch) {
        plan.table_columns *= 2;
    }
    plan.token_bytes = 8 + (plan.rotated > 0 ? 8 * axes : 0);
    for (int i = 0; i < plan.per_axis && plan.rotated > 0; ++i) {
        plan.turns[i] = std::pow(static_cast<double>(theta), -static_cast<double>(i) / plan.per_axis) / 6.283185307179586476925;
        plan.near = std::min(i == 0 ? HUGE_VALF : plan.near, static_cast<float>(kNearTurns / plan.turns[i]));
    }
    const int v = vector_width(sides, dtype, batch, dim, plan.rotated, axes, pairs);
    const int units = v == 1 ? 4 : v == 2 && dim > 64 ? 2 : 1;
    const int lanes = v == 1 ? 32 : lanes_for(dim, v);
    const int groups = kThreads / lanes;
    const int in_flight = rows_in_flight(units, back);
    int most = 0;
    with_kernel(dtype, v, units, back, [&](auto kernel, std::atomic<int>* cache) {
        const int device = current_device();
        most = device_sm_count(device) * std::min(kMostResident, resident_ctas(reinterpret_cast<const void*>(kernel), kThreads, kTableBytes, cache, device));
    });
    long long tiles[2] = {0, 0};
    int table_tokens = 1;
    for (int i = 0; i < 2; ++i) {
        const spectral_heads* s = sides[i];
        if (s == nullptr || batch * s->tokens == 0) {
            continue;
        }
        Side& t = plan.side[i];
        t.x = s->x;
        t.dy = s->dy;
        t.out = s->out;
        t.weight = s->weight;
        t.positions = plan.rotated > 0 ? s->positions : nullptr;
        t.position_type = s->position_type;
        std::copy(s->stride, s->stride + 3, t.stride);
        std::copy(s->position_stride, s->position_stride + 3, t.position_stride);
        t.heads = s->heads;
        t.tokens = s->tokens;
        t.total = batch * s->tokens;
        // As many tokens as the table holds, fewer if that leaves CTAs without any, but enough to keep all lanes busy.
        const long long cap = kTableBytes / (plan.table_pitch * 8 + plan.token_bytes);
        const long long busy = std::max(1, groups * in_flight / s->heads);
        const long long share = (t.total + most - 1) / most;
        t.tile_tokens = static_cast<int>(std::min(cap, std::min(t.total, std::max(busy, share))));
        tiles[i] = (t.total + t.tile_tokens - 1) / t.tile_tokens;
        table_tokens = std::max(table_tokens, t.tile_tokens);
    }
    // CTAs in proportion to the sides' values.
    const long long all = tiles[0] + tiles[1];
    if (all > 0) {
        const long long ctas = std::min<long long>(all, most);
        for (int i = 0; i < 2; ++i) {
            plan.side[i].ctas = tiles[i] == 0 ? 0 : static_cast<int>(std::max(1LL, std::min(tiles[i], (ctas * tiles[i] + all / 2) / all)));
        }
    }
    Sums sums{};
    sums.dim = dim;
    float* at = work;
    for (int i = 0; i < 2; ++i) {
        if (back && sides[i] != nullptr && sides[i]->dweight != nullptr) {
            sums.partial[i] = at;
            sums.out[i] = sides[i]->dweight;
            sums.rows[i] = plan.side[i].ctas;
            plan.side[i].partial = at;
            at += static_cast<long long>(plan.side[i].ctas) * dim;
        }
    }
    const int ctas = plan.side[0].ctas + plan.side[1].ctas;
    if (ctas > 0) {
        std::size_t smem = static_cast<std::size_t>(table_tokens) * (plan.table_pitch * 8 + plan.token_bytes) + 16;
        if (back) {
            smem = std::max(smem, static_cast<std::size_t>(groups) * dim * sizeof(float));
        }
        with_kernel(dtype, v, units, back, [&](auto kernel, std::atomic<int>*) {
            launch_pdl(kernel, dim3(ctas), dim3(kThreads), smem, stream, plan, lanes);
        });
    }
    if (sums.out[0] != nullptr || sums.out[1] != nullptr) {
        launch_pdl(weight_sum_kernel, dim3((dim + 31) / 32, 2), dim3(256), 0, stream, sums);
    }
}

int entry(const char* op, const spectral_heads* q, const spectral_heads* k, bool back, int dtype, long long batch, int dim, int rotated,
          int axes, int pairs, float eps, float theta, void* work, void* stream)
{
    const spectral_heads* const sides[2] = {q, k};
    const int status = check(op, sides, back, dtype, batch, dim, rotated, axes, pairs, eps, theta);
    if (status != SPECTRAL_OK) {
        return status;
    }
    const bool sums = back && ((q != nullptr && q->dweight != nullptr) || (k != nullptr && k->dweight != nullptr));
    if (sums && (work == nullptr || !aligned_to(work, 8))) {
        return invalid(std::string(op) + ": needs a workspace, 8-byte aligned");
    }
    try {
        run(sides, back, dtype, batch, dim, rotated, axes, pairs, eps, theta, static_cast<float*>(work), static_cast<cudaStream_t>(stream));
        return SPECTRAL_OK;
    } catch (const InvalidArgument& e) {
        return invalid(e.what());
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}

}  // namespace
}  // namespace spectral

extern "C" int spectral_qk_norm_rotary(const spectral_heads* q, const spectral_heads* k, int dtype, long long batch, int dim,
                                       int rotated, int axes, int pairs, float eps, float theta, void* stream)
{
    return spectral::entry("qk_norm_rotary", q, k, false, dtype, batch, dim, rotated, axes, pairs, eps, theta, nullptr, stream);
}

extern "C" int spectral_qk_norm_rotary_backward_workspace(int dim, size_t* count)
{
    using namespace spectral;
    if (count == nullptr || dim < 1 || dim > kMaxDim) {
        return invalid("qk_norm_rotary_backward_workspace: need 1 <= dim <= " + std::to_string(kMaxDim) + " and a count");
    }
    try {
        *count = (static_cast<std::size_t>(most_ctas() + 2) * dim + 1) / 2;
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}

extern "C" int spectral_qk_norm_rotary_backward(const spectral_heads* q, const spectral_heads* k, int dtype, long long batch, int dim,
                                                int rotated, int axes, int pairs, float eps, float theta, void* work, void* stream)
{
    return spectral::entry("qk_norm_rotary_backward", q, k, true, dtype, batch, dim, rotated, axes, pairs, eps, theta, work, stream);
}
