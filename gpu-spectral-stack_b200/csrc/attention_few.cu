// Attention of up to eight rows per key head: a single query's heads, while serving.
//
// The keys and values are all there is to read, once, and two multiply-adds per value and row all there is to compute: memory
// bounds it, and the CUDA cores keep up. (On the tensor cores such a tile leaves 120 of 128 rows empty, and its
// softmax runs in one warp: 16 samples x 4 x 16384 keys x 64 bf16, a quarter of them cut off, took 111 us; here
// 70 us.) A key
// head's keys are cut into ranges, one per CTA, and a range among its warps. `lanes` lanes hold a key, 16 bytes each
// where rows allow; each such group of lanes walks over keys of its own with the running maximum, sum and result of
// every row, four keys at a time: four scores by shuffles, one rescaling, four weighted values, with the next two
// fours copied to shared memory meanwhile. Groups, warps and ranges are joined at the end, in a fixed order.

#include "attention.cuh"

#include <algorithm>

namespace spectral::attention {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSms = 148;
constexpr int kBatch = 4;   // keys of a group at a time
constexpr int kStages = 3;  // batches on their way or being worked on

// Shared memory of a batch of a warp: every lane's pieces of K and V.
template <class T, int V, int U>
constexpr int kStageBytes = 2 * kBatch * U * 32 * V * static_cast<int>(sizeof(T));

struct Few {
    Call c;
    int lanes = 1;      // per key
    int splits = 1;
    float factor = 1.0f;
    float* partial = nullptr;    // (split, pair, row, dim)
    float2* stats = nullptr;     // (split, pair, row)
};

template <class T, int V, int U, int R>
__global__ void __launch_bounds__(kThreads, R >= 8 ? 1 : 2) few_kernel(const Few g)
{
    using Piece = Vec<T, V>;
    const Call& c = g.c;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float m_of[kWarps][R], sum_of[kWarps][R];
    __shared__ float acc_of[kWarps][R][SPECTRAL_HEAD_DIM_MAX];
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int lanes = g.lanes;
    const int sub = lane & (lanes - 1);
    const int groups = 32 / lanes;
    const int group = lane / lanes;
    const int at = blockIdx.x;
    const int b = at / c.kv_heads, head = at - b * c.kv_heads;
    const int rows = static_cast<int>(c.rows());
    allow_next_grid();
    wait_for_previous_grid();
    const int length = length_of(c, b);
    // This CTA's keys, and its warps' turns at them.
    const long long span = ((static_cast<long long>(length) + g.splits - 1) / g.splits + 31) / 32 * 32;
    const long long begin = min(static_cast<long long>(length), blockIdx.y * span);
    const long long end = min(static_cast<long long>(length), begin + span);

    Floats<V> q[R][U], acc[R][U];
    float m[R], sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        sum[r] = 0.0f;
        const int t = min(r, rows - 1) / c.group;
        const T* from = static_cast<const T*>(c.q) + b * c.qs.sample + t * c.qs.token + (head * c.group + min(r, rows - 1) - t * c.group) * c.qs.head;
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int d = (sub + k * lanes) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                q[r][k].set(j, d + j < c.dim ? to_float(from[d + j]) * g.factor : 0.0f);
            }
            if (V == 1) {
                q[r][k].p[0].y = 0.0f;
            }
            acc[r][k].fill(0.0f);
        }
    }
    const T* keys = static_cast<const T*>(c.k) + b * c.ks.sample + head * c.ks.head;
    const T* values = static_cast<const T*>(c.v) + b * c.vs.sample + head * c.vs.head;
    const unsigned char* mask = c.mask == nullptr ? nullptr : c.mask + static_cast<long long>(b) * c.keys;
    // Each lane copies its own pieces ahead and reads them back: [stage][K, V][key][unit][lane].
    Piece* const ring = reinterpret_cast<Piece*>(smem) + warp * kStages * (kStageBytes<T, V, U> / static_cast<int>(sizeof(Piece))) + lane;
    const auto slot = [&](int stage, int which, int i, int k) -> Piece& { return ring[(((stage * 2 + which) * kBatch + i) * U + k) * 32]; };
    const int step = kWarps * groups * kBatch;
    const long long first = begin + warp * groups * kBatch + group;
    const auto counting = [&](long long key0) {  // bit i: key i of the batch counts
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const long long key = key0 + i * groups;
            bits |= (key < end && (mask == nullptr || mask[key] != 0) ? 1u : 0u) << i;
        }
        return bits;
    };
    const auto ask = [&](int stage, long long key0, unsigned bits) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const T* k_row = keys + (key0 + i * groups) * c.ks.token;
            const T* v_row = values + (key0 + i * groups) * c.vs.token;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int d = (sub + k * lanes) * V;
                if ((bits >> i & 1u) != 0 && d < c.dim) {
                    copy_async<sizeof(Piece)>(&slot(stage, 0, i, k), k_row + d);
                    copy_async<sizeof(Piece)>(&slot(stage, 1, i, k), v_row + d);
                } else {  // what does not count may be anything
                    slot(stage, 0, i, k) = Piece{};
                    slot(stage, 1, i, k) = Piece{};
                }
            }
        }
        cp_async_commit();
    };
    unsigned bits_of[kStages];
    long long ahead = first;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        bits_of[i] = counting(ahead);
        ask(i, ahead, bits_of[i]);
        ahead += step;
    }
    unsigned next = counting(ahead);
    int stage = 0;
    for (long long key0 = first - group; key0 < end; key0 += step) {
        // The batch two ahead, into the place of the one that was left last; its mask was read a turn ago.
        const unsigned bits = bits_of[0];
#pragma unroll
        for (int i = 0; i + 2 < kStages; ++i) {
            bits_of[i] = bits_of[i + 1];
        }
        bits_of[kStages - 2] = next;
        ask(stage == 0 ? kStages - 1 : stage - 1, ahead, next);
        ahead += step;
        next = counting(ahead);
        cp_async_wait<kStages - 1>();
        Piece k_piece[kBatch][U];
        bool counts[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            counts[i] = (bits >> i & 1u) != 0;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                k_piece[i][k] = slot(stage, 0, i, k);
            }
        }
        float s[R][kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            float2 dot[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                dot[r] = pair(0.0f);
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const Floats<V> f = widen(k_piece[i][k]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int j = 0; j < Floats<V>::kPairs; ++j) {
                        dot[r] = fma2(f.p[j], q[r][k].p[j], dot[r]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                s[r][i] = dot[r].x + dot[r].y;
            }
        }
        for (int o = lanes / 2; o > 0; o /= 2) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    s[r][i] += __shfl_xor_sync(0xffffffffu, s[r][i], o);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float now = m[r];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                s[r][i] = counts[i] ? s[r][i] : -INFINITY;
                now = fmaxf(now, s[r][i]);
            }
            const float base = now == -INFINITY ? 0.0f : now;
            const float keep = exp2_fast(m[r] - base);
            m[r] = now;
            sum[r] *= keep;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                s[r][i] = exp2_fast(s[r][i] - base);
                sum[r] += s[r][i];
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
#pragma unroll
                for (int j = 0; j < Floats<V>::kPairs; ++j) {
                    acc[r][k].p[j] = acc[r][k].p[j] * pair(keep);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const Floats<V> f = widen(slot(stage, 1, i, k));
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int j = 0; j < Floats<V>::kPairs; ++j) {
                        acc[r][k].p[j] = fma2(f.p[j], pair(s[r][i]), acc[r][k].p[j]);
                    }
                }
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    cp_async_wait_all();
    // The groups of a warp.
    for (int o = lanes; o < 32; o *= 2) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float other = __shfl_xor_sync(0xffffffffu, m[r], o);
            const float now = fmaxf(m[r], other);
            const float base = now == -INFINITY ? 0.0f : now;
            const float mine = exp2_fast(m[r] - base), theirs = exp2_fast(other - base);
            m[r] = now;
            sum[r] = sum[r] * mine + __shfl_xor_sync(0xffffffffu, sum[r], o) * theirs;
#pragma unroll
            for (int k = 0; k < U; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float v = acc[r][k].at(j);
                    acc[r][k].set(j, v * mine + __shfl_xor_sync(0xffffffffu, v, o) * theirs);
                }
            }
        }
    }
    if (group == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (sub == 0) {
                m_of[warp][r] = m[r];
                sum_of[warp][r] = sum[r];
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int d = (sub + k * lanes) * V + j;
                    if (d < c.dim) {
                        acc_of[warp][r][d] = acc[r][k].at(j);
                    }
                }
            }
        }
    }
    __syncthreads();
    // The warps of the CTA: a value a thread.
    for (int i = threadIdx.x; i < rows * c.dim; i += kThreads) {
        const int r = i / c.dim, d = i - r * c.dim;
        float now = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            now = fmaxf(now, m_of[w][r]);
        }
        const float base = now == -INFINITY ? 0.0f : now;
        float total = 0.0f, result = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2_fast(m_of[w][r] - base);
            total = fmaf(sum_of[w][r], f, total);
            result = fmaf(acc_of[w][r][d], f, result);
        }
        if (g.splits > 1) {
            const long long to = (static_cast<long long>(blockIdx.y) * c.pairs() + at) * rows + r;
            g.partial[to * c.dim + d] = result;
            if (d == 0) {
                g.stats[to] = make_float2(now, total);
            }
        } else {
            const float o = total == 0.0f ? 0.0f : result / total;
            const long long to = c.row_at(b, head, r) + d;
            static_cast<T*>(c.out)[to] = from_float<T>(o);
            if constexpr (sizeof(T) == 2) {
                if (c.rest != nullptr) {
                    c.rest[to] = static_cast<unsigned char>(rest_of<T>(make_float2(o, 0.0f)));
                }
            }
            if (c.stats != nullptr && d == 0) {
                c.stats[static_cast<long long>(at) * rows + r] = make_float2(base, total);
            }
        }
    }
}

// --- host ------------------------------------------------------------------------------------------------

// Values of a piece: 16 bytes where every row allows it, else two or one.
int piece_of(const Call& c)
{
    const int size = static_cast<int>(dtype_size(c.dtype));
    for (int v : {16 / size, 2}) {
        bool ok = c.dim % v == 0;
        const Strides* strides[2] = {&c.ks, &c.vs};
        const void* arrays[2] = {c.k, c.v};
        for (int i = 0; i < 2; ++i) {
            ok = ok && aligned_to(arrays[i], v * size) && strides[i]->sample % v == 0 && strides[i]->token % v == 0 && strides[i]->head % v == 0;
        }
        if (ok) {
            return v;
        }
    }
    return 1;
}

// Ranges of a key head's keys: one for each resident CTA (twice and four times as many were 3 and 9 % slower on the ragged
// case above), each with a few turns of its warps.
int splits_of(const Call& c)
{
    const long long most = std::max(1LL, (static_cast<long long>(c.keys) + 127) / 128);
    const long long wanted = (2LL * kSms + c.pairs() - 1) / c.pairs();
    return static_cast<int>(std::min({most, wanted, 256LL}));
}

template <class T, int V, int U>
void launch(const Few& g, cudaStream_t stream)
{
    const int rows = static_cast<int>(g.c.rows());
    const dim3 grid(static_cast<unsigned>(g.c.pairs()), g.splits);
    const auto run = [&](auto r) {
        constexpr int kSmem = kWarps * kStages * kStageBytes<T, V, U>;
        const auto kernel = few_kernel<T, V, U, decltype(r)::value>;
        static std::atomic<bool> ready[kMaxDevices];
        const int device = current_device();
        if (!ready[device].load(std::memory_order_relaxed)) {
            const auto* f = reinterpret_cast<const void*>(kernel);
            SPECTRAL_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
            SPECTRAL_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
            ready[device].store(true, std::memory_order_relaxed);
        }
        launch_pdl(kernel, grid, dim3(kThreads), kSmem, stream, g);
    };
    if (rows == 1) {
        run(std::integral_constant<int, 1>{});
    } else if (rows == 2) {
        run(std::integral_constant<int, 2>{});
    } else if (rows <= 4) {
        run(std::integral_constant<int, 4>{});
    } else {
        run(std::integral_constant<int, 8>{});
    }
}

std::size_t stats_at(const Call& c, int splits)
{
    Arena arena;
    arena.take(static_cast<std::size_t>(c.pairs()) * c.rows() * splits * c.dim * sizeof(float));
    return arena.size();
}

}  // namespace

bool few_rows(const Call& c) { return c.rows() <= 8 && c.keys > 0; }

std::size_t few_workspace(const Call& c)
{
    const int splits = splits_of(c);
    return splits == 1 ? 0 : stats_at(c, splits) + static_cast<std::size_t>(c.pairs()) * c.rows() * splits * sizeof(float2);
}

void few_forward(const Call& c, char* work, cudaStream_t stream)
{
    Few g;
    g.c = c;
    g.splits = splits_of(c);
    g.factor = c.scale * kLog2e;
    g.partial = reinterpret_cast<float*>(work);
    g.stats = reinterpret_cast<float2*>(work + stats_at(c, g.splits));
    const int v = piece_of(c);
    const int units = v == 1 ? 4 : v == 2 ? 2 : 1;
    while (g.lanes < 32 && g.lanes * v * units < c.dim) {
        g.lanes *= 2;
    }
    with_dtype(c.dtype, [&](auto t) {
        using T = decltype(t);
        if (v == 1) {
            launch<T, 1, 4>(g, stream);
        } else if (v == 2) {
            launch<T, 2, 2>(g, stream);
        } else {
            launch<T, 16 / sizeof(T), 1>(g, stream);
        }
    });
    if (g.splits > 1) {
        join_splits(c, g.partial, g.stats, g.splits, stream);
    }
}

}  // namespace spectral::attention
