// Attention for float32 on the tensor cores, forward and backward.
//
// Every operand is split into three bf16 parts (their sum is the value to 2^-24 of it), every product into the six
// that matter, the small ones first: FP32-level error. q, k, v and the upstream gradient are split by a kernel before
// (with zeros for keys that do not count); the weights and the score gradients are split by the threads that compute them,
// into three operands in tensor memory. The tensor core cuts its FP32 sum once per 16 terms, so no sum stays in one
// accumulator for longer than a tile: each tile's products start from zero and are added up in registers.
//
// Otherwise the kernels are those of the 16-bit types: forward, two row tiles a CTA that take turns between the
// tensor cores and the softmax, a thread per row; backward, one kernel that owns keys and one that owns rows.
//
// Measured: 2 samples, 8 heads, 2048 x 2048 keys, 64 values 129 us (the CUDA cores took 625), with gradients 573; 128 values
// 290 and 1308. The tensor pipe is busy 43 to 53 % of the time: a step's products and its threads wait for each other.

#include "attention_tc.cuh"

#include <algorithm>

namespace spectral::attention {
namespace {

constexpr int kSms = 148;
constexpr int kPlanes = 3;
constexpr int kProducts = 6;

// Three operands of a pair of values: 16-bit pairs as they lie in tensor memory.
__device__ __forceinline__ void split_pair(float2 v, uint32_t& hi, uint32_t& mid, uint32_t& lo)
{
    const auto wide = [](uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); };
    hi = pack2<bf16>(v);
    const float2 r = v - wide(hi);
    mid = pack2<bf16>(r);
    lo = pack2<bf16>(r - wide(mid));
}

__device__ __forceinline__ void store8(uint32_t taddr, const uint32_t (&v)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// 32 columns of a row into operands: parts 0 and 1 over the scores they came from, part 2 into `rest`.
__device__ __forceinline__ void store_parts(uint32_t scores, uint32_t rest, const float (&v)[32])
{
    uint32_t part[kPlanes][16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        split_pair(make_float2(v[2 * k], v[2 * k + 1]), part[0][k], part[1][k], part[2][k]);
    }
    store16(scores, part[0]);
    store16(scores + 16, part[1]);
    store16(rest, part[2]);
}

// The same of 16 columns.
__device__ __forceinline__ void store_parts(uint32_t scores, uint32_t rest, const float (&v)[16])
{
    uint32_t part[kPlanes][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        split_pair(make_float2(v[2 * k], v[2 * k + 1]), part[0][k], part[1][k], part[2][k]);
    }
    store8(scores, part[0]);
    store8(scores + 8, part[1]);
    store8(rest, part[2]);
}

// Where the operand's part p of the s-th 16 columns lies, if threads hold Columns of them.
template <int Columns>
__device__ __forceinline__ uint32_t part_at(uint32_t scores, uint32_t rest, int p, int s)
{
    return p == 2 ? rest + s * 8 : Columns == 32 ? scores + (s >> 1) * 32 + p * 16 + (s & 1) * 8 : scores + s * 16 + p * 8;
}

// --- forward -------------------------------------------------------------------------------------------

struct Forward {
    HeadMap q, k, v;
    Call c;
    int tokens_per_tile = 0;  // 128 / group
    unsigned row_items = 0;   // pairs of row tiles
    unsigned splits = 1;
    int split_tiles = 0;
    unsigned items = 0;
    float factor = 1.0f;
    float* partial = nullptr;
    float2* part_stats = nullptr;
    unsigned* fault = nullptr;
};

struct Item {
    int b;
    int head;
    int split;
    int row_tile;
    int tiles;
    int key0;
    int end;
    int slots;
};

// Heads of up to 64 values: two row tiles and 128 keys at a time. Wider ones: their parts fill the shared memory with one row
// tile and 64 keys.
template <int Boxes>
struct ForwardConfig {
    static constexpr int kSlots = Boxes == 1 ? 2 : 1;
    static constexpr int kKeys = Boxes == 1 ? 128 : 64;
    static constexpr int kWarps = 4 * kSlots;
    static constexpr int kThreads = 32 * (kWarps + 2);
    static constexpr int kPlaneBytes = Boxes * kBox;     // of 128 rows
    static constexpr int kTileBytes = kPlanes * kPlaneBytes;
    static constexpr int kKeyBox = kKeys * umma::kRowBytes;
    static constexpr int kKeyPlane = Boxes * kKeyBox;
    static constexpr int kKeyBytes = kPlanes * kKeyPlane;
    static constexpr int kSmem = kSlots * kTileBytes + 2 * kKeyBytes + 1024;  // Q, K, V
    // Tensor memory of a row tile: scores (parts 0 and 1 of the weights), part 2, O.
    static constexpr int kRest = kKeys;
    static constexpr int kO = kKeys + kKeys / 2;
    static constexpr int kSlotCols = 256;
    static_assert(kSmem <= kSmemMost - 1024 && kO + Boxes * 64 <= kSlotCols, "shared and tensor memory");
};

template <int Boxes>
__device__ __forceinline__ Item item_at(const Forward& g, unsigned i)
{
    using Cfg = ForwardConfig<Boxes>;
    Item it;
    const unsigned r = i / g.row_items;
    it.row_tile = static_cast<int>(i - r * g.row_items) * Cfg::kSlots;
    const unsigned pair = r / g.splits;
    it.split = static_cast<int>(r - pair * g.splits);
    it.b = static_cast<int>(pair / static_cast<unsigned>(g.c.kv_heads));
    it.head = static_cast<int>(pair) - it.b * g.c.kv_heads;
    it.key0 = it.split * g.split_tiles * Cfg::kKeys;
    const int length = length_of(g.c, it.b);
    const int span = g.split_tiles * Cfg::kKeys;
    it.end = length - it.key0 > span ? it.key0 + span : length;  // the last split's nominal end may pass 2^31
    it.tiles = it.end > it.key0 ? (it.end - it.key0 + Cfg::kKeys - 1) / Cfg::kKeys : 0;
    it.slots = Cfg::kSlots == 2 && (it.row_tile + 1) * g.tokens_per_tile < g.c.queries ? 2 : 1;
    return it;
}

template <int Boxes>
__global__ void __launch_bounds__(ForwardConfig<Boxes>::kThreads, 1) forward_kernel(const __grid_constant__ Forward g)
{
    using Cfg = ForwardConfig<Boxes>;
    constexpr int kWarps = Cfg::kWarps;
    constexpr int kKeys = Cfg::kKeys;
    extern __shared__ unsigned char smem_base[];
    const uint32_t base = (tma::smem_addr(smem_base) + 1023u) & ~1023u;
    const uint32_t kv = base + Cfg::kSlots * Cfg::kTileBytes;  // K, then V
    __shared__ uint64_t q_full, q_empty, full[2], empty[2], s_full[2], p_full[2], o_full[2], o_free[2], drain;
    __shared__ uint32_t tmem_slot;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == kWarps) {
        umma::alloc<512>(&tmem_slot);
    }
    if (threadIdx.x == 0) {
        tma::mbar_init(&q_full, 1);
        tma::mbar_init(&q_empty, 1);
        for (int x = 0; x < 2; ++x) {
            tma::mbar_init(&full[x], 1);
            tma::mbar_init(&empty[x], 1);
            tma::mbar_init(&s_full[x], 1);
            tma::mbar_init(&p_full[x], 4);
            tma::mbar_init(&o_full[x], 1);
            tma::mbar_init(&o_free[x], 4);
        }
        tma::mbar_init(&drain, 1);
        tma::fence_mbar_init();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    // The next grid may start from here: its CTAs cannot take this one's tensor memory any more.
    allow_next_grid();
    wait_for_previous_grid();
    const Call& c = g.c;
    bool ok = true;

    if (warp == kWarps) {
        // The TMA warp.
        asm volatile("fence.proxy.async.global;" ::: "memory");
        const unsigned q_bytes = static_cast<unsigned>(g.tokens_per_tile * c.group) * umma::kRowBytes * kPlanes * Boxes;
        unsigned issued[2] = {0, 0}, items = 0;  // K, V
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<Boxes>(g, i);
            if (it.tiles == 0) {
                continue;
            }
            ok = tma::mbar_wait(&q_empty, (items & 1u) ^ 1u);
            if (!ok) {
                break;
            }
            if (umma::elect_one()) {
                tma::mbar_arrive_expect_tx(&q_full, q_bytes * it.slots);
                for (int x = 0; x < it.slots; ++x) {
                    for (int p = 0; p < kPlanes; ++p) {
                        for (int j = 0; j < Boxes; ++j) {
                            load_heads(base + x * Cfg::kTileBytes + p * Cfg::kPlaneBytes + j * kBox, g.q, j * umma::kAtom, it.head * c.group,
                                       (it.row_tile + x) * g.tokens_per_tile, p * c.batch + it.b, &q_full);
                        }
                    }
                }
            }
            __syncwarp();
            ++items;
            for (int t = 0; ok && t < it.tiles; ++t) {
                for (int x = 0; x < 2; ++x) {
                    ok = ok && tma::mbar_wait(&empty[x], (issued[x] & 1u) ^ 1u);
                    if (!ok) {
                        break;
                    }
                    if (umma::elect_one()) {
                        tma::mbar_arrive_expect_tx(&full[x], Cfg::kKeyBytes);
                        for (int p = 0; p < kPlanes; ++p) {
                            for (int j = 0; j < Boxes; ++j) {
                                load_heads(kv + x * Cfg::kKeyBytes + p * Cfg::kKeyPlane + j * Cfg::kKeyBox, x == 0 ? g.k : g.v, j * umma::kAtom, it.head,
                                           it.key0 + t * kKeys, p * c.batch + it.b, &full[x]);
                            }
                        }
                    }
                    __syncwarp();
                    ++issued[x];
                }
            }
        }
        if (!ok) {  // the loads in flight land (bounded) before the shared memory is given up
            bool drained = items == 0 || tma::mbar_wait(&q_full, (items - 1) & 1u);
            for (int x = 0; x < 2; ++x) {
                drained = (issued[x] == 0 || tma::mbar_wait(&full[x], (issued[x] - 1) & 1u)) && drained;
            }
            if (lane == 0) {
                atomicOr(g.fault, drained ? tma::kFaultWaitTimeout : tma::kFaultWaitTimeout | tma::kFaultDrainTimeout);
            }
        }
    } else if (warp == kWarps + 1) {
        // The MMA warp, one elected lane issues.
        const int steps = (c.dim + 15) / 16;
        const uint32_t score = umma::instruction(true, false, false, kTile, kKeys);
        const uint32_t weigh = umma::instruction(true, false, true, kTile, steps * 16);
        unsigned used = 0, items = 0;
        unsigned p_phases[2] = {0, 0}, slot_items[2] = {0, 0};
        const auto scores = [&](int x) {
            if (umma::elect_one()) {
                for (int p = 0; p < kProducts; ++p) {
                    const uint64_t a = umma::desc_k(base + x * Cfg::kTileBytes + mlp::part_a<float>(p) * Cfg::kPlaneBytes);
                    const uint64_t b = umma::desc_k(kv + mlp::part_b<float>(p) * Cfg::kKeyPlane);
                    for (int s = 0; s < steps; ++s) {
                        const uint64_t step = (s & 3) * umma::kStepK;
                        umma::mma(tmem + x * Cfg::kSlotCols, a + step + (s >> 2) * (kBox >> 4), b + step + (s >> 2) * (Cfg::kKeyBox >> 4), score, p > 0 || s > 0);
                    }
                }
                umma::commit(&s_full[x]);
            }
            __syncwarp();
        };
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<Boxes>(g, i);
            if (it.tiles == 0) {
                continue;
            }
            ok = tma::mbar_wait(&q_full, items & 1u) && tma::mbar_wait(&full[0], used & 1u);
            if (!ok) {
                break;
            }
            ++items;
            umma::fence_after_sync();
            for (int x = 0; x < it.slots; ++x) {
                scores(x);
            }
            if (umma::elect_one()) {
                umma::commit(&empty[0]);
                if (it.tiles == 1) {
                    umma::commit(&q_empty);
                }
            }
            __syncwarp();
            for (int t = 0; ok && t < it.tiles; ++t) {
                const bool more = t + 1 < it.tiles;
                ok = tma::mbar_wait(&full[1], used & 1u) && (!more || tma::mbar_wait(&full[0], (used + 1) & 1u));
                ++used;
                for (int x = 0; ok && x < it.slots; ++x) {
                    ok = tma::mbar_wait(&p_full[x], p_phases[x]) && (t > 0 || tma::mbar_wait(&o_free[x], (slot_items[x] & 1u) ^ 1u));
                    if (!ok) {
                        break;
                    }
                    p_phases[x] ^= 1u;
                    umma::fence_after_sync();
                    if (umma::elect_one()) {
                        const uint32_t at = tmem + x * Cfg::kSlotCols;
                        for (int p = 0; p < kProducts; ++p) {
                            const uint64_t b = umma::desc_mn<Cfg::kKeyBox>(kv + Cfg::kKeyBytes + mlp::part_b<float>(p) * Cfg::kKeyPlane);
#pragma unroll
                            for (int s = 0; s < kKeys / 16; ++s) {
                                mma_tmem(at + Cfg::kO, part_at<32>(at, at + Cfg::kRest, mlp::part_a<float>(p), s), b + umma::kStepMn * s, weigh, p > 0 || s > 0);
                            }
                        }
                        if (!more) {
                            umma::commit(&o_full[x]);
                        }
                    }
                    __syncwarp();
                    if (more) {
                        scores(x);
                    }
                }
                if (!ok) {
                    break;
                }
                if (umma::elect_one()) {
                    umma::commit(&empty[1]);
                    if (more) {
                        umma::commit(&empty[0]);
                        if (t + 2 == it.tiles) {
                            umma::commit(&q_empty);
                        }
                    }
                }
                __syncwarp();
            }
            for (int x = 0; x < it.slots; ++x) {
                ++slot_items[x];
            }
        }
        if (!ok) {
            if (umma::elect_one()) {
                umma::commit(&drain);
            }
            __syncwarp();
            const bool drained = tma::mbar_wait(&drain, 0);
            if (lane == 0) {
                atomicOr(g.fault, drained ? tma::kFaultWaitTimeout : tma::kFaultWaitTimeout | tma::kFaultDrainTimeout);
            }
        }
    } else {
        // A thread per row: warps 0 to 3 the first tile's, 4 to 7 the second's.
        const int x = warp >> 2;
        const int quad = warp & 3;
        const uint32_t s_at = tmem + (static_cast<uint32_t>(quad * 32) << 16) + x * Cfg::kSlotCols;
        const int local = quad * 32 + lane;
        const int row_token = local / c.group;
        const int row_head = local - row_token * c.group;
        unsigned s_phase = 0, o_phase = 0;
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<Boxes>(g, i);
            if (x >= it.slots) {
                continue;
            }
            const int first_token = (it.row_tile + x) * g.tokens_per_tile;
            const int token = first_token + row_token;
            const int row = token * c.group + row_head;
            const bool live = row_token < g.tokens_per_tile && token < c.queries;
            const bool idle = quad * 32 >= min(g.tokens_per_tile, c.queries - first_token) * c.group;
            float m = -INFINITY, sum = 0.0f;
            MaskBytes<kKeys / 32> coming = mask_bytes<kKeys / 32>(c, it.b, it.end, it.key0);
            float o[2 * Boxes][32];
#pragma unroll
            for (int j = 0; j < 2 * Boxes; ++j) {
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    o[j][k] = 0.0f;
                }
            }
            // The products of the tile before, when they are done.
            const auto collect = [&](float keep) {
#pragma unroll
                for (int j = 0; j < 2 * Boxes; ++j) {
                    if (32 * j < c.dim) {
                        float v[32];
                        umma::load32(s_at + Cfg::kO + 32 * j, v);
                        umma::load_wait(v);
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            o[j][k] = (o[j][k] + v[k]) * keep;
                        }
                    }
                }
            };
            for (int t = 0; ok && t < it.tiles; ++t) {
                uint32_t w[4];
                tile_bits<kKeys / 32>(c, coming, it.end, it.key0 + t * kKeys, w);
                coming = mask_bytes<kKeys / 32>(c, it.b, it.end, it.key0 + (t + 1) * kKeys);
                ok = tma::mbar_wait(&s_full[x], s_phase);
                if (!ok) {
                    break;
                }
                s_phase ^= 1u;
                umma::fence_after_sync();
                if (!idle) {
                    const auto scores = [&](int j, float (&s)[32]) {
                        umma::load32(s_at + 32 * j, s);
                        umma::load_wait(s);
                        if (w[j] != 0xffffffffu) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                s[k] = (w[j] >> k & 1u) != 0 ? s[k] * g.factor : -INFINITY;
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                s[k] *= g.factor;
                            }
                        }
                    };
                    float now = m;
#pragma unroll
                    for (int j = 0; j < kKeys / 32; ++j) {
                        float s[32];
                        scores(j, s);
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            now = fmaxf(now, s[k]);
                        }
                    }
                    const float keep = m == -INFINITY ? 0.0f : exp2f(m - now);
                    m = now;
                    sum *= keep;
                    if (t > 0) {  // their commit came with these scores
                        collect(keep);
                    }
                    const float shift = m == -INFINITY ? 0.0f : m;
                    float2 total = pair(0.0f);
#pragma unroll
                    for (int j = 0; j < kKeys / 32; ++j) {
                        float s[32];
                        scores(j, s);
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            s[k] = exp2_fast(s[k] - shift);
                            s[k + 1] = exp2_fast(s[k + 1] - shift);
                            total = total + make_float2(s[k], s[k + 1]);
                        }
                        store_parts(s_at + 32 * j, s_at + Cfg::kRest + 16 * j, s);
                    }
                    sum += total.x + total.y;
                    store_wait();
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    umma::arrive(&p_full[x]);
                }
            }
            if (!ok) {
                break;
            }
            if (it.tiles > 0) {
                ok = tma::mbar_wait(&o_full[x], o_phase);
                if (!ok) {
                    break;
                }
                o_phase ^= 1u;
                umma::fence_after_sync();
                if (!idle) {
                    collect(1.0f);
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    umma::arrive(&o_free[x]);
                }
            }
            if (!idle) {
                const long long at = static_cast<long long>(it.b) * c.kv_heads + it.head;
                const float base_m = m == -INFINITY && g.splits == 1 ? 0.0f : m;
                const float factor = g.splits > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
                const bool sectors = whole_sectors(g.splits > 1 ? g.partial : c.out, c.dim, 4);
                const long long part_row = (it.split * c.pairs() + at) * c.rows() + row;
                float* to = g.splits > 1 ? g.partial + part_row * c.dim
                                         : static_cast<float*>(c.out)
                                               + ((static_cast<long long>(it.b) * c.queries + token) * c.kv_heads + it.head) * c.group * c.dim
                                               + row_head * c.dim;
#pragma unroll
                for (int j = 0; j < 2 * Boxes; ++j) {
                    if (32 * j < c.dim) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            o[j][k] *= factor;
                        }
                        store_lanes<float>(to + 32 * j, nullptr, live, o[j], min(32, c.dim - 32 * j), sectors);
                    }
                }
                if (live && g.splits > 1) {
                    g.part_stats[part_row] = make_float2(base_m, sum);
                } else if (live && c.stats != nullptr) {
                    c.stats[at * c.rows() + row] = make_float2(base_m, sum);
                }
            }
        }
        if (!ok && lane == 0) {
            atomicOr(g.fault, tma::kFaultWaitTimeout);
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (warp == kWarps) {
        umma::dealloc<512>(tmem);
    }
}

// --- backward ------------------------------------------------------------------------------------------

constexpr int kWidth = 64;  // entries of the walk at a time
constexpr int kConstants = 2 * kWidth;

// Heads of up to 64 values: the owned tiles stay in shared memory, a thread holds 32 columns. Wider ones: the parts of the owned
// tiles take turns in it, the first for S, the second for D of every step, read again from L2; a thread holds 16 columns,
// so that the results' 128 fit in the registers of sixteen warps.
template <int Boxes>
struct BackwardConfig {
    static constexpr int kColumns = Boxes == 1 ? 32 : 16;
    static constexpr int kParts = kWidth / kColumns;     // of a row
    static constexpr int kWarps = 4 * kParts;
    static constexpr int kThreads = 32 * (kWarps + 2);
    static constexpr int kOwnedPlane = Boxes * kBox;
    static constexpr int kOwnedBytes = kPlanes * kOwnedPlane;
    static constexpr int kOwned = Boxes == 1 ? 2 : 1;    // owned tiles that are there at a time
    static constexpr int kWalkedBox = kWidth * umma::kRowBytes;
    static constexpr int kWalkedPlane = Boxes * kWalkedBox;
    static constexpr int kWalkedBytes = kPlanes * kWalkedPlane;
    static constexpr int kStages = Boxes == 1 ? 2 : 1;
    static constexpr int kSmem = kOwned * kOwnedBytes + kStages * (2 * kWalkedBytes + kConstants * 4) + 1024;
    // Tensor memory: S (parts 0, 1 of P), part 2 of P, D (parts 0, 1 of dS), part 2 of dS, A0, A1.
    static constexpr int kSRest = 64, kD = 96, kDRest = 160, kA0 = 192, kA1 = 192 + Boxes * 64;
    static_assert(kSmem <= kSmemMost - 1024 && kA1 + Boxes * 64 <= 512, "shared and tensor memory");
};

struct Backward {
    HeadMap x0, x1, y0, y1;
    Call c;
    int owned_tokens = 0;
    int walked_tokens = 0;
    unsigned owned = 0;
    int walked = 0;
    int row_walks = 0;
    unsigned parts = 1;
    int part_tiles = 0;
    unsigned items = 0;
    float factor = 1.0f;
    const float* constants = nullptr;
    float* partial0 = nullptr;
    float* partial1 = nullptr;
    unsigned* fault = nullptr;
};

struct Walk {
    int b;
    int head;
    int part;
    int tile;
    int first;
    int tiles;
    int end;
};

template <bool Rows>
__device__ __forceinline__ Walk walk_at(const Backward& g, unsigned i)
{
    Walk it;
    const unsigned r = i / g.owned;
    it.tile = static_cast<int>(i - r * g.owned);
    const unsigned pair = r / g.parts;
    it.part = static_cast<int>(r - pair * g.parts);
    it.b = static_cast<int>(pair / static_cast<unsigned>(g.c.kv_heads));
    it.head = static_cast<int>(pair) - it.b * g.c.kv_heads;
    it.end = length_of(g.c, it.b);
    it.first = it.part * g.part_tiles;
    const int walked = Rows ? (it.end + kWidth - 1) / kWidth : it.tile * kTile < it.end ? g.walked : 0;
    it.tiles = max(0, min(g.part_tiles, walked - it.first));
    return it;
}

template <bool Rows, int Boxes>
__global__ void __launch_bounds__(BackwardConfig<Boxes>::kThreads, 1) backward_kernel(const __grid_constant__ Backward g)
{
    using Cfg = BackwardConfig<Boxes>;
    constexpr int kWarps = Cfg::kWarps;
    constexpr int kStages = Cfg::kStages;
    constexpr int kColumns = Cfg::kColumns;
    extern __shared__ unsigned char smem_base[];
    const uint32_t base = (tma::smem_addr(smem_base) + 1023u) & ~1023u;
    unsigned char* const generic = smem_base + (base - tma::smem_addr(smem_base));
    const uint32_t ring = base + Cfg::kOwned * Cfg::kOwnedBytes;
    float* const constants = reinterpret_cast<float*>(generic + Cfg::kOwned * Cfg::kOwnedBytes + kStages * 2 * Cfg::kWalkedBytes);
    __shared__ uint64_t x_full, x_empty, full[kStages], empty[kStages], s_full, d_full, p_ready, ds_ready, acc_full, acc_free, drain;
    __shared__ uint32_t tmem_slot;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == kWarps) {
        umma::alloc<512>(&tmem_slot);
    }
    if (threadIdx.x == 0) {
        tma::mbar_init(&x_full, 1);
        tma::mbar_init(&x_empty, 1);
        for (int s = 0; s < kStages; ++s) {
            tma::mbar_init(&full[s], 1);
            tma::mbar_init(&empty[s], 1);
        }
        tma::mbar_init(&s_full, 1);
        tma::mbar_init(&d_full, 1);
        tma::mbar_init(&p_ready, kWarps);
        tma::mbar_init(&ds_ready, kWarps);
        tma::mbar_init(&acc_full, 1);
        tma::mbar_init(&acc_free, kWarps);
        tma::mbar_init(&drain, 1);
        tma::fence_mbar_init();
    }
    if constexpr (!Rows) {
        // Rows of a tile that no box writes (64 % group) are reduced over: zeros, once.
        const int used = g.walked_tokens * g.c.group;
        const int spare = kWidth - used;
        for (int i = threadIdx.x; i < kStages * 2 * kPlanes * Boxes * spare * 8; i += Cfg::kThreads) {
            const int box = i / (spare * 8), at = i - box * spare * 8;
            *reinterpret_cast<uint4*>(generic + Cfg::kOwned * Cfg::kOwnedBytes + box * Cfg::kWalkedBox + (used + at / 8) * umma::kRowBytes + at % 8 * 16) =
                make_uint4(0, 0, 0, 0);
        }
        tma::fence_proxy_async();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    allow_next_grid();
    wait_for_previous_grid();
    const Call& c = g.c;
    bool ok = true;

    if (warp == kWarps) {
        // The TMA warp.
        asm volatile("fence.proxy.async.global;" ::: "memory");
        const unsigned token_bytes = static_cast<unsigned>(c.group) * umma::kRowBytes * kPlanes * Boxes;
        const unsigned owned_bytes = Rows ? g.owned_tokens * token_bytes : Cfg::kOwnedBytes;  // of one
        const unsigned walked_bytes = 2 * (Rows ? Cfg::kWalkedBytes : g.walked_tokens * token_bytes) + (Rows ? 0 : kConstants * 4);
        int stage = 0;
        unsigned phase = 0;
        long long issued = 0, x_issued = 0;  // steps, loads of owned tiles
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Walk it = walk_at<Rows>(g, i);
            if (it.tiles == 0) {
                continue;
            }
            const int x_head = Rows ? it.head * c.group : it.head;
            const int y_head = Rows ? it.head : it.head * c.group;
            const int x_token = it.tile * (Rows ? g.owned_tokens : kTile);
            // Both owned tiles (which < 0) or one, when the ones before are done with.
            const auto load_owned = [&](int which) {
                ok = tma::mbar_wait(&x_empty, (static_cast<unsigned>(x_issued) & 1u) ^ 1u);
                if (ok && umma::elect_one()) {
                    tma::mbar_arrive_expect_tx(&x_full, which < 0 ? 2 * owned_bytes : owned_bytes);
                    for (int k = 0; k < 2; ++k) {
                        if (which >= 0 && k != which) {
                            continue;
                        }
                        const uint32_t to = base + (which < 0 ? k * Cfg::kOwnedBytes : 0);
                        for (int p = 0; p < kPlanes; ++p) {
                            for (int j = 0; j < Boxes; ++j) {
                                load_heads(to + p * Cfg::kOwnedPlane + j * kBox, k == 0 ? g.x0 : g.x1, j * umma::kAtom, x_head, x_token, p * c.batch + it.b,
                                           &x_full);
                            }
                        }
                    }
                }
                __syncwarp();
                x_issued += ok ? 1 : 0;
            };
            if (Cfg::kOwned == 2) {
                load_owned(-1);
            }
            for (int t = it.first; ok && t < it.first + it.tiles; ++t) {
                if (Cfg::kOwned == 1) {
                    load_owned(0);
                }
                ok = ok && tma::mbar_wait(&empty[stage], phase ^ 1u);
                if (!ok) {
                    break;
                }
                if (umma::elect_one()) {
                    const uint32_t y = ring + stage * 2 * Cfg::kWalkedBytes;
                    const int token = t * (Rows ? kWidth : g.walked_tokens);
                    tma::mbar_arrive_expect_tx(&full[stage], walked_bytes);
                    for (int p = 0; p < kPlanes; ++p) {
                        for (int j = 0; j < Boxes; ++j) {
                            const uint32_t to = y + p * Cfg::kWalkedPlane + j * Cfg::kWalkedBox;
                            load_heads(to, g.y0, j * umma::kAtom, y_head, token, p * c.batch + it.b, &full[stage]);
                            load_heads(to + Cfg::kWalkedBytes, g.y1, j * umma::kAtom, y_head, token, p * c.batch + it.b, &full[stage]);
                        }
                    }
                    if constexpr (!Rows) {
                        const long long at = (static_cast<long long>(it.b) * c.kv_heads + it.head) * g.row_walks + t;
                        tma::bulk_g2s(constants + stage * kConstants, g.constants + row_constants_at(at, kWidth), kConstants * 4, &full[stage]);
                    }
                }
                __syncwarp();
                ++issued;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
                if (Cfg::kOwned == 1) {
                    load_owned(1);
                }
            }
        }
        if (!ok) {  // the loads in flight land (bounded) before the shared memory is given up
            bool drained = x_issued == 0 || tma::mbar_wait(&x_full, static_cast<unsigned>(x_issued - 1) & 1u);
            for (long long i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                drained = tma::mbar_wait(&full[i % kStages], static_cast<unsigned>(i / kStages) & 1u) && drained;
            }
            if (lane == 0) {
                atomicOr(g.fault, drained ? tma::kFaultWaitTimeout : tma::kFaultWaitTimeout | tma::kFaultDrainTimeout);
            }
        }
    } else if (warp == kWarps + 1) {
        // The MMA warp, one elected lane issues.
        const int steps = (c.dim + 15) / 16;
        const uint32_t score = umma::instruction(true, false, false, kTile, kWidth);
        const uint32_t weigh = umma::instruction(true, false, true, kTile, steps * 16);
        int stage = 0;
        unsigned phase = 0, x_phase = 0, step_phase = 0, acc_phase = 0;
        // S (k = 0) or D (k = 1) from the owned tiles and a stage's.
        const auto scores = [&](int k, int y_stage, uint64_t* done) {
            if (umma::elect_one()) {
                for (int p = 0; p < kProducts; ++p) {
                    const uint64_t a = umma::desc_k(base + (Cfg::kOwned == 2 ? k * Cfg::kOwnedBytes : 0) + mlp::part_a<float>(p) * Cfg::kOwnedPlane);
                    const uint64_t b = umma::desc_k(ring + (2 * y_stage + k) * Cfg::kWalkedBytes + mlp::part_b<float>(p) * Cfg::kWalkedPlane);
                    for (int s = 0; s < steps; ++s) {
                        const uint64_t step = (s & 3) * umma::kStepK;
                        umma::mma(tmem + k * Cfg::kD, a + step + (s >> 2) * (kBox >> 4), b + step + (s >> 2) * (Cfg::kWalkedBox >> 4), score, p > 0 || s > 0);
                    }
                }
                umma::commit(done);
            }
            __syncwarp();
        };
        // A0 = dS Y0 (k = 0), A1 = P Y1 (k = 1), of this tile alone.
        const auto weighed = [&](int k, int y_stage) {
            const uint32_t from = tmem + (k == 0 ? Cfg::kD : 0), rest = tmem + (k == 0 ? Cfg::kDRest : Cfg::kSRest);
            for (int p = 0; p < kProducts; ++p) {
                const uint64_t b = umma::desc_mn<Cfg::kWalkedBox>(ring + (2 * y_stage + k) * Cfg::kWalkedBytes + mlp::part_b<float>(p) * Cfg::kWalkedPlane);
#pragma unroll
                for (int s = 0; s < kWidth / 16; ++s) {
                    mma_tmem(tmem + (k == 0 ? Cfg::kA0 : Cfg::kA1), part_at<kColumns>(from, rest, mlp::part_a<float>(p), s), b + umma::kStepMn * s, weigh, p > 0 || s > 0);
                }
            }
        };
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Walk it = walk_at<Rows>(g, i);
            if (it.tiles == 0) {
                continue;
            }
            if constexpr (Cfg::kOwned == 1) {
                // The owned tiles take turns, so the steps follow each other.
                const auto turn = [&](int k, uint64_t* done) {
                    ok = tma::mbar_wait(&x_full, x_phase) && tma::mbar_wait(&full[stage], phase);
                    if (ok) {
                        x_phase ^= 1u;
                        umma::fence_after_sync();
                        scores(k, stage, done);
                        if (umma::elect_one()) {
                            umma::commit(&x_empty);
                        }
                        __syncwarp();
                    }
                };
                for (int t = 0; ok && t < it.tiles; ++t) {
                    turn(0, &s_full);
                    if (ok) {
                        turn(1, &d_full);
                    }
                    ok = ok && tma::mbar_wait(&p_ready, step_phase) && (t > 0 || tma::mbar_wait(&acc_free, acc_phase ^ 1u));
                    if (!ok) {
                        break;
                    }
                    umma::fence_after_sync();
                    if constexpr (!Rows) {
                        if (umma::elect_one()) {
                            weighed(1, stage);
                        }
                        __syncwarp();
                    }
                    ok = tma::mbar_wait(&ds_ready, step_phase);
                    if (!ok) {
                        break;
                    }
                    step_phase ^= 1u;
                    umma::fence_after_sync();
                    if (umma::elect_one()) {
                        weighed(0, stage);
                        umma::commit(&empty[stage]);
                        if (t + 1 == it.tiles) {
                            umma::commit(&acc_full);
                        }
                    }
                    __syncwarp();
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                acc_phase ^= 1u;
                continue;
            }
            ok = tma::mbar_wait(&x_full, x_phase) && tma::mbar_wait(&full[stage], phase);
            if (!ok) {
                break;
            }
            x_phase ^= 1u;
            umma::fence_after_sync();
            scores(0, stage, &s_full);
            scores(1, stage, &d_full);
            // After its last scores an item has no more use for the owned tiles.
            const auto release = [&](int t) {
                if (t + 1 == it.tiles && umma::elect_one()) {
                    umma::commit(&x_empty);
                }
                __syncwarp();
            };
            release(0);
            for (int t = 0; ok && t < it.tiles; ++t) {
                const bool more = t + 1 < it.tiles;
                const int now = stage;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
                ok = tma::mbar_wait(&p_ready, step_phase) && (t > 0 || tma::mbar_wait(&acc_free, acc_phase ^ 1u))
                     && (!more || tma::mbar_wait(&full[stage], phase));
                if (!ok) {
                    break;
                }
                umma::fence_after_sync();
                if constexpr (!Rows) {
                    if (umma::elect_one()) {
                        weighed(1, now);
                    }
                    __syncwarp();
                }
                if (more) {
                    scores(0, stage, &s_full);
                }
                ok = tma::mbar_wait(&ds_ready, step_phase);
                if (!ok) {
                    break;
                }
                step_phase ^= 1u;
                umma::fence_after_sync();
                if (umma::elect_one()) {
                    weighed(0, now);
                    umma::commit(&empty[now]);
                    if (!more) {
                        umma::commit(&acc_full);
                    }
                }
                __syncwarp();
                if (more) {
                    scores(1, stage, &d_full);
                    release(t + 1);
                }
            }
            acc_phase ^= 1u;
        }
        if (!ok) {
            if (umma::elect_one()) {
                umma::commit(&drain);
            }
            __syncwarp();
            const bool drained = tma::mbar_wait(&drain, 0);
            if (lane == 0) {
                atomicOr(g.fault, drained ? tma::kFaultWaitTimeout : tma::kFaultWaitTimeout | tma::kFaultDrainTimeout);
            }
        }
    } else {
        // A thread per owned row and kColumns columns of scores, and 32 of the results: warps 4 k to 4 k + 3 the k-th.
        const int part = warp >> 2;
        const int local = (warp & 3) * 32 + lane;
        const uint32_t at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int row_token = local / c.group;
        const int row_head = local - row_token * c.group;
        const bool holds = part * 32 < c.dim;
        int stage = 0;
        unsigned phase = 0, step_phase = 0, acc_phase = 0;
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Walk it = walk_at<Rows>(g, i);
            const long long pair_at = static_cast<long long>(it.b) * c.kv_heads + it.head;
            // Rows: this row's -lse and -delta. Keys: whether this key counts.
            float2 shift = pair(0.0f), delta = pair(0.0f);
            bool counts = true;
            const int token = it.tile * g.owned_tokens + row_token;
            const int row = Rows ? token * c.group + row_head : it.tile * kTile + local;
            const bool live = Rows ? row_token < g.owned_tokens && token < c.queries : row < c.keys;
            if constexpr (Rows) {
                if (live) {
                    const int tile = token / g.walked_tokens;
                    const float* from = g.constants + row_constants_at(pair_at * g.row_walks + tile, kWidth) + (token - tile * g.walked_tokens) * c.group + row_head;
                    shift = pair(from[0]);
                    delta = pair(from[kWidth]);
                }
            } else {
                counts = row < it.end && (c.mask == nullptr || c.mask[static_cast<long long>(it.b) * c.keys + row] != 0);
            }
            float a0[32], a1[Rows ? 1 : 32];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                a0[k] = 0.0f;
                if constexpr (!Rows) {
                    a1[k] = 0.0f;
                }
            }
            const auto collect = [&](int column, auto& sum) {
                if (holds) {
                    float v[32];
                    umma::load32(at + column + 32 * part, v);
                    umma::load_wait(v);
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        sum[k] += v[k];
                    }
                }
            };
            MaskBytes<2> mask{};
            if constexpr (Rows) {
                mask = mask_bytes<2>(c, it.b, it.end, it.first * kWidth);
            }
            for (int t = it.first; ok && t < it.first + it.tiles; ++t) {
                uint32_t w[4] = {0, 0, 0, 0};
                if constexpr (Rows) {
                    tile_bits<2>(c, mask, it.end, t * kWidth, w);
                    mask = mask_bytes<2>(c, it.b, it.end, (t + 1) * kWidth);
                }
                constexpr uint32_t kAll = kColumns == 32 ? 0xffffffffu : (1u << (kColumns % 32)) - 1u;
                const uint32_t word = (Rows ? w[part * kColumns / 32] >> (part * kColumns % 32) : counts ? 0xffffffffu : 0u) & kAll;
                ok = tma::mbar_wait(&full[stage], phase) && tma::mbar_wait(&s_full, step_phase);
                if (!ok) {
                    break;
                }
                umma::fence_after_sync();
                const float* less = constants + stage * kConstants + part * kColumns;  // -lse, then -delta
                if constexpr (!Rows) {
                    if (t > it.first) {  // its commit came before these scores'
                        collect(Cfg::kA1, a1);
                    }
                }
                float p[kColumns];
                umma::load_run(at + part * kColumns, p);
                umma::load_wait(p);
#pragma unroll
                for (int k = 0; k < kColumns; k += 2) {
                    const float2 l = Rows ? shift : *reinterpret_cast<const float2*>(less + k);
                    const float2 e = fma2(make_float2(p[k], p[k + 1]), pair(g.factor), l);
                    p[k] = exp2_fast(e.x);
                    p[k + 1] = exp2_fast(e.y);
                }
                if (word != kAll) {
#pragma unroll
                    for (int k = 0; k < kColumns; ++k) {
                        p[k] = (word >> k & 1u) != 0 ? p[k] : 0.0f;
                    }
                }
                if constexpr (!Rows) {
                    store_parts(at + part * kColumns, at + Cfg::kSRest + part * (kColumns / 2), p);
                    store_wait();
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    umma::arrive(&p_ready);
                }
                ok = tma::mbar_wait(&d_full, step_phase);
                if (!ok) {
                    break;
                }
                step_phase ^= 1u;
                umma::fence_after_sync();
                if (t > it.first) {
                    collect(Cfg::kA0, a0);
                }
                float d[kColumns];
                umma::load_run(at + Cfg::kD + part * kColumns, d);
                umma::load_wait(d);
#pragma unroll
                for (int k = 0; k < kColumns; k += 2) {
                    const float2 l = Rows ? delta : *reinterpret_cast<const float2*>(less + kWidth + k);
                    const float2 v = (make_float2(d[k], d[k + 1]) + l) * make_float2(p[k], p[k + 1]);
                    d[k] = v.x;
                    d[k + 1] = v.y;
                }
                if (word != kAll) {  // a key that does not count may have made D anything
#pragma unroll
                    for (int k = 0; k < kColumns; ++k) {
                        d[k] = (word >> k & 1u) != 0 ? d[k] : 0.0f;
                    }
                }
                store_parts(at + Cfg::kD + part * kColumns, at + Cfg::kDRest + part * (kColumns / 2), d);
                store_wait();
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    umma::arrive(&ds_ready);
                }
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) {
                break;
            }
            if (it.tiles > 0) {
                ok = tma::mbar_wait(&acc_full, acc_phase);
                if (!ok) {
                    break;
                }
                acc_phase ^= 1u;
                umma::fence_after_sync();
                collect(Cfg::kA0, a0);
                if constexpr (!Rows) {
                    collect(Cfg::kA1, a1);
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    umma::arrive(&acc_free);
                }
            }
            if (holds) {
                const long long part_row = (it.part * c.pairs() + pair_at) * (Rows ? c.rows() : c.keys) + row;
                const long long to = (g.parts > 1 ? part_row * c.dim
                                      : Rows
                                          ? ((static_cast<long long>(it.b) * c.queries + token) * c.kv_heads + it.head) * c.group * c.dim + row_head * c.dim
                                          : ((static_cast<long long>(it.b) * c.keys + row) * c.kv_heads + it.head) * c.dim)
                                     + part * 32;
                const int valid = min(32, c.dim - part * 32);
                const float scale = g.parts > 1 ? 1.0f : c.scale;
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    a0[k] = counts ? a0[k] * scale : 0.0f;
                }
                float* result = g.parts > 1 ? g.partial0 : static_cast<float*>(Rows ? c.dq : c.dk);
                store_lanes<float>(result + to, nullptr, live, a0, valid, whole_sectors(result, c.dim, 4));
                if constexpr (!Rows) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        a1[k] = counts ? a1[k] : 0.0f;
                    }
                    result = g.parts > 1 ? g.partial1 : static_cast<float*>(c.dv);
                    store_lanes<float>(result + to, nullptr, live, a1, valid, whole_sectors(result, c.dim, 4));
                }
            }
        }
        if (!ok && lane == 0) {
            atomicOr(g.fault, tma::kFaultWaitTimeout);
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (warp == kWarps) {
        umma::dealloc<512>(tmem);
    }
}

// --- splitting the operands ----------------------------------------------------------------------------

struct SplitJob {
    const float* source;
    bf16* target;
    Strides stride;
    long long tokens;
    int heads;
    bool keys;  // zeros for keys that do not count
    bool vectors;
    long long rows;
};
struct SplitJobs {
    SplitJob job[4];
    Call c;
    int pitch;  // a multiple of 8
    int lanes;  // of 8 values each, a power of two
};

// A head takes `lanes` lanes of eight values.
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ SplitJobs g)
{
    allow_next_grid();
    wait_for_previous_grid();
    const SplitJob& j = g.job[blockIdx.y];
    const Call& c = g.c;
    const int per_cta = 256 / g.lanes;
    const int d = (threadIdx.x % g.lanes) * 8;
    const unsigned heads = j.heads, tokens = static_cast<unsigned>(j.tokens);
    for (long long row = static_cast<long long>(blockIdx.x) * per_cta + threadIdx.x / g.lanes; row < j.rows;
         row += static_cast<long long>(gridDim.x) * per_cta) {
        long long token, b;
        if (j.rows < (1LL << 31)) {
            token = static_cast<unsigned>(row) / heads;
            b = static_cast<unsigned>(token) / tokens;
        } else {
            token = row / heads;
            b = token / tokens;
        }
        const long long in = token - b * tokens;
        const bool counts = !j.keys || (in < length_of(c, static_cast<int>(b)) && (c.mask == nullptr || c.mask[b * c.keys + in] != 0));
        if (d >= g.pitch) {
            continue;
        }
        const float* from = j.source + b * j.stride.sample + in * j.stride.token + (row - token * heads) * j.stride.head + d;
        float v[8];
        if (j.vectors && d + 8 <= c.dim) {
            const float4 a = counts ? *reinterpret_cast<const float4*>(from) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float4 e = counts ? *reinterpret_cast<const float4*>(from + 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = e.x, v[5] = e.y, v[6] = e.z, v[7] = e.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = counts && d + k < c.dim ? from[k] : 0.0f;
            }
        }
        Vec<bf16, 8> part[kPlanes];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            mlp::split3(v[k], part[0].v[k], part[1].v[k], part[2].v[k]);
            // An infinity (or NaN) as the last part: that one meets the other side's first part alone, so a product is what it is of the
            // whole values. As the first it would meet parts of either sign and zeros, and be NaN.
            if (!(fabsf(v[k]) <= 3.4028234663852886e38f)) {
                part[2].v[k] = part[0].v[k];
                part[0].v[k] = from_float<bf16>(0.0f);
            }
        }
#pragma unroll
        for (int p = 0; p < kPlanes; ++p) {
            *reinterpret_cast<Vec<bf16, 8>*>(j.target + (p * j.rows + row) * g.pitch + d) = part[p];
        }
    }
}

// --- host ------------------------------------------------------------------------------------------------

struct Planes {
    std::size_t at = 0;
    long long tokens = 0;
    int heads = 0;
};

int pitch_of(int dim) { return (dim + 7) / 8 * 8; }

Planes planes(Arena& arena, const Call& c, long long tokens, int heads)
{
    Planes p;
    p.tokens = tokens;
    p.heads = heads;
    p.at = arena.take(static_cast<std::size_t>(kPlanes) * c.batch * tokens * heads * pitch_of(c.dim) * 2);
    return p;
}

HeadMap plane_map(const Call& c, const Planes& p, char* work, int box_heads, int box_tokens)
{
    const long long pitch = pitch_of(c.dim);
    const Strides s{p.tokens * p.heads * pitch, p.heads * pitch, pitch};
    return head_map(work + p.at, true, s, static_cast<long long>(kPlanes) * c.batch, p.tokens, p.heads, c.dim, box_heads, box_tokens);
}

struct Source {
    const void* base;
    Strides stride;
    const Planes* planes;
    bool keys;
};

void split_all(const Call& c, const Source* sources, int count, char* work, cudaStream_t stream)
{
    SplitJobs g;
    g.c = c;
    g.pitch = pitch_of(c.dim);
    g.lanes = 1;
    while (g.lanes * 8 < g.pitch) {
        g.lanes *= 2;
    }
    long long most = 0;
    int jobs = 0;
    for (int i = 0; i < count; ++i) {
        const Source& s = sources[i];
        const long long rows = c.batch * s.planes->tokens * s.planes->heads;
        if (rows == 0) {
            continue;
        }
        const bool vectors = aligned_to(s.base, 16) && s.stride.sample % 4 == 0 && s.stride.token % 4 == 0 && s.stride.head % 4 == 0;
        g.job[jobs++] = {static_cast<const float*>(s.base), reinterpret_cast<bf16*>(work + s.planes->at), s.stride, s.planes->tokens,
                         s.planes->heads, s.keys, vectors, rows};
        most = std::max(most, rows);
    }
    const long long per_cta = 256 / g.lanes;
    const auto grid = static_cast<unsigned>(std::min<long long>((most + per_cta - 1) / per_cta, kSms * 8));
    launch_pdl(split_kernel, dim3(grid, jobs), dim3(256), 0, stream, g);
}

// How many parts an axis of `walked` tiles is cut into for `owned` items of one part each: the fewest turns of the busiest
// CTA, counted in tiles, of which an item costs about `extra` more.
void cut(long long owned, int walked, double extra, int& parts, int& part_tiles)
{
    double best = 0.0;
    parts = 1;
    part_tiles = std::max(1, walked);
    for (int s = 1; s <= std::min(walked, 64); ++s) {
        const int span = (walked + s - 1) / s;
        if ((walked + span - 1) / span != s) {
            continue;
        }
        const double turns = static_cast<double>((owned * s + kSms - 1) / kSms) * (span + extra) + (s > 1 ? 3.0 + 0.1 * s : 0.0);
        if (s == 1 || turns < best) {
            best = turns;
            parts = s;
            part_tiles = span;
        }
    }
}

unsigned item_count(long long items)
{
    if (items >= (1LL << 31)) {
        throw InvalidArgument("cross_attention: too many tiles for one call");
    }
    return static_cast<unsigned>(items);
}

template <class K, class G>
void launch(K kernel, const G& g, int threads, int smem, cudaStream_t stream)
{
    SPECTRAL_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const unsigned grid = std::min(g.items, static_cast<unsigned>(device_sm_count(current_device())));
    launch_pdl(kernel, dim3(grid), dim3(threads), smem, stream, g);
}

int forward_keys(const Call& c) { return c.dim <= 64 ? ForwardConfig<1>::kKeys : ForwardConfig<2>::kKeys; }

struct ForwardPlan {
    Planes q, k, v;
    int row_items = 0, splits = 1, split_tiles = 0;
    std::size_t partial = 0, stats = 0;
    Arena arena;

    explicit ForwardPlan(const Call& c)
    {
        q = planes(arena, c, c.queries, c.kv_heads * c.group);
        k = planes(arena, c, c.keys, c.kv_heads);
        v = planes(arena, c, c.keys, c.kv_heads);
        const int slots = c.dim <= 64 ? ForwardConfig<1>::kSlots : ForwardConfig<2>::kSlots;
        row_items = pieces(pieces(c.queries, kTile / c.group), slots);
        cut(c.pairs() * row_items, pieces(c.keys, forward_keys(c)), 2.0, splits, split_tiles);
        if (splits > 1) {
            const std::size_t all = static_cast<std::size_t>(c.pairs()) * c.rows() * splits;
            partial = arena.take(all * c.dim * sizeof(float));
            stats = arena.take(all * sizeof(float2));
        }
    }
};

struct BackwardPlan {
    Planes q, k, v, dout;
    int owned_tokens = 0, walked_tokens = 0;
    int row_tiles = 0, key_tiles = 0, row_walks = 0, key_walks = 0;
    int row_parts = 1, row_span = 0, key_parts = 1, key_span = 0;
    std::size_t constants = 0, dq = 0, dk = 0, dv = 0;
    Arena arena;

    explicit BackwardPlan(const Call& c)
    {
        const int heads = c.kv_heads * c.group;
        q = planes(arena, c, c.queries, heads);
        k = planes(arena, c, c.keys, c.kv_heads);
        v = planes(arena, c, c.keys, c.kv_heads);
        dout = planes(arena, c, c.queries, heads);
        owned_tokens = kTile / c.group;
        walked_tokens = kWidth / c.group;
        row_tiles = pieces(c.queries, owned_tokens);
        key_tiles = pieces(c.keys, kTile);
        row_walks = pieces(c.queries, walked_tokens);
        key_walks = pieces(c.keys, kWidth);
        cut(c.pairs() * key_tiles, row_walks, 2.0, row_parts, row_span);
        cut(c.pairs() * row_tiles, key_walks, 2.0, key_parts, key_span);
        constants = arena.take(static_cast<std::size_t>(c.pairs()) * row_walks * kConstants * sizeof(float));
        if (key_parts > 1) {
            dq = arena.take(static_cast<std::size_t>(c.pairs()) * c.rows() * c.dim * key_parts * sizeof(float));
        }
        if (row_parts > 1) {
            dk = arena.take(static_cast<std::size_t>(c.pairs()) * c.keys * c.dim * row_parts * sizeof(float));
            dv = arena.take(static_cast<std::size_t>(c.pairs()) * c.keys * c.dim * row_parts * sizeof(float));
        }
    }
};

}  // namespace

std::size_t split_forward_workspace(const Call& c) { return ForwardPlan(c).arena.size(); }
std::size_t split_backward_workspace(const Call& c) { return BackwardPlan(c).arena.size(); }

void split_forward(const Call& c, char* work, cudaStream_t stream)
{
    const ForwardPlan plan(c);
    const Source sources[3] = {{c.q, c.qs, &plan.q, false}, {c.k, c.ks, &plan.k, true}, {c.v, c.vs, &plan.v, true}};
    split_all(c, sources, 3, work, stream);
    Forward g;
    g.c = c;
    g.tokens_per_tile = kTile / c.group;
    g.row_items = plan.row_items;
    g.splits = plan.splits;
    g.split_tiles = plan.split_tiles;
    g.items = item_count(c.pairs() * plan.row_items * plan.splits);
    g.factor = c.scale * kLog2e;
    g.partial = reinterpret_cast<float*>(work + plan.partial);
    g.part_stats = reinterpret_cast<float2*>(work + plan.stats);
    g.fault = device_fault_word();
    g.q = plane_map(c, plan.q, work, c.group, g.tokens_per_tile);
    g.k = plane_map(c, plan.k, work, 1, forward_keys(c));
    g.v = plane_map(c, plan.v, work, 1, forward_keys(c));
    if (c.dim <= 64) {
        launch(forward_kernel<1>, g, ForwardConfig<1>::kThreads, ForwardConfig<1>::kSmem, stream);
    } else {
        launch(forward_kernel<2>, g, ForwardConfig<2>::kThreads, ForwardConfig<2>::kSmem, stream);
    }
    if (plan.splits > 1) {
        join_splits(c, g.partial, g.part_stats, plan.splits, stream);
    }
}

void split_backward(const Call& c, char* work, cudaStream_t stream)
{
    const BackwardPlan plan(c);
    const int heads = c.kv_heads * c.group;
    const Strides dense{static_cast<long long>(c.queries) * heads * c.dim, static_cast<long long>(heads) * c.dim, c.dim};
    const Source sources[4] = {{c.q, c.qs, &plan.q, false}, {c.k, c.ks, &plan.k, true}, {c.v, c.vs, &plan.v, true}, {c.dout, dense, &plan.dout, false}};
    split_all(c, sources, 4, work, stream);
    Backward g;
    g.c = c;
    g.owned_tokens = plan.owned_tokens;
    g.walked_tokens = plan.walked_tokens;
    g.walked = plan.row_walks;
    g.row_walks = plan.row_walks;
    g.factor = c.scale * kLog2e;
    auto* constants = reinterpret_cast<float*>(work + plan.constants);
    g.constants = constants;
    g.fault = device_fault_word();
    row_constants(c, constants, kWidth, plan.walked_tokens, plan.row_walks, stream);
    // dk and dv.
    g.x0 = plane_map(c, plan.k, work, 1, kTile);
    g.x1 = plane_map(c, plan.v, work, 1, kTile);
    g.y0 = plane_map(c, plan.q, work, c.group, plan.walked_tokens);
    g.y1 = plane_map(c, plan.dout, work, c.group, plan.walked_tokens);
    g.owned = plan.key_tiles;
    g.parts = plan.row_parts;
    g.part_tiles = plan.row_span;
    g.items = item_count(c.pairs() * plan.key_tiles * plan.row_parts);
    g.partial0 = reinterpret_cast<float*>(work + plan.dk);
    g.partial1 = reinterpret_cast<float*>(work + plan.dv);
    if (c.dim <= 64) {
        launch(backward_kernel<false, 1>, g, BackwardConfig<1>::kThreads, BackwardConfig<1>::kSmem, stream);
    } else {
        launch(backward_kernel<false, 2>, g, BackwardConfig<2>::kThreads, BackwardConfig<2>::kSmem, stream);
    }
    // dq.
    g.x0 = plane_map(c, plan.q, work, c.group, plan.owned_tokens);
    g.x1 = plane_map(c, plan.dout, work, c.group, plan.owned_tokens);
    g.y0 = plane_map(c, plan.k, work, 1, kWidth);
    g.y1 = plane_map(c, plan.v, work, 1, kWidth);
    g.owned = plan.row_tiles;
    g.parts = plan.key_parts;
    g.part_tiles = plan.key_span;
    g.items = item_count(c.pairs() * plan.row_tiles * plan.key_parts);
    g.partial0 = reinterpret_cast<float*>(work + plan.dq);
    if (c.dim <= 64) {
        launch(backward_kernel<true, 1>, g, BackwardConfig<1>::kThreads, BackwardConfig<1>::kSmem, stream);
    } else {
        launch(backward_kernel<true, 2>, g, BackwardConfig<2>::kThreads, BackwardConfig<2>::kSmem, stream);
    }
    Sums sums;
    if (plan.row_parts > 1) {
        sums.add(reinterpret_cast<const float*>(work + plan.dk), plan.row_parts, true, c.dk, c.scale);
        sums.add(reinterpret_cast<const float*>(work + plan.dv), plan.row_parts, true, c.dv, 1.0f);
    }
    if (plan.key_parts > 1) {
        sums.add(reinterpret_cast<const float*>(work + plan.dq), plan.key_parts, false, c.dq, c.scale);
    }
    add_parts(c, sums, stream);
}

}  // namespace spectral::attention
