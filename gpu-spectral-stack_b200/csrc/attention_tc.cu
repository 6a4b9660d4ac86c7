// Attention forward for 16-bit values on the 5th-generation tensor cores.
//
// A CTA keeps two or four tiles of 128 query rows and walks over tiles of 128 or 64 keys. Both products run on tcgen05: the
// scores S = Q K^T into tensor memory, from where a thread per row takes them to registers, and
// O += P V with the weights P written back over S as the 16-bit operand. While one row tile's threads work on
// their scores the tensor cores multiply for the others. A warp brings tiles of K and V in by TMA through a ring, a
// warp issues the products.
//
// Softmax in one pass: a row's weights are 2^(c s - m) with m the largest c s when it was last moved, and m moves only
// if a later score passes it by more than 2^8; then O in tensor memory and the sum are scaled. Weights reach 2^8 that way,
// which changes nothing in bf16; float16 has them times 2^7, so that the smallest it keeps is 2^-31 of the largest.
//
// Work items are (row tiles, split of the keys, sample and key head); CTAs, one per SM, stay and take every
// 148th. Few rows over many keys are split so that all SMs read, and the parts joined by a second kernel.
//
// Measured in bf16: 64 x 16384 x 256 keys, 2 heads of 32, 297 us (XU 39 %, issue 39 %: the softmax bounds it); 4 x 4096 x 4096, 16
// and 4 heads of 128, 597 us, 922 TFLOP/s (tensor pipe 44 %).

#include "attention_tc.cuh"

#include <algorithm>

namespace spectral::attention {
namespace {

constexpr float kSlack = 8.0f;  // in powers of two, see above

struct Forward {
    HeadMap q, k, v;
    Call c;
    int tokens_per_tile = 0;  // 128 / group
    unsigned row_items = 0;   // groups of Config::kSlots row tiles
    unsigned splits = 1;
    int split_tiles = 0;      // key tiles of a split
    unsigned items = 0;
    float factor = 1.0f;      // |scale| log2(e)
    bool negative = false;    // scale < 0
    float* partial = nullptr;
    float2* part_stats = nullptr;
    unsigned* fault = nullptr;
};

struct Item {
    int b;
    int head;
    int split;
    int row_tile;   // the first
    int tiles;      // of keys
    int key0;
    int end;        // keys before this count, but for the mask
    int slots;      // row tiles with rows
};

template <int Slots, int Keys>
__device__ __forceinline__ Item item_at(const Forward& g, unsigned i)
{
    Item it;
    const unsigned r = i / g.row_items;
    it.row_tile = static_cast<int>(i - r * g.row_items) * Slots;
    const unsigned pair = r / g.splits;
    it.split = static_cast<int>(r - pair * g.splits);
    it.b = static_cast<int>(pair / static_cast<unsigned>(g.c.kv_heads));
    it.head = static_cast<int>(pair) - it.b * g.c.kv_heads;
    it.key0 = it.split * g.split_tiles * Keys;
    const int length = length_of(g.c, it.b);
    const int span = g.split_tiles * Keys;
    it.end = length - it.key0 > span ? it.key0 + span : length;  // the last split's nominal end may pass 2^31
    it.tiles = it.end > it.key0 ? (it.end - it.key0 + Keys - 1) / Keys : 0;
    it.slots = min(Slots, (g.c.queries - it.row_tile * g.tokens_per_tile + g.tokens_per_tile - 1) / g.tokens_per_tile);
    return it;
}

// Heads of up to 64 values: four row tiles and 64 keys at a time, wider ones two and 128. Either way tensor memory is full; the
// more warps, the better they fill each other's waits (128 keys and two tiles for all: 64 x 2 x 16384 x 256 x 32 took
// 400 us, this takes 297).
template <int Boxes>
struct Config {
    static constexpr int kSlots = Boxes == 1 ? 4 : 2;
    static constexpr int kKeys = Boxes == 1 ? 64 : 128;
    static constexpr int kWarps = 4 * kSlots;            // of the softmax
    static constexpr int kThreads = 32 * (kWarps + 2);
    static constexpr int kQBytes = Boxes * kBox;
    static constexpr int kKeyBox = kKeys * umma::kRowBytes;
    static constexpr int kTileBytes = Boxes * kKeyBox;
    static constexpr int kStages = Boxes == 1 ? 8 : 5;   // of K and V tiles
    static constexpr int kQueries = Boxes == 1 ? 2 : 1;  // items whose queries are kept
    static constexpr int kSmem = kSlots * kQueries * kQBytes + kStages * kTileBytes + 1024;
    static constexpr int kO = kSlots * kKeys;            // tensor memory: S and P of each row tile, then O of each
    static constexpr int kCols = 512;
    static_assert(kSmem <= kSmemMost - 1024, "shared memory");
    static_assert(kO + kSlots * Boxes * 64 <= kCols, "tensor memory");
};

template <class T, int Boxes>
__global__ void __launch_bounds__(Config<Boxes>::kThreads, 1) forward_kernel(const __grid_constant__ Forward g)
{
    using Cfg = Config<Boxes>;
    constexpr bool kBf16 = std::is_same_v<T, bf16>;
    constexpr float kOffset = kBf16 ? 0.0f : 7.0f;  // weights times 2^7
    constexpr int kStages = Cfg::kStages;
    constexpr int kSlots = Cfg::kSlots;
    constexpr int kKeys = Cfg::kKeys;
    constexpr int kWarps = Cfg::kWarps;
    extern __shared__ unsigned char smem_base[];
    const uint32_t base = (tma::smem_addr(smem_base) + 1023u) & ~1023u;
    const uint32_t ring = base + kSlots * Cfg::kQueries * Cfg::kQBytes;
    __shared__ uint64_t q_full[2], q_empty[2], full[kStages], empty[kStages], s_full[kSlots], p_full[kSlots], o_full[kSlots], o_free[kSlots], drain;
    __shared__ uint32_t tmem_slot;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == kWarps) {
        umma::alloc<Cfg::kCols>(&tmem_slot);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            tma::mbar_init(&full[s], 1);
            tma::mbar_init(&empty[s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            tma::mbar_init(&q_full[x], 1);
            tma::mbar_init(&q_empty[x], 1);
        }
        for (int x = 0; x < kSlots; ++x) {
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
        // The TMA warp: Q of an item as soon as the one before is read, then its K and V tiles in turn.
        asm volatile("fence.proxy.async.global;" ::: "memory");
        const unsigned q_bytes = static_cast<unsigned>(g.tokens_per_tile * c.group) * umma::kRowBytes * Boxes;
        int stage = 0;
        unsigned phase = 0;
        long long issued = 0, q_issued = 0;
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<kSlots, kKeys>(g, i);
            if (it.tiles == 0) {
                continue;
            }
            const int kept = static_cast<int>(q_issued % Cfg::kQueries);
            ok = tma::mbar_wait(&q_empty[kept], (static_cast<unsigned>(q_issued / Cfg::kQueries) & 1u) ^ 1u);
            if (!ok) {
                break;
            }
            if (umma::elect_one()) {
                tma::mbar_arrive_expect_tx(&q_full[kept], q_bytes * it.slots);
                for (int x = 0; x < it.slots; ++x) {
#pragma unroll
                    for (int j = 0; j < Boxes; ++j) {
                        load_heads(base + (kSlots * kept + x) * Cfg::kQBytes + j * kBox, g.q, j * umma::kAtom, it.head * c.group,
                                   (it.row_tile + x) * g.tokens_per_tile, it.b, &q_full[kept]);
                    }
                }
            }
            __syncwarp();
            ++q_issued;
            for (int t = 0; ok && t < 2 * it.tiles; ++t) {
                ok = tma::mbar_wait(&empty[stage], phase ^ 1u);
                if (!ok) {
                    break;
                }
                if (umma::elect_one()) {
                    tma::mbar_arrive_expect_tx(&full[stage], Cfg::kTileBytes);
#pragma unroll
                    for (int j = 0; j < Boxes; ++j) {
                        load_heads(ring + stage * Cfg::kTileBytes + j * Cfg::kKeyBox, (t & 1) != 0 ? g.v : g.k, j * umma::kAtom, it.head,
                                   it.key0 + (t >> 1) * kKeys, it.b, &full[stage]);
                    }
                }
                __syncwarp();
                ++issued;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        if (!ok) {  // the loads in flight land (bounded) before the shared memory is given up
            bool drained = true;
            for (long long i = q_issued > Cfg::kQueries ? q_issued - Cfg::kQueries : 0; i < q_issued; ++i) {
                drained = tma::mbar_wait(&q_full[i % Cfg::kQueries], static_cast<unsigned>(i / Cfg::kQueries) & 1u) && drained;
            }
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
        const uint32_t score = umma::instruction(kBf16, false, false, kTile, kKeys);
        const uint32_t weigh = umma::instruction(kBf16, false, true, kTile, steps * 16);
        int stage = 0;
        unsigned phase = 0, taken = 0;  // items
        unsigned slot_items = 0, p_phases = 0;  // a bit per row tile
        int kept = 0;
        const auto scores = [&](int x, uint32_t k_tile) {
            if (umma::elect_one()) {
                const uint64_t a = umma::desc_k(base + (kSlots * kept + x) * Cfg::kQBytes), b = umma::desc_k(k_tile);
                for (int s = 0; s < steps; ++s) {
                    const uint64_t step = (s & 3) * umma::kStepK;
                    umma::mma(tmem + x * kKeys, a + step + (s >> 2) * (kBox >> 4), b + step + (s >> 2) * (Cfg::kKeyBox >> 4), score, s > 0);
                }
                umma::commit(&s_full[x]);
            }
            __syncwarp();
        };
        const auto advance = [&] {
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1u;
            }
        };
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<kSlots, kKeys>(g, i);
            if (it.tiles == 0) {
                continue;
            }
            kept = static_cast<int>(taken % Cfg::kQueries);
            ok = tma::mbar_wait(&q_full[kept], taken / Cfg::kQueries & 1u) && tma::mbar_wait(&full[stage], phase);
            if (!ok) {
                break;
            }
            ++taken;
            umma::fence_after_sync();
            for (int x = 0; x < it.slots; ++x) {
                scores(x, ring + stage * Cfg::kTileBytes);
            }
            if (umma::elect_one()) {
                umma::commit(&empty[stage]);
                if (it.tiles == 1) {
                    umma::commit(&q_empty[kept]);
                }
            }
            __syncwarp();
            advance();
            for (int t = 0; ok && t < it.tiles; ++t) {
                const int v_stage = stage;
                ok = tma::mbar_wait(&full[stage], phase);
                advance();
                const bool more = t + 1 < it.tiles;
                const int k_stage = stage;
                if (ok && more) {
                    ok = tma::mbar_wait(&full[stage], phase);
                    advance();
                }
                if (!ok) {
                    break;
                }
                for (int x = 0; ok && x < it.slots; ++x) {
                    ok = tma::mbar_wait(&p_full[x], p_phases >> x & 1u) && (t > 0 || tma::mbar_wait(&o_free[x], (slot_items >> x & 1u) ^ 1u));
                    if (!ok) {
                        break;
                    }
                    p_phases ^= 1u << x;
                    umma::fence_after_sync();
                    if (umma::elect_one()) {
                        const uint64_t b = umma::desc_mn<Cfg::kKeyBox>(ring + v_stage * Cfg::kTileBytes);
#pragma unroll
                        for (int s = 0; s < kKeys / 16; ++s) {
                            mma_tmem(tmem + Cfg::kO + x * Boxes * 64, tmem + x * kKeys + s * 8, b + umma::kStepMn * s, weigh, t > 0 || s > 0);
                        }
                        if (!more) {
                            umma::commit(&o_full[x]);
                        }
                    }
                    __syncwarp();
                    if (more) {
                        scores(x, ring + k_stage * Cfg::kTileBytes);
                    }
                }
                if (!ok) {
                    break;
                }
                if (umma::elect_one()) {
                    umma::commit(&empty[v_stage]);
                    if (more) {
                        umma::commit(&empty[k_stage]);
                        if (t + 2 == it.tiles) {
                            umma::commit(&q_empty[kept]);
                        }
                    }
                }
                __syncwarp();
            }
            slot_items ^= (1u << it.slots) - 1u;
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
        // A thread per row: warps 4 x to 4 x + 3 the x-th tile's.
        const int x = warp >> 2;
        const int quad = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t s_at = tmem + lanes + x * kKeys;
        const uint32_t o_at = tmem + lanes + Cfg::kO + x * Boxes * 64;
        const int local = quad * 32 + lane;
        const int row_token = local / c.group;
        const int row_head = local - row_token * c.group;
        unsigned s_phase = 0, o_phase = 0;
        unsigned entry = 0;  // of the ring: the next K tile
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<kSlots, kKeys>(g, i);
            if (x >= it.slots) {
                entry += 2 * it.tiles;
                continue;
            }
            const int first_token = (it.row_tile + x) * g.tokens_per_tile;
            const int token = first_token + row_token;
            const int row = token * c.group + row_head;
            const bool live = row_token < g.tokens_per_tile && token < c.queries;
            // A warp without rows only keeps the barriers going; what lies in its lanes reaches no one.
            const bool idle = quad * 32 >= min(g.tokens_per_tile, c.queries - first_token) * c.group;
            float m = -INFINITY, sum = 0.0f;
            MaskBytes<kKeys / 32> coming = mask_bytes<kKeys / 32>(c, it.b, it.end, it.key0);
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
                    // 32 scores at a time, fetched twice: for the largest, then for the weights.
                    const auto scores = [&](int j, float (&s)[32]) {
                        umma::load32(s_at + 32 * j, s);
                        umma::load_wait(s);
                        if (g.negative) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                s[k] = -s[k];
                            }
                        }
                        if (w[j] != 0xffffffffu) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                s[k] = (w[j] >> k & 1u) != 0 ? s[k] : -INFINITY;
                            }
                        }
                    };
                    float largest = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kKeys / 32; ++j) {
                        float s[32];
                        scores(j, s);
                        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (int k = 4; k < 32; ++k) {
                            top[k % 4] = fmaxf(top[k % 4], s[k]);
                        }
                        largest = fmaxf(largest, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                    }
                    largest *= g.factor;
                    const bool move = largest > m + kSlack || (m == -INFINITY && largest > -INFINITY);
                    if (__any_sync(0xffffffffu, move)) {
                        // Each row by its own scores alone: its bits do not depend on its neighbours.
                        const float keep = !move ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - largest);
                        m = move ? largest : m;
                        sum *= keep;
                        if (t > 0) {  // the products before are done: their commit came with these scores
                            for (int d = 0; d < c.dim; d += 16) {
                                float o[16];
                                umma::load16(o_at + d, o);
                                umma::load_wait(o);
#pragma unroll
                                for (int k = 0; k < 16; ++k) {
                                    o[k] *= keep;
                                }
                                store16(o_at + d, o);
                            }
                        }
                    }
                    const float2 shift = pair((m == -INFINITY ? 0.0f : -m) + kOffset);
                    float2 total = pair(0.0f);
#pragma unroll
                    for (int j = 0; j < kKeys / 32; ++j) {
                        float s[32];
                        scores(j, s);
                        uint32_t p[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float2 e = fma2(make_float2(s[2 * k], s[2 * k + 1]), pair(g.factor), shift);
                            const float2 v = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                            total = total + v;
                            p[k] = pack2<T>(v);
                        }
                        store16(s_at + 16 * j, p);
                    }
                    sum += total.x + total.y;
                    store_wait();
                }
                if (!all_count<kKeys / 32>(w)) {
                    // Each row tile's warps wipe all of V: another's products may come first.
                    const unsigned v_entry = entry + 1;
                    ok = tma::mbar_wait(&full[v_entry % kStages], v_entry / kStages & 1u);
                    wipe_rows<kKeys, 4>(ring + v_entry % kStages * Cfg::kTileBytes, Boxes, w, quad);
                }
                entry += 2;
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
            }
            const long long at = static_cast<long long>(it.b) * c.kv_heads + it.head;
            const float base_m = m == -INFINITY ? (g.splits > 1 ? m : 0.0f) : m - kOffset;
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
            const long long part_row = (it.split * c.pairs() + at) * c.rows() + row;
            const long long out_at = ((static_cast<long long>(it.b) * c.queries + token) * c.kv_heads + it.head) * c.group * c.dim + row_head * c.dim;
            T* out = static_cast<T*>(c.out) + out_at;
            const bool sectors = g.splits > 1 ? whole_sectors(g.partial, c.dim, 4)
                                              : whole_sectors(c.out, c.dim, 2) && (c.rest == nullptr || whole_sectors(c.rest, c.dim * 2, 1));
            if (!idle) {
                for (int d = 0; d < c.dim; d += 16) {
                    float o[16];
                    if (it.tiles > 0) {
                        umma::load16(o_at + d, o);
                        umma::load_wait(o);
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            o[k] = 0.0f;
                        }
                    }
                    const int valid = min(16, c.dim - d);
                    if (g.splits > 1) {
                        store_lanes<float>(g.partial + part_row * c.dim + d, nullptr, live, o, valid, sectors);
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            o[k] *= inverse;
                        }
                        store_lanes<T>(out + d, c.rest == nullptr ? nullptr : c.rest + out_at + d, live, o, valid, sectors);
                    }
                }
                if (live && g.splits > 1) {
                    g.part_stats[part_row] = make_float2(base_m, sum);
                } else if (live && c.stats != nullptr) {
                    c.stats[at * c.rows() + row] = make_float2(base_m, sum);
                }
            }
            if (it.tiles > 0) {
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    umma::arrive(&o_free[x]);
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
        umma::dealloc<Cfg::kCols>(tmem);
    }
}

// --- staging -------------------------------------------------------------------------------------------

struct StageJob {
    const void* source;
    void* target;
    Strides stride;
    long long tokens;
    int heads;
    long long rows;  // heads of all tokens
};
struct StageJobs {
    StageJob job[4];
    int dim;
    int pitch;
};

// 16-bit values, whatever their type: a warp takes four heads at a time, all their values asked for before one is stored.
__global__ void __launch_bounds__(256) stage_kernel(const __grid_constant__ StageJobs g)
{
    constexpr int kHeads = 4;
    constexpr int kPer = SPECTRAL_HEAD_DIM_MAX / 32;
    allow_next_grid();
    wait_for_previous_grid();
    const StageJob& j = g.job[blockIdx.y];
    const auto* __restrict__ source = static_cast<const unsigned short*>(j.source);
    auto* __restrict__ target = static_cast<unsigned short*>(j.target);
    const int lane = threadIdx.x & 31;
    const unsigned heads = j.heads, tokens = static_cast<unsigned>(j.tokens);
    for (long long first = (static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * kHeads; first < j.rows;
         first += static_cast<long long>(gridDim.x) * 8 * kHeads) {
        unsigned short v[kHeads][kPer];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const long long row = first + h;
            long long token, b;
            if (j.rows < (1LL << 31)) {
                token = static_cast<unsigned>(row) / heads;
                b = static_cast<unsigned>(token) / tokens;
            } else {
                token = row / heads;
                b = token / tokens;
            }
            const auto* from = source + b * j.stride.sample + (token - b * tokens) * j.stride.token + (row - token * heads) * j.stride.head;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int d = lane + 32 * k;
                v[h][k] = row < j.rows && d < g.dim ? from[d] : static_cast<unsigned short>(0);
            }
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int d = lane + 32 * k;
                if (first + h < j.rows && d < g.pitch) {
                    target[(first + h) * g.pitch + d] = v[h][k];
                }
            }
        }
    }
}

// --- host ------------------------------------------------------------------------------------------------

constexpr int kSms = 148;

struct Plan {
    Operand q, k, v;
    int row_items = 0;
    int splits = 1;
    int split_tiles = 0;
    std::size_t partial = 0, stats = 0;
    Arena arena;

    explicit Plan(const Call& c)
    {
        q = operand(arena, c.q, c.qs, c.batch, c.queries, c.kv_heads * c.group, c.dim, false);
        k = operand(arena, c.k, c.ks, c.batch, c.keys, c.kv_heads, c.dim, true);
        v = operand(arena, c.v, c.vs, c.batch, c.keys, c.kv_heads, c.dim, true);
        const int width = c.dim <= 64 ? Config<1>::kKeys : Config<2>::kKeys;
        row_items = pieces(pieces(c.queries, kTile / c.group), c.dim <= 64 ? Config<1>::kSlots : Config<2>::kSlots);
        // Splits of the keys: the fewest turns of the busiest CTA, counted in key tiles, where an item costs about two
        // more (its first loads and scores, its last products and stores); parts are written and joined.
        const long long tiles = pieces(c.keys, width);
        const long long base = c.pairs() * row_items;
        const long long least = std::max(1LL, (tiles + kLongestSum / width - 1) / (kLongestSum / width));
        double best = 0.0;
        for (long long s = least; s <= std::max(least, std::min(tiles, 128LL)); ++s) {
            const long long span = (tiles + s - 1) / s;
            if (s > least && (tiles + span - 1) / span != s) {
                continue;  // the same span as fewer splits
            }
            const double turns = static_cast<double>((base * s + kSms - 1) / kSms) * (static_cast<double>(span) + 2.0) + (s > 1 ? 4.0 + 0.02 * s : 0.0);
            if (s == least || turns < best) {
                best = turns;
                splits = static_cast<int>(s);
                split_tiles = static_cast<int>(span);
            }
        }
        splits = static_cast<int>(std::max(1LL, split_tiles == 0 ? 1LL : (tiles + split_tiles - 1) / split_tiles));
        if (splits > 1) {
            const std::size_t all = static_cast<std::size_t>(c.pairs()) * c.rows() * splits;
            partial = arena.take(all * c.dim * sizeof(float));
            stats = arena.take(all * sizeof(float2));
        }
    }
};

template <class T, int Boxes>
void launch(const Forward& g, cudaStream_t stream)
{
    using Cfg = Config<Boxes>;
    const auto kernel = forward_kernel<T, Boxes>;
    static std::atomic<int> cache[kMaxDevices];
    const unsigned grid = persistent_grid(reinterpret_cast<const void*>(kernel), Cfg::kThreads, Cfg::kSmem, cache, g.items);
    launch_pdl(kernel, dim3(grid), dim3(Cfg::kThreads), Cfg::kSmem, stream, g);
}

}  // namespace

void stage(const Operand* const* operands, int count, int batch, int dim, char* work, cudaStream_t stream)
{
    StageJobs g;
    g.dim = dim;
    g.pitch = (dim + 7) / 8 * 8;
    int jobs = 0;
    long long most = 0;
    for (int i = 0; i < count; ++i) {
        const Operand& o = *operands[i];
        if (o.staged && batch * o.tokens > 0) {
            const long long rows = batch * o.tokens * o.heads;
            g.job[jobs++] = {o.source, work + o.at, o.stride, o.tokens, o.heads, rows};
            most = std::max(most, rows);
        }
    }
    if (jobs > 0) {
        const auto grid = static_cast<unsigned>(std::min<long long>((most + 31) / 32, kSms * 8));
        launch_pdl(stage_kernel, dim3(grid, jobs), dim3(256), 0, stream, g);
    }
}

std::size_t tensor_forward_workspace(const Call& c) { return Plan(c).arena.size(); }

void tensor_forward(const Call& c, char* work, cudaStream_t stream)
{
    const Plan plan(c);
    const Operand* const operands[3] = {&plan.q, &plan.k, &plan.v};
    stage(operands, 3, c.batch, c.dim, work, stream);
    const bool is_bf16 = c.dtype == SPECTRAL_BFLOAT16;
    Forward g;
    g.c = c;
    g.tokens_per_tile = kTile / c.group;
    g.row_items = plan.row_items;
    g.splits = plan.splits;
    g.split_tiles = plan.split_tiles;
    const long long items = c.pairs() * plan.row_items * plan.splits;
    if (items >= (1LL << 31)) {
        throw InvalidArgument("cross_attention: too many tiles for one call");
    }
    g.items = static_cast<unsigned>(items);
    g.negative = c.scale < 0.0f;
    // A factor of 0 would turn the -infinity of a key that does not count into a NaN.
    g.factor = std::max(std::abs(c.scale) * kLog2e, 1.17549435e-38f);
    g.partial = reinterpret_cast<float*>(work + plan.partial);
    g.part_stats = reinterpret_cast<float2*>(work + plan.stats);
    g.fault = device_fault_word();
    g.q = head_map(plan.q.base(work), is_bf16, plan.q.strides(c.dim), c.batch, c.queries, c.kv_heads * c.group, c.dim, c.group, g.tokens_per_tile);
    const int width = c.dim <= 64 ? Config<1>::kKeys : Config<2>::kKeys;
    const void* keys[2] = {plan.k.base(work), plan.v.base(work)};
    if (c.keys > 0) {
        g.k = head_map(keys[0], is_bf16, plan.k.strides(c.dim), c.batch, c.keys, c.kv_heads, c.dim, 1, width);
        g.v = head_map(keys[1], is_bf16, plan.v.strides(c.dim), c.batch, c.keys, c.kv_heads, c.dim, 1, width);
    }
    const auto with_boxes = [&](auto t) {
        if (c.dim <= 64) {
            launch<decltype(t), 1>(g, stream);
        } else {
            launch<decltype(t), 2>(g, stream);
        }
    };
    if (is_bf16) {
        with_boxes(bf16{});
    } else {
        with_boxes(f16{});
    }
    if (plan.splits > 1) {
        join_splits(c, g.partial, g.part_stats, plan.splits, stream);
    }
}

}  // namespace spectral::attention
