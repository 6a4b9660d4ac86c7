// Attention backward for 16-bit values on the 5th-generation tensor cores.
//
// With p = 2^(c s - lse) (c = scale log2(e), lse = m + log2(sum) of the forward pass), g the upstream gradient,
// delta = sum over dim of g out and ds = p (g v^T - delta):
//   dv = p^T g,   dk = scale ds^T q,   dq = scale ds k
// Two kernels of one form, each sum with one owner, so that nothing is atomic and equal inputs give equal bits. A CTA
// owns 128 keys (their k and v stay in shared memory) and walks over row tiles for dk and dv, or owns 128 rows (q
// and g) and walks over key tiles for dq; the scores are computed in both. Per step, on tcgen05:
//   S = X0 Y0^T and D = X1 Y1^T into tensor memory (X owned, Y the tiles of the walk)
//   P over S and dS over D, as 16-bit operands; A1 += P Y1 (keys), A0 += dS Y0, accumulators in tensor memory.
// Warps with a thread per owned row and 32 columns first turn S to P, then D to dS; the products that
// need P and the next S run under the second half of that, those that need dS and the next D under the first half of the
// next step. A warp brings the tiles by TMA, one issues the products.
//
// float16 keeps p times 2^15 and ds times a power of two that no |ds| takes past 2^15: |g v - delta| is at most
// 2 max|g| max|v| (norms of rows and keys that count), which the kernel before these finds. Unscaled, weights of 2^-14 and
// less (16384 keys and more) would be subnormal, and small gradients zero.
//
// Measured, forward and backward in bf16: 64 x 16384 x 256 keys, 2 heads of 32, 1228 us (both kernels issue in 44 to 48 % of
// their slots: instructions of dependent chains); 4 x 4096 x 4096, 16 and 4 heads of 128, 2567 us (tensor pipe 48 to 54 %).

#include "attention_tc.cuh"

#include <algorithm>

namespace spectral::attention {
namespace {

constexpr int kSms = 148;
constexpr int kNormCtas = 4 * kSms;          // of the constants kernel, at most
constexpr float kWeightPower = 15.0f;        // float16's p times 2^15

struct Backward {
    HeadMap x0, x1, y0, y1;
    Call c;
    // Rows come in whole tokens: of the tiles that are owned, and of those walked over.
    int owned_tokens = 0;
    int walked_tokens = 0;
    unsigned owned = 0;        // tiles that are owned
    int walked = 0;            // tiles of rows to walk over (keys' kernel)
    int row_walks = 0;         // tiles of rows in `constants`
    unsigned parts = 1;
    int part_tiles = 0;        // tiles walked over per part
    unsigned items = 0;
    float factor = 1.0f;       // c
    const float* constants = nullptr;  // (pair, tile of walked_tokens): -lse of its rows, then -delta
    const float* norms = nullptr;      // float16: the CTAs' largest squares of rows of g, then of v
    int norm_count = 0;
    float* partial0 = nullptr;
    float* partial1 = nullptr;
    unsigned* fault = nullptr;
};

struct Item {
    int b;
    int head;
    int part;
    int tile;    // owned
    int first;   // tile walked over first
    int tiles;   // how many
    int end;     // keys before this count, but for the mask
};

// Rows: the CTA owns rows and walks over keys, `Width` at a time.
template <bool Rows, int Width>
__device__ __forceinline__ Item item_at(const Backward& g, unsigned i)
{
    Item it;
    const unsigned r = i / g.owned;
    it.tile = static_cast<int>(i - r * g.owned);
    const unsigned pair = r / g.parts;
    it.part = static_cast<int>(r - pair * g.parts);
    it.b = static_cast<int>(pair / static_cast<unsigned>(g.c.kv_heads));
    it.head = static_cast<int>(pair) - it.b * g.c.kv_heads;
    it.end = length_of(g.c, it.b);
    it.first = it.part * g.part_tiles;
    const int walked = Rows ? (it.end + Width - 1) / Width : it.tile * kTile < it.end ? g.walked : 0;
    it.tiles = max(0, min(g.part_tiles, walked - it.first));
    return it;
}

// Heads of up to 64 values: 64 entries of the walk at a time and two CTAs per SM that fill each other's waits. Wider heads: 128
// at a time, one CTA. Either way sixteen warps of an SM work on scores: their instructions follow from each other, and
// with eight (64 columns a thread) an SM issued one in four cycles per scheduler.
template <int Boxes, bool Rows>
struct Config {
    static constexpr int kWidth = Boxes == 1 ? 64 : 128;
    static constexpr int kCtas = Boxes == 1 ? 2 : 1;
    static constexpr int kParts = kWidth / 32;           // of a row of scores: a thread per owned row and 32 columns
    static constexpr int kWarps = 4 * kParts;            // that turn scores
    static constexpr int kThreads = 32 * (kWarps + 2);
    static constexpr int kOwnedBytes = Boxes * kBox;
    static constexpr int kWalkedBox = kWidth * umma::kRowBytes;
    static constexpr int kWalkedBytes = Boxes * kWalkedBox;
    static constexpr int kConstants = 2 * kWidth;        // floats per tile of rows
    static constexpr int kConstantBytes = Rows ? 0 : kConstants * 4;
    static constexpr int kStageBytes = 2 * kWalkedBytes;  // Y0, Y1
    static constexpr int kStages = Boxes == 1 ? 4 : 2;
    static constexpr int kSmem = 2 * kOwnedBytes + kStages * (kStageBytes + kConstantBytes) + 1024;
    static constexpr int kD = kWidth;                    // tensor memory: S and P, D and dS, A0, A1
    static constexpr int kA0 = 2 * kWidth;
    static constexpr int kA1 = 2 * kWidth + Boxes * 64;
    static constexpr int kCols = Boxes == 1 ? 256 : 512;
    static_assert(kCtas * (kSmem + 1024) <= kSmemMost, "shared memory");
    static_assert(kCtas * kCols <= 512 && kA1 + Boxes * 64 <= kCols, "tensor memory");
};

template <class T, int Boxes, bool Rows>
__global__ void __launch_bounds__(Config<Boxes, Rows>::kThreads, Config<Boxes, Rows>::kCtas) backward_kernel(const __grid_constant__ Backward g)
{
    using Cfg = Config<Boxes, Rows>;
    constexpr bool kBf16 = std::is_same_v<T, bf16>;
    constexpr int kStages = Cfg::kStages;
    constexpr int kWidth = Cfg::kWidth;
    constexpr int kWarps = Cfg::kWarps;
    extern __shared__ unsigned char smem_base[];
    const uint32_t base = (tma::smem_addr(smem_base) + 1023u) & ~1023u;
    unsigned char* const generic = smem_base + (base - tma::smem_addr(smem_base));
    const uint32_t ring = base + 2 * Cfg::kOwnedBytes;
    const float* const constants = reinterpret_cast<const float*>(generic + 2 * Cfg::kOwnedBytes + kStages * Cfg::kStageBytes);
    __shared__ uint64_t x_full, x_empty, full[kStages], empty[kStages], s_full, d_full, p_ready, ds_ready, acc_full, acc_free, drain;
    __shared__ uint32_t tmem_slot;
    __shared__ float norm_of[2][20];
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == kWarps) {
        umma::alloc<Cfg::kCols>(&tmem_slot);
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
        // Rows of a tile that no box writes (width % group) are reduced over: zeros, once.
        const int used = g.walked_tokens * g.c.group;
        const int spare = kWidth - used;
        for (int i = threadIdx.x; i < 2 * kStages * Boxes * spare * 8; i += Cfg::kThreads) {
            const int box = i / (spare * 8), at = i - box * spare * 8;
            *reinterpret_cast<uint4*>(generic + 2 * Cfg::kOwnedBytes + box * Cfg::kWalkedBox + (used + at / 8) * umma::kRowBytes + at % 8 * 16) =
                make_uint4(0, 0, 0, 0);
        }
        tma::fence_proxy_async();
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

    // float16: the power of two that ds is held in.
    float ds_scale = 1.0f;
    if constexpr (!kBf16) {
        float top[2] = {0.0f, 0.0f};
        for (int i = threadIdx.x; i < 2 * g.norm_count; i += Cfg::kThreads) {
            const int which = i >= g.norm_count ? 1 : 0;
            top[which] = fmaxf(top[which], g.norms[i]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int o = 16; o > 0; o /= 2) {
                top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
            }
            if (lane == 0) {
                norm_of[k][warp] = top[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            top[k] = 0.0f;
            for (int i = 0; i < Cfg::kThreads / 32; ++i) {
                top[k] = fmaxf(top[k], norm_of[k][i]);
            }
        }
        const float most = 2.0f * sqrtf(top[0]) * sqrtf(top[1]);
        // 2^(14 - floor(log2(most))) times most is below 2^15.
        const int power = most > 0.0f ? 14 - ilogbf(most) : 0;
        ds_scale = exp2f(static_cast<float>(max(-60, min(60, power))));
    }

    if (warp == kWarps) {
        // The TMA warp: the owned tiles as soon as the item before has no more use for its own, then Y0, Y1 in turn.
        asm volatile("fence.proxy.async.global;" ::: "memory");
        const unsigned token_bytes = static_cast<unsigned>(c.group) * umma::kRowBytes * Boxes;
        const unsigned owned_bytes = 2 * (Rows ? g.owned_tokens * token_bytes : Cfg::kOwnedBytes);
        const unsigned walked_bytes = 2 * (Rows ? Cfg::kWalkedBytes : g.walked_tokens * token_bytes) + Cfg::kConstantBytes;
        int stage = 0;
        unsigned phase = 0, x_phase = 0;
        long long issued = 0, x_issued = 0;
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<Rows, kWidth>(g, i);
            if (it.tiles == 0) {
                continue;
            }
            ok = tma::mbar_wait(&x_empty, x_phase ^ 1u);
            if (!ok) {
                break;
            }
            x_phase ^= 1u;
            const int x_head = Rows ? it.head * c.group : it.head;
            const int y_head = Rows ? it.head : it.head * c.group;
            const int x_token = it.tile * (Rows ? g.owned_tokens : kTile);
            if (umma::elect_one()) {
                tma::mbar_arrive_expect_tx(&x_full, owned_bytes);
#pragma unroll
                for (int j = 0; j < Boxes; ++j) {
                    load_heads(base + j * kBox, g.x0, j * umma::kAtom, x_head, x_token, it.b, &x_full);
                    load_heads(base + Cfg::kOwnedBytes + j * kBox, g.x1, j * umma::kAtom, x_head, x_token, it.b, &x_full);
                }
            }
            __syncwarp();
            ++x_issued;
            for (int t = it.first; ok && t < it.first + it.tiles; ++t) {
                ok = tma::mbar_wait(&empty[stage], phase ^ 1u);
                if (!ok) {
                    break;
                }
                if (umma::elect_one()) {
                    const uint32_t y = ring + stage * Cfg::kStageBytes;
                    const int y_token = t * (Rows ? kWidth : g.walked_tokens);
                    tma::mbar_arrive_expect_tx(&full[stage], walked_bytes);
#pragma unroll
                    for (int j = 0; j < Boxes; ++j) {
                        load_heads(y + j * Cfg::kWalkedBox, g.y0, j * umma::kAtom, y_head, y_token, it.b, &full[stage]);
                        load_heads(y + Cfg::kWalkedBytes + j * Cfg::kWalkedBox, g.y1, j * umma::kAtom, y_head, y_token, it.b, &full[stage]);
                    }
                    if constexpr (!Rows) {
                        const long long at = (static_cast<long long>(it.b) * c.kv_heads + it.head) * g.row_walks + t;
                        tma::bulk_g2s(const_cast<float*>(constants) + stage * Cfg::kConstants, g.constants + row_constants_at(at, kWidth), Cfg::kConstantBytes,
                                      &full[stage]);
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
        const uint32_t score = umma::instruction(kBf16, false, false, kTile, kWidth);
        const uint32_t weigh = umma::instruction(kBf16, false, true, kTile, steps * 16);
        int stage = 0;
        unsigned phase = 0, x_phase = 0, step_phase = 0, acc_phase = 0;
        // S (k = 0) or D (k = 1) from the owned tiles and a stage's.
        const auto scores = [&](int k, int y_stage, uint64_t* done) {
            if (umma::elect_one()) {
                const uint64_t a = umma::desc_k(base + k * Cfg::kOwnedBytes);
                const uint64_t b = umma::desc_k(ring + y_stage * Cfg::kStageBytes + k * Cfg::kWalkedBytes);
                for (int s = 0; s < steps; ++s) {
                    const uint64_t step = (s & 3) * umma::kStepK;
                    umma::mma(tmem + k * Cfg::kD, a + step + (s >> 2) * (kBox >> 4), b + step + (s >> 2) * (Cfg::kWalkedBox >> 4), score, s > 0);
                }
                umma::commit(done);
            }
            __syncwarp();
        };
        // A0 += dS Y0 (k = 0), A1 += P Y1 (k = 1). Each 32 columns of scores leave theirs in the first 16 of the same place.
        const auto weighed = [&](int k, int y_stage, bool accumulate) {
            const uint64_t b = umma::desc_mn<Cfg::kWalkedBox>(ring + y_stage * Cfg::kStageBytes + k * Cfg::kWalkedBytes);
            const uint32_t a = tmem + (k == 0 ? Cfg::kD : 0);
#pragma unroll
            for (int s = 0; s < kWidth / 16; ++s) {
                mma_tmem(tmem + (k == 0 ? Cfg::kA0 : Cfg::kA1), a + (s >> 1) * 32 + (s & 1) * 8, b + umma::kStepMn * s, weigh, accumulate || s > 0);
            }
        };
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<Rows, kWidth>(g, i);
            if (it.tiles == 0) {
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
                ok = tma::mbar_wait(&p_ready, step_phase) && (t > 0 || tma::mbar_wait(&acc_free, acc_phase ^ 1u)) && (!more || tma::mbar_wait(&full[stage], phase));
                if (!ok) {
                    break;
                }
                umma::fence_after_sync();
                if constexpr (!Rows) {
                    if (umma::elect_one()) {
                        weighed(1, now, t > 0);
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
                    weighed(0, now, t > 0);
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
        // A thread per owned row and 32 columns: warps 4 k to 4 k + 3 the k-th.
        const int part = warp >> 2;
        const int local = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + part * 32;
        const uint32_t d_at = s_at + Cfg::kD;
        int stage = 0;
        unsigned phase = 0, step_phase = 0, acc_phase = 0;
        const float power = kBf16 ? 0.0f : kWeightPower;
        // Where an owned row lies: token and head in the group.
        const int row_token = local / c.group;
        const int row_head = local - row_token * c.group;
        for (unsigned i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
            const Item it = item_at<Rows, kWidth>(g, i);
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
            const bool whole = __all_sync(0xffffffffu, counts);
            MaskBytes<kWidth / 32> mask{};
            if constexpr (Rows) {
                mask = mask_bytes<kWidth / 32>(c, it.b, it.end, it.first * kWidth);
            }
            for (int t = it.first; ok && t < it.first + it.tiles; ++t) {
                uint32_t w[4] = {0, 0, 0, 0};
                if constexpr (Rows) {
                    tile_bits<kWidth / 32>(c, mask, it.end, t * kWidth, w);
                    mask = mask_bytes<kWidth / 32>(c, it.b, it.end, (t + 1) * kWidth);
                }
                ok = tma::mbar_wait(&full[stage], phase);
                const float* less = constants + stage * Cfg::kConstants + part * 32;  // -lse, then -delta
                const uint32_t word = Rows ? (part == 0 ? w[0] : part == 1 ? w[1] : part == 2 ? w[2] : w[3]) : counts ? 0xffffffffu : 0u;
                const bool all = Rows ? word == 0xffffffffu : whole;
                ok = ok && tma::mbar_wait(&s_full, step_phase);
                if (!ok) {
                    break;
                }
                umma::fence_after_sync();
                float p[32];
                umma::load32(s_at, p);
                umma::load_wait(p);
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float2 a = shift, b = shift;
                    if constexpr (!Rows) {
                        const float4 l = *reinterpret_cast<const float4*>(less + k);
                        a = make_float2(l.x, l.y);
                        b = make_float2(l.z, l.w);
                    }
                    a = fma2(make_float2(p[k], p[k + 1]), pair(g.factor), a);
                    b = fma2(make_float2(p[k + 2], p[k + 3]), pair(g.factor), b);
                    p[k] = exp2_fast(a.x);
                    p[k + 1] = exp2_fast(a.y);
                    p[k + 2] = exp2_fast(b.x);
                    p[k + 3] = exp2_fast(b.y);
                }
                if (!all) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        p[k] = (word >> k & 1u) != 0 ? p[k] : 0.0f;
                    }
                }
                if constexpr (!Rows) {
                    uint32_t out[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 v = make_float2(p[2 * k], p[2 * k + 1]);
                        if constexpr (!kBf16) {
                            v = v * pair(32768.0f);  // 2^kWeightPower
                        }
                        out[k] = pack2<T>(v);
                    }
                    store16(s_at, out);
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
                float d[32];
                umma::load32(d_at, d);
                umma::load_wait(d);
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float2 a = delta, b = delta;
                    if constexpr (!Rows) {
                        const float4 l = *reinterpret_cast<const float4*>(less + kWidth + k);
                        a = make_float2(l.x, l.y);
                        b = make_float2(l.z, l.w);
                    }
                    a = (make_float2(d[k], d[k + 1]) + a) * make_float2(p[k], p[k + 1]);
                    b = (make_float2(d[k + 2], d[k + 3]) + b) * make_float2(p[k + 2], p[k + 3]);
                    if constexpr (!kBf16) {
                        a = a * pair(ds_scale);
                        b = b * pair(ds_scale);
                    }
                    d[k] = a.x;
                    d[k + 1] = a.y;
                    d[k + 2] = b.x;
                    d[k + 3] = b.y;
                }
                // A key that does not count may have made D anything.
                if (!all) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        d[k] = (word >> k & 1u) != 0 ? d[k] : 0.0f;
                    }
                }
                {
                    uint32_t out[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        out[k] = pack2<T>(make_float2(d[2 * k], d[2 * k + 1]));
                    }
                    store16(d_at, out);
                    store_wait();
                }
                if constexpr (Rows) {  // of k, which ds meets; v has only been read for scores that were dropped
                    if (!all_count<kWidth / 32>(w)) {
                        wipe_rows<kWidth, kWarps>(ring + stage * Cfg::kStageBytes, Boxes, w, warp);
                    }
                }
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
            }
            // The warps share the stores: rows, each part some of dq; keys, the first half of the parts dk, the others dv.
            constexpr int kSharers = Rows ? Cfg::kParts : Cfg::kParts / 2;
            const int span = ((c.dim + 15) / 16 + kSharers - 1) / kSharers * 16;
            const long long part_row = (it.part * c.pairs() + pair_at) * (Rows ? c.rows() : c.keys) + row;
            const long long at = Rows ? ((static_cast<long long>(it.b) * c.queries + token) * c.kv_heads + it.head) * c.group * c.dim + row_head * c.dim
                                      : ((static_cast<long long>(it.b) * c.keys + row) * c.kv_heads + it.head) * c.dim;
            {
                const bool of_v = !Rows && part >= kSharers;
                const int from = part % kSharers * span;
                const float factor = of_v ? exp2f(-power) : (g.parts > 1 ? 1.0f : c.scale) / ds_scale;
                float* partial = of_v ? g.partial1 : g.partial0;
                T* result = static_cast<T*>(Rows ? c.dq : of_v ? c.dv : c.dk);
                for (int d = from; d < min(from + span, c.dim); d += 16) {
                    float a[16];
                    if (it.tiles > 0) {
                        umma::load16(tmem + lanes + (of_v ? Cfg::kA1 : Cfg::kA0) + d, a);
                        umma::load_wait(a);
                    }
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        a[k] = it.tiles == 0 || !counts ? 0.0f : a[k] * factor;
                    }
                    if (g.parts > 1) {
                        store_lanes<float>(partial + part_row * c.dim + d, nullptr, live, a, min(16, c.dim - d), whole_sectors(partial, c.dim, 4));
                    } else {
                        store_lanes<T>(result + at + d, nullptr, live, a, min(16, c.dim - d), whole_sectors(result, c.dim, 2));
                    }
                }
            }
            if (it.tiles > 0) {
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    umma::arrive(&acc_free);
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

// --- the rows' constants -----------------------------------------------------------------------------------

// -lse (infinite for rows that are not there or have no keys, so that their weights are 0) and -delta of every entry of
// every row tile, `lanes` lanes of eight values a row. float16: also the largest squares of g's rows and v's
// keys that this CTA met (finite ones).
template <class T, bool Vectors>
__global__ void __launch_bounds__(256) constants_kernel(const Call c, float* __restrict__ out, float* __restrict__ norms, int width, int rows_per_tile,
                                                        int row_tiles, int lanes)
{
    __shared__ float top_of[2][8];
    allow_next_grid();
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31;
    const int sub = lane & (lanes - 1);
    const int per_cta = 256 / lanes;
    const T* __restrict__ o = static_cast<const T*>(c.out);
    const T* __restrict__ g = static_cast<const T*>(c.dout);
    const auto fetch = [&](const T* p) {
        Vec<T, 8> v{};
        if (sub * 8 < c.dim) {
            if constexpr (Vectors) {
                v = *reinterpret_cast<const Vec<T, 8>*>(p + sub * 8);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v.v[j] = sub * 8 + j < c.dim ? p[sub * 8 + j] : from_float<T>(0.0f);
                }
            }
        }
        return widen(v);
    };
    const auto total = [&](float2 v) {
        float s = v.x + v.y;
        for (int k = lanes / 2; k > 0; k /= 2) {
            s += __shfl_xor_sync(0xffffffffu, s, k);
        }
        return s;
    };
    float top[2] = {0.0f, 0.0f};
    const long long all = c.pairs() * row_tiles * width;
    // Whole warps stay in the loops together: they shuffle.
    for (long long base = static_cast<long long>(blockIdx.x) * per_cta; base < all; base += static_cast<long long>(gridDim.x) * per_cta) {
        const long long i = base + threadIdx.x / lanes;
        const int local = static_cast<int>(i & (width - 1));  // 64 or 128
        const auto tile = static_cast<unsigned>(i / width);     // below 2^32: their constants are 512 bytes each and more
        const unsigned pair_at = tile / static_cast<unsigned>(row_tiles);
        const int r = static_cast<int>(tile - pair_at * row_tiles) * rows_per_tile + local;
        const bool there = i < all && local < rows_per_tile && r < c.rows();
        float2 dot = pair(0.0f), square = pair(0.0f);
        if (there) {
            const unsigned b = pair_at / static_cast<unsigned>(c.kv_heads), token = static_cast<unsigned>(r) / static_cast<unsigned>(c.group);
            const long long at = ((static_cast<long long>(b) * c.queries + token) * c.kv_heads + (pair_at - b * c.kv_heads)) * c.group * c.dim
                                 + (r - static_cast<int>(token) * c.group) * c.dim;
            Floats<8> x = fetch(o + at);
            const Floats<8> y = fetch(g + at);
            if (sizeof(T) == 2 && c.rest != nullptr && sub * 8 < c.dim) {
                Vec<unsigned char, 8> code{};
                if constexpr (Vectors) {
                    code = *reinterpret_cast<const Vec<unsigned char, 8>*>(c.rest + at + sub * 8);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        code.v[j] = sub * 8 + j < c.dim ? c.rest[at + sub * 8 + j] : static_cast<unsigned char>(0);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x.p[j] = with_rest<T>(x.p[j], reinterpret_cast<const unsigned short*>(&code)[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                dot = fma2(x.p[j], y.p[j], dot);
                square = fma2(y.p[j], y.p[j], square);
            }
        }
        const float delta = total(dot);
        if constexpr (std::is_same_v<T, f16>) {
            const float s = total(square);
            top[0] = s < INFINITY ? fmaxf(top[0], s) : top[0];
        }
        if (sub == 0 && i < all) {
            float lse = INFINITY;
            if (there) {
                const float2 s = c.stats[pair_at * c.rows() + r];
                lse = s.y == 0.0f ? INFINITY : s.x + log2f(s.y);
            }
            float* at = out + row_constants_at(tile, width) + local;
            at[0] = -lse;
            at[width] = -delta;
        }
    }
    if constexpr (std::is_same_v<T, f16>) {
        const T* __restrict__ v = static_cast<const T*>(c.v);
        const long long keys = c.pairs() * c.keys;
        for (long long base = static_cast<long long>(blockIdx.x) * per_cta; base < keys; base += static_cast<long long>(gridDim.x) * per_cta) {
            const long long i = base + threadIdx.x / lanes;
            const long long pair_at = i / c.keys;
            const int key = static_cast<int>(i - pair_at * c.keys);
            const int b = static_cast<int>(pair_at / c.kv_heads);
            float2 square = pair(0.0f);
            if (i < keys && key < length_of(c, b) && (c.mask == nullptr || c.mask[static_cast<long long>(b) * c.keys + key] != 0)) {
                const T* at = v + b * c.vs.sample + key * c.vs.token + (pair_at - static_cast<long long>(b) * c.kv_heads) * c.vs.head;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = sub * 8 + j < c.dim ? to_float(at[sub * 8 + j]) : 0.0f;
                    square.x = fmaf(x, x, square.x);
                }
            }
            const float s = total(square);
            top[1] = s < INFINITY ? fmaxf(top[1], s) : top[1];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int s = 16; s > 0; s /= 2) {
                top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], s));
            }
            if (lane == 0) {
                top_of[k][threadIdx.x >> 5] = top[k];
            }
        }
        __syncthreads();
        if (threadIdx.x < 2) {
            float m = 0.0f;
            for (int w = 0; w < 8; ++w) {
                m = fmaxf(m, top_of[threadIdx.x][w]);
            }
            norms[threadIdx.x * gridDim.x + blockIdx.x] = m;
        }
    }
}

// --- host --------------------------------------------------------------------------------------------------

// How many parts `walked` tiles are cut into for `owned` items of one part each: the fewest turns of the busiest CTA,
// counted in tiles (an item costs about two more), at most kLongestSum entries a part.
void cut(long long owned, int walked, int width, int ctas, int& parts, int& part_tiles)
{
    const int most = kLongestSum / width;
    const long long least = std::max(1, (walked + most - 1) / most);
    double best = 0.0;
    for (long long s = least; s <= std::max<long long>(least, std::min(walked, 64)); ++s) {
        const long long span = (walked + s - 1) / s;
        if (s > least && (walked + span - 1) / span != s) {
            continue;
        }
        const double turns = static_cast<double>((owned * s + ctas - 1) / ctas) * (static_cast<double>(span) + 2.0) + (s > 1 ? 3.0 + 0.1 * s : 0.0);
        if (s == least || turns < best) {
            best = turns;
            parts = static_cast<int>(s);
            part_tiles = static_cast<int>(span);
        }
    }
    parts = std::max(1, (walked + part_tiles - 1) / part_tiles);
}

struct Plan {
    Operand q, k, v, dout;
    int boxes = 1, width = 64;
    int owned_tokens = 0, walked_tokens = 0;
    int row_tiles = 0, key_tiles = 0;  // owned
    int row_walks = 0, key_walks = 0;
    int row_parts = 1, row_span = 0;   // keys' kernel: parts of the rows
    int key_parts = 1, key_span = 0;   // rows' kernel: parts of the keys
    std::size_t constants = 0, norms = 0, dq = 0, dk = 0, dv = 0;
    Arena arena;

    explicit Plan(const Call& c)
    {
        const int heads = c.kv_heads * c.group;
        const Strides dense{static_cast<long long>(c.queries) * heads * c.dim, static_cast<long long>(heads) * c.dim, c.dim};
        q = operand(arena, c.q, c.qs, c.batch, c.queries, heads, c.dim, false);
        k = operand(arena, c.k, c.ks, c.batch, c.keys, c.kv_heads, c.dim, true);
        v = operand(arena, c.v, c.vs, c.batch, c.keys, c.kv_heads, c.dim, true);
        dout = operand(arena, c.dout, dense, c.batch, c.queries, heads, c.dim, false);
        boxes = c.dim <= 64 && c.group <= 64 ? 1 : 2;  // a tile that is walked over holds a token's heads
        width = boxes == 1 ? 64 : 128;
        owned_tokens = kTile / c.group;
        walked_tokens = width / c.group;
        row_tiles = pieces(c.queries, owned_tokens);
        key_tiles = pieces(c.keys, kTile);
        row_walks = pieces(c.queries, walked_tokens);
        key_walks = pieces(c.keys, width);
        const int ctas = kSms * (boxes == 1 ? 2 : 1);
        cut(c.pairs() * key_tiles, row_walks, width, ctas, row_parts, row_span);
        cut(c.pairs() * row_tiles, key_walks, width, ctas, key_parts, key_span);
        constants = arena.take(static_cast<std::size_t>(c.pairs()) * row_walks * 2 * width * sizeof(float));
        norms = arena.take(2 * kNormCtas * sizeof(float));
        if (key_parts > 1) {
            dq = arena.take(static_cast<std::size_t>(c.pairs()) * c.rows() * c.dim * key_parts * sizeof(float));
        }
        if (row_parts > 1) {
            dk = arena.take(static_cast<std::size_t>(c.pairs()) * c.keys * c.dim * row_parts * sizeof(float));
            dv = arena.take(static_cast<std::size_t>(c.pairs()) * c.keys * c.dim * row_parts * sizeof(float));
        }
    }
};

unsigned item_count(long long items)
{
    if (items >= (1LL << 31)) {
        throw InvalidArgument("cross_attention_backward: too many tiles for one call");
    }
    return static_cast<unsigned>(items);
}

template <class T, int Boxes, bool Rows>
void launch(const Backward& g, cudaStream_t stream)
{
    using Cfg = Config<Boxes, Rows>;
    const auto kernel = backward_kernel<T, Boxes, Rows>;
    static std::atomic<bool> ready[kMaxDevices];
    const int device = current_device();
    if (!ready[device].load(std::memory_order_relaxed)) {
        const auto* f = reinterpret_cast<const void*>(kernel);
        SPECTRAL_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
        // All of the SM's memory, or the occupancy is one CTA where two fit.
        SPECTRAL_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        ready[device].store(true, std::memory_order_relaxed);
    }
    const unsigned grid = std::min(g.items, static_cast<unsigned>(device_sm_count(device) * Cfg::kCtas));
    launch_pdl(kernel, dim3(grid), dim3(Cfg::kThreads), Cfg::kSmem, stream, g);
}

template <class T, int Boxes>
void both(Backward g, const Plan& plan, const HeadMap (&rows)[2], const HeadMap (&row_walk)[2], const HeadMap (&keys)[2], const HeadMap (&key_walk)[2],
          char* work, cudaStream_t stream)
{
    const Call& c = g.c;
    // dk and dv.
    g.x0 = keys[0];
    g.x1 = keys[1];
    g.y0 = row_walk[0];
    g.y1 = row_walk[1];
    g.owned = plan.key_tiles;
    g.parts = plan.row_parts;
    g.part_tiles = plan.row_span;
    g.items = item_count(c.pairs() * plan.key_tiles * plan.row_parts);
    g.partial0 = reinterpret_cast<float*>(work + plan.dk);
    g.partial1 = reinterpret_cast<float*>(work + plan.dv);
    launch<T, Boxes, false>(g, stream);
    // dq.
    g.x0 = rows[0];
    g.x1 = rows[1];
    g.y0 = key_walk[0];
    g.y1 = key_walk[1];
    g.owned = plan.row_tiles;
    g.parts = plan.key_parts;
    g.part_tiles = plan.key_span;
    g.items = item_count(c.pairs() * plan.row_tiles * plan.key_parts);
    g.partial0 = reinterpret_cast<float*>(work + plan.dq);
    launch<T, Boxes, true>(g, stream);
}

// `norms` (float16): 2 x the returned count of floats.
int launch_constants(const Call& c, float* constants, float* norms, int width, int rows_per_tile, int row_tiles, cudaStream_t stream)
{
    int lanes = 1;
    while (lanes * 8 < c.dim) {
        lanes *= 2;
    }
    const long long entries = std::max(c.pairs() * row_tiles * width, c.dtype == SPECTRAL_FLOAT16 ? c.pairs() * c.keys : 0LL);
    const auto grid = static_cast<unsigned>(std::min<long long>((entries * lanes + 255) / 256, kNormCtas));
    const std::size_t piece = 8 * dtype_size(c.dtype);
    const bool vectors = c.dim % 8 == 0 && aligned_to(c.out, piece) && aligned_to(c.dout, piece) && aligned_to(c.rest, 8);
    with_dtype(c.dtype, [&](auto t) {
        using T = decltype(t);
        launch_pdl(vectors ? constants_kernel<T, true> : constants_kernel<T, false>, dim3(grid), dim3(256), 0, stream, c, constants, norms, width,
                   rows_per_tile, row_tiles, lanes);
    });
    return static_cast<int>(grid);
}

}  // namespace

void row_constants(const Call& c, float* out, int width, int tokens, int tiles, cudaStream_t stream)
{
    launch_constants(c, out, nullptr, width, tokens * c.group, tiles, stream);
}

std::size_t tensor_backward_workspace(const Call& c) { return Plan(c).arena.size(); }

void tensor_backward(const Call& c, char* work, cudaStream_t stream)
{
    const Plan plan(c);
    const Operand* const operands[4] = {&plan.q, &plan.k, &plan.v, &plan.dout};
    stage(operands, 4, c.batch, c.dim, work, stream);
    const bool is_bf16 = c.dtype == SPECTRAL_BFLOAT16;
    Backward g;
    g.c = c;
    g.owned_tokens = plan.owned_tokens;
    g.walked_tokens = plan.walked_tokens;
    g.walked = plan.row_walks;
    g.row_walks = plan.row_walks;
    g.factor = c.scale * kLog2e;
    auto* constants = reinterpret_cast<float*>(work + plan.constants);
    auto* norms = reinterpret_cast<float*>(work + plan.norms);
    g.constants = constants;
    g.norms = norms;
    g.fault = device_fault_word();
    g.norm_count = launch_constants(c, constants, norms, plan.width, plan.walked_tokens * c.group, plan.row_walks, stream);
    const int heads = c.kv_heads * c.group;
    const auto rows_map = [&](const Operand& o, int tokens) {
        return head_map(o.base(work), is_bf16, o.strides(c.dim), c.batch, c.queries, heads, c.dim, c.group, tokens);
    };
    const auto keys_map = [&](const Operand& o, int keys) {
        return head_map(o.base(work), is_bf16, o.strides(c.dim), c.batch, c.keys, c.kv_heads, c.dim, 1, keys);
    };
    const HeadMap rows[2] = {rows_map(plan.q, plan.owned_tokens), rows_map(plan.dout, plan.owned_tokens)};
    const HeadMap row_walk[2] = {rows_map(plan.q, plan.walked_tokens), rows_map(plan.dout, plan.walked_tokens)};
    const HeadMap keys[2] = {keys_map(plan.k, kTile), keys_map(plan.v, kTile)};
    const HeadMap key_walk[2] = {keys_map(plan.k, plan.width), keys_map(plan.v, plan.width)};
    const auto run = [&](auto t) {
        using T = decltype(t);
        if (plan.boxes == 1) {
            both<T, 1>(g, plan, rows, row_walk, keys, key_walk, work, stream);
        } else {
            both<T, 2>(g, plan, rows, row_walk, keys, key_walk, work, stream);
        }
    };
    if (is_bf16) {
        run(bf16{});
    } else {
        run(f16{});
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
