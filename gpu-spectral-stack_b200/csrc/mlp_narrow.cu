// The feed-forward block where it is narrow, as between the spectral convolutions of an FNO: few
// channels, very many tokens. Its weights fit in shared memory and its hidden values never leave the
// SM, so HBM carries only x and y (backward: x, dy and dx).
//
// Both kernels are persistent, one CTA per SM, tiles of 128 tokens: a TMA warp, two MMA warps (one for
// the products that lead to the hidden values, one for those that use them, so that the first run
// ahead while the epilogue works) and sixteen epilogue warps; the hidden values in chunks of 64.
// Every wait is bounded (tma.cuh).
//
// Forward, chunk j:  [G U] = x [Wg_j; Wu_j]^T   (N = 128, one accumulator set of two)
//                    h = act(G) * U, rounded, into shared memory as the next A operand
//                    y += h Wd_j^T              (N = outputs, one accumulator of two)
// Backward, chunk j: [G U] as above and dh = dy Wd_j
//                    dG, dU and h, rounded, into shared memory
//                    dx += dG Wg_j + dU Wu_j
//                    [dWg; dWu]_j += [dG dU]^T x     (M = 128, K = 128 tokens)
//          per tile: dWd^T += [h_0 h_1]^T dy
// The weight gradients stay in tensor memory over all of a CTA's tiles (512 columns in all: 192 for a
// chunk's three products, 2 x 64 for dx, 128 and 64 for the gradients) and leave it once, as the
// CTA's part of a sum that a last kernel adds up in order. (Past 64 tiles a CTA, ranges of tokens are launched
// one by one.)
// x, dy, the weights and the hidden tiles each serve as K-major and as MN-major operands from the
// one copy in shared memory (umma.cuh).
//
// What bounds them (262144 tokens, 64 channels, 128 hidden). Forward: a chunk's way from one stage to the next
// (accumulator, activation, shared memory, second product; 30 us with gelu, 28 us with silu, 18 us with no activation;
// HBM alone 10 us): the issue slots are 46 % busy, the tensor pipe 19 %, and the warps wait longest for tensor memory and barriers.
// gelu without special functions, a polynomial, and with one reciprocal for two values measured the same. Backward: the
// tensor cores' reads of shared memory; a tile's 56 MMAs of N = 64 or 128 take some 85 cycles each, 4800 in all, which is
// a tile's period (with the sum of the CTAs' parts 58 us with gelu, 51 us without).

#include "mlp.cuh"

#include <algorithm>

namespace spectral::mlp {
namespace {

constexpr int kHiddenChunk = 64;
constexpr int kTileBytes = kTileM * umma::kRowBytes;  // 128 tokens x 64 values: 16 KiB
constexpr int kWeightBytes = kHiddenChunk * umma::kRowBytes;  // 64 x 64 weights: 8 KiB

// Sixteen epilogue warps, the TMA warp, and two that issue MMAs. The latter run as one lane each from
// start to end: a wait costs it some 75 to 100 cycles even where nothing is left to wait for, a
// commit 50, and as one warp with an elected lane per step the two products of a chunk took 1500 cycles
// to issue, three times what they take to run.
constexpr int kWarps = 16;
constexpr int kNarrowThreads = 32 * (kWarps + 3);

struct NarrowMaps {
    CUtensorMap x;
    CUtensorMap dy;
    CUtensorMap wg;
    CUtensorMap wu;
    CUtensorMap wd;
};

struct NarrowArgs {
    long long tokens = 0;
    int tiles = 0;
    int channels = 0;
    int hidden = 0;
    int outputs = 0;
    void* out = nullptr;      // y or dx
    float* partial = nullptr;
    long long part_size = 0;
    unsigned* fault = nullptr;
};

// Byte offset of the 16-byte piece `piece` of row `row` in a tile with the 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int piece)
{
    return static_cast<uint32_t>(row * umma::kRowBytes + ((piece ^ (row & 7)) << 4));
}

// N (16 or 32) values of one row, rounded to T, into columns [N part, N part + N) of a tile at shared
// address `tile`.
template <class T, int N>
__device__ __forceinline__ void put_row(uint32_t tile, int row, int part, const float (&v)[N])
{
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
        Floats<8> f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f.p[j] = make_float2(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
        }
        const Vec<T, 8> w = narrow<T>(f);
        const auto* u = reinterpret_cast<const uint32_t*>(&w);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + swizzled(row, N / 8 * part + i)), "r"(u[0]),
                     "r"(u[1]), "r"(u[2]), "r"(u[3])
                     : "memory");
    }
}

// A ring position of N places.
template <int N>
struct Turn {
    int at = 0;
    unsigned phase = 0;
    __device__ __forceinline__ void next()
    {
        if (++at == N) {
            at = 0;
            phase ^= 1u;
        }
    }
};

// This warp is done with what `bar` guards; `writes`: its stores to shared memory come before the
// tensor core's reads.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, bool writes)
{
    if (writes) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    umma::fence_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
        umma::arrive(bar);
    }
}

// The end of an MMA warp that gave up: waits (bounded) for the MMAs it issued.
__device__ __forceinline__ void drain_on_failure(bool ok, uint64_t* bar, unsigned* fault)
{
    if (!ok) {
        umma::commit(bar);
        if (!tma::mbar_wait(bar, 0)) {
            atomicOr(fault, tma::kFaultDrainTimeout);
        }
    }
}

// --- forward -------------------------------------------------------------------------------------------

// The epilogue warps work in two groups of eight, on every second chunk each: a chunk's way from the
// accumulator through the activation to shared memory is mostly latency (one group took 1650 cycles a
// chunk with no activation at all).
constexpr int kGroupWarps = kWarps / 2;

// CK and DK: channels and outputs in 64s (1 or 2).
template <int CK, int DK>
struct Forward {
    static constexpr int kXBytes = CK * kTileBytes;
    static constexpr int kXStages = CK == 1 ? 4 : 2;  // tiles of x in flight or in use
    static constexpr int kChunkBytes = CK * 2 * kWeightBytes + DK * kWeightBytes;  // [Wg; Wu] per 64 channels, Wd
    static constexpr int kFixed = kXStages * kXBytes + 2 * kTileBytes + 2048;
    static constexpr int kYCols = DK * 64;
    static constexpr int smem(int chunks) { return kFixed + chunks * kChunkBytes; }
    // Each CTA takes all of tensor memory: no second one fits an SM's 228 KiB beside it.
    static_assert(2 * (kFixed + kChunkBytes) > 228 * 1024, "one CTA per SM");
};

template <class T, int Act, int CK, int DK>
__global__ void __launch_bounds__(kNarrowThreads, 1)
    narrow_forward_kernel(const __grid_constant__ NarrowMaps maps, const __grid_constant__ NarrowArgs g)
{
    using F = Forward<CK, DK>;
    constexpr bool kBf16 = std::is_same_v<T, bf16>;
    constexpr uint32_t kFirst = umma::instruction(kBf16, false, false, kTileM, 128);
    constexpr uint32_t kSecond = umma::instruction(kBf16, false, false, kTileM, F::kYCols);
    allow_next_grid();
    extern __shared__ unsigned char smem_base[];
    const uint32_t base = (tma::smem_addr(smem_base) + 1023u) & ~1023u;
    const uint32_t xs = base;                       // tiles of x
    const uint32_t hs = xs + F::kXStages * F::kXBytes;  // two chunks of h
    const uint32_t ws = hs + 2 * kTileBytes;        // the weights, by chunk
    __shared__ uint64_t weights_full, x_full[F::kXStages], x_empty[F::kXStages], gu_full[2], gu_empty[2], h_full[2], h_empty[2], y_full[2],
        y_empty[2], drain[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == kWarps) {
        umma::alloc<512>(&tmem_slot);
    }
    if (threadIdx.x == 0) {
        tma::mbar_init(&weights_full, 1);
        for (int i = 0; i < 2; ++i) {
            tma::mbar_init(&drain[i], 1);
            tma::mbar_init(&gu_full[i], 1);
            tma::mbar_init(&gu_empty[i], kGroupWarps);
            tma::mbar_init(&h_full[i], kGroupWarps);
            tma::mbar_init(&h_empty[i], 1);
            tma::mbar_init(&y_full[i], 1);
            tma::mbar_init(&y_empty[i], kGroupWarps);
        }
        for (int i = 0; i < F::kXStages; ++i) {
            tma::mbar_init(&x_full[i], 1);
            tma::mbar_init(&x_empty[i], 1);
        }
        gave_up = 0;
        tma::fence_mbar_init();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    const uint32_t tmem_y = tmem + 256;
    const int chunks = (g.hidden + kHiddenChunk - 1) / kHiddenChunk;
    const int stride = static_cast<int>(gridDim.x);
    const int mine = g.tiles > static_cast<int>(blockIdx.x) ? (g.tiles - static_cast<int>(blockIdx.x) + stride - 1) / stride : 0;
    wait_for_previous_grid();
    bool ok = true;

    if (warp == kWarps) {
        asm volatile("fence.proxy.async.global;" ::: "memory");
        if (umma::elect_one()) {
            tma::mbar_arrive_expect_tx(&weights_full, static_cast<unsigned>(chunks * F::kChunkBytes));
            for (int j = 0; j < chunks; ++j) {
                const uint32_t w = ws + j * F::kChunkBytes;
                for (int c = 0; c < CK; ++c) {
                    umma::load_3d(w + c * 2 * kWeightBytes, &maps.wg, 64 * c, 64 * j, 0, &weights_full);
                    umma::load_3d(w + c * 2 * kWeightBytes + kWeightBytes, &maps.wu, 64 * c, 64 * j, 0, &weights_full);
                }
                for (int d = 0; d < DK; ++d) {
                    umma::load_3d(w + CK * 2 * kWeightBytes + d * kWeightBytes, &maps.wd, 64 * j, 64 * d, 0, &weights_full);
                }
            }
        }
        __syncwarp();
        Turn<F::kXStages> x;
        int issued = 0;
        for (int t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
            ok = tma::mbar_wait(&x_empty[x.at], x.phase ^ 1u);
            if (ok) {
                if (umma::elect_one()) {
                    tma::mbar_arrive_expect_tx(&x_full[x.at], F::kXBytes);
                    for (int c = 0; c < CK; ++c) {
                        umma::load_3d(xs + x.at * F::kXBytes + c * kTileBytes, &maps.x, 64 * c, t * kTileM, 0, &x_full[x.at]);
                    }
                }
                __syncwarp();
                ++issued;
                x.next();
            }
        }
        if (!ok) {  // let the loads in flight land (bounded) before the shared memory is given up
            bool drained = tma::mbar_wait(&weights_full, 0);
            for (int i = issued > F::kXStages ? issued - F::kXStages : 0; i < issued; ++i) {
                drained = tma::mbar_wait(&x_full[i % F::kXStages], static_cast<unsigned>(i / F::kXStages) & 1u) && drained;
            }
            if (lane == 0 && !drained) {
                atomicOr(g.fault, tma::kFaultDrainTimeout);
            }
        }
    } else if (warp == kWarps + 1) {
        if (lane == 0) {  // [G U] of every chunk; a tile's last chunk releases its x
            Turn<F::kXStages> x;
            Turn<2> gu;
            ok = tma::mbar_wait(&weights_full, 0);
            for (int k = 0; ok && k < mine; ++k) {
                ok = tma::mbar_wait(&x_full[x.at], x.phase);
                for (int j = 0; ok && j < chunks; ++j) {
                    ok = tma::mbar_wait(&gu_empty[gu.at], gu.phase ^ 1u);
                    if (!ok) {
                        break;
                    }
                    umma::fence_after_sync();
#pragma unroll
                    for (int c = 0; c < CK; ++c) {
                        const uint64_t da = umma::desc_k(xs + x.at * F::kXBytes + c * kTileBytes);
                        const uint64_t db = umma::desc_k(ws + j * F::kChunkBytes + c * 2 * kWeightBytes);
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            umma::mma(tmem + gu.at * 128, da + umma::kStepK * s, db + umma::kStepK * s, kFirst, c > 0 || s > 0);
                        }
                    }
                    umma::commit(&gu_full[gu.at]);
                    gu.next();
                }
                if (ok) {
                    umma::commit(&x_empty[x.at]);
                    x.next();
                }
            }
            drain_on_failure(ok, &drain[0], g.fault);
        }
    } else if (warp == kWarps + 2) {
        if (lane == 0) {  // y += h Wd^T of every chunk
            Turn<2> h, y;
            ok = tma::mbar_wait(&weights_full, 0);
            for (int k = 0; ok && k < mine; ++k) {
                ok = tma::mbar_wait(&y_empty[y.at], y.phase ^ 1u);
                for (int j = 0; ok && j < chunks; ++j) {
                    ok = tma::mbar_wait(&h_full[h.at], h.phase);
                    if (!ok) {
                        break;
                    }
                    umma::fence_after_sync();
                    const uint64_t da = umma::desc_k(hs + h.at * kTileBytes);
                    const uint64_t db = umma::desc_k(ws + j * F::kChunkBytes + CK * 2 * kWeightBytes);
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        umma::mma(tmem_y + y.at * F::kYCols, da + umma::kStepK * s, db + umma::kStepK * s, kSecond, j > 0 || s > 0);
                    }
                    umma::commit(&h_empty[h.at]);
                    h.next();
                }
                if (ok) {
                    umma::commit(&y_full[y.at]);
                    y.next();
                }
            }
            drain_on_failure(ok, &drain[1], g.fault);
        }
    } else {
        const int group = warp / kGroupWarps;
        const int quad = warp & 3;
        const int half = warp % kGroupWarps >> 2;
        const int row = quad * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const int total = mine * chunks;
        // The outputs of this CTA's k-th tile, once its last product is done. Group k % 2 stores them from
        // accumulator k % 2.
        const auto store_y = [&](int k) {
            ok = tma::mbar_wait(&y_full[group], static_cast<unsigned>(k >> 1) & 1u);
            if (!ok) {
                return;
            }
            umma::fence_after_sync();
            const long long token = (static_cast<long long>(blockIdx.x) + static_cast<long long>(k) * stride) * kTileM + row;
#pragma unroll
            for (int d = 0; d < DK; ++d) {
                float v[32];
                const int col = 64 * d + 32 * half;
                umma::load32(tmem_y + lanes + group * F::kYCols + col, v);
                umma::load_wait(v);
                store_rows(static_cast<T*>(g.out) + (token - lane) * g.outputs + col, g.outputs, v, g.tokens - (token - lane),
                           g.outputs - col);
            }
            warp_arrive(&y_empty[group], false);
        };
        int stored = group;  // the group's next tile to store
        for (int n = group; ok && n < total; n += 2) {
            const unsigned phase = static_cast<unsigned>(n >> 1) & 1u;  // buffer n % 2 is this group's
            ok = tma::mbar_wait(&gu_full[group], phase);
            if (!ok) {
                break;
            }
            umma::fence_after_sync();
            float a[32], u[32];
            umma::load32(tmem + lanes + group * 128 + 32 * half, a);
            umma::load32(tmem + lanes + group * 128 + 64 + 32 * half, u);
            umma::load_wait(a);
            umma::load_wait(u);
            warp_arrive(&gu_empty[group], false);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const float2 v = activate2<Act, T>(make_float2(a[i], a[i + 1])) * make_float2(u[i], u[i + 1]);
                a[i] = v.x;
                a[i + 1] = v.y;
            }
            ok = tma::mbar_wait(&h_empty[group], phase ^ 1u);
            if (!ok) {
                break;
            }
            put_row<T>(hs + group * kTileBytes, row, half, a);
            warp_arrive(&h_full[group], true);
            // A tile whose last chunk is behind this one needs nothing more of this group.
            if ((stored + 1) * chunks <= n) {
                store_y(stored);
                stored += 2;
            }
        }
        for (; ok && stored < mine; stored += 2) {
            store_y(stored);
        }
    }
    if (!ok && lane == 0) {
        gave_up = 1;
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (threadIdx.x == 0 && gave_up != 0) {
        atomicOr(g.fault, tma::kFaultWaitTimeout);
    }
    if (warp == kWarps) {
        umma::dealloc<512>(tmem);
    }
}

// --- backward ------------------------------------------------------------------------------------------

constexpr int kBackHidden = 128;   // at most: two chunks
constexpr int kBackWidth = 64;     // channels and outputs, at most
// Shared memory: three stages of x and dy (a tile's stage is held until its weight gradients are done), the weights (Wg, Wu, Wd of each chunk), one chunk's dG
// and dU, both chunks' h.
constexpr int kBackStages = 3;
constexpr int kBackChunkWeights = 3 * kWeightBytes;
constexpr int kBackSmem = 2 * kBackStages * kTileBytes + 2 * kBackChunkWeights + 4 * kTileBytes + 2048;
static_assert(kBackSmem <= kMaxSmem, "shared memory");
static_assert(2 * kBackSmem > 228 * 1024, "one CTA per SM, which takes all of tensor memory");
// Tensor memory columns.
constexpr int kColDx = 192;        // two accumulators of 64
constexpr int kColGateUp = 320;    // two chunks of 64
constexpr int kColDown = 448;

template <class T, int Act>
__global__ void __launch_bounds__(kNarrowThreads, 1)
    narrow_backward_kernel(const __grid_constant__ NarrowMaps maps, const __grid_constant__ NarrowArgs g)
{
    constexpr bool kBf16 = std::is_same_v<T, bf16>;
    constexpr uint32_t kGateUp = umma::instruction(kBf16, false, false, kTileM, 128);  // x [Wg; Wu]^T
    constexpr uint32_t kThrough = umma::instruction(kBf16, false, true, kTileM, 64);   // dy Wd, dG Wg, dU Wu
    constexpr uint32_t kGradient = umma::instruction(kBf16, true, true, 128, 64);      // [dG dU]^T x, h^T dy
    allow_next_grid();
    extern __shared__ unsigned char smem_base[];
    const uint32_t base = (tma::smem_addr(smem_base) + 1023u) & ~1023u;
    const uint32_t ins = base;                          // [stage][x, dy]
    const uint32_t ws = ins + 2 * kBackStages * kTileBytes;  // [chunk][Wg, Wu, Wd]
    const uint32_t dgs = ws + 2 * kBackChunkWeights;    // [dG, dU]
    const uint32_t hs = dgs + 2 * kTileBytes;           // [chunk]
    __shared__ uint64_t weights_full, in_full[kBackStages], in_empty[kBackStages], acc_full, acc_empty, hidden_full[2], dgu_empty, h_empty,
        dx_full[2], dx_empty[2], all_done, drain[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == kWarps) {
        umma::alloc<512>(&tmem_slot);
    }
    if (threadIdx.x == 0) {
        tma::mbar_init(&weights_full, 1);
        tma::mbar_init(&acc_full, 1);
        tma::mbar_init(&acc_empty, kWarps);
        tma::mbar_init(&all_done, 1);
        tma::mbar_init(&h_empty, 1);
        tma::mbar_init(&dgu_empty, 1);
        for (int i = 0; i < kBackStages; ++i) {
            tma::mbar_init(&in_full[i], 1);
            tma::mbar_init(&in_empty[i], 2);  // both MMA warps
        }
        for (int i = 0; i < 2; ++i) {
            tma::mbar_init(&drain[i], 1);
            tma::mbar_init(&hidden_full[i], kWarps);
            tma::mbar_init(&dx_full[i], 1);
            tma::mbar_init(&dx_empty[i], kWarps);
        }
        gave_up = 0;
        tma::fence_mbar_init();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    const int chunks = (g.hidden + kHiddenChunk - 1) / kHiddenChunk;
    const int first_tile = static_cast<int>(blockIdx.x);
    const int stride = static_cast<int>(gridDim.x);
    const int mine = g.tiles > first_tile ? (g.tiles - first_tile + stride - 1) / stride : 0;
    wait_for_previous_grid();
    bool ok = true;

    if (warp == kWarps) {
        asm volatile("fence.proxy.async.global;" ::: "memory");
        if (umma::elect_one()) {
            tma::mbar_arrive_expect_tx(&weights_full, static_cast<unsigned>(chunks * kBackChunkWeights));
            for (int j = 0; j < chunks; ++j) {
                const uint32_t w = ws + j * kBackChunkWeights;
                umma::load_3d(w, &maps.wg, 0, 64 * j, 0, &weights_full);
                umma::load_3d(w + kWeightBytes, &maps.wu, 0, 64 * j, 0, &weights_full);
                umma::load_3d(w + 2 * kWeightBytes, &maps.wd, 64 * j, 0, 0, &weights_full);
            }
        }
        __syncwarp();
        Turn<kBackStages> in;
        int issued = 0;
        for (int k = 0; ok && k < mine; ++k) {
            ok = tma::mbar_wait(&in_empty[in.at], in.phase ^ 1u);
            if (ok) {
                const int row = (first_tile + k * stride) * kTileM;
                const uint32_t dst = ins + in.at * 2 * kTileBytes;
                if (umma::elect_one()) {
                    tma::mbar_arrive_expect_tx(&in_full[in.at], 2 * kTileBytes);
                    umma::load_3d(dst, &maps.x, 0, row, 0, &in_full[in.at]);
                    umma::load_3d(dst + kTileBytes, &maps.dy, 0, row, 0, &in_full[in.at]);
                }
                __syncwarp();
                ++issued;
                in.next();
            }
        }
        if (!ok) {
            bool drained = tma::mbar_wait(&weights_full, 0);
            for (int i = issued > kBackStages ? issued - kBackStages : 0; i < issued; ++i) {
                drained = tma::mbar_wait(&in_full[i % kBackStages], static_cast<unsigned>(i / kBackStages) & 1u) && drained;
            }
            if (lane == 0 && !drained) {
                atomicOr(g.fault, tma::kFaultDrainTimeout);
            }
        }
    } else if (warp == kWarps + 1) {
        if (lane == 0) {  // G, U and dh of every chunk
            Turn<kBackStages> in;
            Turn<1> acc;
            ok = tma::mbar_wait(&weights_full, 0);
            for (int k = 0; ok && k < mine; ++k) {
                ok = tma::mbar_wait(&in_full[in.at], in.phase);
                const uint64_t dx = umma::desc_k(ins + in.at * 2 * kTileBytes);
                const uint64_t ddy = umma::desc_k(ins + in.at * 2 * kTileBytes + kTileBytes);
                for (int j = 0; ok && j < chunks; ++j) {
                    ok = tma::mbar_wait(&acc_empty, acc.phase ^ 1u);
                    if (!ok) {
                        break;
                    }
                    umma::fence_after_sync();
                    const uint64_t dw = umma::desc_k(ws + j * kBackChunkWeights);
                    const uint64_t dwd = umma::desc_mn<kWeightBytes>(ws + j * kBackChunkWeights + 2 * kWeightBytes);
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        umma::mma(tmem, dx + umma::kStepK * s, dw + umma::kStepK * s, kGateUp, s > 0);
                    }
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        umma::mma(tmem + 128, ddy + umma::kStepK * s, dwd + umma::kStepMn * s, kThrough, s > 0);
                    }
                    umma::commit(&acc_full);
                    acc.next();
                }
                if (ok) {
                    umma::commit(&in_empty[in.at]);
                    in.next();
                }
            }
            drain_on_failure(ok, &drain[0], g.fault);
        }
    } else if (warp == kWarps + 2) {
        if (lane == 0) {  // dx and the weight gradients
            Turn<kBackStages> in;
            Turn<2> dx;
            Turn<1> hidden;
            ok = tma::mbar_wait(&weights_full, 0);
            for (int k = 0; ok && k < mine; ++k) {
                ok = tma::mbar_wait(&in_full[in.at], in.phase) && tma::mbar_wait(&dx_empty[dx.at], dx.phase ^ 1u);
                const uint32_t x = ins + in.at * 2 * kTileBytes;
                const uint64_t x_mn = umma::desc_mn<kTileBytes>(x);
                for (int j = 0; ok && j < chunks; ++j) {
                    ok = tma::mbar_wait(&hidden_full[j], hidden.phase);
                    if (!ok) {
                        break;
                    }
                    umma::fence_after_sync();
                    if (j == chunks - 1) {
                        // First, as the next tile's first hidden values wait for it. With one chunk only,
                        // the second half of M reads the other chunk's tile, which the epilogue zeroed.
                        const uint64_t dh = umma::desc_mn<kTileBytes>(hs), dy_mn = umma::desc_mn<kTileBytes>(x + kTileBytes);
#pragma unroll
                        for (int s = 0; s < 8; ++s) {
                            umma::mma(tmem + kColDown, dh + umma::kStepMn * s, dy_mn + umma::kStepMn * s, kGradient,
                                      k > 0 || s > 0);
                        }
                        umma::commit(&h_empty);
                    }
                    const uint32_t w = ws + j * kBackChunkWeights;
                    const uint32_t dg = dgs;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // dG Wg, then dU Wu
                        const uint64_t da = umma::desc_k(dg + i * kTileBytes);
                        const uint64_t db = umma::desc_mn<kWeightBytes>(w + i * kWeightBytes);
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            umma::mma(tmem + kColDx + dx.at * 64, da + umma::kStepK * s, db + umma::kStepMn * s, kThrough,
                                      j > 0 || i > 0 || s > 0);
                        }
                    }
                    if (j == chunks - 1) {
                        umma::commit(&dx_full[dx.at]);
                    }
                    const uint64_t dgu = umma::desc_mn<kTileBytes>(dg);
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        umma::mma(tmem + kColGateUp + j * 64, dgu + umma::kStepMn * s, x_mn + umma::kStepMn * s, kGradient,
                                  k > 0 || s > 0);
                    }
                    umma::commit(&dgu_empty);
                }
                if (!ok) {
                    break;
                }
                umma::commit(&in_empty[in.at]);
                in.next();
                dx.next();
                hidden.next();
            }
            if (ok) {
                umma::commit(&all_done);
            }
            drain_on_failure(ok, &drain[1], g.fault);
        }
    } else {
        const int quad = warp & 3;
        const int part = warp >> 2;  // 16 of a chunk's 64 columns
        const int row = quad * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        if (chunks == 1) {  // the other chunk's h takes part in the last product
            const float zero[16] = {};
            put_row<T>(hs + kTileBytes, row, part, zero);
        }
        Turn<1> acc, dgu, hidden;
        Turn<2> dx;
        const auto store_dx = [&](int t) {
            ok = tma::mbar_wait(&dx_full[dx.at], dx.phase);
            if (!ok) {
                return;
            }
            umma::fence_after_sync();
            float v[16];
            umma::load16(tmem + lanes + kColDx + dx.at * 64 + 16 * part, v);
            umma::load_wait(v);
            warp_arrive(&dx_empty[dx.at], false);
            dx.next();
            const long long token = static_cast<long long>(t) * kTileM + row;
            const int col = 16 * part;
            store_rows(static_cast<T*>(g.out) + (token - lane) * g.channels + col, g.channels, v, g.tokens - (token - lane),
                       g.channels - col);
        };
        int before = -1;
        for (int k = 0; ok && k < mine; ++k) {
            for (int j = 0; ok && j < chunks; ++j) {
                ok = tma::mbar_wait(&acc_full, acc.phase);
                if (!ok) {
                    break;
                }
                umma::fence_after_sync();
                float a[16], u[16], dh[16];
                umma::load16(tmem + lanes + 16 * part, a);
                umma::load16(tmem + lanes + 64 + 16 * part, u);
                umma::load16(tmem + lanes + 128 + 16 * part, dh);
                umma::load_wait(a);
                umma::load_wait(u);
                umma::load_wait(dh);
                warp_arrive(&acc_empty, false);
                acc.next();
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float2 slope;
                    const float2 up = make_float2(u[i], u[i + 1]);
                    const float2 d = make_float2(dh[i], dh[i + 1]);
                    const float2 v = activate_slope2<Act, T>(make_float2(a[i], a[i + 1]), slope);
                    const float2 dg = d * up * slope, h = v * up, du = d * v;
                    a[i] = dg.x;
                    a[i + 1] = dg.y;
                    u[i] = h.x;
                    u[i + 1] = h.y;
                    dh[i] = du.x;
                    dh[i + 1] = du.y;
                }
                ok = tma::mbar_wait(&dgu_empty, dgu.phase ^ 1u);
                if (!ok) {
                    break;
                }
                dgu.next();
                put_row<T>(dgs, row, part, a);
                put_row<T>(dgs + kTileBytes, row, part, dh);
                ok = j > 0 || tma::mbar_wait(&h_empty, hidden.phase ^ 1u);
                if (!ok) {
                    break;
                }
                put_row<T>(hs + j * kTileBytes, row, part, u);
                warp_arrive(&hidden_full[j], true);
                if (j == 0 && before >= 0) {
                    store_dx(before);
                    before = -1;
                }
            }
            hidden.next();
            before = first_tile + k * stride;
        }
        if (ok && before >= 0) {
            store_dx(before);
        }
        // The CTA's part of the weight gradients: lanes 0-63 of a chunk's accumulator are dWg's rows,
        // 64-127 dWu's; the last one is dWd transposed.
        if (ok && mine > 0) {
            ok = tma::mbar_wait(&all_done, 0);
        }
        if (ok) {
            umma::fence_after_sync();
            float* sums = g.partial + blockIdx.x * g.part_size;
            const long long size = static_cast<long long>(g.hidden) * g.channels;
            const int col = 16 * part;
            for (int j = 0; j < chunks; ++j) {
                float v[16] = {};
                if (mine > 0) {
                    umma::load16(tmem + lanes + kColGateUp + 64 * j + col, v);
                    umma::load_wait(v);
                }
                const int f = 64 * j + (row & 63);
                if (f < g.hidden && col < g.channels) {
                    store_values<float>(sums + (row >> 6) * size + static_cast<long long>(f) * g.channels + col, v,
                                        min(16, g.channels - col));
                }
            }
            float v[16] = {};
            if (mine > 0) {
                umma::load16(tmem + lanes + kColDown + col, v);
                umma::load_wait(v);
            }
            if (row < g.hidden) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (col + i < g.outputs) {
                        sums[2 * size + static_cast<long long>(col + i) * g.hidden + row] = v[i];
                    }
                }
            }
        }
    }
    if (!ok && lane == 0) {
        gave_up = 1;
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (threadIdx.x == 0 && gave_up != 0) {
        atomicOr(g.fault, tma::kFaultWaitTimeout);
    }
    if (warp == kWarps) {
        umma::dealloc<512>(tmem);
    }
}

// --- host ----------------------------------------------------------------------------------------------

int tile_count(const MlpShape& n) { return static_cast<int>((n.tokens + kTileM - 1) / kTileM); }

NarrowArgs arguments(const MlpShape& n, void* out)
{
    NarrowArgs g;
    g.tokens = n.tokens;
    g.tiles = tile_count(n);
    g.channels = n.channels;
    g.hidden = n.hidden;
    g.outputs = n.outputs;
    g.out = out;
    g.fault = device_fault_word();
    return g;
}

template <auto Kernel>
void launch(int ctas, int smem, const NarrowMaps& maps, const NarrowArgs& g, cudaStream_t stream)
{
    static std::atomic<bool> opted[kMaxDevices];
    const int device = current_device();
    if (!opted[device].load(std::memory_order_relaxed)) {
        SPECTRAL_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem - 1024));
        opted[device].store(true, std::memory_order_relaxed);
    }
    launch_pdl(Kernel, dim3(static_cast<unsigned>(ctas)), dim3(kNarrowThreads), static_cast<std::size_t>(smem), stream, maps, g);
}

int forward_smem(const MlpShape& n)
{
    const int chunks = (n.hidden + kHiddenChunk - 1) / kHiddenChunk;
    const bool c2 = n.channels > 64, d2 = n.outputs > 64;
    return c2 ? (d2 ? Forward<2, 2>::smem(chunks) : Forward<2, 1>::smem(chunks))
              : (d2 ? Forward<1, 2>::smem(chunks) : Forward<1, 1>::smem(chunks));
}

template <class F>
void with_16_bits(int dtype, F&& f)
{
    if (dtype == SPECTRAL_BFLOAT16) {
        f(bf16{});
    } else {
        f(f16{});
    }
}

}  // namespace

bool narrow_forward_fits(const MlpShape& n, int dtype)
{
    return dtype != SPECTRAL_FLOAT32 && n.channels <= 128 && n.outputs <= 128 && n.hidden <= 1024
           && forward_smem(n) <= kMaxSmem - 1024;
}

void narrow_forward(const Matrix& x, const Matrix& wg, const Matrix& wu, const Matrix& wd, void* y, int dtype,
                    const MlpShape& n, cudaStream_t stream)
{
    NarrowMaps maps{};
    maps.x = x.map(kTileM);
    maps.wg = wg.map(kHiddenChunk);
    maps.wu = wu.map(kHiddenChunk);
    maps.wd = wd.map(64);
    const NarrowArgs g = arguments(n, y);
    const int ctas = std::min(g.tiles, device_sm_count(current_device()));
    const int smem = forward_smem(n);
    with_16_bits(dtype, [&](auto type) {
        using T = decltype(type);
        with_activation(n.act, [&](auto act) {
            constexpr int Act = decltype(act)::value;
            const bool c2 = n.channels > 64, d2 = n.outputs > 64;
            if (c2 && d2) {
                launch<narrow_forward_kernel<T, Act, 2, 2>>(ctas, smem, maps, g, stream);
            } else if (c2) {
                launch<narrow_forward_kernel<T, Act, 2, 1>>(ctas, smem, maps, g, stream);
            } else if (d2) {
                launch<narrow_forward_kernel<T, Act, 1, 2>>(ctas, smem, maps, g, stream);
            } else {
                launch<narrow_forward_kernel<T, Act, 1, 1>>(ctas, smem, maps, g, stream);
            }
        });
    });
}

bool narrow_backward_fits(const MlpShape& n, int dtype)
{
    return dtype != SPECTRAL_FLOAT32 && n.channels <= kBackWidth && n.outputs <= kBackWidth && n.hidden <= kBackHidden;
}

// The weight gradients' accumulators take 8 MMAs per tile (128 tokens) over all of a CTA's tiles, so a call of very
// many tokens is cut into ranges of as many tiles each, a launch with parts of its own (kLongSum; 1.2 M tokens).
constexpr int kBackCtas = 148;
constexpr int kRangeTiles = kLongSum / (kTileM / 16) * kBackCtas;
int backward_ranges(const MlpShape& n) { return std::max(1, (tile_count(n) + kRangeTiles - 1) / kRangeTiles); }
int range_tiles(const MlpShape& n) { return (tile_count(n) + backward_ranges(n) - 1) / backward_ranges(n); }

int narrow_backward_parts(const MlpShape& n)
{
    const int ranges = backward_ranges(n), each = range_tiles(n);
    return (ranges - 1) * std::min(each, kBackCtas) + std::min(tile_count(n) - (ranges - 1) * each, kBackCtas);
}

void narrow_backward(const Matrix& dy, const Matrix& x, const Matrix& wg, const Matrix& wu, const Matrix& wd, void* dx,
                     float* partial, int dtype, const MlpShape& n, cudaStream_t stream)
{
    const int each = range_tiles(n);
    for (int first = 0; first < tile_count(n); first += each) {
        const long long start = static_cast<long long>(first) * kTileM;
        MlpShape part = n;
        part.tokens = std::min(n.tokens - start, static_cast<long long>(each) * kTileM);
        const auto rows = [&](Matrix m) {  // the range's rows of x or dy
            m.base = static_cast<const char*>(m.base) + start * m.pitch * 2;
            m.rows = part.tokens;
            return m.map(kTileM);
        };
        NarrowMaps maps{};
        maps.x = rows(x);
        maps.dy = rows(dy);
        maps.wg = wg.map(kHiddenChunk);
        maps.wu = wu.map(kHiddenChunk);
        maps.wd = wd.map(64);
        NarrowArgs g = arguments(part, static_cast<char*>(dx) + start * n.channels * 2);
        const int ctas = std::min(g.tiles, kBackCtas);
        g.partial = partial;
        g.part_size = 2LL * n.hidden * n.channels + static_cast<long long>(n.outputs) * n.hidden;
        with_16_bits(dtype, [&](auto type) {
            using T = decltype(type);
            with_activation(n.act, [&](auto act) {
                constexpr int Act = decltype(act)::value;
                launch<narrow_backward_kernel<T, Act>>(ctas, kBackSmem, maps, g, stream);
            });
        });
        partial += ctas * g.part_size;
    }
}

}  // namespace spectral::mlp
