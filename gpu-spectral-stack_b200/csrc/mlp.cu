// The gated feed-forward block, y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its gradients, as tcgen05
// matrix products with the pointwise work in their epilogues.
//
// Forward (M tokens, C channels, F hidden, D outputs):
//   gate       G = x Wg^T and U = x Wu^T in one kernel (one MMA of N = 256 over the stacked tiles
//              [Wg; Wu]); its epilogue stores h = act(G) * U, so neither product reaches HBM
//   down       y = h Wd^T
// Backward, from x (or its 8-bit checkpoint) and dy alone:
//   gate back  G, U and dh = dy Wd in one kernel; its epilogue stores dU = dh act(G),
//              dG = dh U act'(G) and h
//   input      dx = dG Wg + dU Wu, one sum over both products
//   weights    dWg = dG^T x, dWu = dU^T x, dWd = dy^T h, K = tokens: the token range is cut into
//              parts, FP32 partial products are added up in a fixed order by a last kernel
// Weights and activations are used as they lie: a product that needs a transposed operand reads
// the same TMA tile through an MN-major descriptor (umma.cuh), nothing is transposed in memory.
//
// One kernel template serves the products: persistent CTAs (one per SM), a TMA warp, an MMA warp
// (one elected lane issues) and eight or sixteen epilogue warps; tiles of 128 rows (256 where that pays), K in
// chunks of 64, kStages chunks in flight; two accumulator sets in tensor memory where they fit, so a
// tile's epilogue runs under the next tile's products. 8192 x 512 x 2048 bf16: forward 43 us (51.5
// GFLOP, 1.2 PFLOP/s), backward 146 us (with the recomputed products 137 GFLOP, 0.94 PFLOP/s). Every wait is bounded (tma.cuh).
//
// Types: bf16 and f16 run as they are, accumulated in FP32; h, dG and dU are rounded once to the
// type, as they feed the next product. With the rounding of the result that is 1.4 times the error of
// rounding the result alone; a second 16-bit part of them would double those products. float32 operands are split into three bf16 parts
// (24 significand bits, bf16 has FP32's range) and the six products of order up to 2 (hi hi, hi
// mid, mid hi, mid mid, hi lo, lo hi) are taken: the dropped ones are below 2^-24 of the product.
// The tensor core cuts its FP32 accumulator once per MMA, an error that grows with K, so float32
// products run in passes of 128 values of K: the five small products first, hi hi last, and the
// epilogue warps add the passes up in registers (rounded to nearest). One pass over all of K left
// an error of 4.3e-6 at K = 100 and 270.
//
// A few tokens: matrix tiles would be mostly padding, and the weights are all there is to read.
// Two kernels read each weight row once with 16-byte loads, all lanes of a warp on one row, h
// in FP32 in between.

#include "../../include/spectral_b200.h"

#include "mlp.cuh"

#include <algorithm>

namespace spectral {

void unpack8(const signed char* codes, const float* scales, void* x, int dtype, long long rows, int width,
             cudaStream_t stream);

namespace {

using namespace mlp;

constexpr long long kMaxTokens = 0x7fffff00LL;  // 32-bit TMA coordinates

// --- staging ---------------------------------------------------------------------------------------

// Matrices of T to copy into the operand form: planes of the operand type, `pitch` values a row (a
// multiple of 8). For arrays TMA cannot read as they lie: float32, or rows that are not 16-byte
// pieces. One launch for all of a call's (blockIdx.y).
struct StageJob {
    const void* src;
    void* dst;
    long long rows;
    int cols;
    int pitch;
};
struct StageJobs {
    StageJob job[5];
    int count = 0;
};

// A warp copies 256 values at a time, some whole rows or a part of one: single values loaded in a row,
// through shared memory, eight stored at once. (Eight loads side by side per thread took 262 us for 47519 x 895
// bf16.)
constexpr int kStageValues = 256;

template <class T>
__global__ void __launch_bounds__(256) stage_kernel(const __grid_constant__ StageJobs jobs)
{
    __shared__ float rows_of[8][kStageValues];
    const StageJob& job = jobs.job[blockIdx.y];
    const T* __restrict__ src = static_cast<const T*>(job.src);
    auto* __restrict__ dst = static_cast<typename Operand<T>::Type*>(job.dst);
    const long long rows = job.rows;
    const int cols = job.cols;
    const int pitch = job.pitch;
    allow_next_grid();
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31;
    float* buf = rows_of[threadIdx.x >> 5];
    const int at_once = pitch <= kStageValues ? kStageValues / pitch : 1;  // rows
    const int parts = (pitch + kStageValues - 1) / kStageValues;           // of a row
    const long long total = (rows + at_once - 1) / at_once * parts;
    // This lane's eight values, among the rows at once or in the part.
    const int r = parts == 1 ? lane * 8 / pitch : 0;
    const int c = lane * 8 - r * pitch;
    for (long long i = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); i < total;
         i += static_cast<long long>(gridDim.x) * 8) {
        const long long first = i / parts;
        const long long row0 = first * at_once;
        const int c0 = static_cast<int>(i - first * parts) * kStageValues;
        const int have = parts == 1 ? static_cast<int>(min(static_cast<long long>(at_once), rows - row0)) * cols
                                    : min(kStageValues, cols - c0);
        const T* from = src + row0 * cols + c0;
#pragma unroll
        for (int j = 0; j < kStageValues / 32; ++j) {
            const int e = 32 * j + lane;
            buf[e] = e < have ? to_float(from[e]) : 0.0f;
        }
        __syncwarp();
        const long long row = row0 + r;
        if (r < at_once && row < rows && c0 + c < pitch) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = c0 + c + j < cols ? buf[r * cols + c + j] : 0.0f;
            }
            const long long at = row * pitch + c0 + c;
            if constexpr (sizeof(T) == 4) {
                Vec<bf16, 8> hi, mid, lo;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    split3(v[j], hi.v[j], mid.v[j], lo.v[j]);
                }
                *reinterpret_cast<Vec<bf16, 8>*>(dst + at) = hi;
                *reinterpret_cast<Vec<bf16, 8>*>(dst + rows * pitch + at) = mid;
                *reinterpret_cast<Vec<bf16, 8>*>(dst + 2 * rows * pitch + at) = lo;
            } else {
                Vec<T, 8> out;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    out.v[j] = from_float<T>(v[j]);
                }
                *reinterpret_cast<Vec<T, 8>*>(dst + at) = out;
            }
        }
        __syncwarp();
    }
}

// --- epilogue stores ---------------------------------------------------------------------------------

// A run of hidden values in the operand form (planes `plane` values apart).
template <class T, int N>
__device__ __forceinline__ void store_hidden(typename Operand<T>::Type* p, long long plane, const float (&v)[N], int valid)
{
    if constexpr (sizeof(T) == 4) {
        bf16 hi[N], mid[N], lo[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            split3(v[j], hi[j], mid[j], lo[j]);
        }
        store_run(p, hi, valid);
        store_run(p + plane, mid, valid);
        store_run(p + 2 * plane, lo, valid);
    } else {
        T out[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            out[j] = from_float<T>(v[j]);
        }
        store_run(p, out, valid);
    }
}

// --- the matrix-product kernel -----------------------------------------------------------------------

enum class Kind {
    kGate,      // A = x, B = [Wg; Wu] (K-major): h
    kGateBack,  // A = x, B = [Wg; Wu], then A = dy, B = Wd (MN-major): dG, dU, h
    kDown,      // A = h, B = Wd (K-major): y
    kInput,     // A = dG, B = Wg, then A = dU, B = Wu (MN-major): dx
    kWeight,    // three problems, A and B MN-major, K = tokens: FP32 partial products
};

struct Maps {
    CUtensorMap a[3];
    CUtensorMap b[3];
};

struct Args {
    int rows = 0;         // of the output (M)
    int cols = 0;         // per accumulator (N)
    int m_tiles = 0;
    int n_tiles = 0;
    long long tiles = 0;
    int chunks[2] = {0, 0};  // K chunks of the one or two operand pairs
    void* out[3] = {nullptr, nullptr, nullptr};
    long long pitch = 0;  // of the output rows, in values
    long long plane = 0;  // of the hidden arrays, in values
    // kWeight: problem p is rows_of[p] x cols_of[p]; tiles [first[p], first[p + 1]) of one part.
    int rows_of[3] = {0, 0, 0};
    int cols_of[3] = {0, 0, 0};
    int n_tiles_of[3] = {0, 0, 0};
    long long first[4] = {0, 0, 0, 0};
    int parts = 1;
    int part_chunks = 0;
    long long part_size = 0;  // floats of one part's three products
    long long offset[3] = {0, 0, 0};
    unsigned* fault = nullptr;
};

// A tile is MT x 128 rows by BN columns (of each accumulator). Two accumulator sets where tensor memory
// holds them, so that a tile's epilogue runs under the next tile's products.
template <Kind K, int BN, int MT, class T>
struct Config {
    // The activation's epilogues wait on special functions and tensor memory: sixteen warps in 16-bit types, each
    // a quarter of the columns in runs of 16 (16384 x 256 x 1024 backward 100 us, with eight 115 us; float32
    // sums need the registers of eight).
    static constexpr bool kActs = sizeof(T) == 2 && (K == Kind::kGate || K == Kind::kGateBack);
    static constexpr int kEpilogueWarps = kActs ? 16 : 8;
    static constexpr int kThreads = 32 * (kEpilogueWarps + 2);
    static constexpr int kRun = kActs ? 16 : 32;                   // columns of a row at a time
    static constexpr int kColumns = BN / (kEpilogueWarps / 4);     // a warp's
    static constexpr bool kAMn = K == Kind::kWeight;
    static constexpr int kSets = K == Kind::kGate ? 2 : K == Kind::kGateBack ? 3 : 1;  // accumulators of BN columns
    static constexpr int kBRows = K == Kind::kGate || K == Kind::kGateBack ? 2 * BN : BN;
    static constexpr int kRows = MT * kTileM;
    static constexpr int kABytes = MT * kTileABytes;
    static constexpr int kBBytes = kBRows * umma::kRowBytes;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = (kMaxSmem - 2048) / kStageBytes > 6 ? 6 : (kMaxSmem - 2048) / kStageBytes;
    static constexpr int kCols = kSets * BN * MT;
    static constexpr int kSlots = 2 * kCols <= 512 ? 2 : 1;
    static constexpr int kUsed = kSlots * kCols;
    static constexpr int kTmemCols = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static constexpr int kSmem = kStages * kStageBytes + 2048;  // barriers, and slack for the 1 KiB base
    static_assert(kUsed <= 512, "tensor memory");
    static_assert(MT == 1 || kSets == 1, "row tiles of one accumulator each");
};

// Tile t: output rows from m0, columns from n0, chunks [k0, k1) (kWeight: of problem p and part `part`).
struct Tile {
    int m0;
    int n0;
    int k0;
    int k1;
    int problem;
    int part;
    int passes;
};

// float32 dx: its two products take passes of their own, alternately, or the second's small products
// would be cut against the first's sum (an error of 1.3e-6 instead of 3e-7).
template <Kind K, class T>
constexpr bool kApart = K == Kind::kInput && sizeof(T) == 4;

// Chunks of K whose products share an accumulator.
template <Kind K, class T>
constexpr int kPass = K == Kind::kWeight && sizeof(T) == 2 ? kLongSum * 16 / kChunk : Operand<T>::kPassChunks;

// The chunks of operand pair `pair` that pass `pass` of a tile covers.
template <Kind K, class T>
__device__ __forceinline__ void pass_range(const Args& g, const Tile& tile, int pair, int pass, int& begin, int& end)
{
    constexpr int kStep = kPass<K, T>;
    const int last = pair == 0 ? tile.k1 : g.chunks[1];
    begin = min((pair == 0 ? tile.k0 : 0) + pass * kStep, last);
    end = min(begin + kStep, last);
}

template <Kind K, int BN, int MT, class T>
__device__ __forceinline__ Tile locate(const Args& g, long long t)
{
    Tile tile{0, 0, 0, g.chunks[0], 0, 0, 1};
    if constexpr (K == Kind::kWeight) {
        tile.part = static_cast<int>(t / g.first[3]);
        const long long r = t - tile.part * g.first[3];
        tile.problem = r >= g.first[2] ? 2 : r >= g.first[1] ? 1 : 0;
        const int i = static_cast<int>(r - g.first[tile.problem]);
        tile.m0 = i / g.n_tiles_of[tile.problem] * (MT * kTileM);
        tile.n0 = i % g.n_tiles_of[tile.problem] * BN;
        tile.k0 = tile.part * g.part_chunks;
        tile.k1 = min(tile.k0 + g.part_chunks, g.chunks[0]);
    } else {
        tile.m0 = static_cast<int>(t / g.n_tiles) * (MT * kTileM);
        tile.n0 = static_cast<int>(t % g.n_tiles) * BN;
    }
    if constexpr (sizeof(T) == 4 || K == Kind::kWeight) {
        constexpr int kStep = kPass<K, T>;
        tile.passes = (max(tile.k1 - tile.k0, g.chunks[1]) + kStep - 1) / kStep;
    }
    return tile;
}

// Results of one accumulator: the warp's 32 rows from row - lane on, 32 columns from col on; `add` (kWeight): to those
// of the passes before.
template <Kind K, class T>
__device__ __forceinline__ void store_results(const Args& g, const Tile& tile, int row, int rows, int col, int cols, float (&acc)[32],
                                              bool add = false)
{
    using Out = std::conditional_t<K == Kind::kWeight, float, T>;
    const int lane = threadIdx.x & 31;
    const long long pitch = K == Kind::kWeight ? cols : g.pitch;
    Out* out = static_cast<Out*>(g.out[0]) + (K == Kind::kWeight ? tile.part * g.part_size + g.offset[tile.problem] : 0);
    const int first = row - lane;
    store_rows(out + static_cast<long long>(first) * pitch + col, pitch, acc, rows - first, cols - col,
               K == Kind::kWeight && add);
}

// The epilogue of the gate kernels, N columns of one row from col on: acc holds each accumulator's values.
template <Kind K, class T, int Act, int Sets, int N>
__device__ __forceinline__ void finish(const Args& g, const Tile& tile, int row, int col, int cols, float (&acc)[Sets][N])
{
    using Op = typename Operand<T>::Type;
    const int valid = min(N, cols - col);
    const long long at = row * g.pitch + col;
    if constexpr (K == Kind::kGate) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float2 h = activate2<Act, T>(make_float2(acc[0][j], acc[0][j + 1])) * make_float2(acc[1][j], acc[1][j + 1]);
            acc[0][j] = h.x;
            acc[0][j + 1] = h.y;
        }
        store_hidden<T>(static_cast<Op*>(g.out[0]) + at, g.plane, acc[0], valid);
    } else if constexpr (K == Kind::kGateBack) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            float2 slope;
            const float2 up = make_float2(acc[1][j], acc[1][j + 1]);
            const float2 dh = make_float2(acc[2][j], acc[2][j + 1]);
            const float2 a = activate_slope2<Act, T>(make_float2(acc[0][j], acc[0][j + 1]), slope);
            const float2 dg = dh * up * slope, h = a * up, du = dh * a;
            acc[0][j] = dg.x;
            acc[0][j + 1] = dg.y;
            acc[1][j] = h.x;
            acc[1][j + 1] = h.y;
            acc[2][j] = du.x;
            acc[2][j + 1] = du.y;
        }
        store_hidden<T>(static_cast<Op*>(g.out[0]) + at, g.plane, acc[0], valid);
        store_hidden<T>(static_cast<Op*>(g.out[1]) + at, g.plane, acc[2], valid);
        store_hidden<T>(static_cast<Op*>(g.out[2]) + at, g.plane, acc[1], valid);
    }
}

template <Kind K, int BN, int MT, class T, int Act>
__global__ void __launch_bounds__(Config<K, BN, MT, T>::kThreads, 1) product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g)
{
    using Cfg = Config<K, BN, MT, T>;
    using Op = Operand<T>;
    constexpr bool kBf16 = std::is_same_v<typename Op::Type, bf16>;
    constexpr int kStages = Cfg::kStages;
    allow_next_grid();
    extern __shared__ unsigned char smem_base[];
    const uint32_t base = (tma::smem_addr(smem_base) + 1023u) & ~1023u;
    __shared__ uint64_t full[kStages], empty[kStages], done[2], freed[2], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == Cfg::kEpilogueWarps) {
        umma::alloc<Cfg::kTmemCols>(&tmem_slot);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            tma::mbar_init(&full[s], 1);
            tma::mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            tma::mbar_init(&done[s], 1);
            tma::mbar_init(&freed[s], Cfg::kEpilogueWarps);
        }
        tma::mbar_init(&drain, 1);
        gave_up = 0;
        tma::fence_mbar_init();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot;
    wait_for_previous_grid();

    if (warp == Cfg::kEpilogueWarps) {
        // The TMA warp. The previous kernels' plain stores come before these async-proxy reads.
        asm volatile("fence.proxy.async.global;" ::: "memory");
        int stage = 0;
        unsigned phase = 0;
        long long issued = 0;
        bool ok = true;
        for (long long t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
            const Tile tile = locate<K, BN, MT, T>(g, t);
            constexpr int kPairs = K == Kind::kGateBack || K == Kind::kInput ? 2 : 1;
            for (int turn = 0; ok && turn < tile.passes * kPairs; ++turn) {
                const int pair = turn % kPairs;
                int k0, k1;
                pass_range<K, T>(g, tile, pair, turn / kPairs, k0, k1);
                for (int p = 0; ok && p < Op::kProducts; ++p) {
                    const int pa = part_a<T>(p), pb = part_b<T>(p);
                    for (int k = k0; k < k1; ++k) {
                        ok = tma::mbar_wait(&empty[stage], phase ^ 1u);
                        if (!ok) {
                            break;
                        }
                        const uint32_t a = base + stage * Cfg::kStageBytes;
                        const uint32_t b = a + Cfg::kABytes;
                        uint64_t* bar = &full[stage];
                        if (umma::elect_one()) {
                            const int kc = k * kChunk;
                            if constexpr (K == Kind::kWeight) {
                                const int q = tile.problem;
                                tma::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
#pragma unroll
                                for (int j = 0; j < MT * kTileM / 64; ++j) {
                                    umma::load_3d(a + j * 8192, &maps.a[q], tile.m0 + 64 * j, kc, pa, bar);
                                }
#pragma unroll
                                for (int j = 0; j < BN / 64; ++j) {
                                    umma::load_3d(b + j * 8192, &maps.b[q], tile.n0 + 64 * j, kc, pb, bar);
                                }
                            } else if constexpr (K == Kind::kInput) {
                                tma::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
                                umma::load_3d(a, &maps.a[pair], kc, tile.m0, pa, bar);
#pragma unroll
                                for (int j = 0; j < BN / 64; ++j) {
                                    umma::load_3d(b + j * 8192, &maps.b[pair], tile.n0 + 64 * j, kc, pb, bar);
                                }
                            } else if constexpr (K == Kind::kDown) {
                                tma::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
                                umma::load_3d(a, &maps.a[0], kc, tile.m0, pa, bar);
                                umma::load_3d(b, &maps.b[0], kc, tile.n0, pb, bar);
                            } else if (pair == 0) {
                                tma::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
                                umma::load_3d(a, &maps.a[0], kc, tile.m0, pa, bar);
                                umma::load_3d(b, &maps.b[0], kc, tile.n0, pb, bar);
                                umma::load_3d(b + BN * umma::kRowBytes, &maps.b[1], kc, tile.n0, pb, bar);
                            } else {
                                tma::mbar_arrive_expect_tx(bar, Cfg::kABytes + BN * umma::kRowBytes);
                                umma::load_3d(a, &maps.a[1], kc, tile.m0, pa, bar);
#pragma unroll
                                for (int j = 0; j < BN / 64; ++j) {
                                    umma::load_3d(b + j * 8192, &maps.b[2], tile.n0 + 64 * j, kc, pb, bar);
                                }
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
            }
        }
        if (!ok) {
            // Let the loads in flight land (bounded) before the shared memory is given up.
            bool drained = true;
            for (long long i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                drained = tma::mbar_wait(&full[i % kStages], static_cast<unsigned>(i / kStages) & 1u) && drained;
            }
            if (lane == 0) {
                gave_up = 1;
                if (!drained) {
                    atomicOr(g.fault, tma::kFaultDrainTimeout);
                }
            }
        }
    } else if (warp == Cfg::kEpilogueWarps + 1) {
        // The MMA warp: converged, so that addresses and descriptors stay warp-uniform, one elected lane
        // issues (one lane throughout measured 10 % slower).
        constexpr bool kBMnFirst = K == Kind::kWeight || K == Kind::kInput;
        constexpr uint32_t kFirst = umma::instruction(kBf16, Cfg::kAMn, kBMnFirst, kTileM, Cfg::kBRows);
        constexpr uint32_t kSecond =
            K == Kind::kGateBack ? umma::instruction(kBf16, false, true, kTileM, BN) : kFirst;
        int stage = 0;
        unsigned phase = 0;
        int slot = 0;
        unsigned slot_phase = 0;
        bool ok = true;
        for (long long t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
            const Tile tile = locate<K, BN, MT, T>(g, t);
            constexpr int kPairs = K == Kind::kGateBack || K == Kind::kInput ? 2 : 1;
            const int passes = tile.passes * (kApart<K, T> ? 2 : 1);
            for (int pass = 0; ok && pass < passes; ++pass) {
                ok = tma::mbar_wait(&freed[slot], slot_phase ^ 1u);
                if (!ok) {
                    break;
                }
                umma::fence_after_sync();
                const int first = kApart<K, T> ? pass & 1 : 0;
                for (int pair = first; ok && pair < (kApart<K, T> ? first + 1 : kPairs); ++pair) {
                    int k0, k1;
                    pass_range<K, T>(g, tile, pair, kApart<K, T> ? pass >> 1 : pass, k0, k1);
                    const int steps = (k1 - k0) * Op::kProducts;
                    // kInput's two products share an accumulator (16-bit types); kGateBack's second has its own.
                    const bool fresh = kApart<K, T> || pair == 0 || K == Kind::kGateBack;
                    const uint32_t d = tmem + slot * Cfg::kCols + (K == Kind::kGateBack && pair == 1 ? 2 * BN : 0);
                    for (int i = 0; i < steps; ++i) {
                        ok = tma::mbar_wait(&full[stage], phase);
                        if (!ok) {
                            break;
                        }
                        umma::fence_after_sync();
                        const uint32_t a = base + stage * Cfg::kStageBytes;
                        const uint32_t b = a + Cfg::kABytes;
                        if (umma::elect_one()) {
                            const uint64_t da = Cfg::kAMn ? umma::desc_mn<8192>(a) : umma::desc_k(a);
                            constexpr uint64_t kStepA = Cfg::kAMn ? umma::kStepMn : umma::kStepK;
                            if (K == Kind::kGateBack && pair == 1) {
                                const uint64_t db = umma::desc_mn<8192>(b);
#pragma unroll
                                for (int s = 0; s < kChunk / 16; ++s) {
                                    umma::mma(d, da + kStepA * s, db + umma::kStepMn * s, kSecond, !fresh || i > 0 || s > 0);
                                }
                            } else {
                                const uint64_t db = kBMnFirst ? umma::desc_mn<8192>(b) : umma::desc_k(b);
                                constexpr uint64_t kStepB = kBMnFirst ? umma::kStepMn : umma::kStepK;
#pragma unroll
                                for (int s = 0; s < kChunk / 16; ++s) {
#pragma unroll
                                    for (int m = 0; m < MT; ++m) {
                                        umma::mma(d + m * BN, da + kStepA * s + m * (kTileABytes >> 4), db + kStepB * s, kFirst,
                                                  !fresh || i > 0 || s > 0);
                                    }
                                }
                            }
                            umma::commit(&empty[stage]);
                        }
                        __syncwarp();
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
                if (ok) {
                    if (umma::elect_one()) {
                        umma::commit(&done[slot]);
                    }
                    __syncwarp();
                    slot = (slot + 1) % Cfg::kSlots;
                    slot_phase ^= slot == 0 ? 1u : 0u;
                }
            }
        }
        if (!ok) {
            if (umma::elect_one()) {
                umma::commit(&drain);
            }
            __syncwarp();
            const bool drained = tma::mbar_wait(&drain, 0);
            if (lane == 0) {
                gave_up = 1;
                if (!drained) {
                    atomicOr(g.fault, tma::kFaultDrainTimeout);
                }
            }
        }
    } else {
        // The epilogue warps: warp w reads lanes 32 (w % 4) .. + 31 (rows of the tile) and its kColumns
        // columns of each accumulator.
        const int quad = warp & 3;
        const int first = (warp >> 2) * Cfg::kColumns;
        int slot = 0;
        unsigned slot_phase = 0;
        bool ok = true;
        for (long long t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
            const Tile tile = locate<K, BN, MT, T>(g, t);
            const int row = tile.m0 + quad * 32 + lane;
            const int rows = K == Kind::kWeight ? g.rows_of[tile.problem] : g.rows;
            const int cols = K == Kind::kWeight ? g.cols_of[tile.problem] : g.cols;
            if constexpr (sizeof(T) == 4) {
                // The passes' accumulators add up in registers: BN / 2 columns of each per warp, in runs of 32.
                static_assert(MT == 1 && Cfg::kSets * BN <= 256, "the sums fit in registers");
                constexpr int kRuns = BN / 64;
                float acc[kRuns][Cfg::kSets][32];
#pragma unroll
                for (int r = 0; r < kRuns; ++r) {
#pragma unroll
                    for (int q = 0; q < Cfg::kSets; ++q) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            acc[r][q][j] = 0.0f;
                        }
                    }
                }
                const int passes = tile.passes * (kApart<K, T> ? 2 : 1);
                for (int pass = 0; ok && pass < passes; ++pass) {
                    ok = tma::mbar_wait(&done[slot], slot_phase);
                    if (!ok) {
                        break;
                    }
                    umma::fence_after_sync();
                    const uint32_t d = tmem + slot * Cfg::kCols + (static_cast<uint32_t>(quad * 32) << 16) + first;
#pragma unroll
                    for (int q = 0; q < Cfg::kSets; ++q) {
                        // An operand pair that ended in an earlier pass has nothing new here.
                        int begin, end;
                        pass_range<K, T>(g, tile, kApart<K, T> ? pass & 1 : K == Kind::kGateBack && q == 2 ? 1 : 0,
                                      kApart<K, T> ? pass >> 1 : pass, begin, end);
                        if (begin < end) {
#pragma unroll
                            for (int r = 0; r < kRuns; ++r) {
                                float v[32];
                                umma::load32(d + q * BN + 32 * r, v);
                                umma::load_wait(v);
#pragma unroll
                                for (int j = 0; j < 32; ++j) {
                                    acc[r][q][j] += v[j];
                                }
                            }
                        }
                    }
                    release(&freed[slot], lane);
                    slot = (slot + 1) % Cfg::kSlots;
                    slot_phase ^= slot == 0 ? 1u : 0u;
                }
#pragma unroll
                for (int r = 0; r < kRuns; ++r) {
                    const int col = tile.n0 + first + 32 * r;
                    if (!ok || col >= cols) {
                        continue;
                    }
                    if constexpr (Cfg::kSets == 1) {
                        store_results<K, T>(g, tile, row, rows, col, cols, acc[r][0]);
                    } else if (row < rows) {
                        finish<K, T, Act>(g, tile, row, col, cols, acc[r]);
                    }
                }
            } else {
                for (int pass = 0; ok && pass < tile.passes; ++pass) {
                    ok = tma::mbar_wait(&done[slot], slot_phase);
                    if (!ok) {
                        break;
                    }
                    umma::fence_after_sync();
                    const uint32_t d = tmem + slot * Cfg::kCols + (static_cast<uint32_t>(quad * 32) << 16);
#pragma unroll 1
                    for (int i = 0; i < MT * (Cfg::kColumns / Cfg::kRun); ++i) {
                        const int m = i / (Cfg::kColumns / Cfg::kRun);  // row tile
                        const int c = first + i % (Cfg::kColumns / Cfg::kRun) * Cfg::kRun;
                        if (tile.n0 + c >= cols) {
                            continue;
                        }
                        float acc[Cfg::kSets][Cfg::kRun];
#pragma unroll
                        for (int q = 0; q < Cfg::kSets; ++q) {
                            umma::load_run(d + (m * Cfg::kSets + q) * BN + c, acc[q]);
                        }
#pragma unroll
                        for (int q = 0; q < Cfg::kSets; ++q) {
                            umma::load_wait(acc[q]);
                        }
                        if constexpr (Cfg::kSets == 1) {
                            store_results<K, T>(g, tile, row + m * kTileM, rows, tile.n0 + c, cols, acc[0], pass > 0);
                        } else if (row + m * kTileM < rows) {
                            finish<K, T, Act>(g, tile, row + m * kTileM, tile.n0 + c, cols, acc);
                        }
                        __syncwarp();
                    }
                    release(&freed[slot], lane);
                    slot = (slot + 1) % Cfg::kSlots;
                    slot_phase ^= slot == 0 ? 1u : 0u;
                }
            }
        }
        if (!ok && lane == 0) {
            gave_up = 1;
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (threadIdx.x == 0 && gave_up != 0) {
        atomicOr(g.fault, tma::kFaultWaitTimeout);
    }
    if (warp == Cfg::kEpilogueWarps) {
        umma::dealloc<Cfg::kTmemCols>(tmem);
    }
}

// The parts of the three weight products, added up and rounded once. Many parts (a narrow block's CTAs):
// 32 values side by side, eight warps taking every eighth part, joined in order. Few parts of large
// products: a thread per value (with the eight warps, 80 us instead of 6 for three parts of 3 M values).
template <class T, bool Many>
__global__ void __launch_bounds__(256)
    weight_sum_kernel(const float* __restrict__ partial, T* __restrict__ w0, T* __restrict__ w1, T* __restrict__ w2,
                      long long size0, long long size2, long long part_size, int parts)
{
    allow_next_grid();
    const long long total = 2 * size0 + size2;
    const auto put = [&](long long i, float s) {
        if (i < size0) {
            w0[i] = from_float<T>(s);
        } else if (i < 2 * size0) {
            w1[i - size0] = from_float<T>(s);
        } else {
            w2[i - 2 * size0] = from_float<T>(s);
        }
    };
    wait_for_previous_grid();
    if constexpr (Many) {
        __shared__ float sums[8][32];
        const int lane = threadIdx.x & 31;
        const int warp = threadIdx.x >> 5;
        for (long long i0 = static_cast<long long>(blockIdx.x) * 32; i0 < total; i0 += static_cast<long long>(gridDim.x) * 32) {
            const long long i = i0 + lane;
            float s = 0.0f;
            if (i < total) {
#pragma unroll 8
                for (int p = warp; p < parts; p += 8) {
                    s += partial[p * part_size + i];
                }
            }
            sums[warp][lane] = s;
            __syncthreads();
            if (warp == 0 && i < total) {
#pragma unroll
                for (int k = 1; k < 8; ++k) {
                    s += sums[k][lane];
                }
                put(i, s);
            }
            __syncthreads();
        }
    } else {
        for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total;
             i += static_cast<long long>(gridDim.x) * 256) {
            float s = partial[i];
#pragma unroll 4
            for (int p = 1; p < parts; ++p) {
                s += partial[p * part_size + i];
            }
            put(i, s);
        }
    }
}

// --- a few tokens --------------------------------------------------------------------------------------

constexpr int kFewAtOnce = 8;  // tokens of one launch
constexpr int kFewThreads = 256;

// The most tokens that take this path: past them the tensor cores are faster. float32, whose weights would
// have to be split first, stays here longer (four launches).
template <class T>
constexpr int kFewTokens = sizeof(T) == 4 ? 32 : 8;

// N consecutive values as floats, by 16-byte loads.
template <class X, int N>
__device__ __forceinline__ void load_floats(const X* p, float (&v)[N])
{
    constexpr int kPer = 16 / static_cast<int>(sizeof(X));
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) {
        const Vec<X, kPer> q = reinterpret_cast<const Vec<X, kPer>*>(p)[i];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            v[i * kPer + j] = to_float(q.v[j]);
        }
    }
}

// acc[r][m] += the share of lane `first` of `step` of w[r][0 .. n) . v[m][0 .. n), for R rows of weights at
// once: lanes stride 16-byte pieces, or single values where rows are not whole aligned pieces.
template <class W, class X, int R, int M>
__device__ __forceinline__ void row_dots(const W* const (&w)[R], const X* __restrict__ v, long long pitch, int n, int first,
                                         int step, bool wide, float (&acc)[R][M])
{
    constexpr int kV = 16 / static_cast<int>(sizeof(W));
    if (wide) {
#pragma unroll 2
        for (int c = first * kV; c < n; c += step * kV) {
            float p[R][kV];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                load_floats<W, kV>(w[r] + c, p[r]);
            }
#pragma unroll
            for (int m = 0; m < M; ++m) {
                float q[kV];
                load_floats<X, kV>(v + m * pitch + c, q);
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int j = 0; j < kV; ++j) {
                        acc[r][m] = fmaf(p[r][j], q[j], acc[r][m]);
                    }
                }
            }
        }
    } else {
        for (int c = first; c < n; c += step) {
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const float q = to_float(v[m * pitch + c]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    acc[r][m] = fmaf(to_float(w[r][c]), q, acc[r][m]);
                }
            }
        }
    }
}

// One warp per hidden value: h[m][f] = act(x_m . Wg_f) * (x_m . Wu_f), in FP32.
template <class T, int Act, int M>
__global__ void __launch_bounds__(kFewThreads)
    few_gate_kernel(const T* __restrict__ x, const T* __restrict__ w_gate, const T* __restrict__ w_up, float* __restrict__ h,
                    int channels, int hidden, bool wide)
{
    allow_next_grid();
    wait_for_previous_grid();
    const int f = static_cast<int>(blockIdx.x) * (kFewThreads / 32) + static_cast<int>(threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (f >= hidden) {
        return;
    }
    float acc[2][M] = {};
    const T* const rows[2] = {w_gate + static_cast<long long>(f) * channels, w_up + static_cast<long long>(f) * channels};
    row_dots<T, T, 2, M>(rows, x, channels, channels, lane, 32, wide, acc);
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            acc[0][m] += __shfl_xor_sync(0xffffffffu, acc[0][m], o);
            acc[1][m] += __shfl_xor_sync(0xffffffffu, acc[1][m], o);
        }
        if (lane == 0) {
            h[static_cast<long long>(m) * hidden + f] = activate<Act>(acc[0][m]) * acc[1][m];
        }
    }
}

// One CTA per output: its warps share the row of Wd, the partial sums meet in shared memory.
template <class T, int M>
__global__ void __launch_bounds__(kFewThreads)
    few_down_kernel(const float* __restrict__ h, const T* __restrict__ w_down, T* __restrict__ y, int hidden, int outputs,
                    bool wide)
{
    __shared__ float sums[kFewThreads / 32][M];
    allow_next_grid();
    wait_for_previous_grid();
    const int o = blockIdx.x;
    float acc[1][M] = {};
    const T* const row[1] = {w_down + static_cast<long long>(o) * hidden};
    row_dots<T, float, 1, M>(row, h, hidden, hidden, static_cast<int>(threadIdx.x), kFewThreads, wide, acc);
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) {
            acc[0][m] += __shfl_xor_sync(0xffffffffu, acc[0][m], k);
        }
        if ((threadIdx.x & 31) == 0) {
            sums[threadIdx.x >> 5][m] = acc[0][m];
        }
    }
    __syncthreads();
    if (threadIdx.x < M) {
        float s = 0.0f;
        for (int k = 0; k < kFewThreads / 32; ++k) {
            s += sums[k][threadIdx.x];
        }
        y[static_cast<long long>(threadIdx.x) * outputs + o] = from_float<T>(s);
    }
}

// --- host side -----------------------------------------------------------------------------------------

int round_up(int v, int to) { return (v + to - 1) / to * to; }
int tiles_of(long long v, int tile) { return static_cast<int>((v + tile - 1) / tile); }
int hidden_pitch(const MlpShape& n) { return round_up(n.hidden, 16); }  // 32-byte rows for the epilogue's stores
int planes_of(int dtype) { return dtype == SPECTRAL_FLOAT32 ? 3 : 1; }

// A workspace handed out piece by piece, each 256-byte aligned. A call lays its pieces out in the same steps
// in which the workspace queries counted them (then at an address that nothing reads or writes).
struct Arena {
    std::uintptr_t base = 256;
    std::size_t used = 0;

    Arena() = default;
    explicit Arena(void* work) : base((reinterpret_cast<std::uintptr_t>(work) + 255) & ~std::uintptr_t{255}) {}
    void* take(std::size_t bytes)
    {
        void* p = reinterpret_cast<void*>(base + used);
        used += (bytes + 255) / 256 * 256;
        return p;
    }
    std::size_t total() const { return used + 256; }  // whatever the workspace's own alignment
};

// TMA reads the array as it lies: 16-bit values in 16-byte aligned rows. (A workspace query that does not know
// the array passes nullptr.)
template <class T>
bool direct(const void* p, int cols)
{
    return sizeof(T) == 2 && cols % 8 == 0 && p != nullptr && aligned_to(p, 16);
}

template <class T>
std::size_t staged_bytes(long long rows, int cols)
{
    return static_cast<std::size_t>(rows) * round_up(cols, 8) * 2 * Operand<T>::kPlanes;
}

// The operand form of a rows x cols array; where TMA cannot read it in place, in the arena, filled once
// `jobs` have run.
template <class T>
Matrix operand(const void* p, long long rows, int cols, Arena& arena, StageJobs& jobs)
{
    constexpr bool kBf16 = std::is_same_v<typename Operand<T>::Type, bf16>;
    if (direct<T>(p, cols)) {
        return {p, rows, cols, cols, 1, kBf16};
    }
    const int pitch = round_up(cols, 8);
    void* dst = arena.take(staged_bytes<T>(rows, cols));
    jobs.job[jobs.count++] = {p, dst, rows, cols, pitch};
    return {dst, rows, cols, pitch, Operand<T>::kPlanes, kBf16};
}

template <class T>
void run_jobs(const StageJobs& jobs, cudaStream_t stream)
{
    if (jobs.count == 0) {
        return;
    }
    long long pieces = 1;
    for (int i = 0; i < jobs.count; ++i) {
        pieces = std::max(pieces, jobs.job[i].rows * (jobs.job[i].pitch / 8));
    }
    const unsigned grid = static_cast<unsigned>(std::min<long long>((pieces + 255) / 256, 148 * 16));
    launch_pdl(stage_kernel<T>, dim3(grid, static_cast<unsigned>(jobs.count)), dim3(256), 0, stream, jobs);
}

// hidden values (tokens x hidden) in the arena, in the operand form.
template <class T>
Matrix hidden_matrix(const MlpShape& n, Arena& arena)
{
    const int pitch = hidden_pitch(n);
    void* p = arena.take(static_cast<std::size_t>(n.tokens) * pitch * 2 * Operand<T>::kPlanes);
    return {p, n.tokens, n.hidden, pitch, Operand<T>::kPlanes, std::is_same_v<typename Operand<T>::Type, bf16>};
}

template <Kind K, int BN, int MT, class T, int Act>
void launch_product(const Maps& maps, Args& g, cudaStream_t stream)
{
    using Cfg = Config<K, BN, MT, T>;
    static std::atomic<bool> opted[kMaxDevices];
    const int device = current_device();
    const auto kernel = product_kernel<K, BN, MT, T, Act>;
    if (!opted[device].load(std::memory_order_relaxed)) {
        SPECTRAL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
        opted[device].store(true, std::memory_order_relaxed);
    }
    g.fault = device_fault_word();
    const long long grid = std::min<long long>(g.tiles, device_sm_count(device));
    launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(Cfg::kThreads), static_cast<std::size_t>(Cfg::kSmem), stream, maps, g);
}

// Calls f(integral_constant<BN>) with the widest tile of 64, 128 or 256 columns that `cols` fills and that
// still leaves about two thirds of the SMs a tile: wider tiles read each row of A fewer times and run
// longer MMAs (float32 8192 x 512 x 2048 forward 440 us at 64 columns, 255 us at 256), but few tokens
// would leave SMs idle (float32 128 x 512 x 2048: 83 us at 64, 110 us at 256).
constexpr long long kEnoughTiles = 96;
template <class F>
void with_width(long long rows, int cols, F&& f)
{
    const auto enough = [&](int bn) { return static_cast<long long>(tiles_of(rows, kTileM)) * tiles_of(cols, bn) >= kEnoughTiles; };
    if (cols > 128 && enough(256)) {
        f(std::integral_constant<int, 256>{});
    } else if (cols > 64 && enough(128)) {
        f(std::integral_constant<int, 128>{});
    } else {
        f(std::integral_constant<int, 64>{});
    }
}

void set_tiles(Args& g, long long rows, int cols, int bn)
{
    g.rows = static_cast<int>(rows);
    g.cols = cols;
    g.m_tiles = tiles_of(rows, kTileM);
    g.n_tiles = tiles_of(cols, bn);
    g.tiles = static_cast<long long>(g.m_tiles) * g.n_tiles;
}

template <class T, int Act>
void mlp_few(const T* x, const T* wg, const T* wu, const T* wd, T* y, const MlpShape& n, float* h, cudaStream_t stream)
{
    constexpr int kV = 16 / static_cast<int>(sizeof(T));
    const bool wide_c = n.channels % kV == 0 && aligned_to(x, 16) && aligned_to(wg, 16) && aligned_to(wu, 16);
    const bool wide_f = n.hidden % 8 == 0 && aligned_to(wd, 16);  // h: rows of whole 16-byte pieces too
    for (long long t = 0; t < n.tokens; t += kFewAtOnce) {
        const auto run = [&](auto m) {
            constexpr int M = decltype(m)::value;
            launch_pdl(few_gate_kernel<T, Act, M>, dim3(static_cast<unsigned>(tiles_of(n.hidden, kFewThreads / 32))),
                       dim3(kFewThreads), 0, stream, x + t * n.channels, wg, wu, h, n.channels, n.hidden, wide_c);
            launch_pdl(few_down_kernel<T, M>, dim3(static_cast<unsigned>(n.outputs)), dim3(kFewThreads), 0, stream,
                       static_cast<const float*>(h), wd, y + t * n.outputs, n.hidden, n.outputs, wide_f);
        };
        switch (std::min<long long>(n.tokens - t, kFewAtOnce)) {
            case 1: run(std::integral_constant<int, 1>{}); break;
            case 2: run(std::integral_constant<int, 2>{}); break;
            case 3: run(std::integral_constant<int, 3>{}); break;
            case 4: run(std::integral_constant<int, 4>{}); break;
            case 5: run(std::integral_constant<int, 5>{}); break;
            case 6: run(std::integral_constant<int, 6>{}); break;
            case 7: run(std::integral_constant<int, 7>{}); break;
            default: run(std::integral_constant<int, 8>{}); break;
        }
    }
}

// The arrays a call gives.
struct Arrays {
    const void* dy = nullptr;  // backward
    const void* x = nullptr;
    const void* wg = nullptr;
    const void* wu = nullptr;
    const void* wd = nullptr;
};

// A forward call's workspace: the few-token form's hidden values, or the operands TMA does not read in place and,
// unless they stay on chip, the hidden values.
template <class T>
struct ForwardLayout {
    bool few = false, narrow = false;
    float* few_hidden = nullptr;
    StageJobs jobs;
    Matrix x, wg, wu, wd, h;

    ForwardLayout(Arena& arena, const Arrays& in, int dtype, const MlpShape& n)
        : few(n.tokens <= kFewTokens<T>), narrow(narrow_forward_fits(n, dtype))
    {
        if (few) {
            few_hidden = static_cast<float*>(arena.take(sizeof(float) * kFewAtOnce * static_cast<std::size_t>(n.hidden)));
            return;
        }
        x = operand<T>(in.x, n.tokens, n.channels, arena, jobs);
        wg = operand<T>(in.wg, n.hidden, n.channels, arena, jobs);
        wu = operand<T>(in.wu, n.hidden, n.channels, arena, jobs);
        wd = operand<T>(in.wd, n.outputs, n.hidden, arena, jobs);
        if (!narrow) {
            h = hidden_matrix<T>(n, arena);
        }
    }
};

template <class T>
void mlp_forward(const Arrays& in, void* y, int dtype, const MlpShape& n, void* work, cudaStream_t stream)
{
    Arena arena(work);
    const ForwardLayout<T> lay(arena, in, dtype, n);
    if (lay.few) {
        with_activation(n.act, [&](auto act) {
            mlp_few<T, decltype(act)::value>(static_cast<const T*>(in.x), static_cast<const T*>(in.wg),
                                             static_cast<const T*>(in.wu), static_cast<const T*>(in.wd), static_cast<T*>(y), n,
                                             lay.few_hidden, stream);
        });
        return;
    }
    const Matrix &mx = lay.x, &mg = lay.wg, &mu = lay.wu, &md = lay.wd, &mh = lay.h;
    run_jobs<T>(lay.jobs, stream);
    if constexpr (sizeof(T) == 2) {
        if (lay.narrow) {
            narrow_forward(mx, mg, mu, md, y, dtype, n, stream);
            return;
        }
    }
    const auto gate = [&](auto width) {
        constexpr int BN = decltype(width)::value;
        Maps maps;
        maps.a[0] = mx.map(kTileM);
        maps.b[0] = mg.map(BN);
        maps.b[1] = mu.map(BN);
        Args g;
        set_tiles(g, n.tokens, n.hidden, BN);
        g.chunks[0] = tiles_of(n.channels, kChunk);
        g.out[0] = const_cast<void*>(mh.base);
        g.pitch = mh.pitch;
        g.plane = mh.rows * mh.pitch;
        with_activation(n.act, [&](auto act) { launch_product<Kind::kGate, BN, 1, T, decltype(act)::value>(maps, g, stream); });
    };
    // As with_width, up to 128; float32 with short products is bound by its epilogue, which two narrow tiles
    // overlap better (262144 x 64 x 128: 166 us at 64 columns, 184 us at 128).
    const bool wide = n.hidden > 64 && static_cast<long long>(tiles_of(n.tokens, kTileM)) * tiles_of(n.hidden, 128) >= kEnoughTiles
                      && (sizeof(T) == 2 || n.channels >= 128);
    if (wide) {
        gate(std::integral_constant<int, 128>{});
    } else {
        gate(std::integral_constant<int, 64>{});
    }
    with_width(n.tokens, n.outputs, [&](auto width) {
        constexpr int BN = decltype(width)::value;
        Maps maps;
        maps.a[0] = mh.map(kTileM);
        maps.b[0] = md.map(BN);
        Args g;
        set_tiles(g, n.tokens, n.outputs, BN);
        g.chunks[0] = tiles_of(n.hidden, kChunk);
        g.out[0] = y;
        g.pitch = n.outputs;
        launch_product<Kind::kDown, BN, 1, T, SPECTRAL_ACT_NONE>(maps, g, stream);
    });
}

// Tiles of the weight products: 256 x 256 where every side is longer than that (a tile of 128 x 128 reads
// twice as much per product), else 128 x 128, whose epilogue overlaps. Backward passes measured with the large
// and the small tiles, us: 8192 x 512 x 2048 146 and 156, 8192 x 1024 x 4096 519 and 538, 8192 x 448 x 1792 140 and 152, but
// 32768 x 256 x 512 114 and 106. From 257 to 384 neither wins by much (8192 x 384 x 1536 113 and 112, 8192 x 320 x 1280 89 and 85,
// 65536 x 384 x 768 405 and 418).
template <class T>
bool large_weight_tiles(const MlpShape& n)
{
    return sizeof(T) == 2 && n.hidden > 256 && n.channels > 256 && n.outputs > 256;
}

// The weight products' tiles and parts: as many parts as keep the SMs busy over whole waves, each
// at least eight chunks (512 tokens) long.
template <class T>
void set_weight_tiles(Args& g, const MlpShape& n)
{
    const bool large = large_weight_tiles<T>(n);
    const int tile_rows = large ? 256 : 128;
    const int tile_cols = large ? 256 : 128;
    const int rows[3] = {n.hidden, n.hidden, n.outputs};
    const int cols[3] = {n.channels, n.channels, n.hidden};
    g.first[0] = 0;
    for (int p = 0; p < 3; ++p) {
        g.rows_of[p] = rows[p];
        g.cols_of[p] = cols[p];
        g.n_tiles_of[p] = tiles_of(cols[p], tile_cols);
        g.first[p + 1] = g.first[p] + static_cast<long long>(tiles_of(rows[p], tile_rows)) * g.n_tiles_of[p];
    }
    const long long size = static_cast<long long>(n.hidden) * n.channels;
    g.offset[0] = 0;
    g.offset[1] = size;
    g.offset[2] = 2 * size;
    g.part_size = 2 * size + static_cast<long long>(n.outputs) * n.hidden;
    g.chunks[0] = std::max(1, tiles_of(n.tokens, kChunk));  // no tokens: sized for, never launched
    // A part of k chunks costs its tiles k units and an epilogue of about four (eight for a large tile).
    const int epilogue = large ? 8 : 4;
    double best = 0.0;
    for (int parts = 1; parts <= 148 && (parts == 1 || g.chunks[0] / parts >= 8); ++parts) {
        const int k = tiles_of(g.chunks[0], parts);
        const long long waves = (g.first[3] * tiles_of(g.chunks[0], k) + 147) / 148;
        const double cost = static_cast<double>(waves) * (k + epilogue);
        if (parts == 1 || cost < 0.97 * best) {
            best = cost;
            g.parts = tiles_of(g.chunks[0], k);
            g.part_chunks = k;
        }
    }
    g.tiles = g.first[3] * g.parts;
}

// A backward call's workspace: x restored from its checkpoint, the operands TMA does not read in place, the hidden
// values and their gradients unless they stay on chip, and the FP32 parts of the weight gradients.
template <class T>
struct BackwardLayout {
    bool narrow = false;
    int parts = 0;
    void* restored = nullptr;
    StageJobs jobs;
    Matrix dy, x, wg, wu, wd, dg, du, h;
    Args weights;  // the weight products' tiles, where they are products of their own
    float* partial = nullptr;

    BackwardLayout(Arena& arena, const Arrays& in, bool packed, int dtype, const MlpShape& n)
        : narrow(narrow_backward_fits(n, dtype))
    {
        if (packed) {
            restored = arena.take(static_cast<std::size_t>(n.tokens) * n.channels * sizeof(T));
        }
        x = operand<T>(packed ? restored : in.x, n.tokens, n.channels, arena, jobs);
        dy = operand<T>(in.dy, n.tokens, n.outputs, arena, jobs);
        wg = operand<T>(in.wg, n.hidden, n.channels, arena, jobs);
        wu = operand<T>(in.wu, n.hidden, n.channels, arena, jobs);
        wd = operand<T>(in.wd, n.outputs, n.hidden, arena, jobs);
        if (narrow) {
            parts = narrow_backward_parts(n);
        } else {
            dg = hidden_matrix<T>(n, arena);
            du = hidden_matrix<T>(n, arena);
            h = hidden_matrix<T>(n, arena);
            set_weight_tiles<T>(weights, n);
            parts = weights.parts;
        }
        const std::size_t part = static_cast<std::size_t>(n.hidden) * (2 * static_cast<std::size_t>(n.channels) + n.outputs);
        partial = static_cast<float*>(arena.take(sizeof(float) * part * parts));
    }
};

template <class T>
void mlp_backward(const Arrays& in, const signed char* codes, const float* scales, void* dx, void* dwg, void* dwu, void* dwd,
                  int dtype, const MlpShape& n, void* work, cudaStream_t stream)
{
    Arena arena(work);
    BackwardLayout<T> lay(arena, in, codes != nullptr, dtype, n);
    if (codes != nullptr) {
        unpack8(codes, scales, lay.restored, dtype, n.tokens, n.channels, stream);
    }
    const Matrix &mx = lay.x, &mdy = lay.dy, &mg = lay.wg, &mu = lay.wu, &md = lay.wd;
    const Matrix &mdg = lay.dg, &mdu = lay.du, &mh = lay.h;
    float* const partial = lay.partial;
    run_jobs<T>(lay.jobs, stream);
    const long long size0 = static_cast<long long>(n.hidden) * n.channels;
    const long long size2 = static_cast<long long>(n.outputs) * n.hidden;
    const long long part_size = 2 * size0 + size2;
    const auto add_parts = [&](int parts) {
        const auto launch = [&](auto many, int per_cta) {
            const unsigned grid = static_cast<unsigned>(std::min<long long>((part_size + per_cta - 1) / per_cta, 148 * 16));
            launch_pdl(weight_sum_kernel<T, decltype(many)::value>, dim3(grid), dim3(256), 0, stream,
                       static_cast<const float*>(partial), static_cast<T*>(dwg), static_cast<T*>(dwu), static_cast<T*>(dwd), size0, size2, part_size, parts);
        };
        if (parts > 8) {
            launch(std::true_type{}, 32);
        } else {
            launch(std::false_type{}, 256);
        }
    };
    if constexpr (sizeof(T) == 2) {
        if (lay.narrow) {
            narrow_backward(mdy, mx, mg, mu, md, dx, partial, dtype, n, stream);
            add_parts(lay.parts);
            return;
        }
    }
    const auto gate_back = [&](auto width) {
        constexpr int BN = decltype(width)::value;
        Maps maps;
        maps.a[0] = mx.map(kTileM);
        maps.b[0] = mg.map(BN);
        maps.b[1] = mu.map(BN);
        maps.a[1] = mdy.map(kTileM);
        maps.b[2] = md.map(kChunk);
        Args g;
        set_tiles(g, n.tokens, n.hidden, BN);
        g.chunks[0] = tiles_of(n.channels, kChunk);
        g.chunks[1] = tiles_of(n.outputs, kChunk);
        g.out[0] = const_cast<void*>(mdg.base);
        g.out[1] = const_cast<void*>(mdu.base);
        g.out[2] = const_cast<void*>(mh.base);
        g.pitch = mh.pitch;
        g.plane = mh.rows * mh.pitch;
        with_activation(n.act,
                        [&](auto act) { launch_product<Kind::kGateBack, BN, 1, T, decltype(act)::value>(maps, g, stream); });
    };
    // 128 columns leave one accumulator set (384 of 512), so the epilogue does not overlap, but an MMA of N = 64
    // takes nearly as long as one of 128 and a wider tile reads its tokens fewer times: worth it where the
    // products are long. Backward passes with 128 and 64 columns, us: 8192 x 1024 x 4096 536 and 557,
    // 8192 x 512 x 2048 146 and 149, 8192 x 448 x 1792 150 and 142, 8192 x 384 x 1536 118 and 113, 32768 x 256 x 512 105 and 99;
    // unequal sides, 16384 x 1024 x 300 with 512 outputs 118 and 120. At 128 the tiles' operands are what counts:
    // 650 MB from L2 to shared memory in the 72 us of 8192 x 512 x 2048, 9 TB/s.
    if constexpr (sizeof(T) == 4) {
        gate_back(std::integral_constant<int, 64>{});  // the passes' sums stay in registers
    } else if (n.channels + n.outputs >= 1024) {
        gate_back(std::integral_constant<int, 128>{});
    } else {
        gate_back(std::integral_constant<int, 64>{});
    }
    with_width(n.tokens, n.channels, [&](auto width) {
        constexpr int BN = decltype(width)::value;
        Maps maps;
        maps.a[0] = mdg.map(kTileM);
        maps.a[1] = mdu.map(kTileM);
        maps.b[0] = mg.map(kChunk);
        maps.b[1] = mu.map(kChunk);
        Args g;
        set_tiles(g, n.tokens, n.channels, BN);
        g.chunks[0] = tiles_of(n.hidden, kChunk);
        g.chunks[1] = g.chunks[0];
        g.out[0] = dx;
        g.pitch = n.channels;
        launch_product<Kind::kInput, BN, 1, T, SPECTRAL_ACT_NONE>(maps, g, stream);
    });
    {
        Maps maps;
        maps.a[0] = mdg.map(kChunk);
        maps.a[1] = mdu.map(kChunk);
        maps.a[2] = mdy.map(kChunk);
        maps.b[0] = mx.map(kChunk);
        maps.b[1] = mx.map(kChunk);
        maps.b[2] = mh.map(kChunk);
        Args& g = lay.weights;
        g.out[0] = partial;
        if constexpr (sizeof(T) == 2) {
            if (large_weight_tiles<T>(n)) {
                launch_product<Kind::kWeight, 256, 2, T, SPECTRAL_ACT_NONE>(maps, g, stream);
            } else {
                launch_product<Kind::kWeight, 128, 1, T, SPECTRAL_ACT_NONE>(maps, g, stream);
            }
        } else {
            launch_product<Kind::kWeight, 128, 1, T, SPECTRAL_ACT_NONE>(maps, g, stream);
        }
        add_parts(lay.parts);
    }
}

int invalid(const std::string& message)
{
    set_last_error(message);
    return SPECTRAL_INVALID_ARGUMENT;
}

int check(const char* op, int dtype, long long tokens, int channels, int hidden, int outputs)
{
    const std::string name(op);
    if (!dtype_known(dtype)) {
        return invalid(name + ": dtype must be SPECTRAL_FLOAT32, SPECTRAL_BFLOAT16 or SPECTRAL_FLOAT16");
    }
    constexpr int kMost = 1 << 20;
    if (tokens < 0 || tokens > kMaxTokens || channels < 1 || hidden < 1 || outputs < 1 || channels > kMost || hidden > kMost
        || outputs > kMost) {
        return invalid(name + ": need 0 <= tokens < 2^31 - 256 and channels, hidden and outputs from 1 to 2^20");
    }
    return SPECTRAL_OK;
}

bool overlap(const void* a, unsigned long long a_bytes, const void* b, unsigned long long b_bytes)
{
    const auto p = reinterpret_cast<unsigned long long>(a);
    const auto q = reinterpret_cast<unsigned long long>(b);
    return p < q + b_bytes && q < p + a_bytes;
}

}  // namespace
}  // namespace spectral

extern "C" int spectral_gated_mlp_workspace_for(const void* x, const void* w_gate, const void* w_up, const void* w_down,
                                                int dtype, long long tokens, int channels, int hidden, int outputs,
                                                size_t* count)
{
    using namespace spectral;
    const int status = check("gated_mlp_workspace", dtype, tokens, channels, hidden, outputs);
    if (status != SPECTRAL_OK || count == nullptr) {
        return status != SPECTRAL_OK ? status : invalid("gated_mlp_workspace: null count");
    }
    const MlpShape n{tokens, channels, hidden, outputs, 0};
    with_dtype(dtype, [&](auto t) {
        Arena arena;
        const ForwardLayout<decltype(t)> lay(arena, {nullptr, x, w_gate, w_up, w_down}, dtype, n);
        *count = (arena.total() + 7) / 8;
    });
    return SPECTRAL_OK;
}

extern "C" int spectral_gated_mlp_workspace(int dtype, long long tokens, int channels, int hidden, int outputs, size_t* count)
{
    return spectral_gated_mlp_workspace_for(nullptr, nullptr, nullptr, nullptr, dtype, tokens, channels, hidden, outputs, count);
}

extern "C" int spectral_gated_mlp_backward_workspace_for(const void* dy, const void* x, int packed, const void* w_gate,
                                                         const void* w_up, const void* w_down, int dtype, long long tokens,
                                                         int channels, int hidden, int outputs, size_t* count)
{
    using namespace spectral;
    const int status = check("gated_mlp_backward_workspace", dtype, tokens, channels, hidden, outputs);
    if (status != SPECTRAL_OK || count == nullptr) {
        return status != SPECTRAL_OK ? status : invalid("gated_mlp_backward_workspace: null count");
    }
    const MlpShape n{tokens, channels, hidden, outputs, 0};
    with_dtype(dtype, [&](auto t) {
        Arena arena;
        const BackwardLayout<decltype(t)> lay(arena, {dy, x, w_gate, w_up, w_down}, packed != 0, dtype, n);
        *count = (arena.total() + 7) / 8;
    });
    return SPECTRAL_OK;
}

extern "C" int spectral_gated_mlp_backward_workspace(int dtype, long long tokens, int channels, int hidden, int outputs,
                                                     size_t* count)
{
    size_t plain = 0, packed = 0;
    for (size_t* c : {&plain, &packed}) {
        const int status = spectral_gated_mlp_backward_workspace_for(nullptr, nullptr, c == &packed, nullptr, nullptr, nullptr, dtype,
                                                                     tokens, channels, hidden, outputs, count != nullptr ? c : nullptr);
        if (status != SPECTRAL_OK) {
            return status;
        }
    }
    *count = std::max(plain, packed);
    return SPECTRAL_OK;
}

extern "C" int spectral_gated_mlp(const void* x, const void* w_gate, const void* w_up, const void* w_down, void* y, int dtype,
                                  long long tokens, int channels, int hidden, int outputs, int activation, void* work,
                                  void* stream)
{
    using namespace spectral;
    const int status = check("gated_mlp", dtype, tokens, channels, hidden, outputs);
    if (status != SPECTRAL_OK) {
        return status;
    }
    if (!activation_known(activation)) {
        return invalid("gated_mlp: activation must be SPECTRAL_ACT_NONE, _SILU or _GELU");
    }
    if (tokens == 0) {
        return SPECTRAL_OK;
    }
    if (x == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr || y == nullptr || work == nullptr) {
        return invalid("gated_mlp: null array");
    }
    const std::size_t size = dtype_size(dtype);
    for (const void* p : {x, w_gate, w_up, w_down, static_cast<const void*>(y)}) {
        if (!aligned_to(p, size)) {
            return invalid("gated_mlp: arrays must be aligned to their element size");
        }
    }
    if (overlap(x, tokens * channels * size, y, tokens * outputs * size)) {
        return invalid("gated_mlp: x and y must not overlap");
    }
    try {
        const MlpShape n{tokens, channels, hidden, outputs, activation};
        with_dtype(dtype, [&](auto t) {
            mlp_forward<decltype(t)>({nullptr, x, w_gate, w_up, w_down}, y, dtype, n, work, static_cast<cudaStream_t>(stream));
        });
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}

extern "C" int spectral_gated_mlp_backward(const void* dy, const void* x, const void* codes, const float* scales,
                                           const void* w_gate, const void* w_up, const void* w_down, void* dx,
                                           void* dw_gate, void* dw_up, void* dw_down, int dtype, long long tokens,
                                           int channels, int hidden, int outputs, int activation, void* work, void* stream)
{
    using namespace spectral;
    const int status = check("gated_mlp_backward", dtype, tokens, channels, hidden, outputs);
    if (status != SPECTRAL_OK) {
        return status;
    }
    if (!activation_known(activation)) {
        return invalid("gated_mlp_backward: activation must be SPECTRAL_ACT_NONE, _SILU or _GELU");
    }
    if (dw_gate == nullptr || dw_up == nullptr || dw_down == nullptr) {
        return invalid("gated_mlp_backward: null array");
    }
    const std::size_t size = dtype_size(dtype);
    const auto s = static_cast<cudaStream_t>(stream);
    try {
        if (tokens == 0) {  // sums over nothing
            SPECTRAL_CUDA(cudaMemsetAsync(dw_gate, 0, size * hidden * channels, s));
            SPECTRAL_CUDA(cudaMemsetAsync(dw_up, 0, size * hidden * channels, s));
            SPECTRAL_CUDA(cudaMemsetAsync(dw_down, 0, size * outputs * hidden, s));
            return SPECTRAL_OK;
        }
        if (dy == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr || dx == nullptr || work == nullptr
            || (x == nullptr) == (codes == nullptr) || (codes == nullptr) != (scales == nullptr)) {
            return invalid("gated_mlp_backward: every array must be given, and either x or codes with scales");
        }
        for (const void* p : {dy, x, w_gate, w_up, w_down, static_cast<const void*>(dx), static_cast<const void*>(dw_gate),
                              static_cast<const void*>(dw_up), static_cast<const void*>(dw_down)}) {
            if (!aligned_to(p, size)) {
                return invalid("gated_mlp_backward: arrays must be aligned to their element size");
            }
        }
        if (!aligned_to(scales, sizeof(float))) {
            return invalid("gated_mlp_backward: scales must be aligned to 4 bytes");
        }
        if (overlap(dx, tokens * channels * size, dy, tokens * outputs * size)
            || (x != nullptr && overlap(dx, tokens * channels * size, x, tokens * channels * size))) {
            return invalid("gated_mlp_backward: dx must not overlap dy or x");
        }
        const MlpShape n{tokens, channels, hidden, outputs, activation};
        with_dtype(dtype, [&](auto t) {
            mlp_backward<decltype(t)>({dy, x, w_gate, w_up, w_down}, static_cast<const signed char*>(codes), scales, dx, dw_gate,
                                      dw_up, dw_down, dtype, n, work, s);
        });
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}
