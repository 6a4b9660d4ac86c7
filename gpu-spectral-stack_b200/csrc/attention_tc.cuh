#pragma once

// What the tensor-core attention kernels (16-bit values) share: tensor maps over strided heads, tensor-memory
// operands, which keys of a tile count, and wiping those that do not.
//
// A tile of queries is 128 rows: 128 / group tokens with the `group` query heads of a key head side by side
// (the last 128 % group rows stay unused), fetched by one box of (64 values, group heads, tokens). A tile of keys is
// 128 keys. Heads are padded with zeros to 64 or 128 values by the copy; products run over whole 16s of `dim`.

#include "attention.cuh"
#include "mlp.cuh"
#include "umma.cuh"

namespace spectral::attention {

constexpr int kTile = 128;              // rows, keys
constexpr int kBox = kTile * umma::kRowBytes;  // bytes of 128 rows of 64 values
constexpr int kSmemMost = 227 * 1024;

// Strided heads as a tensor map: (value, head, token, sample), boxes of 64 values x heads x tokens. An axis of
// stride 0 (a broadcast) has one entry and its coordinate is always 0.
struct HeadMap {
    CUtensorMap map;
    int head_step = 1;
    int sample_step = 1;
};

__device__ __forceinline__ void load_heads(uint32_t dst, const HeadMap& m, int value, int head, int token, int sample, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(&m.map), "r"(value), "r"(head * m.head_step), "r"(token), "r"(sample * m.sample_step), "r"(tma::smem_addr(bar))
        : "memory");
}

// D = A B with A, 16-bit pairs in 32-bit columns, in tensor memory.
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

// 16 or 32 columns of this warp's 32 lanes, one lane per thread; store_wait before others read them.
__device__ __forceinline__ void store16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void store16(uint32_t taddr, const float (&v)[16])
{
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        w[i] = __float_as_uint(v[i]);
    }
    store16(taddr, w);
}
__device__ __forceinline__ void store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <class T>
__device__ __forceinline__ uint32_t pack2(float2 v)
{
    const Vec<T, 2> two = narrow<T>(Floats<2>{{v}});
    return *reinterpret_cast<const uint32_t*>(&two);
}

// A lane's bytes of the mask over a tile of 32 Words keys, asked for a tile ahead of their use.
template <int Words>
struct MaskBytes {
    unsigned char v[Words];
};

template <int Words>
__device__ __forceinline__ MaskBytes<Words> mask_bytes(const Call& c, int b, int end, int key0)
{
    MaskBytes<Words> m;
    if (c.mask != nullptr) {
        const unsigned char* at = c.mask + static_cast<long long>(b) * c.keys + key0;
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < Words; ++i) {
            m.v[i] = 32 * i + lane < end - key0 ? at[32 * i + lane] : 0;
        }
    }
    return m;
}

// One bit per key of the tile at key0 that counts: bit i of word w is key0 + 32 w + i. The whole warp calls it.
template <int Words>
__device__ __forceinline__ void tile_bits(const Call& c, const MaskBytes<Words>& m, int end, int key0, uint32_t (&w)[4])
{
    const int left = end - key0;
#pragma unroll
    for (int i = 0; i < Words; ++i) {
        const int n = left - 32 * i;
        w[i] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
    }
    if (c.mask != nullptr) {
#pragma unroll
        for (int i = 0; i < Words; ++i) {
            w[i] = __ballot_sync(0xffffffffu, m.v[i] != 0);
        }
    }
}

// Whether the first 32 Words keys all do.
template <int Words = 4>
__device__ __forceinline__ bool all_count(const uint32_t (&w)[4])
{
    return (Words == 4 ? w[0] & w[1] & w[2] & w[3] : w[0] & w[1]) == 0xffffffffu;
}

// Zeros into the rows of a tile (`boxes` boxes of Rows rows) whose keys do not count: a masked weight of 0 times an infinity
// or NaN would be a NaN. The Warps warps that are about to hand over the weights each take a share, `warp` of them;
// the tile has landed, and the product that reads it comes after their arrivals.
template <int Rows, int Warps>
__device__ __forceinline__ void wipe_rows(uint32_t tile, int boxes, const uint32_t (&w)[4], int warp)
{
    const int lane = threadIdx.x & 31;
    for (int r = warp * (Rows / Warps) + lane / 8; r < (warp + 1) * (Rows / Warps); r += 4) {
        const uint32_t word = r < 64 ? (r < 32 ? w[0] : w[1]) : (r < 96 ? w[2] : w[3]);
        if ((word >> (r & 31) & 1u) == 0) {
            for (int box = 0; box < boxes; ++box) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + (box * Rows + r) * umma::kRowBytes + (lane & 7) * 16), "r"(0)
                             : "memory");
            }
        }
    }
    tma::fence_proxy_async();
}

// N columns of 32 rows, a row a lane: lane l's at its own p (if it is `live`), `valid` of them. `sectors` (the same in all
// lanes): every row's run is whole 32-byte sectors, and each lane stores its own; else the values change lanes first, so that
// a row's are stored side by side. `rest` (16-bit types, or NULL): the bytes that out's rounding leaves, at the same places.
template <class T, int N>
__device__ __forceinline__ void store_lanes(T* p, unsigned char* rest, bool live, float (&v)[N], int valid, bool sectors)
{
    if (sectors) {
        if (live) {
            mlp::store_values<T>(p, v, valid);
            if constexpr (sizeof(T) == 2) {
                if (rest != nullptr) {
                    Vec<unsigned char, N> bytes;
#pragma unroll
                    for (int j = 0; j < N / 2; ++j) {
                        reinterpret_cast<unsigned short*>(&bytes)[j] = rest_of<T>(make_float2(v[2 * j], v[2 * j + 1]));
                    }
                    *reinterpret_cast<Vec<unsigned char, N>*>(rest) = bytes;  // dim is a multiple of 16 then
                }
            }
        }
        return;
    }
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int s = N / 2; s > 0; s >>= 1) {
        const bool upper = (lane & s) != 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if ((j & s) == 0) {
                const float other = __shfl_xor_sync(0xffffffffu, upper ? v[j] : v[j | s], s);
                v[j] = upper ? other : v[j];
                v[j | s] = upper ? v[j | s] : other;
            }
        }
    }
    const int first = lane & ~(N - 1);  // N lanes hold the columns of N rows
    const int col = lane & (N - 1);
    const unsigned there = __ballot_sync(0xffffffffu, live);
    const auto at = reinterpret_cast<unsigned long long>(p);
    const auto rest_at = reinterpret_cast<unsigned long long>(rest);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        T* row = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, at, first + j));
        const bool stores = (there >> (first + j) & 1u) != 0 && col < valid;
        if (stores) {
            row[col] = from_float<T>(v[j]);
        }
        if constexpr (sizeof(T) == 2) {
            if (rest != nullptr) {
                auto* bytes = reinterpret_cast<unsigned char*>(__shfl_sync(0xffffffffu, rest_at, first + j));
                if (stores) {
                    bytes[col] = static_cast<unsigned char>(rest_of<T>(make_float2(v[j], 0.0f)));
                }
            }
        }
    }
}

// Whether rows of dim values of `size` bytes from `base` on are whole sectors.
__device__ __forceinline__ bool whole_sectors(const void* base, int dim, int size)
{
    return ((reinterpret_cast<std::uintptr_t>(base) | static_cast<std::uintptr_t>(dim * size)) & 31u) == 0;
}

// --- host ------------------------------------------------------------------------------------------

// Whether a tensor map can read the array as it lies: 16-byte steps on every axis that is walked. (An axis of stride 0
// is not walked if its box takes one entry.)
inline bool mappable(const void* base, const Strides& s, long long samples, long long tokens, long long heads, bool one_head)
{
    const auto whole = [](long long stride) { return stride > 0 && stride % 8 == 0 && stride < (1LL << 39); };
    return base != nullptr && aligned_to(base, 16) && (samples <= 1 || s.sample == 0 || whole(s.sample)) && (tokens <= 1 || whole(s.token))
           && (heads <= 1 || (one_head && s.head == 0) || whole(s.head));
}

inline HeadMap head_map(const void* base, bool is_bf16, const Strides& s, long long samples, long long tokens, long long heads, int dim,
                        int box_heads, int box_tokens)
{
    HeadMap m;
    const bool one_sample = samples > 1 && s.sample == 0;
    const bool one_head = heads > 1 && s.head == 0;
    m.sample_step = one_sample ? 0 : 1;
    m.head_step = one_head ? 0 : 1;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(one_head ? 1 : heads),
                                static_cast<cuuint64_t>(tokens < 1 ? 1 : tokens), static_cast<cuuint64_t>(one_sample ? 1 : samples)};
    // The stride of an axis with one entry is never used, but has to be a valid one.
    const cuuint64_t row = (static_cast<cuuint64_t>(dim) * 2 + 15) / 16 * 16;
    const auto bytes = [&](long long stride, cuuint64_t entries) { return entries <= 1 ? row : static_cast<cuuint64_t>(2 * stride); };
    const cuuint64_t strides[3] = {bytes(s.head, dims[1]), bytes(s.token, dims[2]), bytes(s.sample, dims[3])};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(umma::kAtom), static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens), 1};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    const CUresult r = umma::encode_fn()(&m.map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                         const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        throw CudaError("cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(r)) + ")");
    }
    return m;
}

// An array for a tensor map: as it lies, or copied to rows of whole 16 bytes.
struct Operand {
    const void* source = nullptr;
    Strides stride;
    long long tokens = 0;
    int heads = 0;
    bool one_head = false;  // its boxes take one head
    bool staged = false;
    std::size_t at = 0;  // in the workspace

    // Before the launch: `work` is the call's workspace.
    const void* base(char* work) const { return staged ? work + at : source; }
    Strides strides(int dim) const
    {
        if (!staged) {
            return stride;
        }
        const long long pitch = (dim + 7) / 8 * 8;
        return {tokens * heads * pitch, heads * pitch, pitch};
    }
};

inline Operand operand(Arena& arena, const void* base, const Strides& s, long long samples, long long tokens, int heads, int dim, bool one_head)
{
    Operand o;
    o.source = base;
    o.stride = s;
    o.tokens = tokens;
    o.heads = heads;
    o.one_head = one_head;
    o.staged = !mappable(base, s, samples, tokens, heads, one_head);
    if (o.staged) {
        o.at = arena.take(static_cast<std::size_t>(samples) * tokens * heads * ((dim + 7) / 8 * 8) * 2);
    }
    return o;
}

// Copies the operands that need it.
void stage(const Operand* const* operands, int count, int batch, int dim, char* work, cudaStream_t stream);

// The most keys (rows) whose products share an accumulator: the tensor core cuts its FP32 sum once per 16 of
// them, which pulls a sum of one sign down by 1.1e-7 each time; 512 times is 5.5e-5, a fifth of a rounding to f16. Longer
// sums are split, and their parts added in FP32.
constexpr int kLongestSum = 8192;

}  // namespace spectral::attention
