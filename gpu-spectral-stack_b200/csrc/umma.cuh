#pragma once

// The tcgen05 pieces of the 16-bit matrix-product kernels: shared-memory and instruction
// descriptors, the MMA and its commit, accumulator reads, tiled TMA loads, and the tensor maps.
//
// Operand tiles are 64 values (128 bytes) wide along the contiguous dimension and stored by TMA
// with the 128-byte swizzle, 1 KiB aligned. The same tile serves as either kind of operand:
//   K-major   rows are M or N, the 64 contiguous values are K: 8-row groups 1 KiB apart; 16 values
//             of K are 32 bytes further along the row;
//   MN-major  the 64 contiguous values are M or N, rows are K: 8 rows of K 1 KiB apart, the
//             next 64 values of M or N one tile further; 16 rows of K are 2 KiB further.
// No load is multicast, and every tensor map covers this GPU's own memory.

#include "common.cuh"
#include "tma.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <string>

namespace spectral::umma {

constexpr int kAtom = 64;          // 16-bit values per 128-byte row
constexpr int kRowBytes = 128;
constexpr int kGroupBytes = 1024;  // 8 rows

// Shared-memory matrix descriptors: start address, leading and stride byte offsets (16-byte units),
// version 1 at bit 46, 128-byte swizzle (2) at bit 61. Everything but the address is a constant, and a
// step of 16 along K adds a constant to the address field: one descriptor per tile, one addition per
// MMA. (Building each from its byte address cost the issuing warp some 150 cycles an MMA, more than
// the MMA itself.)
constexpr uint64_t constant_bits(uint32_t leading)
{
    return (static_cast<uint64_t>(leading >> 4) << 16) | (static_cast<uint64_t>(kGroupBytes >> 4) << 32) | (1ull << 46)
           | (2ull << 61);
}

// A K-major tile at `addr`; K step s is + kStepK * s.
constexpr uint64_t kStepK = 32 >> 4;
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return constant_bits(16) | (addr >> 4); }

// An MN-major tile at `addr` whose next 64 rows of M or N are Next bytes further; K step s is
// + kStepMn * s.
constexpr uint64_t kStepMn = 2 * kGroupBytes >> 4;
template <uint32_t Next>
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr)
{
    return constant_bits(Next) | (addr >> 4);
}

// Instruction descriptor of kind::f16 with an FP32 accumulator: operand type (0 f16, 1 bf16) at
// bits 7 and 10, majors (1: MN) at 15 and 16, N / 8 at 17, M / 16 at 24.
constexpr uint32_t instruction(bool is_bf16, bool a_mn, bool b_mn, int m, int n)
{
    return (1u << 4) | ((is_bf16 ? 1u : 0u) << 7) | ((is_bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15)
           | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n / 8) << 17) | (static_cast<uint32_t>(m / 16) << 24);
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

// `bar` completes once every MMA this thread has issued so far has.
__device__ __forceinline__ void commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tma::smem_addr(bar))
                 : "memory");
}

__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <int Cols>
__device__ __forceinline__ void alloc(uint32_t* slot)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tma::smem_addr(slot)), "n"(Cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

template <int Cols>
__device__ __forceinline__ void dealloc(uint32_t tmem)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Cols) : "memory");
}

// True in exactly one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one()
{
    uint32_t pred = 0;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
    return pred != 0;
}

__device__ __forceinline__ void arrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tma::smem_addr(bar)) : "memory");
}

// Starts the read of 32 accumulator columns of this warp's 32 lanes (one lane per thread);
// load_wait makes the registers usable.
__device__ __forceinline__ void load32(uint32_t taddr, float (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}

// 16 columns, as load32.
__device__ __forceinline__ void load16(uint32_t taddr, float (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr));
}
__device__ __forceinline__ void load_run(uint32_t taddr, float (&v)[16]) { load16(taddr, v); }
__device__ __forceinline__ void load_run(uint32_t taddr, float (&v)[32]) { load32(taddr, v); }
__device__ __forceinline__ void load_wait(float (&v)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
}

// Waits for this thread's accumulator reads; v's registers are in-out operands, so no use of them
// moves above the wait.
__device__ __forceinline__ void load_wait(float (&v)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                   "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
                   "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 :
                 : "memory");
}

// One tiled TMA load of `map`'s box at (c0, c1, c2) into shared `dst`, completing on `bar`. c0 is
// a multiple of 64 values (128 bytes).
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(tma::smem_addr(bar))
        : "memory");
}

// --- host ------------------------------------------------------------------------------------------

inline PFN_cuTensorMapEncodeTiled encode_fn()
{
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess
            && q == cudaDriverEntryPointSuccess) {
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled>(p);
        }
    });
    if (fn == nullptr) {
        throw CudaError("cuTensorMapEncodeTiled is not available from the driver");
    }
    return fn;
}

// A matrix of 16-bit values: `planes` matrices of rows x cols, `pitch` values a row (a multiple of
// 8), plane_stride values apart; boxes of 64 values x box_rows rows, zero outside.
inline CUtensorMap matrix_map(const void* base, bool is_bf16, long long rows, long long cols, long long pitch, int planes,
                              long long plane_stride, int box_rows)
{
    CUtensorMap map;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch) * 2,
                                   static_cast<cuuint64_t>(planes > 1 ? plane_stride : pitch * rows) * 2};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(kAtom), static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult r =
        encode_fn()(&map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                    const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        throw CudaError("cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(r)) + ")");
    }
    return map;
}

}  // namespace spectral::umma
