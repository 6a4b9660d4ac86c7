// 8-bit activation checkpoints: an activation kept for the backward pass as one byte per value.
//
// Each row is cut into blocks of 64 values (the last one may be shorter). Per block, in FP32:
//     m = max(|v|, 2^-100),  scale = m / 127,  code = round(v * (127 / m)),  value = code * scale,
// so the error is at most half a step, m / 254. A block that holds an infinity or a NaN gets the
// scale NaN and restores as NaN throughout: a fault in the forward pass stays visible.
//
// Both directions are one pass over the data and HBM-bound (a 16-bit value: 3 + 1/16 bytes moved
// per direction). Eight or sixteen lanes with 16 bytes each share a block, its maximum goes
// through shuffles, and each thread has four blocks in flight. Rows that are not whole 16-byte
// pieces, or whose arrays are not aligned, take 32 lanes per block with single values.

#include "../../include/spectral_b200.h"

#include "backend.hpp"
#include "launch.cuh"
#include "pointwise.cuh"

#include <climits>

namespace spectral {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // blocks in flight per thread

// Values per lane and lanes per block.
template <class T, bool Wide>
struct Shape {
    static constexpr int kValues = Wide ? 16 / static_cast<int>(sizeof(T)) : 2;
    static constexpr int kLanes = kPackBlock / kValues;
};

// Unpacking moves 16 codes per lane to a 16-bit type (one 32-byte store: 50 us against 57 us with 8 for
// 67 M values), 4 to float32 (64 us against 83 us with 8).
template <class T, bool Wide>
struct UnpackShape {
    static constexpr int kValues = Wide ? (sizeof(T) == 2 ? 16 : 4) : 2;
    static constexpr int kLanes = kPackBlock / kValues;
};

// The row and first column of block q of `per_row` blocks a row.
__device__ __forceinline__ void locate(long long q, int per_row, long long& row, int& col)
{
    if (per_row == 1) {
        row = q;
        col = 0;
    } else if (q <= 0x7fffffffLL) {
        const unsigned r = static_cast<unsigned>(q) / static_cast<unsigned>(per_row);
        row = r;
        col = static_cast<int>(static_cast<unsigned>(q) - r * static_cast<unsigned>(per_row)) * kPackBlock;
    } else {
        row = q / per_row;
        col = static_cast<int>(q - row * per_row) * kPackBlock;
    }
}

template <class T, bool Wide>
__global__ void __launch_bounds__(kThreads)
    pack_kernel(const T* __restrict__ x, signed char* __restrict__ codes, float* __restrict__ scales, int width,
                int per_row, long long blocks)
{
    constexpr int kV = Shape<T, Wide>::kValues;
    constexpr int kLanes = Shape<T, Wide>::kLanes;
    allow_next_grid();
    wait_for_previous_grid();
    const int sub = static_cast<int>(threadIdx.x) % kLanes;
    const long long first = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
    const long long step = static_cast<long long>(gridDim.x) * kThreads / kLanes;
    // A block's lanes agree on q0, so whole lane groups leave together; the shuffles name only them.
    for (long long q0 = first; q0 < blocks; q0 += step * kUnroll) {
        Vec<T, kV> raw[kUnroll];
        long long at[kUnroll];
        int have[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long q = q0 + u * step;
            have[u] = 0;
            at[u] = 0;
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                raw[u].v[j] = from_float<T>(0.0f);
            }
            if (q < blocks) {
                long long row;
                int col;
                locate(q, per_row, row, col);
                at[u] = row * width + col;
                const int left = width - col;
                if constexpr (Wide) {
                    have[u] = sub * kV < left ? kV : 0;  // the row is whole pieces
                    at[u] += sub * kV;
                    if (have[u] != 0) {
                        raw[u] = *reinterpret_cast<const Vec<T, kV>*>(x + at[u]);
                    }
                } else {
                    at[u] += sub;
                    have[u] = (sub < left) + (sub + 32 < left);
                    if (have[u] > 0) {
                        raw[u].v[0] = x[at[u]];
                    }
                    if (have[u] > 1) {
                        raw[u].v[1] = x[at[u] + 32];
                    }
                }
            }
        }
        pack_blocks(
            raw, [&](int u) { return q0 + u * step < blocks ? scales + (q0 + u * step) : nullptr; },
            [&](int u, const Vec<signed char, kV>& c) {
                if constexpr (Wide) {
                    if (have[u] != 0) {
                        *reinterpret_cast<Vec<signed char, kV>*>(codes + at[u]) = c;
                    }
                } else {
                    if (have[u] > 0) {
                        codes[at[u]] = c.v[0];
                    }
                    if (have[u] > 1) {
                        codes[at[u] + 32] = c.v[1];
                    }
                }
            });
    }
}

template <class T, bool Wide>
__global__ void __launch_bounds__(kThreads)
    unpack_kernel(const signed char* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ x,
                  int width, int per_row, long long blocks)
{
    constexpr int kV = UnpackShape<T, Wide>::kValues;
    constexpr int kLanes = UnpackShape<T, Wide>::kLanes;
    allow_next_grid();
    wait_for_previous_grid();
    const int sub = static_cast<int>(threadIdx.x) % kLanes;
    const long long first = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
    const long long step = static_cast<long long>(gridDim.x) * kThreads / kLanes;
    for (long long q0 = first; q0 < blocks; q0 += step * kUnroll) {
        Vec<signed char, kV> raw[kUnroll] = {};
        float scale[kUnroll];
        long long at[kUnroll];
        int have[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long q = q0 + u * step;
            have[u] = 0;
            scale[u] = 0.0f;
            if (q < blocks) {
                long long row;
                int col;
                locate(q, per_row, row, col);
                const int left = width - col;
                scale[u] = scales[q];
                at[u] = row * width + col + (Wide ? sub * kV : sub);
                if constexpr (Wide) {
                    have[u] = sub * kV < left ? kV : 0;
                    if (have[u] != 0) {
                        raw[u] = *reinterpret_cast<const Vec<signed char, kV>*>(codes + at[u]);
                    }
                } else {
                    have[u] = (sub < left) + (sub + 32 < left);
                    if (have[u] > 0) {
                        raw[u].v[0] = codes[at[u]];
                    }
                    if (have[u] > 1) {
                        raw[u].v[1] = codes[at[u] + 32];
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const Vec<T, kV> out = narrow<T>(restored<T, kV>(raw[u], scale[u]));
            if constexpr (Wide) {
                if (have[u] != 0) {
                    if constexpr (sizeof(out) == 32) {
                        store32(x + at[u], *reinterpret_cast<const uint32_t(*)[8]>(&out));
                    } else {
                        *reinterpret_cast<Vec<T, kV>*>(x + at[u]) = out;
                    }
                }
            } else {
                if (have[u] > 0) {
                    x[at[u]] = out.v[0];
                }
                if (have[u] > 1) {
                    x[at[u] + 32] = out.v[1];
                }
            }
        }
    }
}

unsigned grid_for(long long blocks, int lanes)
{
    const long long per_cta = static_cast<long long>(kThreads) / lanes * kUnroll;
    const long long ctas = (blocks + per_cta - 1) / per_cta;
    return static_cast<unsigned>(ctas < (1LL << 30) ? ctas : (1LL << 30));
}

// Rows of whole pieces of 16 (times `pieces`) bytes of values, and the codes' pieces aligned.
bool wide_fits(const void* x, const void* codes, int dtype, int width, int pieces)
{
    const int values = 16 / static_cast<int>(dtype_size(dtype)) * pieces;
    return width % values == 0 && aligned_to(x, 16 * static_cast<std::size_t>(pieces)) && aligned_to(codes, static_cast<std::size_t>(values));
}

int check(const char* op, const void* x, const void* codes, const void* scales, int dtype, long long rows, int width)
{
    const std::string name(op);
    if (!dtype_known(dtype)) {
        set_last_error(name + ": dtype must be SPECTRAL_FLOAT32, SPECTRAL_BFLOAT16 or SPECTRAL_FLOAT16");
        return SPECTRAL_INVALID_ARGUMENT;
    }
    if (rows < 0 || width < 0 || (width > 0 && rows > (1LL << 46) / width)) {
        set_last_error(name + ": need rows >= 0, width >= 0 and at most 2^46 values");
        return SPECTRAL_INVALID_ARGUMENT;
    }
    if (rows == 0 || width == 0) {
        return SPECTRAL_OK;
    }
    if (x == nullptr || codes == nullptr || scales == nullptr) {
        set_last_error(name + ": null array");
        return SPECTRAL_INVALID_ARGUMENT;
    }
    if (!aligned_to(x, dtype_size(dtype)) || !aligned_to(scales, 4)) {
        set_last_error(name + ": arrays must be aligned to their element size");
        return SPECTRAL_INVALID_ARGUMENT;
    }
    return SPECTRAL_OK;
}

}  // namespace

void pack8(const void* x, int dtype, signed char* codes, float* scales, long long rows, int width, cudaStream_t stream)
{
    const int per_row = (width - 1) / kPackBlock + 1;
    const long long blocks = rows * per_row;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const auto launch = [&](auto wide) {
            constexpr bool kWide = decltype(wide)::value;
            launch_pdl(pack_kernel<T, kWide>, dim3(grid_for(blocks, Shape<T, kWide>::kLanes)), dim3(kThreads), 0, stream,
                       static_cast<const T*>(x), codes, scales, width, per_row, blocks);
        };
        if (wide_fits(x, codes, dtype, width, 1)) {
            launch(std::true_type{});
        } else {
            launch(std::false_type{});
        }
    });
}

void unpack8(const signed char* codes, const float* scales, void* x, int dtype, long long rows, int width,
             cudaStream_t stream)
{
    const int per_row = (width - 1) / kPackBlock + 1;
    const long long blocks = rows * per_row;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const auto launch = [&](auto wide) {
            constexpr bool kWide = decltype(wide)::value;
            launch_pdl(unpack_kernel<T, kWide>, dim3(grid_for(blocks, UnpackShape<T, kWide>::kLanes)), dim3(kThreads), 0,
                       stream, codes, scales, static_cast<T*>(x), width, per_row, blocks);
        };
        if (wide_fits(x, codes, dtype, width, sizeof(T) == 2 ? 2 : 1)) {
            launch(std::true_type{});
        } else {
            launch(std::false_type{});
        }
    });
}

}  // namespace spectral

extern "C" int spectral_pack8(const void* x, int dtype, void* codes, float* scales, long long rows, int width,
                              void* stream)
{
    using namespace spectral;
    const int status = check("pack8", x, codes, scales, dtype, rows, width);
    if (status != SPECTRAL_OK || rows == 0 || width == 0) {
        return status;
    }
    try {
        pack8(x, dtype, static_cast<signed char*>(codes), scales, rows, width, static_cast<cudaStream_t>(stream));
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}

extern "C" int spectral_unpack8(const void* codes, const float* scales, void* x, int dtype, long long rows, int width,
                                void* stream)
{
    using namespace spectral;
    const int status = check("unpack8", x, codes, scales, dtype, rows, width);
    if (status != SPECTRAL_OK || rows == 0 || width == 0) {
        return status;
    }
    try {
        unpack8(static_cast<const signed char*>(codes), scales, x, dtype, rows, width,
                static_cast<cudaStream_t>(stream));
        return SPECTRAL_OK;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SPECTRAL_CUDA_ERROR;
    }
}
