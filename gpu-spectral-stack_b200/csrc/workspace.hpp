// Workspaces cut into arrays, for the host and for tests of it.
#pragma once

#include <cstddef>
#include <cstdint>

namespace spectral {

// Every array of a workspace starts on this many bytes: bulk copies, tensor maps and 16-byte accesses need 16 of them.
constexpr std::size_t kWorkAlign = 256;

// A workspace's arrays, as offsets in bytes from its first whole kWorkAlign.
class Arena {
public:
    std::size_t take(std::size_t bytes)
    {
        const std::size_t at = size_;
        size_ += (bytes + kWorkAlign - 1) / kWorkAlign * kWorkAlign;
        return at;
    }
    std::size_t size() const { return size_; }

private:
    std::size_t size_ = 0;
};

// Where the arrays of a workspace start, whatever its own alignment, and what the caller has to bring for `bytes` of them.
inline char* work_base(void* work)
{
    return reinterpret_cast<char*>((reinterpret_cast<std::uintptr_t>(work) + kWorkAlign - 1) & ~static_cast<std::uintptr_t>(kWorkAlign - 1));
}
inline std::size_t work_bytes(std::size_t bytes)
{
    return bytes == 0 ? 0 : (bytes + 7) / 8 * 8 + kWorkAlign;
}

// Attention backward, an array of floats: where a tile of rows keeps its constants, `width` of one kind and `width` of the other.
// (In 64 bits: 2^25 tiles of 64 rows, one token of 33 heads each, are 2^32 floats.)
constexpr long long row_constants_at(long long tile, int width) { return tile * 2 * width; }

}  // namespace spectral
