// The memory that an array can touch, for checks of arguments.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace spectral {

struct Extent {
    std::uintptr_t first = 0, last = 0;  // bytes [first, last); empty for NULL or no bytes

    Extent() = default;
    Extent(const void* p, unsigned long long bytes)
        : first(reinterpret_cast<std::uintptr_t>(p)), last(p == nullptr ? first : first + bytes)
    {
    }
    // A strided view of (sample, token, head) with `dim` values of `size` bytes side by side; strides of either sign.
    Extent(const void* p, const long long (&stride)[3], const long long (&count)[3], int dim, std::size_t size)
    {
        first = last = reinterpret_cast<std::uintptr_t>(p);
        if (p == nullptr || count[0] <= 0 || count[1] <= 0 || count[2] <= 0) {
            return;
        }
        long long low = 0, high = dim;
        for (int i = 0; i < 3; ++i) {
            (stride[i] < 0 ? low : high) += stride[i] * (count[i] - 1);
        }
        first += low * static_cast<long long>(size);
        last += high * static_cast<long long>(size);
    }
    bool meets(const Extent& o) const { return first < last && o.first < o.last && first < o.last && o.first < last; }
};

// Whether one of the written arrays shares memory with another of them or with one of those read.
inline bool any_overlap(std::initializer_list<Extent> written, std::initializer_list<Extent> read)
{
    for (const Extent* w = written.begin(); w != written.end(); ++w) {
        for (const Extent& r : read) {
            if (w->meets(r)) {
                return true;
            }
        }
        for (const Extent* o = w + 1; o != written.end(); ++o) {
            if (w->meets(*o)) {
                return true;
            }
        }
    }
    return false;
}

}  // namespace spectral
