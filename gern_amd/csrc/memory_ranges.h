// Whether the buffers of a call share memory.  Addresses and sizes only; nothing is read.
#pragma once

#include <cstdint>

namespace gern_detail {

// Whether [a, a + na) and [b, b + nb), sizes in bytes, share memory.
inline bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    return na > 0 && nb > 0 && pa < pb + (uintptr_t)nb && pb < pa + (uintptr_t)na;
}

// Rows of `width` bytes, `stride` bytes apart (stride >= width).
struct Rows {
    const void *at;
    int64_t rows, stride, width;

    // From the first byte to the last one, at most what is left of the address space.
    int64_t bytes() const {
        if (rows <= 0) {
            return 0;
        }
        const unsigned __int128 n = (unsigned __int128)(rows - 1) * (uint64_t)stride + (uint64_t)width, room = UINTPTR_MAX - reinterpret_cast<uintptr_t>(at);
        const unsigned __int128 most = room < INT64_MAX ? room : INT64_MAX;
        return (int64_t)(n < most ? n : most);
    }
};

inline bool overlap(const Rows &a, const void *b, int64_t nb) {
    return overlap(a.at, a.bytes(), b, nb);
}

// Two arrays of as many rows, which may stand side by side in wider rows: of the same stride, they share no memory if no
// row of one reaches into a row of the other.
inline bool overlap(const Rows &a, const Rows &b) {
    if (!overlap(a.at, a.bytes(), b.at, b.bytes())) {
        return false;
    }
    if (a.stride != b.stride || a.rows <= 1) {
        return true;
    }
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.at), pb = reinterpret_cast<uintptr_t>(b.at);
    const bool a_first = pa <= pb;
    const uint64_t at = (uint64_t)(a_first ? pb - pa : pa - pb) % (uint64_t)a.stride;  // of the later one's rows in the earlier one's
    const int64_t first = a_first ? a.width : b.width, second = a_first ? b.width : a.width;
    return at < (uint64_t)first || at + (uint64_t)second > (uint64_t)a.stride;
}

}  // namespace gern_detail
