// Argument checks shared by the 8-bit operators: row arrays, their extents and
// whether two of them share bytes.
#pragma once

#include <cstdint>

#include "../../include/ridge_b200.h"

namespace ridge_b200 {

inline int type_size(int32_t type) {
    switch (type) {
        case RIDGE_F16: case RIDGE_BF16: return 2;
        case RIDGE_F32: return 4;
        default: return 0;
    }
}

// `rows` rows of `width` bytes, `pitch` bytes apart.
struct RowArray {
    const void* p;
    int64_t rows, pitch, width;
};

// A pitch (unused with one row) and, unless the array is empty, a pointer
// aligned to its elements. The whole array stays below 2^60 bytes, so that no
// offset in it can pass 63 bits.
inline bool array_ok(const void* p, int64_t M, int64_t D, int64_t ld, int size) {
    if (M > 1 && (ld < D || ld > (int64_t(1) << 58) / M)) return false;
    if (M == 0 || D == 0) return true;
    return p != nullptr && reinterpret_cast<uintptr_t>(p) % uintptr_t(size) == 0;
}

// Whether two arrays share bytes: their address ranges meet, and they are not
// columns of one wider array (same pitch, disjoint windows of a row).
inline bool overlaps(const RowArray& a, const RowArray& b) {
    if (!a.p || !b.p || a.rows == 0 || b.rows == 0 || a.width == 0 || b.width == 0) return false;
    const uint64_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
    const uint64_t a1 = a0 + uint64_t(a.rows - 1) * uint64_t(a.pitch) + uint64_t(a.width);
    const uint64_t b1 = b0 + uint64_t(b.rows - 1) * uint64_t(b.pitch) + uint64_t(b.width);
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.pitch != b.pitch || a.pitch < a.width || a.pitch < b.width) return true;
    const uint64_t ld = uint64_t(a.pitch);
    const uint64_t d = b0 >= a0 ? (b0 - a0) % ld : ld - 1 - (a0 - b0 - 1) % ld;
    return !(d >= uint64_t(a.width) && d + uint64_t(b.width) <= ld);
}

}  // namespace ridge_b200
