// Sequences of packed rows (uzu_row_sequence): the host's checks, and the table of them that a launch takes along. Plain C++.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <vector>

#include "../../include/uzu_b200.h"

namespace uzu {

constexpr uint32_t kLaunchSequences = 128;      // of one launch (a kernel's arguments end at 4 KB); more take more launches

struct PackedSequence {
    uint32_t first, rows, slot_fresh, tile0;      // tile0: the first of the launch's tiles that is this sequence's
#ifdef __CUDACC__
    __host__ __device__
#endif
    uint32_t slot() const { return slot_fresh & 0x7fffffffu; }
#ifdef __CUDACC__
    __host__ __device__
#endif
    bool fresh() const { return slot_fresh >> 31 != 0; }
};
struct SequenceTable {
    uint32_t count, tiles;
    PackedSequence s[kLaunchSequences];
};

// null, or what is wrong with them
inline const char* check_sequences(const uzu_row_sequence* s, uint32_t count, uint32_t rows, uint32_t slots) {
    if (!count) return nullptr;
    if (!s) return "null sequences";
    if (slots >> 31) return "at most 2^31 - 1 slots";
    try {
        std::vector<uint32_t> named(count);
        std::vector<std::pair<uint32_t, uint32_t>> spans;
        spans.reserve(count);
        for (uint32_t i = 0; i < count; ++i) {
            if (s[i].slot >= slots) return "a sequence's slot is not below slots";
            if ((uint64_t)s[i].first_row + s[i].rows > rows) return "a sequence ends behind the last row";
            named[i] = s[i].slot;
            if (s[i].rows) spans.emplace_back(s[i].first_row, s[i].rows);
        }
        std::sort(named.begin(), named.end());
        if (std::adjacent_find(named.begin(), named.end()) != named.end()) return "two sequences name the same slot";
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            if (spans[i - 1].first + spans[i - 1].second > spans[i].first) return "two sequences share a row";
    } catch (const std::bad_alloc&) {
        return "out of host memory";
    }
    return nullptr;
}

// sequences [begin, min(count, begin + kLaunchSequences)) with as many tiles as `tiles_of(rows)` says, and the next begin
template <typename F>
inline uint32_t fill_sequences(SequenceTable& t, const uzu_row_sequence* s, uint32_t count, uint32_t begin, F tiles_of) {
    const uint32_t end = std::min(count, begin + kLaunchSequences);
    t.count = end - begin;
    t.tiles = 0;
    for (uint32_t i = begin; i < end; ++i) {
        t.s[i - begin] = {s[i].first_row, s[i].rows, s[i].slot | (s[i].fresh ? 0x80000000u : 0u), t.tiles};
        t.tiles += tiles_of(s[i].rows);
    }
    return end;
}

// bytes of `rows` rows of `width` elements, `stride` elements apart
inline uint64_t rows_extent(uint64_t rows, uint64_t stride, uint64_t width, uint64_t size) { return rows ? ((rows - 1) * stride + width) * size : 0; }
// Whether two arrays of rows share bytes. Slices of the same wide rows, side by side, do not.
inline bool rows_overlap(uint64_t a, uint64_t a_stride, uint64_t a_width, uint64_t b, uint64_t b_stride, uint64_t b_width, uint64_t rows, uint64_t size) {
    if (!rows || a + rows_extent(rows, a_stride, a_width, size) <= b || b + rows_extent(rows, b_stride, b_width, size) <= a) return false;
    if (a_stride != b_stride || !a_stride) return true;
    const uint64_t pitch = a_stride * size, off = (b >= a ? (b - a) % pitch : (pitch - (a - b) % pitch) % pitch);      // from a slice of `a` to the next of `b`
    return off < a_width * size || off + b_width * size > pitch;
}
inline bool bytes_overlap(uint64_t a, uint64_t a_bytes, uint64_t b, uint64_t b_bytes) { return a && b && a_bytes && b_bytes && a < b + b_bytes && b < a + a_bytes; }

}  // namespace uzu
