// Index arithmetic of the head-wise kernels and the paged cache: division by a launch's
// constants, slot -> (page, place) and output row -> (page, place).  Plain C++ apart from the function qualifiers, so that every guard below is
// also compiled and tested on the host.  No function reads outside the arrays it is
// given, whatever the indices in them say.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define B2K_HD __host__ __device__ __forceinline__
#else
#define B2K_HD inline
#endif

namespace paging {

// Division of n < 2^31 by a constant of the launch: with s = ceil(log2 d) and
// m = ceil(2^(31 + s) / d), which fits 32 bits, floor(n m / 2^(31 + s)) = floor(n / d),
// because m d - 2^(31 + s) < 2^s keeps the error of n m / 2^(31 + s) below 1 / d.
struct Divisor {
    uint32_t d, m, shift;
    B2K_HD uint32_t quotient(uint32_t n) const { return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> shift); }
};
inline Divisor divisor(uint32_t d) {
    uint32_t s = 0;
    while (s < 31 && (1u << s) < d) ++s;
    return Divisor{d, static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + d - 1) / d), 31 + s};
}

struct Place {
    int64_t page, slot;
    bool ok;
};

B2K_HD int64_t load_index(const void *p, int bytes, int64_t i) {
    return bytes == 4 ? static_cast<int64_t>(static_cast<const int32_t *>(p)[i]) : static_cast<const int64_t *>(p)[i];
}

// Quotient and remainder of non-negative numbers; a 64-bit division costs about 100
// instructions, so the common case takes 32-bit ones.
B2K_HD void divide(int64_t n, int64_t d, int64_t &quotient, int64_t &rest) {
    if (((n | d) >> 32) == 0) {
        const uint32_t q = static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
        quotient = q;
        rest = static_cast<uint32_t>(n) - q * static_cast<uint32_t>(d);
    } else {
        quotient = n / d;
        rest = n - quotient * d;
    }
}

// pages * page_size fits 63 bits (checked by the caller).
B2K_HD Place place_of_slot(int64_t slot, int64_t pages, int64_t page_size) {
    Place at{0, 0, slot >= 0 && slot < pages * page_size};
    if (at.ok) divide(slot, page_size, at.page, at.slot);
    return at;
}

// The sequence b with offsets[b] <= row < offsets[b + 1], or -1.  offsets holds
// seqs + 1 values; empty sequences (equal neighbours) own no row.
B2K_HD int64_t sequence_of_row(const void *offsets, int bytes, int64_t seqs, int64_t row) {
    if (row < load_index(offsets, bytes, 0)) return -1;
    int64_t lo = 0, hi = seqs + 1;        // offsets[lo] <= row, and offsets[hi] > row as far as it was looked at
    while (hi - lo > 1) {
        const int64_t mid = lo + (hi - lo) / 2;
        if (load_index(offsets, bytes, mid) <= row) lo = mid;
        else hi = mid;
    }
    return lo < seqs ? lo : -1;
}

B2K_HD Place place_in_sequence(int64_t position, const void *table, int64_t table_stride, int64_t table_width,
                               int table_bytes, int64_t sequence, int64_t pages, int64_t page_size) {
    Place at{0, 0, false};
    if (position < 0) return at;
    int64_t column;
    divide(position, page_size, column, at.slot);
    if (column >= table_width) return at;
    at.page = load_index(table, table_bytes, sequence * table_stride + column);
    at.ok = at.page >= 0 && at.page < pages;
    return at;
}

}  // namespace paging
