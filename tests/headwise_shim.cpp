// Host build of the cache's index arithmetic and of the argument structs' layout, for
// tests without a GPU.
#include <stddef.h>

#include "../include/b2k.h"
#include "../numba_cuda_b200/csrc/b2k_pages.cuh"

extern "C" {

int64_t shim_size(int which) {
    switch (which) {
        case 0: return sizeof(b2k_heads);
        case 1: return sizeof(b2k_rotation);
        case 2: return sizeof(b2k_cache);
        case 3: return offsetof(b2k_rotation, eps);
        case 4: return offsetof(b2k_rotation, positions_dev);
        case 5: return offsetof(b2k_cache, v);
    }
    return -1;
}

int shim_place_of_slot(int64_t slot, int64_t pages, int64_t page_size, int64_t *page, int64_t *place) {
    const paging::Place at = paging::place_of_slot(slot, pages, page_size);
    *page = at.page;
    *place = at.slot;
    return at.ok;
}

int64_t shim_sequence_of_row(const void *offsets, int bytes, int64_t seqs, int64_t row) {
    return paging::sequence_of_row(offsets, bytes, seqs, row);
}

int shim_place_in_sequence(int64_t position, const void *table, int64_t stride, int64_t width, int bytes, int64_t sequence,
                           int64_t pages, int64_t page_size, int64_t *page, int64_t *place) {
    const paging::Place at = paging::place_in_sequence(position, table, stride, width, bytes, sequence, pages, page_size);
    *page = at.page;
    *place = at.slot;
    return at.ok;
}
}

extern "C" uint32_t shim_quotient(uint32_t n, uint32_t d) { return paging::divisor(d).quotient(n); }
