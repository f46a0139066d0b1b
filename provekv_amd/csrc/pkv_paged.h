// pkv_paged.h -- paged caches and packed prompts: what the host half
// (pkv_paged.cpp) hands to the kernels (pkv_paged.hip).  Not part of the C ABI.
#pragma once
#include <stdint.h>

#include "../../include/pkv_codec.h"

namespace pkv {

// Packed rows of sequences and where their slots are (pkv_sequences).
struct SeqsDev {
    bool paged;              // false: packed prompts, slot j is the sequence's row j
    const int32_t* tables;
    uint64_t table;          // words from a sequence to the next
    const int32_t* lens;     // null: a sequence's length is its rows
    const int32_t* starts;   // null: `each` rows a sequence
    uint32_t seqs, pages, shift, rows, each;   // shift: log2 of a page's slots
    uint32_t max_len;
};

struct PagedDev {
    SeqsDev seq;
    const uint8_t* k;
    const uint8_t* v;
    const uint8_t* ks;
    const uint8_t* vs;
    uint64_t page;                             // elements, as all strides
    uint64_t k_head, k_slot, v_head, v_slot;   // pages: the same for both
    const uint8_t* q;
    uint8_t* out;
    uint64_t q_row, q_head, o_row, o_head;
    float* lse;
    uint32_t heads, group, max_rows, window, sinks;
    uint32_t reach;          // window, 2^31 at most and where there is none: a row sees slots less than this behind it
    float scale2;            // scale * log2 e
    uint32_t clear;          // nobody's rows of out become 0
};

struct PagedRowsDev {
    SeqsDev seq;
    uint8_t* k;
    uint8_t* v;
    uint8_t* ks;
    uint8_t* vs;
    uint64_t p_layer, page, p_head, slot;      // strides of the pages
    uint8_t* keys;
    uint8_t* values;
    uint64_t layer, row, head;                 // strides of keys / values
    uint32_t layers, heads;
};

// Launchers (pkv_paged.hip); a hipError_t as int.  dim 64 or 128.
uint64_t paged_workspace(const PagedDev& a, uint32_t dim, int cache_dtype);
bool paged_fits(const PagedDev& a, uint32_t dim, int cache_dtype);   // the launches are within the device's limits
int launch_paged(const PagedDev& a, uint32_t dim, int cache_dtype, int dtype, uint8_t* workspace, void* stream);
int launch_paged_store(const PagedRowsDev& r, uint32_t dim, int cache_dtype, int dtype, void* stream);
int launch_paged_load(const PagedRowsDev& r, uint32_t dim, int cache_dtype, int dtype, void* stream);

}  // namespace pkv
