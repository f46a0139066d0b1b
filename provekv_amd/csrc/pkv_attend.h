// pkv_attend.h -- live caches: what the host half (pkv_attend.cpp) hands to the
// kernels (pkv_attend.hip).  Not part of the C ABI.
#pragma once
#include <stdint.h>

#include "../../include/pkv_codec.h"

namespace pkv {

// A cache view as the kernels read it: pkv_kv_view's pointers and strides
// (elements), one layer's or several layers'.
struct KvDev {
    const uint8_t* k;
    const uint8_t* v;
    const uint8_t* ks;
    const uint8_t* vs;
    uint64_t copy, layer, head, slot;   // strides, elements
};

struct AttendDev {
    KvDev kv;
    const uint8_t* q;
    uint8_t* out;
    uint64_t q_copy, q_row, q_head, o_copy, o_row, o_head;   // elements
    const int32_t* lens;
    const int32_t* q_lens;
    float* lse;
    float* weights;
    uint64_t w_copy, w_head;
    float* stats;          // [copy][kv head][row i * group + g] (base, factor): weight 2^(s * scale2 + base) * factor
    uint32_t copies, heads, group, nq, max_len, window, sinks;
    uint32_t reach;        // window, 2^31 at most and where there is none: a row sees slots less than this behind it
    float scale2;          // scale * log2 e
};

struct RowsDev {
    KvDev kv;
    uint8_t* keys;
    uint8_t* values;
    uint64_t copy, layer, head, row;    // strides of keys / values, elements
    const int32_t* first;
    const int32_t* counts;
    uint32_t copies, layers, heads, slots, rows;
};

struct EvictDev {
    KvDev kv, into;
    const int32_t* lens;
    int32_t* new_lens;
    int32_t* kept;
    const float* w;
    float* w_out;
    uint64_t ws[3], os[3];
    uint32_t copies, layers, heads, slots, into_slots, budget, sinks, recent;
    uint32_t in_place;
};

// Launchers (pkv_attend.hip); a hipError_t as int.  dim 64 or 128.
uint64_t attend_workspace(const AttendDev& a, uint32_t dim, int cache_dtype, int dtype);
bool attend_fits(const AttendDev& a, uint32_t dim, int cache_dtype);   // the launches are within the device's limits
bool evict_fits(const EvictDev& e, uint32_t dim, int dtype);
int launch_attend(const AttendDev& a, uint32_t dim, int cache_dtype, int dtype, uint8_t* workspace, void* stream);
int launch_fp4_store(const RowsDev& r, uint32_t dim, int dtype, void* stream);
int launch_fp4_load(const RowsDev& r, uint32_t dim, int dtype, void* stream);
int launch_evict(const EvictDev& e, uint32_t dim, int dtype, void* stream);

}  // namespace pkv
