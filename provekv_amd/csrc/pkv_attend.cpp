// pkv_attend.cpp -- host half of the live-cache calls of include/pkv_codec.h:
// argument checks, and the launches on the context's device.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "pkv_attend.h"
#include "pkv_internal.h"

using namespace pkv;

namespace {

using U128 = unsigned __int128;

int hip_rc(int e) {
    if (e == hipSuccess) return PKV_OK;
    return e == hipErrorOutOfMemory ? PKV_ERR_OOM : PKV_ERR_DEVICE;
}

// The context's device for the length of a call; the caller's current device
// comes back afterwards.
struct OnDevice {
    int was = -1, rc = PKV_OK;
    explicit OnDevice(int device) {
        if (hipGetDevice(&was) != hipSuccess) { rc = PKV_ERR_DEVICE; was = -1; return; }
        if (was == device) { was = -1; return; }
        if (hipSetDevice(device) != hipSuccess) rc = PKV_ERR_DEVICE;
    }
    ~OnDevice() {
        if (was >= 0) (void)hipSetDevice(was);
    }
};

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
uint64_t elem_bytes(int dtype) { return dtype == PKV_F32 ? 4 : 2; }

struct Axis {
    uint64_t stride;
    uint32_t count;
};
// Elements from the first row's start to the last row's end; 0: past 2^62.
uint64_t extent(const Axis* a, int n, uint64_t inner) {
    U128 e = inner;
    for (int i = 0; i < n; ++i) e += static_cast<U128>(a[i].stride) * (a[i].count - 1);
    return e >> 62 ? 0 : static_cast<uint64_t>(e);
}
// No two rows of `inner` elements share one: along every axis, in the order of
// their strides, a step is at least what the axes inside it span.
bool distinct(const Axis* a, int n, uint64_t inner) {
    Axis s[4];
    int m = 0;
    for (int i = 0; i < n; ++i)
        if (a[i].count > 1) s[m++] = a[i];
    std::sort(s, s + m, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
    U128 span = inner;
    for (int i = 0; i < m; ++i) {
        if (s[i].stride < span) return false;
        span += static_cast<U128>(s[i].stride) * (s[i].count - 1);
    }
    return true;
}
bool overlap(const void* a, uint64_t an, const void* b, uint64_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bn && y < x + an;
}

constexpr uint32_t kMaxCount = 0x7fffffffu;
constexpr uint32_t kMaxRows = 1u << 30;   // query rows of all copies and query heads
// Elements from a slot to the next: a kernel's tile of 64 slots stays within
// 32-bit offsets of its first.
constexpr uint64_t kMaxSlotStride = 1u << 22;

int check_view(const pkv_kv_view& v, bool written) {
    if (v.dim != 64 && v.dim != 128) return PKV_ERR_UNSUPPORTED;
    if (v.dtype < PKV_F32 || v.dtype > PKV_FP4) return PKV_ERR_INVALID_ARG;
    if (!v.copies || !v.layers || !v.heads || !v.slots) return PKV_ERR_INVALID_ARG;
    if (v.slots > kMaxCount / 2 || static_cast<U128>(v.copies) * v.layers * v.heads > kMaxCount)
        return PKV_ERR_INVALID_ARG;
    if (!v.d_keys || !v.d_values || !aligned(v.d_keys, 16) || !aligned(v.d_values, 16)) return PKV_ERR_INVALID_ARG;
    uint64_t unit = 16 / elem_bytes(v.dtype);
    if (v.dtype == PKV_FP4) {
        unit = v.dim;
        // a row's scale bytes are read as one word of dim / 32 bytes
        if (!v.d_key_scales || !v.d_value_scales || !aligned(v.d_key_scales, v.dim / 32) ||
            !aligned(v.d_value_scales, v.dim / 32))
            return PKV_ERR_INVALID_ARG;
    } else if (v.d_key_scales || v.d_value_scales) {
        return PKV_ERR_INVALID_ARG;
    }
    if (v.slot_stride > kMaxSlotStride) return PKV_ERR_INVALID_ARG;
    if (v.copy_stride % unit || v.layer_stride % unit || v.head_stride % unit || v.slot_stride % unit)
        return PKV_ERR_INVALID_ARG;
    const Axis a[4] = {{v.copy_stride, v.copies}, {v.layer_stride, v.layers}, {v.head_stride, v.heads},
                       {v.slot_stride, v.slots}};
    const uint64_t e = extent(a, 4, v.dim);
    if (!e || e > v.elems) return PKV_ERR_INVALID_ARG;
    if (written && !distinct(a, 4, v.dim)) return PKV_ERR_INVALID_ARG;
    return PKV_OK;
}

KvDev dev(const pkv_kv_view& v) {
    return {static_cast<const uint8_t*>(v.d_keys), static_cast<const uint8_t*>(v.d_values), v.d_key_scales,
            v.d_value_scales, v.copy_stride, v.layer_stride, v.head_stride, v.slot_stride};
}

AttendDev attend_dev(const pkv_attend_op& op) {
    AttendDev a{};
    a.kv = dev(op.cache);
    a.q = static_cast<const uint8_t*>(op.d_q);
    a.out = static_cast<uint8_t*>(op.d_out);
    a.q_copy = op.q_copy_stride; a.q_row = op.q_row_stride; a.q_head = op.q_head_stride;
    a.o_copy = op.out_copy_stride; a.o_row = op.out_row_stride; a.o_head = op.out_head_stride;
    a.lens = op.d_lens;
    a.q_lens = op.d_q_lens;
    a.lse = op.d_lse;
    a.weights = op.d_weights;
    a.w_copy = op.weight_copy_stride; a.w_head = op.weight_head_stride;
    a.copies = op.cache.copies;
    a.heads = op.cache.heads;
    a.group = op.q_heads / op.cache.heads;
    a.nq = op.nq;
    a.max_len = op.max_len ? op.max_len : op.cache.slots;
    a.window = op.window;
    a.sinks = op.sinks;
    a.reach = op.window ? std::min(op.window, 0x80000000u) : 0x80000000u;
    a.scale2 = static_cast<float>(static_cast<double>(op.scale) * 1.4426950408889634074);
    return a;
}

// What pkv_attend_workspace looks at.
int check_attend_shape(const pkv_attend_op& op) {
    const pkv_kv_view& v = op.cache;
    if (v.dim != 64 && v.dim != 128) return PKV_ERR_UNSUPPORTED;
    if (v.dtype < PKV_F32 || v.dtype > PKV_FP4 || op.dtype < PKV_F32 || op.dtype > PKV_F16)
        return PKV_ERR_INVALID_ARG;
    if (v.dtype != PKV_FP4 && op.dtype != v.dtype) return PKV_ERR_INVALID_ARG;
    if (v.layers != 1 || !v.copies || !v.heads || !v.slots || v.slots > kMaxCount / 2 || op.max_len > v.slots)
        return PKV_ERR_INVALID_ARG;
    if (!op.q_heads || op.q_heads % v.heads || op.reserved) return PKV_ERR_INVALID_ARG;
    // a head's rows and some tiles more are counted in 31 bits
    if (op.nq > kMaxCount / 2 || static_cast<U128>(v.copies) * op.q_heads * std::max(op.nq, 1u) > kMaxRows)
        return PKV_ERR_INVALID_ARG;
    if (op.nq && !attend_fits(attend_dev(op), v.dim, v.dtype)) return PKV_ERR_INVALID_ARG;
    return PKV_OK;
}

int check_rows(const pkv_rows_op& op, bool store) {
    const int rc = check_view(op.cache, store);
    if (rc) return rc;
    if (op.cache.dtype != PKV_FP4 || op.dtype < PKV_F32 || op.dtype > PKV_F16) return PKV_ERR_INVALID_ARG;
    if (op.rows > kMaxCount / 2 || !op.d_first ||
        static_cast<U128>(op.cache.copies) * op.cache.layers * op.cache.heads * op.rows > 0xffffffffu)
        return PKV_ERR_INVALID_ARG;
    if (!aligned(op.d_first, 4) || !aligned(op.d_counts, 4))
        return PKV_ERR_INVALID_ARG;
    if (!aligned(op.d_keys, 16) || !aligned(op.d_values, 16)) return PKV_ERR_INVALID_ARG;
    const uint64_t unit = 16 / elem_bytes(op.dtype);
    if (op.copy_stride % unit || op.layer_stride % unit || op.head_stride % unit || op.row_stride % unit)
        return PKV_ERR_INVALID_ARG;
    const Axis a[4] = {{op.copy_stride, op.cache.copies}, {op.layer_stride, op.cache.layers},
                       {op.head_stride, op.cache.heads}, {op.row_stride, std::max(op.rows, 1u)}};
    if (!extent(a, 4, op.cache.dim) || (!store && !distinct(a, 4, op.cache.dim))) return PKV_ERR_INVALID_ARG;
    return PKV_OK;
}

int run_rows(pkv_ctx* ctx, const pkv_rows_op* op, void* stream, bool store) {
    if (!ctx || !op) return PKV_ERR_INVALID_ARG;
    const int rc = check_rows(*op, store);
    if (rc) return rc;
    if (!op->rows || (!op->d_keys && !op->d_values)) return PKV_OK;
    RowsDev r{};
    r.kv = dev(op->cache);
    r.keys = static_cast<uint8_t*>(op->d_keys);
    r.values = static_cast<uint8_t*>(op->d_values);
    r.copy = op->copy_stride; r.layer = op->layer_stride; r.head = op->head_stride; r.row = op->row_stride;
    r.first = op->d_first;
    r.counts = op->d_counts;
    r.copies = op->cache.copies; r.layers = op->cache.layers; r.heads = op->cache.heads; r.slots = op->cache.slots;
    r.rows = op->rows;
    OnDevice on(ctx_device(ctx));
    if (on.rc) return on.rc;
    return hip_rc(store ? launch_fp4_store(r, op->cache.dim, op->dtype, stream)
                        : launch_fp4_load(r, op->cache.dim, op->dtype, stream));
}

// Bytes behind each pointer of a view, codes or elements, and scales.
uint64_t view_bytes(const pkv_kv_view& v) {
    const Axis a[4] = {{v.copy_stride, v.copies}, {v.layer_stride, v.layers}, {v.head_stride, v.heads},
                       {v.slot_stride, v.slots}};
    const uint64_t e = extent(a, 4, v.dim);
    return v.dtype == PKV_FP4 ? e / 2 : e * elem_bytes(v.dtype);
}

bool same_memory(const pkv_kv_view& a, const pkv_kv_view& b) {
    return a.d_keys == b.d_keys && a.d_values == b.d_values && a.d_key_scales == b.d_key_scales &&
           a.d_value_scales == b.d_value_scales && a.copy_stride == b.copy_stride &&
           a.layer_stride == b.layer_stride && a.head_stride == b.head_stride && a.slot_stride == b.slot_stride;
}

bool views_overlap(const pkv_kv_view& a, const pkv_kv_view& b) {
    const uint64_t an = view_bytes(a), bn = view_bytes(b);
    const void* ap[2] = {a.d_keys, a.d_values};
    const void* bp[2] = {b.d_keys, b.d_values};
    const void* as[2] = {a.d_key_scales, a.d_value_scales};
    const void* bs[2] = {b.d_key_scales, b.d_value_scales};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2; ++j) {
            if (overlap(ap[i], an, bp[j], bn)) return true;
            if (a.dtype == PKV_FP4 && overlap(as[i], an / 16, bs[j], bn / 16)) return true;
        }
    return false;
}

}  // namespace

extern "C" {

uint64_t pkv_attend_workspace(const pkv_attend_op* op) {
    if (!op || check_attend_shape(*op) || !op->nq) return 0;
    return attend_workspace(attend_dev(*op), op->cache.dim, op->cache.dtype, op->dtype);
}

int pkv_attend(pkv_ctx* ctx, const pkv_attend_op* op, void* stream) {
    if (!ctx || !op) return PKV_ERR_INVALID_ARG;
    int rc = check_attend_shape(*op);
    if (!rc) rc = check_view(op->cache, false);
    if (rc) return rc;
    if (!(op->scale > 0.0f) || !std::isfinite(attend_dev(*op).scale2)) return PKV_ERR_INVALID_ARG;
    if (!op->d_lens || !aligned(op->d_lens, 4) || !aligned(op->d_q_lens, 4) || !aligned(op->d_lse, 4) ||
        !aligned(op->d_weights, 4))
        return PKV_ERR_INVALID_ARG;
    if (!op->nq) return PKV_OK;
    if (!op->d_q || !op->d_out || !aligned(op->d_q, 16) || !aligned(op->d_out, 16)) return PKV_ERR_INVALID_ARG;
    const uint64_t unit = 16 / elem_bytes(op->dtype);
    if (op->q_copy_stride % unit || op->q_row_stride % unit || op->q_head_stride % unit ||
        op->out_copy_stride % unit || op->out_row_stride % unit || op->out_head_stride % unit)
        return PKV_ERR_INVALID_ARG;
    const uint32_t dim = op->cache.dim;
    const Axis q[3] = {{op->q_copy_stride, op->cache.copies}, {op->q_row_stride, op->nq},
                       {op->q_head_stride, op->q_heads}};
    const Axis o[3] = {{op->out_copy_stride, op->cache.copies}, {op->out_row_stride, op->nq},
                       {op->out_head_stride, op->q_heads}};
    const uint64_t qn = extent(q, 3, dim), on = extent(o, 3, dim);
    if (!qn || !on || !distinct(o, 3, dim)) return PKV_ERR_INVALID_ARG;
    if (overlap(op->d_q, qn * elem_bytes(op->dtype), op->d_out, on * elem_bytes(op->dtype)))
        return PKV_ERR_INVALID_ARG;
    const AttendDev a = attend_dev(*op);
    if (op->d_weights) {
        const Axis w[2] = {{op->weight_copy_stride, a.copies}, {op->weight_head_stride, a.heads}};
        if (!extent(w, 2, a.max_len) || !distinct(w, 2, a.max_len)) return PKV_ERR_INVALID_ARG;
    }
    const uint64_t need = attend_workspace(a, dim, op->cache.dtype, op->dtype);
    if (need && (!op->d_workspace || !aligned(op->d_workspace, 256))) return PKV_ERR_INVALID_ARG;
    if (op->workspace_bytes < need) return PKV_ERR_CAPACITY;
    OnDevice dv(ctx_device(ctx));
    if (dv.rc) return dv.rc;
    return hip_rc(launch_attend(a, dim, op->cache.dtype, op->dtype, static_cast<uint8_t*>(op->d_workspace), stream));
}

int pkv_fp4_store(pkv_ctx* ctx, const pkv_rows_op* op, void* stream) { return run_rows(ctx, op, stream, true); }
int pkv_fp4_load(pkv_ctx* ctx, const pkv_rows_op* op, void* stream) { return run_rows(ctx, op, stream, false); }

int pkv_evict(pkv_ctx* ctx, const pkv_evict_op* op, void* stream) {
    if (!ctx || !op || op->reserved) return PKV_ERR_INVALID_ARG;
    int rc = check_view(op->cache, false);
    if (!rc) rc = check_view(op->into, true);
    if (rc) return rc;
    const pkv_kv_view &c = op->cache, &t = op->into;
    if (t.copies != c.copies || t.layers != c.layers || t.heads != c.heads || t.dim != c.dim || t.dtype != c.dtype)
        return PKV_ERR_INVALID_ARG;
    if (!op->budget || op->budget > kMaxCount || static_cast<uint64_t>(op->sinks) + op->recent > op->budget ||
        t.slots < std::min(op->budget, c.slots))
        return PKV_ERR_INVALID_ARG;
    if (!op->d_lens || !op->d_new_lens || !op->d_kept || !op->d_weights || !op->d_weights_out ||
        !aligned(op->d_lens, 4) || !aligned(op->d_new_lens, 4) || !aligned(op->d_kept, 4) ||
        !aligned(op->d_weights, 4) || !aligned(op->d_weights_out, 4))
        return PKV_ERR_INVALID_ARG;
    if (overlap(op->d_lens, 4ull * c.copies, op->d_new_lens, 4ull * c.copies)) return PKV_ERR_INVALID_ARG;
    const bool in_place = same_memory(c, t);
    if (!in_place && views_overlap(c, t)) return PKV_ERR_INVALID_ARG;
    const Axis w[3] = {{op->weight_strides[0], c.copies}, {op->weight_strides[1], c.layers},
                       {op->weight_strides[2], c.heads}};
    const Axis o[3] = {{op->out_strides[0], c.copies}, {op->out_strides[1], c.layers},
                       {op->out_strides[2], c.heads}};
    const uint64_t wn = extent(w, 3, c.slots), on = extent(o, 3, t.slots);
    if (!wn || !on || !distinct(o, 3, t.slots)) return PKV_ERR_INVALID_ARG;
    bool same_w = op->d_weights == op->d_weights_out && t.slots <= c.slots;
    for (int i = 0; i < 3; ++i) same_w = same_w && (w[i].count == 1 || op->weight_strides[i] == op->out_strides[i]);
    if (!same_w && overlap(op->d_weights, 4 * wn, op->d_weights_out, 4 * on)) return PKV_ERR_INVALID_ARG;
    if (same_w && !distinct(w, 3, c.slots)) return PKV_ERR_INVALID_ARG;
    EvictDev e{};
    e.kv = dev(c);
    e.into = dev(t);
    e.lens = op->d_lens;
    e.new_lens = op->d_new_lens;
    e.kept = op->d_kept;
    e.w = op->d_weights;
    e.w_out = op->d_weights_out;
    for (int i = 0; i < 3; ++i) { e.ws[i] = op->weight_strides[i]; e.os[i] = op->out_strides[i]; }
    e.copies = c.copies; e.layers = c.layers; e.heads = c.heads; e.slots = c.slots; e.into_slots = t.slots;
    e.budget = op->budget; e.sinks = op->sinks; e.recent = op->recent;
    e.in_place = in_place;
    if (!evict_fits(e, c.dim, c.dtype)) return PKV_ERR_INVALID_ARG;
    OnDevice dv(ctx_device(ctx));
    if (dv.rc) return dv.rc;
    return hip_rc(launch_evict(e, c.dim, c.dtype, stream));
}

}  // extern "C"
