// pkv_paged.cpp -- host half of the paged-cache and packed-prompt calls of
// include/pkv_codec.h: argument checks, and the launches on the context's device.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "pkv_check.h"
#include "pkv_internal.h"
#include "pkv_paged.h"

using namespace pkv;

namespace {

constexpr uint32_t kMaxHeads = 1u << 16;

int check_pages(const pkv_page_view& v, bool written) {
    if (v.dim != 64 && v.dim != 128) return PKV_ERR_UNSUPPORTED;
    if (v.dtype != PKV_BF16 && v.dtype != PKV_F16 && v.dtype != PKV_FP8) return PKV_ERR_INVALID_ARG;
    if (!v.layers || !v.pages || !v.heads || v.pages > kMaxCount || v.layers > kMaxCount || v.heads > kMaxHeads)
        return PKV_ERR_INVALID_ARG;
    if (v.page_slots < 16 || v.page_slots > 65536 || (v.page_slots & (v.page_slots - 1))) return PKV_ERR_INVALID_ARG;
    if (!v.d_keys || !v.d_values || !aligned(v.d_keys, 16) || !aligned(v.d_values, 16)) return PKV_ERR_INVALID_ARG;
    uint64_t unit = 8;
    if (v.dtype == PKV_FP8) {
        unit = 16ull * v.dim;   // scale bytes of 16 slots are read 16 bytes at a time
        if (!v.d_key_scales || !v.d_value_scales || !aligned(v.d_key_scales, 16) || !aligned(v.d_value_scales, 16) ||
            v.slot_stride != v.dim)
            return PKV_ERR_INVALID_ARG;
    } else if (v.d_key_scales || v.d_value_scales || v.slot_stride % unit) {
        return PKV_ERR_INVALID_ARG;
    }
    if (v.slot_stride > kMaxSlotStride) return PKV_ERR_INVALID_ARG;
    if (v.layer_stride % unit || v.page_stride % unit || v.head_stride % unit) return PKV_ERR_INVALID_ARG;
    const Axis a[4] = {{v.layer_stride, v.layers}, {v.page_stride, v.pages}, {v.head_stride, v.heads},
                       {v.slot_stride, v.page_slots}};
    const uint64_t e = extent(a, 4, v.dim);
    if (!e || e > v.elems) return PKV_ERR_INVALID_ARG;
    if (written && !distinct(a, 4, v.dim)) return PKV_ERR_INVALID_ARG;
    return PKV_OK;
}

// Whether rows of a call lie on the pages that it reads or writes.
bool over_pages(const pkv_page_view& v, const void* p, uint64_t bytes) {
    const Axis a[4] = {{v.layer_stride, v.layers}, {v.page_stride, v.pages}, {v.head_stride, v.heads},
                       {v.slot_stride, v.page_slots}};
    const uint64_t e = extent(a, 4, v.dim), size = v.dtype == PKV_FP8 ? e : 2 * e;
    if (overlap(v.d_keys, size, p, bytes) || overlap(v.d_values, size, p, bytes)) return true;
    return v.dtype == PKV_FP8 && (overlap(v.d_key_scales, e / 32, p, bytes) || overlap(v.d_value_scales, e / 32, p, bytes));
}

// Counts only: what a workspace's size goes by.
int check_counts(const pkv_sequences& s, uint32_t page_slots) {
    if (!s.seqs || !s.table_pages || s.reserved || s.seqs > 1u << 24 || s.rows > kMaxRows) return PKV_ERR_INVALID_ARG;
    if (static_cast<uint64_t>(s.table_pages) * page_slots > kMaxCount / 2) return PKV_ERR_INVALID_ARG;
    if (!s.d_starts && s.rows % s.seqs) return PKV_ERR_INVALID_ARG;
    return PKV_OK;
}
int check_sequences(const pkv_sequences& s, uint32_t page_slots) {
    const int rc = check_counts(s, page_slots);
    if (rc) return rc;
    if (!s.d_tables || !s.d_lens || !aligned(s.d_tables, 4) || !aligned(s.d_lens, 4) || !aligned(s.d_starts, 4))
        return PKV_ERR_INVALID_ARG;
    const Axis t[1] = {{s.table_stride, s.seqs}};
    return extent(t, 1, s.table_pages) ? PKV_OK : PKV_ERR_INVALID_ARG;
}

uint32_t log2_of(uint32_t x) { return 31 - __builtin_clz(x); }

SeqsDev seqs_dev(const pkv_sequences& s, const pkv_page_view& v) {
    SeqsDev d{};
    d.paged = true;
    d.tables = s.d_tables;
    d.table = s.table_stride;
    d.lens = s.d_lens;
    d.starts = s.d_starts;
    d.seqs = s.seqs;
    d.pages = v.pages;
    d.shift = log2_of(v.page_slots);
    d.rows = s.rows;
    d.each = s.d_starts ? 0 : s.rows / s.seqs;
    d.max_len = s.table_pages * v.page_slots;
    return d;
}

void set_mask(PagedDev& a, uint32_t window, uint32_t sinks, float scale) {
    a.window = window;
    a.sinks = sinks;
    a.reach = window ? std::min(window, 0x80000000u) : 0x80000000u;
    a.scale2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634074);
}

PagedDev paged_dev(const pkv_paged_attend_op& op) {
    const pkv_page_view& v = op.pages;
    PagedDev a{};
    a.seq = seqs_dev(op.seqs, v);
    if (op.max_len) a.seq.max_len = op.max_len;
    a.k = static_cast<const uint8_t*>(v.d_keys);
    a.v = static_cast<const uint8_t*>(v.d_values);
    a.ks = v.d_key_scales;
    a.vs = v.d_value_scales;
    a.page = v.page_stride;
    a.k_head = a.v_head = v.head_stride;
    a.k_slot = a.v_slot = v.slot_stride;
    a.q = static_cast<const uint8_t*>(op.d_q);
    a.out = static_cast<uint8_t*>(op.d_out);
    a.q_row = op.q_row_stride; a.q_head = op.q_head_stride;
    a.o_row = op.out_row_stride; a.o_head = op.out_head_stride;
    a.lse = op.d_lse;
    a.clear = op.clear;
    a.heads = v.heads;
    a.group = op.q_heads / v.heads;
    a.max_rows = a.seq.each ? a.seq.each : op.max_rows ? std::min(op.max_rows, op.seqs.rows) : op.seqs.rows;
    set_mask(a, op.window, op.sinks, op.scale);
    return a;
}

// What pkv_paged_attend_workspace looks at.
int check_paged_shape(const pkv_paged_attend_op& op) {
    const pkv_page_view& v = op.pages;
    if (v.dim != 64 && v.dim != 128) return PKV_ERR_UNSUPPORTED;
    if (op.dtype != PKV_BF16 && op.dtype != PKV_F16) return PKV_ERR_INVALID_ARG;
    if (v.dtype != PKV_FP8 && op.dtype != v.dtype) return PKV_ERR_INVALID_ARG;
    if (v.layers != 1 || !v.heads || v.heads > kMaxHeads || v.page_slots < 16 || v.page_slots > 65536 ||
        (v.page_slots & (v.page_slots - 1)))
        return PKV_ERR_INVALID_ARG;
    if (!op.q_heads || op.q_heads % v.heads || op.clear > 1) return PKV_ERR_INVALID_ARG;
    const int rc = check_counts(op.seqs, v.page_slots);
    if (rc) return rc;
    if (op.max_len > op.seqs.table_pages * v.page_slots) return PKV_ERR_INVALID_ARG;
    if (static_cast<U128>(op.seqs.rows) * op.q_heads > kMaxRows) return PKV_ERR_INVALID_ARG;
    if (op.seqs.rows && !paged_fits(paged_dev(op), v.dim, v.dtype)) return PKV_ERR_INVALID_ARG;
    return PKV_OK;
}

PagedDev prompts_dev(const pkv_prompts_op& op) {
    PagedDev a{};
    a.seq.starts = op.d_starts;
    a.seq.seqs = op.seqs;
    a.seq.rows = op.rows;
    a.max_rows = op.max_rows ? std::min(op.max_rows, op.rows) : op.rows;
    a.seq.max_len = a.max_rows;
    a.k = static_cast<const uint8_t*>(op.d_k);
    a.v = static_cast<const uint8_t*>(op.d_v);
    a.k_head = op.k_head_stride; a.k_slot = op.k_row_stride;
    a.v_head = op.v_head_stride; a.v_slot = op.v_row_stride;
    a.q = static_cast<const uint8_t*>(op.d_q);
    a.out = static_cast<uint8_t*>(op.d_out);
    a.q_row = op.q_row_stride; a.q_head = op.q_head_stride;
    a.o_row = op.out_row_stride; a.o_head = op.out_head_stride;
    a.lse = op.d_lse;
    a.clear = op.clear;
    a.heads = op.heads;
    a.group = op.q_heads / op.heads;
    set_mask(a, op.window, op.sinks, op.scale);
    return a;
}

int check_prompts_shape(const pkv_prompts_op& op) {
    if (op.dim != 64 && op.dim != 128) return PKV_ERR_UNSUPPORTED;
    if (op.dtype != PKV_BF16 && op.dtype != PKV_F16) return PKV_ERR_INVALID_ARG;
    if (!op.heads || op.heads > kMaxHeads || !op.q_heads || op.q_heads % op.heads || op.clear > 1) return PKV_ERR_INVALID_ARG;
    if (!op.seqs || op.seqs > 1u << 24 || op.rows > kMaxRows) return PKV_ERR_INVALID_ARG;
    if (static_cast<U128>(op.rows) * op.q_heads > kMaxRows) return PKV_ERR_INVALID_ARG;
    if (op.rows && !paged_fits(prompts_dev(op), op.dim, op.dtype)) return PKV_ERR_INVALID_ARG;
    return PKV_OK;
}

// Rows of heads that a call reads or writes, 16-bit: their bytes, 0 if they are not such rows.
uint64_t row_bytes(const void* p, uint64_t row, uint64_t head, uint32_t rows, uint32_t heads, uint32_t dim, bool written) {
    if (!p || !aligned(p, 16) || row % 8 || head % 8) return 0;
    const Axis a[2] = {{row, rows}, {head, heads}};
    if (written && !distinct(a, 2, dim)) return 0;
    return 2 * extent(a, 2, dim);
}

int run_rows(pkv_ctx* ctx, const pkv_paged_rows_op* op, void* stream, bool store) {
    if (!ctx || !op || op->reserved) return PKV_ERR_INVALID_ARG;
    const pkv_page_view& v = op->pages;
    int rc = check_pages(v, store);
    if (!rc) rc = check_sequences(op->seqs, v.page_slots);
    if (rc) return rc;
    if (op->dtype < PKV_F32 || op->dtype > PKV_F16) return PKV_ERR_INVALID_ARG;
    if (!aligned(op->d_keys, 16) || !aligned(op->d_values, 16)) return PKV_ERR_INVALID_ARG;
    const uint64_t unit = 16 / elem_bytes(op->dtype);
    if (op->layer_stride % unit || op->row_stride % unit || op->head_stride % unit) return PKV_ERR_INVALID_ARG;
    if (!op->seqs.rows || (!op->d_keys && !op->d_values)) return PKV_OK;
    const Axis a[3] = {{op->layer_stride, v.layers}, {op->row_stride, op->seqs.rows}, {op->head_stride, v.heads}};
    const uint64_t bytes = extent(a, 3, v.dim) * elem_bytes(op->dtype);
    if (!bytes || (!store && !distinct(a, 3, v.dim))) return PKV_ERR_INVALID_ARG;
    for (const void* rows : {op->d_keys, op->d_values})
        if (rows && over_pages(v, rows, bytes)) return PKV_ERR_INVALID_ARG;
    if (!store && op->d_keys && op->d_values && overlap(op->d_keys, bytes, op->d_values, bytes)) return PKV_ERR_INVALID_ARG;
    // the launch: a workgroup of each layer and side for every 16 rows
    if (static_cast<U128>((op->seqs.rows + 15ull) / 16) * v.layers >= 1u << 24) return PKV_ERR_INVALID_ARG;
    PagedRowsDev r{};
    r.seq = seqs_dev(op->seqs, v);
    r.k = static_cast<uint8_t*>(v.d_keys);
    r.v = static_cast<uint8_t*>(v.d_values);
    r.ks = v.d_key_scales;
    r.vs = v.d_value_scales;
    r.p_layer = v.layer_stride; r.page = v.page_stride; r.p_head = v.head_stride; r.slot = v.slot_stride;
    r.keys = static_cast<uint8_t*>(op->d_keys);
    r.values = static_cast<uint8_t*>(op->d_values);
    r.layer = op->layer_stride; r.row = op->row_stride; r.head = op->head_stride;
    r.layers = v.layers;
    r.heads = v.heads;
    OnDevice on(ctx_device(ctx));
    if (on.rc) return on.rc;
    return hip_rc(store ? launch_paged_store(r, v.dim, v.dtype, op->dtype, stream)
                        : launch_paged_load(r, v.dim, v.dtype, op->dtype, stream));
}

// The last checks and the launch of a call whose shape has been checked.
int run_attend(pkv_ctx* ctx, const PagedDev& a, uint32_t dim, int cache_dtype, int dtype, float scale, void* workspace,
               uint64_t workspace_bytes, void* stream) {
    if (!(scale > 0.0f) || !std::isfinite(a.scale2) || !aligned(a.lse, 4)) return PKV_ERR_INVALID_ARG;
    if (!a.seq.rows) return PKV_OK;
    const uint32_t heads = a.heads * a.group;
    const uint64_t qn = row_bytes(a.q, a.q_row, a.q_head, a.seq.rows, heads, dim, false);
    const uint64_t on = row_bytes(a.out, a.o_row, a.o_head, a.seq.rows, heads, dim, true);
    if (!qn || !on || overlap(a.q, qn, a.out, on)) return PKV_ERR_INVALID_ARG;
    const uint64_t need = paged_workspace(a, dim, cache_dtype);
    if (need && (!workspace || !aligned(workspace, 256))) return PKV_ERR_INVALID_ARG;
    if (workspace_bytes < need) return PKV_ERR_CAPACITY;
    OnDevice dv(ctx_device(ctx));
    if (dv.rc) return dv.rc;
    return hip_rc(launch_paged(a, dim, cache_dtype, dtype, static_cast<uint8_t*>(workspace), stream));
}

}  // namespace

extern "C" {

int pkv_paged_store(pkv_ctx* ctx, const pkv_paged_rows_op* op, void* stream) { return run_rows(ctx, op, stream, true); }
int pkv_paged_load(pkv_ctx* ctx, const pkv_paged_rows_op* op, void* stream) { return run_rows(ctx, op, stream, false); }

uint64_t pkv_paged_attend_workspace(const pkv_paged_attend_op* op) {
    if (!op || check_paged_shape(*op) || !op->seqs.rows) return 0;
    return paged_workspace(paged_dev(*op), op->pages.dim, op->pages.dtype);
}

int pkv_paged_attend(pkv_ctx* ctx, const pkv_paged_attend_op* op, void* stream) {
    if (!ctx || !op) return PKV_ERR_INVALID_ARG;
    int rc = check_paged_shape(*op);
    if (!rc) rc = check_pages(op->pages, false);
    if (!rc) rc = check_sequences(op->seqs, op->pages.page_slots);
    if (rc) return rc;
    if (op->seqs.rows) {
        const uint64_t on = row_bytes(op->d_out, op->out_row_stride, op->out_head_stride, op->seqs.rows, op->q_heads,
                                      op->pages.dim, true);
        if (!on || over_pages(op->pages, op->d_out, on)) return PKV_ERR_INVALID_ARG;
    }
    return run_attend(ctx, paged_dev(*op), op->pages.dim, op->pages.dtype, op->dtype, op->scale, op->d_workspace,
                      op->workspace_bytes, stream);
}

uint64_t pkv_prompts_workspace(const pkv_prompts_op* op) {
    if (!op || check_prompts_shape(*op) || !op->rows) return 0;
    return paged_workspace(prompts_dev(*op), op->dim, op->dtype);
}

int pkv_prompts(pkv_ctx* ctx, const pkv_prompts_op* op, void* stream) {
    if (!ctx || !op) return PKV_ERR_INVALID_ARG;
    const int rc = check_prompts_shape(*op);
    if (rc) return rc;
    if (!op->d_starts || !aligned(op->d_starts, 4)) return PKV_ERR_INVALID_ARG;
    if (op->rows) {
        if (op->k_row_stride > kMaxSlotStride || op->v_row_stride > kMaxSlotStride) return PKV_ERR_INVALID_ARG;
        const uint64_t kn = row_bytes(op->d_k, op->k_row_stride, op->k_head_stride, op->rows, op->heads, op->dim, false);
        const uint64_t vn = row_bytes(op->d_v, op->v_row_stride, op->v_head_stride, op->rows, op->heads, op->dim, false);
        if (!kn || !vn) return PKV_ERR_INVALID_ARG;
        const uint64_t on = row_bytes(op->d_out, op->out_row_stride, op->out_head_stride, op->rows, op->q_heads, op->dim,
                                      true);
        if (!on || overlap(op->d_k, kn, op->d_out, on) || overlap(op->d_v, vn, op->d_out, on)) return PKV_ERR_INVALID_ARG;
    }
    return run_attend(ctx, prompts_dev(*op), op->dim, op->dtype, op->dtype, op->scale, op->d_workspace,
                      op->workspace_bytes, stream);
}

}  // extern "C"
