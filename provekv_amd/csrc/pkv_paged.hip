// pkv_paged.hip -- kernels over paged KV caches and packed rows: rows stored
// into pages and loaded from them, attention of packed rows over pages, and
// attention of whole packed prompts on their own rows.  gfx950.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "pkv_attend_tile.h"
#include "pkv_paged.h"

namespace pkv {
namespace {

// ------------------------------------------------------------ packed rows
// A sequence's rows and slots, all within the call's bounds whatever the words hold.
struct Seq {
    int row0, rows, len, first;   // first packed row, rows, slots, slot of row 0 (may be negative)
};
__device__ inline Seq seq_of(const SeqsDev& q, uint32_t s, uint32_t max_rows) {
    Seq o;
    int end;
    if (q.starts) {
        o.row0 = min(max(q.starts[s], 0), static_cast<int>(q.rows));
        end = min(max(q.starts[s + 1], o.row0), static_cast<int>(q.rows));
    } else {
        o.row0 = static_cast<int>(s * q.each);
        end = o.row0 + static_cast<int>(q.each);
    }
    o.rows = min(end - o.row0, static_cast<int>(max_rows));
    o.len = q.lens ? min(max(q.lens[s], 0), static_cast<int>(q.max_len)) : o.rows;
    o.first = o.len - o.rows;
    return o;
}
// The sequence of packed row r (the same in all lanes): the first that ends behind it; -1: nobody's.
__device__ inline int seq_of_row(const SeqsDev& q, int r, uint32_t lane) {
    if (!q.starts) return r / static_cast<int>(q.each);
    uint32_t s = 0;
    for (uint32_t j = 0; j < q.seqs; j += 64)
        s += __popcll(__ballot(j + lane < q.seqs && q.starts[j + lane + 1] <= r));
    return s < q.seqs && q.starts[s] <= r ? static_cast<int>(s) : -1;
}
// The page of sequence s that holds slot j (0 <= j < its length); -1: none.
__device__ inline int page_of(const SeqsDev& q, uint32_t s, int j) {
    const int p = q.tables[s * q.table + (static_cast<uint32_t>(j) >> q.shift)];
    return static_cast<uint32_t>(p) < q.pages ? p : -1;
}

// ------------------------------------------------------------ rows into pages and back
// Exponent byte of a block of 8-bit codes: the smallest e with top <= 448 * 2^e
// = 1.75 * 2^(e + 8), kept in -116 .. 119; 255 when the block holds an infinity
// or NaN.  top's bits, sign off.
__device__ inline uint32_t block_exponent8(uint32_t top) {
    if (top >= 0x7f800000u) return 255;
    const int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(min(max(e, 11), 246));
}

constexpr uint32_t kChunk = 16;   // packed rows of a workgroup

// Element offsets of a chunk's rows in the pages (of layer 0, head 0); -1: nowhere.
__device__ inline void chunk_places(const PagedRowsDev& a, uint32_t first, int64_t* places) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (uint32_t i = wave; i < kChunk; i += 4) {
        const int r = static_cast<int>(first + i);
        int64_t at = -1;
        const int s = r < static_cast<int>(a.seq.rows) ? seq_of_row(a.seq, r, lane) : -1;
        if (s >= 0) {
            const Seq q = seq_of(a.seq, s, a.seq.rows);
            const int j = q.first + r - q.row0;
            const int page = j >= 0 ? page_of(a.seq, s, j) : -1;
            if (page >= 0)
                at = static_cast<int64_t>(page * a.page + (static_cast<uint32_t>(j) & ((1u << a.seq.shift) - 1)) * a.slot);
        }
        if (lane == 0) places[i] = at;
    }
    __syncthreads();
}

// A workgroup takes 16 packed rows of a layer and side, 8 values a thread and
// step, channels fastest, then rows, then heads: rows of a sequence that follow
// each other are neighbours in a page, so that a step writes whole lines.
template <int CT, int QT, int D>
__global__ __launch_bounds__(256) void paged_store_kernel(PagedRowsDev a) {
    using T = typename Elem<QT>::T;
    constexpr uint32_t V = 8, kRow = D / V;
    typedef T Vec __attribute__((ext_vector_type(V)));
    __shared__ int64_t places[kChunk];
    const uint32_t chunk = blockIdx.x / a.layers, layer = blockIdx.x % a.layers;
    const uint8_t* src = blockIdx.y ? a.values : a.keys;
    if (!src) return;
    uint8_t* dst = blockIdx.y ? a.v : a.k;
    uint8_t* dsc = blockIdx.y ? a.vs : a.ks;
    chunk_places(a, chunk * kChunk, places);
    for (uint32_t x = threadIdx.x; x < a.heads * kChunk * kRow; x += 256) {
        const uint32_t d = x % kRow * V, i = x / kRow % kChunk, h = x / kRow / kChunk;
        const bool there = places[i] >= 0;
        // rows without a place read the chunk's first
        const uint64_t from = layer * a.layer + static_cast<uint64_t>(chunk * kChunk + (there ? i : 0)) * a.row + h * a.head;
        const Vec in = *reinterpret_cast<const Vec*>(reinterpret_cast<const T*>(src) + from + d);
        const uint64_t to = layer * a.p_layer + h * a.p_head + (there ? places[i] : 0) + d;
        if constexpr (CT == PKV_FP8) {
            float y[V];
            uint32_t top = 0;
            for (uint32_t e = 0; e < V; ++e) {
                y[e] = static_cast<float>(in[e]);
                top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
            }
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
            const uint32_t b = block_exponent8(top);
            const float s = block_scale(b), most = 448.0f * s;
            u32x2 codes = {};
            if (b != 255) {
                typedef short s16x2 __attribute__((ext_vector_type(2)));
                for (uint32_t e = 0; e < V; ++e) y[e] = fminf(fmaxf(y[e], -most), most);
                for (int w = 0; w < 2; ++w) {
                    s16x2 c = {};
                    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[4 * w], y[4 * w + 1], s, false);
                    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[4 * w + 2], y[4 * w + 3], s, true);
                    codes[w] = __builtin_bit_cast(uint32_t, c);
                }
            }
            if (!there) continue;
            *reinterpret_cast<u32x2*>(dst + to) = codes;
            if (d % 32 == 0) dsc[to / 32] = static_cast<uint8_t>(b);
        } else {
            using P = typename Elem<CT>::T;
            typedef P Out __attribute__((ext_vector_type(V)));
            Out y;
            for (uint32_t e = 0; e < V; ++e) y[e] = static_cast<P>(static_cast<float>(in[e]));
            if (there) *reinterpret_cast<Out*>(reinterpret_cast<P*>(dst) + to) = y;
        }
    }
}

// The same the other way, 16 bytes of the written tensor a thread and step.
template <int CT, int QT, int D>
__global__ __launch_bounds__(256) void paged_load_kernel(PagedRowsDev a) {
    using T = typename Elem<QT>::T;
    constexpr uint32_t V = QT == PKV_F32 ? 4 : 8, kRow = D / V;
    typedef T Vec __attribute__((ext_vector_type(V)));
    __shared__ int64_t places[kChunk];
    const uint32_t chunk = blockIdx.x / a.layers, layer = blockIdx.x % a.layers;
    uint8_t* dst = blockIdx.y ? a.values : a.keys;
    if (!dst) return;
    const uint8_t* src = blockIdx.y ? a.v : a.k;
    const uint8_t* ssc = blockIdx.y ? a.vs : a.ks;
    chunk_places(a, chunk * kChunk, places);
    for (uint32_t x = threadIdx.x; x < a.heads * kChunk * kRow; x += 256) {
        const uint32_t d = x % kRow * V, i = x / kRow % kChunk, h = x / kRow / kChunk;
        if (chunk * kChunk + i >= a.seq.rows) continue;
        const bool there = places[i] >= 0;
        const uint64_t from = layer * a.p_layer + h * a.p_head + (there ? places[i] : 0) + d;   // a place that is read, not used
        float y[V];
        if constexpr (CT == PKV_FP8) {
            const float s = block_scale(ssc[from / 32]);
            for (uint32_t w = 0; w < V / 4; ++w) {
                const uint32_t codes = reinterpret_cast<const uint32_t*>(src + from)[w];
                const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, s, false);
                const f32x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, s, true);
                y[4 * w] = lo[0]; y[4 * w + 1] = lo[1]; y[4 * w + 2] = hi[0]; y[4 * w + 3] = hi[1];
            }
        } else {
            using P = typename Elem<CT>::T;
            typedef P In __attribute__((ext_vector_type(V)));
            const In in = *reinterpret_cast<const In*>(reinterpret_cast<const P*>(src) + from);
            for (uint32_t e = 0; e < V; ++e) y[e] = static_cast<float>(in[e]);
        }
        Vec out;
        for (uint32_t e = 0; e < V; ++e) out[e] = static_cast<T>(there ? y[e] : 0.0f);
        const uint64_t to = layer * a.layer + static_cast<uint64_t>(chunk * kChunk + i) * a.row + h * a.head + d;
        *reinterpret_cast<Vec*>(reinterpret_cast<T*>(dst) + to) = out;
    }
}

// ------------------------------------------------------------ attention
// Element offsets of slot j of sequence s, keys and values; false: no page holds it.
template <bool PAGED>
__device__ inline bool slot_at(const PagedDev& a, uint32_t s, int row0, uint32_t h, int j, uint64_t* k, uint64_t* v) {
    uint64_t kj, vj;
    if constexpr (PAGED) {
        const int page = page_of(a.seq, s, j);
        if (page < 0) return false;
        kj = vj = page * a.page + (static_cast<uint32_t>(j) & ((1u << a.seq.shift) - 1)) * a.k_slot;
    } else {
        kj = static_cast<uint64_t>(row0 + j) * a.k_slot;
        vj = static_cast<uint64_t>(row0 + j) * a.v_slot;
    }
    *k = kj + h * a.k_head;
    *v = vj + h * a.v_head;
    return true;
}
template <int CT>
__device__ inline float element(const uint8_t* p, const uint8_t* scales, uint64_t e) {
    if constexpr (CT == PKV_FP8) {
        const f32x2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(p[e], block_scale(scales[e / 32]), false);
        return x[0];
    } else {
        return static_cast<float>(reinterpret_cast<const typename Elem<CT>::T*>(p)[e]);
    }
}

// Nobody's rows, before the first sequence's and behind the last's, to 0: the
// workgroups behind `work`, kClear of them.
constexpr uint32_t kClear = 64;
template <int QT, int D>
__device__ void clear_rows(const PagedDev& a, uint32_t block) {
    using T = typename Elem<QT>::T;
    const int rows = static_cast<int>(a.seq.rows), heads = static_cast<int>(a.heads * a.group);
    const int first = min(max(a.seq.starts[0], 0), rows);
    int last = first;                                  // the largest end, should starts not ascend
    for (uint32_t s = threadIdx.x % 64; s < a.seq.seqs; s += 64) last = max(last, min(a.seq.starts[s + 1], rows));
    for (int o = 32; o; o >>= 1) last = max(last, __shfl_xor(last, o));
    const int rest = first + rows - last;
    for (int x = static_cast<int>(block); x < rest; x += kClear) {
        T* out = reinterpret_cast<T*>(a.out) + static_cast<uint64_t>(x < first ? x : last + x - first) * a.o_row;
        for (int y = static_cast<int>(threadIdx.x); y < heads * (D / 8); y += 256)
            *reinterpret_cast<u32x4*>(out + static_cast<uint64_t>(y / (D / 8)) * a.o_head + y % (D / 8) * 8) = u32x4{};
    }
}

// A wave a packed row and query head: a slot a lane for the logits, the channels
// over the lanes for the values, one pass with the running maximum and sum.
template <int CT, int QT, int D, bool PAGED>
__global__ __launch_bounds__(256) void row_kernel(PagedDev a, uint32_t work) {
    using T = typename Elem<QT>::T;
    if (blockIdx.x >= work) return clear_rows<QT, D>(a, blockIdx.x - work);
    __shared__ float sq[4][D];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, heads = a.heads * a.group;
    const uint32_t item = blockIdx.x * 4 + wave, r = item / heads, qh = item % heads, h = qh / a.group;
    if (r >= a.seq.rows) return;
    const int s = seq_of_row(a.seq, static_cast<int>(r), lane);
    if (s < 0) return;
    const Seq q = seq_of(a.seq, s, a.max_rows);
    const int i = static_cast<int>(r) - q.row0;
    if (i >= q.rows) return;
    const int pos = q.first + i;
    const T* qp = reinterpret_cast<const T*>(a.q) + static_cast<uint64_t>(r) * a.q_row + qh * a.q_head;
    for (uint32_t d = lane; d < D; d += 64) sq[wave][d] = static_cast<float>(qp[d]);
    float top = -kInf, sum = 0.0f, o[D / 64] = {};
    const Tiles tl = tiles_of(a, pos, pos, 64);
    for (int t = 0; t < tl.count; ++t) {
        const int j0 = tl.slot(t, 64), j = j0 + static_cast<int>(lane);
        uint64_t kj = 0, vj = 0;
        const bool see = j < tl.high && visible(a, pos, j) && slot_at<PAGED>(a, s, q.row0, h, j, &kj, &vj);
        float x = -kInf;
        if (see) {
            x = 0.0f;
            for (uint32_t d = 0; d < D; ++d) x += element<CT>(a.k, a.ks, kj + d) * sq[wave][d];
            x *= a.scale2;
        }
        float m = x;
        for (int y = 32; y; y >>= 1) m = fmaxf(m, __shfl_xor(m, y));
        m = fmaxf(m, top);
        const float f = m == -kInf ? 1.0f : exp2f(top - m), w = see && m != -kInf ? exp2f(x - m) : 0.0f;
        top = m;
        // o is the mean so far: a sum could pass the end of f32 where the mean does not
        const float before = sum * f, all = before + wave_sum(w), part = all == 0.0f ? 0.0f : 1.0f / all;
        sum = all;
        for (int e = 0; e < D / 64; ++e) o[e] *= before * part;
        for (int y = 0; y < 64; ++y) {
            if (!__shfl(static_cast<int>(see), y)) continue;
            const float wy = __shfl(w, y) * part;
            const uint64_t at = static_cast<uint64_t>(__shfl(static_cast<unsigned long long>(vj), y));
            for (int e = 0; e < D / 64; ++e) o[e] += wy * element<CT>(a.v, a.vs, at + 64 * e + lane);
        }
    }
    T* out = reinterpret_cast<T*>(a.out) + static_cast<uint64_t>(r) * a.o_row + qh * a.o_head;
    for (int e = 0; e < D / 64; ++e) out[64 * e + lane] = static_cast<T>(sum == 0.0f ? 0.0f : o[e]);
    if (lane == 0 && a.lse)
        a.lse[static_cast<uint64_t>(qh) * a.seq.rows + r] = sum == 0.0f ? -kInf : (top + log2f(sum)) * kLn2;
}

uint32_t clears(const PagedDev& a) { return a.clear && a.seq.starts ? kClear : 0; }

template <int CT, int QT, int D, bool PAGED>
int attend_typed(const PagedDev& a, uint8_t*, hipStream_t st) {
    const uint32_t work = static_cast<uint32_t>((static_cast<uint64_t>(a.seq.rows) * a.heads * a.group + 3) / 4);
    row_kernel<CT, QT, D, PAGED><<<work + clears(a), 256, 0, st>>>(a, work);
    return hipGetLastError();
}
template <int CT, int QT, bool PAGED>
int attend_dim(const PagedDev& a, uint32_t dim, uint8_t* ws, hipStream_t st) {
    return dim == 64 ? attend_typed<CT, QT, 64, PAGED>(a, ws, st) : attend_typed<CT, QT, 128, PAGED>(a, ws, st);
}

template <int CT, int QT, int D>
int rows_typed(const PagedRowsDev& r, bool store, hipStream_t st) {
    const dim3 grid((r.seq.rows + kChunk - 1) / kChunk * r.layers, 2);
    if (store) paged_store_kernel<CT, QT, D><<<grid, 256, 0, st>>>(r);
    else paged_load_kernel<CT, QT, D><<<grid, 256, 0, st>>>(r);
    return hipGetLastError();
}
template <int CT>
int rows_types(const PagedRowsDev& r, uint32_t dim, int dtype, bool store, hipStream_t st) {
    if (dtype == PKV_F32) return dim == 64 ? rows_typed<CT, PKV_F32, 64>(r, store, st) : rows_typed<CT, PKV_F32, 128>(r, store, st);
    if (dtype == PKV_BF16) return dim == 64 ? rows_typed<CT, PKV_BF16, 64>(r, store, st) : rows_typed<CT, PKV_BF16, 128>(r, store, st);
    return dim == 64 ? rows_typed<CT, PKV_F16, 64>(r, store, st) : rows_typed<CT, PKV_F16, 128>(r, store, st);
}
int launch_rows(const PagedRowsDev& r, uint32_t dim, int cache_dtype, int dtype, bool store, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (cache_dtype == PKV_BF16) return rows_types<PKV_BF16>(r, dim, dtype, store, st);
    if (cache_dtype == PKV_F16) return rows_types<PKV_F16>(r, dim, dtype, store, st);
    return rows_types<PKV_FP8>(r, dim, dtype, store, st);
}

}  // namespace

bool paged_fits(const PagedDev& a, uint32_t, int) {
    return static_cast<uint64_t>(a.seq.rows) * a.heads * a.group < 1u << 26;
}

uint64_t paged_workspace(const PagedDev&, uint32_t, int) { return 0; }

int launch_paged(const PagedDev& a, uint32_t dim, int cache_dtype, int dtype, uint8_t* ws, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (!a.seq.tables)
        return dtype == PKV_BF16 ? attend_dim<PKV_BF16, PKV_BF16, false>(a, dim, ws, st)
                                 : attend_dim<PKV_F16, PKV_F16, false>(a, dim, ws, st);
    if (cache_dtype == PKV_BF16) return attend_dim<PKV_BF16, PKV_BF16, true>(a, dim, ws, st);
    if (cache_dtype == PKV_F16) return attend_dim<PKV_F16, PKV_F16, true>(a, dim, ws, st);
    return dtype == PKV_BF16 ? attend_dim<PKV_FP8, PKV_BF16, true>(a, dim, ws, st)
                             : attend_dim<PKV_FP8, PKV_F16, true>(a, dim, ws, st);
}

int launch_paged_store(const PagedRowsDev& r, uint32_t dim, int cache_dtype, int dtype, void* stream) {
    return launch_rows(r, dim, cache_dtype, dtype, true, stream);
}
int launch_paged_load(const PagedRowsDev& r, uint32_t dim, int cache_dtype, int dtype, void* stream) {
    return launch_rows(r, dim, cache_dtype, dtype, false, stream);
}

}  // namespace pkv
