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
    const int all = end - o.row0;
    o.rows = min(all, static_cast<int>(max_rows));
    o.len = q.lens ? min(max(q.lens[s], 0), static_cast<int>(q.max_len)) : o.rows;
    o.first = q.lens ? o.len - all : 0;     // of all its rows: those past max_rows have their slots too
    return o;
}
// The same of a sequence that all lanes have, in scalar registers.
__device__ inline Seq seq_of_all(const SeqsDev& q, uint32_t s, uint32_t max_rows) {
    const Seq o = seq_of(q, s, max_rows);
    return {__builtin_amdgcn_readfirstlane(o.row0), __builtin_amdgcn_readfirstlane(o.rows),
            __builtin_amdgcn_readfirstlane(o.len), __builtin_amdgcn_readfirstlane(o.first)};
}
// How many of the ascending ends of n things are at most x (both the same in all
// lanes), 64 of them a read: whose x is, or n.
template <class End>
__device__ inline uint32_t ends_up_to(uint32_t n, int x, uint32_t lane, End end) {
    uint32_t lo = 0, left = n;
    while (left) {
        const uint32_t step = (left + 63) / 64, last = (lane + 1) * step - 1;
        lo += __popcll(__ballot(last < left && end(lo + last) <= x)) * step;
        if (step == 1) break;
        left = min(step, n - lo);
    }
    return lo;
}
// The sequence of packed row r (the same in all lanes): the first that ends behind it; -1: nobody's.
__device__ inline int seq_of_row(const SeqsDev& q, int r, uint32_t lane) {
    if (!q.starts) return r / static_cast<int>(q.each);
    const uint32_t s = ends_up_to(q.seqs, r, lane, [&](uint32_t x) { return q.starts[x + 1]; });
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
            const int page = j >= 0 && j < q.len ? page_of(a.seq, s, j) : -1;   // behind it: starts that do not ascend
            if (page >= 0)
                at = static_cast<int64_t>(page * a.page + (static_cast<uint32_t>(j) & ((1u << a.seq.shift) - 1)) * a.slot);
        }
        if (lane == 0) places[i] = at;
    }
    __syncthreads();
}

// A workgroup takes 16 packed rows of a layer and side, 8 values a thread and
// step, channels fastest, then rows, then heads: rows of a sequence that follow
// each other are neighbours in a page, so that a step writes whole lines.  Bound
// by the bytes: 24 x 32 heads x 1,391 rows of 64, keys and values, from f32 in 171 to 183 us and back
// in 141 to 151 (4.1 TB/s; a copy reaches 4.8); 64 single rows take 5 us each way.
template <int CT, int QT, int D>
__global__ __launch_bounds__(256) void paged_store_kernel(PagedRowsDev a, uint32_t heads) {
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
    const uint32_t h0 = blockIdx.z * heads, pieces = min(heads, a.heads - h0) * kChunk * kRow;
    for (uint32_t x = threadIdx.x; x < pieces; x += 256) {
        const uint32_t d = x % kRow * V, i = x / kRow % kChunk, h = h0 + x / kRow / kChunk;
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
__global__ __launch_bounds__(256) void paged_load_kernel(PagedRowsDev a, uint32_t heads) {
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
    const uint32_t h0 = blockIdx.z * heads, pieces = min(heads, a.heads - h0) * kChunk * kRow;
    for (uint32_t x = threadIdx.x; x < pieces; x += 256) {
        const uint32_t d = x % kRow * V, i = x / kRow % kChunk, h = h0 + x / kRow / kChunk;
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
// A cached value.
template <int CT>
__device__ inline float element(const uint8_t* p, const uint8_t* scales, uint64_t e) {
    if constexpr (CT == PKV_FP8) {
        const f32x2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(p[e], block_scale(scales[e / 32]), false);
        return x[0];
    } else {
        return static_cast<float>(reinterpret_cast<const typename Elem<CT>::T*>(p)[e]);
    }
}

// Nobody's rows, before the first sequence's, behind the last's and past a
// sequence's max_rows, to 0: the workgroups behind `work`, kClear of them.
constexpr uint32_t kClear = 64;
template <int QT, int D, int THREADS = 256>
__device__ void clear_rows(const PagedDev& a, uint32_t block) {
    using T = typename Elem<QT>::T;
    const int rows = static_cast<int>(a.seq.rows), most = static_cast<int>(a.max_rows);
    const int heads = static_cast<int>(a.heads * a.group);
    auto clear = [&](int r) {
        T* out = reinterpret_cast<T*>(a.out) + static_cast<uint64_t>(r) * a.o_row;
        for (int y = static_cast<int>(threadIdx.x); y < heads * (D / 8); y += THREADS)
            *reinterpret_cast<u32x4*>(out + static_cast<uint64_t>(y / (D / 8)) * a.o_head + y % (D / 8) * 8) = u32x4{};
    };
    const int first = min(max(a.seq.starts[0], 0), rows);
    int last = first;                                  // the largest end, should starts not ascend
    for (uint32_t s0 = 0; s0 < a.seq.seqs; s0 += 64) {
        const uint32_t s = s0 + threadIdx.x % 64;
        Seq q{};
        if (s < a.seq.seqs) {
            q = seq_of(a.seq, s, a.seq.rows);
            last = max(last, min(a.seq.starts[s + 1], rows));
        }
        for (uint64_t over = __ballot(q.rows > most); over; over &= over - 1) {
            const int i = __ffsll(static_cast<unsigned long long>(over)) - 1;
            const int from = __builtin_amdgcn_readlane(q.row0, i) + most, n = __builtin_amdgcn_readlane(q.rows, i) - most;
            for (int x = static_cast<int>(block); x < n; x += kClear) clear(from + x);
        }
    }
    for (int o = 32; o; o >>= 1) last = max(last, __shfl_xor(last, o));
    const int rest = first + rows - last;
    for (int x = static_cast<int>(block); x < rest; x += kClear) clear(x < first ? x : last + x - first);
}

// Four channels of an output row from their weighted sum (`down` times as large
// as the weights' sum has it), and with the first the row's lse.
template <int QT>
__device__ inline void write_row(const PagedDev& a, uint32_t r, uint32_t qh, uint32_t d, f32x4 o, float base, float sum,
                                 float down) {
    using T = typename Elem<QT>::T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 y;
    const float div = sum * down;
    for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(sum == 0.0f ? 0.0f : o[e] / div);
    *reinterpret_cast<T4*>(reinterpret_cast<T*>(a.out) + static_cast<uint64_t>(r) * a.o_row + qh * a.o_head + d) = y;
    if (d == 0 && a.lse) a.lse[static_cast<uint64_t>(qh) * a.seq.rows + r] = lse_of(base, sum);
}

// ------------------------------------------------------------ few rows: split over the slots
constexpr int kFew = 16;            // rows x group of a KV head that decode_kernel takes
constexpr int kStep = 32;           // slots of its tiles
constexpr int wide_waves(uint32_t dim, int cache_dtype) { return dim == 64 && cache_dtype != PKV_FP8 ? 16 : 8; }
// Units of all heads aimed at.  head_dim 128: two workgroups a CU (a sequence of 32,768 slots of 8 heads: 31 us; 35 with
// fewer, 37 with twice as many, whose start costs more than it hides), and as many as fit where each still has kMany
// tiles (24 such sequences: 541 us, 291 in 8 bits, against 596 and 333; 24 of 700 to 32,768: 168 either way).
constexpr uint32_t fitting_units(uint32_t dim, int cache_dtype) {
    return dim == 64 ? cache_dtype == PKV_FP8 ? 768 : 1024 : 512;
}
constexpr uint32_t kMostUnits = 1024;
static_assert(kMostUnits <= 1u << kJoinDown && fitting_units(64, PKV_BF16) <= kMostUnits && fitting_units(128, PKV_BF16) <= kMostUnits,
              "shares of a row as they are joined");
constexpr int kMany = 96;
constexpr int kLeast = 4;           // tiles of a unit, one a wave
constexpr int kLeastSteps = 8;      // rows_kernel: tiles of 64 slots of a share

// The tiles that a sequence of few rows has; -1: it has no rows, or more.
__device__ inline int few_tiles(const PagedDev& a, uint32_t s) {
    const Seq q = seq_of(a.seq, s, a.max_rows);
    if (!q.rows || static_cast<int64_t>(q.rows) * a.group > kFew) return -1;
    return tiles_of(a, q.first, q.first + q.rows - 1, kStep).count;
}

// The least whole number above all / target, and at least `least`.
__device__ inline int share_of(int64_t all, uint32_t target, int least) {
    const double share = static_cast<double>(all) / target;   // counts stay below 2^53
    return max(least, static_cast<int>(fmin(share, 1e9)) + 1);
}

// A share of a sequence's tiles, as units of about as many tiles for all
// sequences: all their tiles by the units wanted a head, at least kLeast.  Every
// workgroup works this out from the lengths, which only the device knows: a lane
// takes a run of sequences, so up to 64 of them cost one read of their words.
// That work grows with the square of the sequences: more than kCounted are
// counted once, by a kernel ahead, and looked up.
struct Unit {
    int seq, share, shares, first;   // first: the sequence's first unit
};
// Tiles of a unit: no more than target (or most) + sequences units.
__device__ inline int unit_size(int64_t all, uint32_t target, uint32_t most) {
    return share_of(all, all >= static_cast<int64_t>(kMany) * most ? most : target, kLeast);
}
__device__ inline int units_of(int tiles, int size) { return tiles < 0 ? 0 : max(1, (tiles + size - 1) / size); }
__device__ inline bool find_unit(const PagedDev& a, uint32_t u, uint32_t target, uint32_t most, uint32_t lane, Unit* o) {
    const uint32_t per = (a.seq.seqs + 63) / 64, s0 = min(lane * per, a.seq.seqs), s1 = min(s0 + per, a.seq.seqs);
    int mine = -1;                      // of the run's only sequence
    int64_t all = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        mine = few_tiles(a, s);
        all += max(mine, 0);
    }
    for (int x = 32; x; x >>= 1) all += __shfl_xor(static_cast<long long>(all), x);
    const int size = unit_size(all, target, most);
    int n = 0;
    if (per == 1) n = units_of(mine, size);
    else
        for (uint32_t s = s0; s < s1; ++s) n += units_of(few_tiles(a, s), size);
    int end = n;
    for (int x = 1; x < 64; x <<= 1) {
        const int y = __shfl_up(end, x);
        if (static_cast<int>(lane) >= x) end += y;
    }
    const int want = static_cast<int>(u);
    const uint32_t at = __popcll(__ballot(end <= want));
    if (at == 64) return false;
    int first = __shfl(end - n, static_cast<int>(at));
    uint32_t s = at * per;
    for (;; ++s) {
        n = per == 1 ? __shfl(n, static_cast<int>(at)) : units_of(few_tiles(a, s), size);
        if (want < first + n) break;
        first += n;
    }
    *o = {static_cast<int>(s), want - first, n, first};
    return true;
}
// The same by the plan of few_plan_kernel.
__device__ inline bool look_up_unit(const PagedDev& a, const int32_t* plan, uint32_t u, uint32_t lane, Unit* o) {
    const int want = static_cast<int>(u);
    const uint32_t s = ends_up_to(a.seq.seqs, want, lane, [&](uint32_t x) { return plan[2 * x] + plan[2 * x + 1]; });
    if (s >= a.seq.seqs) return false;
    *o = {static_cast<int>(s), want - plan[2 * s], plan[2 * s + 1], plan[2 * s]};
    return true;
}

// What is the same in all lanes, for the compiler to see.
__device__ inline const uint8_t* uniform(const uint8_t* p) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x)),
                   hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
    return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ inline Tiles uniform(const Tiles& t) {
    return {__builtin_amdgcn_readfirstlane(t.first), __builtin_amdgcn_readfirstlane(t.second),
            __builtin_amdgcn_readfirstlane(t.count), __builtin_amdgcn_readfirstlane(t.low),
            __builtin_amdgcn_readfirstlane(t.high)};
}

// Pages of a tile's 16-slot pieces: a lane reads one piece's word.  `last` is the
// last slot that is read; pieces behind its own take its page.
__device__ inline int piece_start(int slot, int piece, int last) { return min(slot + 16 * piece, last & ~15); }
template <int PIECES>
__device__ inline int read_pages(const SeqsDev& q, const int32_t* table, int slot, int last, uint32_t lane) {
    return table[static_cast<uint32_t>(piece_start(slot, lane % PIECES, last)) >> q.shift];
}
// Bit p: piece p of them is on no page.
template <int PIECES>
__device__ inline uint32_t no_page(const SeqsDev& q, int words) {
    return static_cast<uint32_t>(__ballot(static_cast<uint32_t>(words) >= q.pages)) & ((1u << PIECES) - 1);
}
// Elements to the piece that starts at slot `start` (on no page: page 0's, which is not used).
__device__ inline uint64_t piece_at(const PagedDev& a, int words, int piece, int start, uint64_t head) {
    const uint32_t p = __builtin_amdgcn_readlane(words, piece);
    return (p < a.seq.pages ? p : 0) * a.page + head +
           (static_cast<uint32_t>(start) & ((1u << a.seq.shift) - 1)) * a.k_slot;
}

// Eight 8-bit codes under one scale to bf16.
__device__ inline u32x4 expand8(uint32_t lo, uint32_t hi, float s) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true))};
}

// A wave's tile of 32 slots as matrix operands in registers (two pieces of 16):
// of the keys a lane holds slot lane % 16 and a quarter of every 32 channels (8
// bits: a quarter of all), of the values channels kPer (lane % 16) .. of the
// slots 4 (lane / 16) ..: what decode_kernel's products want, every read of 4 to
// 16 bytes in line.
template <int CT, int D>
struct PageTile {
    static constexpr bool k8 = CT == PKV_FP8;
    static constexpr int kKRegs = k8 ? D / 64 : D / 32, kPer = D / 16;
    typedef typename std::conditional<D == 128, uint32_t, uint16_t>::type ScaleRow;   // of a slot
    u32x4 k[2][kKRegs], v[2][4];
    uint32_t ks[2];
    u32x4 vs[2];
    uint32_t missing;                   // pieces on no page

    __device__ void load(const PagedDev& a, uint64_t head, int words, int slot, int last, uint32_t lane) {
        const uint32_t i = lane % 16, g = lane / 16;
        const uint32_t st = static_cast<uint32_t>(a.k_slot);
        constexpr uint32_t kSize = k8 ? 1 : 2;
        missing = no_page<2>(a.seq, words);
        const uint8_t *kt[2], *vt[2], *kst[2], *vst[2];
        int room[2];
        for (int u = 0; u < 2; ++u) {
            const int start = piece_start(slot, u, last);
            const uint64_t e = piece_at(a, words, u, start, head);
            room[u] = last - start;
            kt[u] = a.k + e * kSize;
            vt[u] = a.v + e * kSize;
            if constexpr (k8) { kst[u] = a.ks + e / 32; vst[u] = a.vs + e / 32; }
        }
        for (int u = 0; u < 2; ++u) {
            const uint32_t e = static_cast<uint32_t>(min(static_cast<int>(i), room[u])) * st;
            for (int s = 0; s < kKRegs; ++s)
                k[u][s] = *reinterpret_cast<const u32x4*>(kt[u] + (k8 ? e + D / 4 * g + 16 * s : 2 * e + 64 * s + 16 * g));
            if constexpr (k8) ks[u] = kst[u][e / 32 + (D == 128 ? g : g / 2)];
        }
        for (int u = 0; u < 2; ++u) {
            for (int j = 0; j < 4; ++j) {
                const uint32_t e = static_cast<uint32_t>(min(static_cast<int>(4 * g) + j, room[u])) * st;
                if constexpr (k8 && D == 64) v[u][j][0] = *reinterpret_cast<const uint32_t*>(vt[u] + e + 4 * i);
                else if constexpr (!k8 && D == 128) v[u][j] = *reinterpret_cast<const u32x4*>(vt[u] + 2 * e + 16 * i);
                else {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(vt[u] + kSize * e + 8 * i);
                    v[u][j] = u32x4{x[0], x[1], 0, 0};
                }
            }
            // of the lane group's four slots; slots of the piece past the last: bytes of the page that are not used
            if constexpr (k8 && D == 128) vs[u] = *reinterpret_cast<const u32x4*>(vst[u] + 16 * g);
            else if constexpr (k8) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(vst[u] + 8 * g);
                vs[u] = u32x4{x[0] & 0xffff, x[0] >> 16, x[1] & 0xffff, x[1] >> 16};
            }
        }
    }
    // The operand of step s (32 channels) of piece u's logits.
    __device__ u32x4 keys(int u, int s) const {
        if constexpr (!k8) return k[u][s];
        else {
            const uint32_t lo = k[u][s / 2][s % 2 * 2], hi = k[u][s / 2][s % 2 * 2 + 1];
            return expand8(lo, hi, block_scale(ks[u]));
        }
    }
    __device__ void expand_values(uint32_t lane) {
        if constexpr (k8)
            for (int u = 0; u < 2; ++u)
                for (int j = 0; j < 4; ++j) {
                    const uint32_t row = vs[u][j], lo = v[u][j][0], hi = v[u][j][1];
                    v[u][j] = expand8(lo, hi, block_scale(row >> (lane % 16 / (D == 128 ? 4 : 8) * 8) & 0xff));
                }
    }
    // Infinities and NaN among slot j of piece u's values to 0; true if the lane had any.
    __device__ bool clean(int u, int j) {
        bool odd = false;
        for (int w = 0; w < kPer / 2; ++w) {
            const uint32_t x = v[u][j][w], y = finite_or_0<mat_type(CT)>(x);
            odd |= y != x;
            v[u][j][w] = y;
        }
        return odd;
    }
    // The channel that the lane's keys of step s start at, and that output register (e, r) of lane group g is.
    __device__ static uint32_t channel(int s, uint32_t g) { return k8 ? D / 4 * g + 8 * s : 32 * s + 8 * g; }
    __device__ static uint32_t out_channel(int e, int r, uint32_t g) { return kPer * (4 * g + r) + e; }
};

// Shares of a unit's or a tile's rows on their way to a join.
struct PagedPart {
    float* o;          // [head][unit][rows][D]
    float* ml;         // [head][unit][rows][2]: base, sum of the weights
    int32_t* plan;     // [sequence][2]: first unit, units; of many rows the first that is a share, shares of a tile
    uint32_t units, target, rows, parts;
    uint32_t most;     // decode_kernel: aimed at where they are long
    int32_t* ends;     // [sequence] of many rows, counted ahead: units up to its last
    bool counted;      // plan (and ends) are there before the kernel
};

// The rows of a sequence of few (rows x group up to 16) against a share of its
// slots, both products on the matrix cores with nothing staged in LDS:
//   S^T = K Q^T   A = 16 slots (lane % 16) x 8 channels a lane group (lane /
//                 16); B = 16 rows (lane % 16).  Any order of the channels will
//                 do as long as q has the same.  Result: row lane % 16, slots 4
//                 (lane / 16) + r.
//   O^T = V^T P^T A wants, for one channel a lane, the slots its lane group has
//                 in S^T: the softmax's registers are B as they are, v_perm
//                 gathers each channel across the lane's four (x 2) slots.
// Weights meet the values as two terms of a 16-bit type, which the bytes hide.
// WAVES 4, or 8 or 16 (as registers allow) where a sequence's slots are one
// unit's, so that the call is one launch (a row of 32 heads of 64 on 700 slots:
// 14 us with the host's call, 16 in units of four waves and a join; in a graph 12
// and 9.6, and eight such rows on about 900 slots 16.5 and 19.4).  The next tile
// is on its way while one is worked on, and the words of the pages of the one
// after it, so that no read waits for a page's number.
// Bound by the bytes: 5.9 TB/s of 24 x 32,768 slots of 8 heads of 128, 5.7 in 8
// bits, 5.5 and 5.0 where the 24 sequences have 700 to 32,768; a large copy
// reaches 4.8 on this card, a large sum 4.0.  Of short sequences by the chain
// kernel's start, the lengths, a page's number, a tile, the joins (97 sequences
// of 33 to 3,000 slots of 4 heads in 8 bits: 31 us and 5 of join_kernel for what
// the bytes make 14.5).
template <int CT, int QT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES > 8 ? 4 : 2) void decode_kernel(PagedDev a, PagedPart part) {
    using T = typename Elem<QT>::T;
    using Tile = PageTile<CT, D>;
    constexpr int MT = mat_type(CT), NQ = query_terms(CT, QT), NP = 2, kQ = D / 32, kO = D / 16;
    constexpr int kDownOf = WAVES > 4 ? kPartDown + 2 : kPartDown;   // the waves' outputs together
    const uint32_t work_blocks = a.heads * part.units;
    if (blockIdx.x >= work_blocks) return clear_rows<QT, D, 64 * WAVES>(a, blockIdx.x - work_blocks);
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    // heads fastest, so that a head's workgroups share an XCD's L2 (and the pages of a common prefix) where the heads
    // are a multiple of 8
    const uint32_t h = blockIdx.x % a.heads, u = blockIdx.x / a.heads;
    Unit unit;
    if (!(part.counted ? look_up_unit(a, part.plan, u, lane, &unit) : find_unit(a, u, part.target, part.most, lane, &unit)))
        return;
    unit = {__builtin_amdgcn_readfirstlane(unit.seq), __builtin_amdgcn_readfirstlane(unit.share),
            __builtin_amdgcn_readfirstlane(unit.shares), __builtin_amdgcn_readfirstlane(unit.first)};
    if (h == 0 && unit.share == 0 && threadIdx.x == 0 && !part.counted) {
        part.plan[2 * unit.seq] = unit.first;
        part.plan[2 * unit.seq + 1] = unit.shares;
    }
    const Seq sq = seq_of_all(a.seq, unit.seq, a.max_rows);
    const uint32_t row = lane % 16, g = lane / 16;
    const int R = sq.rows * static_cast<int>(a.group), pos1 = sq.first + sq.rows - 1;
    const bool real = static_cast<int>(row) < R;
    const int qi = row / a.group, pos = real ? sq.first + qi : -1;
    const Tiles tl = uniform(tiles_of(a, sq.first, pos1, kStep));
    const int per = __builtin_amdgcn_readfirstlane((tl.count + unit.shares - 1) / unit.shares);
    const int t0 = unit.share * per, t1 = min(t0 + per, tl.count);
    const int32_t* table = a.seq.tables + unit.seq * a.seq.table;

    const T* qp = reinterpret_cast<const T*>(a.q) + static_cast<uint64_t>(sq.row0 + (real ? qi : 0)) * a.q_row +
                  (h * a.group + (real ? row % a.group : 0)) * a.q_head;
    u32x4 q[NQ][kQ];
    for (int s = 0; s < kQ; ++s) {
        const uint32_t d = Tile::channel(s, g);
        if constexpr (NQ == 1) {
            q[0][s] = real ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{};
        } else {
            for (int w = 0; w < 4; ++w) {
                float x = real ? static_cast<float>(qp[d + 2 * w]) : 0.0f;
                float y = real ? static_cast<float>(qp[d + 2 * w + 1]) : 0.0f;
                for (int n = 0; n < NQ; ++n) q[n][s][w] = pack_query_term(x, y);
            }
        }
    }

    const uint64_t head = h * a.k_head;
    float base = kInf, l = 0.0f;
    f32x4 o[kO] = {};
    auto pages = [&](int t) {   // past the last tile: the last's again, unused
        return read_pages<2>(a.seq, table, tl.slot(min(t, t1 - 1), kStep), tl.high - 1, lane);
    };
    auto fetch = [&](Tile& x, int t, int words) {
        x.load(a, head, words, tl.slot(min(t, t1 - 1), kStep), tl.high - 1, lane);
    };
    auto work = [&](Tile& x, int t, auto again) {
        constexpr bool CLEAN = decltype(again)::value;   // infinities and NaN of the values by themselves
        const int slot = tl.slot(t, kStep);
        f32x4 sc[2] = {};
        for (int p = 0; p < 2; ++p)
            for (int s = 0; s < kQ; ++s) {
                const u32x4 ka = x.keys(p, s);
                for (int n = NQ - 1; n >= 0; --n) sc[p] = mma16<MT>(ka, q[n][s], sc[p]);
            }
        x.expand_values(lane);
        if (x.missing || !all_visible(a, sq.first, pos1, slot, slot + kStep - 1)) {
            for (int p = 0; p < 2; ++p)
                for (int j = 0; j < 4; ++j) {
                    const int key = slot + 16 * p + 4 * static_cast<int>(g) + j;
                    const bool none = x.missing >> p & 1;
                    if (none || !visible(a, pos, key)) sc[p][j] = -kInf;
                    if (none || !any_visible(a, tl, key)) x.v[p][j] = u32x4{};
                }
        }
        bool odd[2][4] = {};
        if constexpr (CLEAN)
            for (int p = 0; p < 2; ++p)
                for (int j = 0; j < 4; ++j) odd[p][j] = x.clean(p, j);
        float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
        top = fmaxf(top, fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
        top = across32(across16(top, larger), larger);
        if (__any(__builtin_fmaf(top, a.scale2, base) > kLift<MT> + kLag<MT>)) {
            const float low = lower_base(a, kLift<MT>, base, top), f = joined(low, base);
            if (low < base) {
                l *= f;
                for (int e = 0; e < kO; ++e) o[e] *= f;
                base = low;
            }
        }
        const float from = base == kInf ? 0.0f : base;
        float p[2][4], r[2][4];
        for (int x2 = 0; x2 < 2; ++x2)
            for (int j = 0; j < 4; ++j) {
                p[x2][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x2][j], a.scale2, from));
                if constexpr (CLEAN) p[x2][j] *= kPower<-kDown<MT>>;
                l += p[x2][j];
                r[x2][j] = p[x2][j];
            }
        u32x4 pt[NP];
        for (int n = 0; n < NP; ++n)
            pt[n] = u32x4{pack_term<MT>(r[0][0], r[0][1]), pack_term<MT>(r[0][2], r[0][3]),
                          pack_term<MT>(r[1][0], r[1][1]), pack_term<MT>(r[1][2], r[1][3])};
        for (int e = 0; e < kO; ++e) {
            const uint32_t sel = e % 2 ? 0x07060302u : 0x05040100u;
            const u32x4 va = {__builtin_amdgcn_perm(x.v[0][1][e / 2], x.v[0][0][e / 2], sel),
                              __builtin_amdgcn_perm(x.v[0][3][e / 2], x.v[0][2][e / 2], sel),
                              __builtin_amdgcn_perm(x.v[1][1][e / 2], x.v[1][0][e / 2], sel),
                              __builtin_amdgcn_perm(x.v[1][3][e / 2], x.v[1][2][e / 2], sel)};
            for (int n = NP - 1; n >= 0; --n) o[e] = mma16<MT>(va, pt[n], o[e]);
        }
        if constexpr (CLEAN)
            for (int x2 = 0; x2 < 2; ++x2)
                for (int j = 0; j < 4; ++j) {
                    const uint64_t has = __ballot(odd[x2][j]);
#pragma unroll 1
                    for (uint32_t g2 = 0; g2 < 4; ++g2) {
                        if (!(has >> 16 * g2 & 0xffff)) continue;
                        const int key = slot + 16 * x2 + 4 * static_cast<int>(g2) + j;
                        const bool sees = real && visible(a, pos, key);
                        // not scaled down: that could make it 0
                        const float w = __shfl(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[x2][j], a.scale2, from)),
                                               static_cast<int>(16 * g2 + row));
                        const int page = page_of(a.seq, unit.seq, min(key, tl.high - 1));
                        const uint64_t at = (page < 0 ? 0 : page) * a.page + head +
                                            (static_cast<uint32_t>(key) & ((1u << a.seq.shift) - 1)) * a.k_slot;
                        for (int e = 0; e < kO; ++e)
                            for (int r2 = 0; r2 < 4; ++r2) {
                                const float v = element<CT>(a.v, a.vs, at + Tile::out_channel(e, r2, g));
                                if (sees && (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[e][r2] += w * v;
                            }
                    }
                }
    };
    // two tiles in turn: one is on its way while the other is worked on
    const int first = t0 + static_cast<int>(wave);
    if (first < t1) {
        Tile even, odd;
        int words = pages(first), next = pages(first + WAVES);
        fetch(even, first, words);
        for (int t = first; t < t1; t += 2 * WAVES) {
            words = pages(t + 2 * WAVES);
            fetch(odd, t + WAVES, next);
            work(even, t, std::false_type());
            if (t + WAVES >= t1) break;
            next = pages(t + 3 * WAVES);
            fetch(even, t + 2 * WAVES, words);
            work(odd, t + WAVES, std::false_type());
        }
        // An infinity or NaN among the values: a row that does not see it has met it with the weight 0, and the terms
        // of a weight that does see it may be 0 or negative.  Again, with those values taken out of the products and
        // each added to the rows that see it; or a sum past the type's end: see kDown.
        bool bad = false;
        for (int e = 0; e < kO; ++e)
            for (int r = 0; r < 4; ++r) bad |= (__float_as_uint(o[e][r]) & 0x7f800000u) == 0x7f800000u;
        if (__builtin_expect(__any(bad && real), 0)) {
            base = kInf;
            l = 0.0f;
            for (int e = 0; e < kO; ++e) o[e] = f32x4{};
#pragma unroll 1
            for (int t = first; t < t1; t += WAVES) {
                fetch(even, t, pages(t));
                work(even, t, std::true_type());
            }
            bool past = false;   // back, unless it does not fit
            for (int e = 0; e < kO; ++e)
                for (int r = 0; r < 4; ++r)
                    past |= fabsf(o[e][r]) < kInf && !(fabsf(o[e][r]) * kPower<kDown<MT>> < kInf);
            if (__any(past && real)) {
                base -= kDown<MT>;
            } else {
                for (int e = 0; e < kO; ++e) o[e] *= kPower<kDown<MT>>;
                l *= kPower<kDown<MT>>;
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' shares joined; a sequence of one unit is done
    __shared__ float so[WAVES][16][D + 4], sb[WAVES][16], sl[WAVES][16];
    for (int r = 0; r < 4; ++r)
        for (int e = 0; e < kO; ++e) so[wave][row][Tile::out_channel(e, r, g)] = o[e][r];
    if (g == 0) { sb[wave][row] = base; sl[wave][row] = l; }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < static_cast<uint32_t>(R) * (D / 4); x += 64 * WAVES) {
        const uint32_t r = x / (D / 4), d = x % (D / 4) * 4;
        float low = sb[0][r];
        for (int w = 1; w < WAVES; ++w) low = fminf(low, sb[w][r]);
        float sum = 0.0f;
        f32x4 acc = {};
        for (int w = 0; w < WAVES; ++w) {
            const float f = joined(low, sb[w][r]);
            sum += sl[w][r] * f;
            acc += *reinterpret_cast<const f32x4*>(&so[w][r][d]) * (f * kPower<-kDownOf>);
        }
        if (unit.shares == 1) {
            write_row<QT>(a, sq.row0 + r / a.group, h * a.group + r % a.group, d, acc, low, sum, kPower<-kDownOf>);
        } else {
            const uint64_t at = (static_cast<uint64_t>(h) * part.units + u) * part.rows + r;
            *reinterpret_cast<f32x4*>(part.o + at * D + d) = acc;
            if (d == 0) {
                part.ml[2 * at] = low;
                part.ml[2 * at + 1] = sum;
            }
        }
    }
}

// The units of a row joined, a workgroup a row: every wave the row's base and
// sum, then 1024 / D units at a time, 4 channels a thread.
template <int QT, int D>
__global__ __launch_bounds__(256) void join_kernel(PagedDev a, PagedPart part) {
    const uint32_t lane = threadIdx.x % 64;
    const uint32_t r = blockIdx.x % part.rows, sh = blockIdx.x / part.rows, s = sh / a.heads, h = sh % a.heads;
    const Seq q = seq_of(a.seq, s, a.max_rows);
    const int64_t all = static_cast<int64_t>(q.rows) * a.group;
    if (r >= all || all > kFew) return;
    const uint32_t first = part.plan[2 * s], shares = part.plan[2 * s + 1];
    if (shares == 1) return;
    const uint64_t at = (static_cast<uint64_t>(h) * part.units + first) * part.rows + r;
    const float* ml = part.ml + 2 * at;
    const uint64_t step = 2ull * part.rows;
    float low = kInf;
    for (uint32_t x = lane; x < shares; x += 64) low = fminf(low, ml[step * x]);
    for (int x = 32; x; x >>= 1) low = fminf(low, __shfl_xor(low, x));
    float sum = 0.0f;
    for (uint32_t x = lane; x < shares; x += 64) sum += ml[step * x + 1] * joined(low, ml[step * x]);
    sum = wave_sum(sum);
    constexpr uint32_t kLanes = D / 4, kShares = 256 / kLanes;
    const uint32_t mine = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
    f32x4 o = {};
    for (uint32_t x = mine; x < shares; x += kShares) {
        const float f = joined(low, ml[step * x]) * kPower<-kJoinDown>;
        o += *reinterpret_cast<const f32x4*>(part.o + (at + static_cast<uint64_t>(part.rows) * x) * D + d) * f;
    }
    __shared__ f32x4 so[256];
    so[threadIdx.x] = o;
    __syncthreads();
    if (mine) return;
    for (uint32_t x = 1; x < kShares; ++x) o += so[threadIdx.x + x * kLanes];
    write_row<QT>(a, q.row0 + r / a.group, h * a.group + r % a.group, d, o, low, sum, kPower<-kPartDown - kJoinDown>);
}

// ------------------------------------------------------------ many rows: tiles of rows through LDS
// A workgroup's part of a head's work: a tile of a sequence's rows against a share
// of the slots' tiles.  Shares are as many for all tiles of a sequence, so that
// one has at least 1 / target of all tiles there are (the last rows' counted for
// all rows) and less than twice that: no more than `target` units are shares.
// Units go from the longest on, of a sequence from the last rows, which see most.
// A lane takes a run of sequences, as in find_unit.
struct RowUnit {
    int seq, tile, share, shares;
    int part;                    // of the units that are shares, the tile's first
};
struct RowWork {
    int tiles, steps;            // row tiles, and the slots' tiles that the last of them sees
};
__device__ inline RowWork row_work(const PagedDev& a, uint32_t s, int64_t few, int rows) {
    const Seq q = seq_of(a.seq, s, a.max_rows);
    const int64_t all = static_cast<int64_t>(q.rows) * a.group;
    RowWork w{};
    if (all <= few) return w;
    w.tiles = static_cast<int>((all + rows - 1) / rows);
    const int first = (w.tiles - 1) * rows / static_cast<int>(a.group);
    w.steps = tiles_of(a, q.first + first, q.first + q.rows - 1, 64).count;
    return w;
}
__device__ inline int rows_size(int64_t all, uint32_t target) {
    return target ? share_of(all, target, kLeastSteps) : 0x7fffffff;
}
__device__ inline int shares_of(const RowWork& w, int size) { return max(1, w.steps / size); }
__device__ inline bool find_rows(const PagedDev& a, uint32_t u, int64_t few, int rows, uint32_t target, uint32_t lane,
                                 RowUnit* o) {
    const uint32_t per = (a.seq.seqs + 63) / 64, s0 = min(lane * per, a.seq.seqs), s1 = min(s0 + per, a.seq.seqs);
    RowWork mine{};
    int64_t all = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        mine = row_work(a, s, few, rows);
        all += static_cast<int64_t>(mine.tiles) * mine.steps;
    }
    if (target)
        for (int x = 32; x; x >>= 1) all += __shfl_xor(static_cast<long long>(all), x);
    const int size = rows_size(all, target);
    auto shares = [&](const RowWork& w) { return shares_of(w, size); };
    int units = 0, parts = 0, longest = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        const RowWork w = per == 1 ? mine : row_work(a, s, few, rows);
        const int n = shares(w);
        units = min(units + w.tiles * n, 1 << 24);   // no launch has as many; more where starts do not ascend
        parts += n > 1 ? w.tiles * n : 0;
        longest = max(longest, w.steps / n);
    }
    // of the lanes with longer units, or as long ones and before this one
    int first = 0, part = 0;
    const uint32_t lanes = (a.seq.seqs + per - 1) / per;
    for (uint32_t x = 0; x < lanes; ++x) {
        const int len = __builtin_amdgcn_readlane(longest, x), n = __builtin_amdgcn_readlane(units, x),
                  m = __builtin_amdgcn_readlane(parts, x);
        const bool ahead = len > longest || (len == longest && x < lane);
        first += ahead ? n : 0;
        part += ahead ? m : 0;
    }
    const int want = static_cast<int>(u);
    const uint64_t found = __ballot(want >= first && want < first + units);
    if (!found) return false;
    const int at = __ffsll(static_cast<unsigned long long>(found)) - 1;
    first = __builtin_amdgcn_readlane(first, at);
    part = __builtin_amdgcn_readlane(part, at);
    for (uint32_t s = at * per;; ++s) {
        const RowWork w = row_work(a, s, few, rows);
        const int n = shares(w);
        if (want < first + w.tiles * n) {
            const int x = (want - first) / n, tile = w.tiles - 1 - x;
            *o = {static_cast<int>(s), tile, want - first - x * n, n, part + tile * n};
            return true;
        }
        first += w.tiles * n;
        part += n > 1 ? w.tiles * n : 0;
    }
}
// The same by the plan of rows_plan_kernel, in the sequences' order.
__device__ inline bool look_up_rows(const PagedDev& a, const int32_t* plan, const int32_t* ends, uint32_t u, int64_t few,
                                    int rows, uint32_t lane, RowUnit* o) {
    const int want = static_cast<int>(u);
    const uint32_t s = ends_up_to(a.seq.seqs, want, lane, [&](uint32_t x) { return ends[x]; });
    if (s >= a.seq.seqs) return false;
    const int n = plan[2 * s + 1], at = want - (s ? ends[s - 1] : 0), x = at / n;
    const int tile = row_work(a, s, few, rows).tiles - 1 - x;
    *o = {static_cast<int>(s), tile, at - x * n, n, plan[2 * s] + tile * n};
    return true;
}

// ------------------------------------------------------------ many sequences: counted once
// More sequences than this are counted by one workgroup ahead of the kernel, whose
// launch costs about what the counting by every workgroup does here: 256 single
// tokens on 20 slots of 8 heads of 64 take 27 us, 23 counted ahead, of 4 heads 17
// and 21; 1,024 of 8 heads 182 and 48, 4,096 prompts of 4 rows 9,900 and 690.
constexpr uint32_t kCounted = 256;
constexpr uint32_t kCounters = 1024;   // its threads

// The sum of x over the workgroup's threads before this one; *all: over all of them.
__device__ inline int64_t sum_before(int64_t x, int64_t* all, int64_t (&waves)[kCounters / 64]) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int64_t end = x;
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(static_cast<long long>(end), o);
        if (lane >= o) end += y;
    }
    __syncthreads();                   // the last call's sums have been read
    if (lane == 63) waves[wave] = end;
    __syncthreads();
    int64_t before = 0;
    *all = 0;
    for (uint32_t w = 0; w < kCounters / 64; ++w) {
        before += w < wave ? waves[w] : 0;
        *all += waves[w];
    }
    return before + end - x;
}

// decode_kernel's units: plan[2 s] the first of sequence s, plan[2 s + 1] how many.
__global__ __launch_bounds__(kCounters) void few_plan_kernel(PagedDev a, PagedPart part) {
    __shared__ int64_t waves[kCounters / 64];
    int64_t mine = 0, all, first = 0;
    for (uint32_t s = threadIdx.x; s < a.seq.seqs; s += kCounters) mine += max(few_tiles(a, s), 0);
    sum_before(mine, &all, waves);
    const int size = unit_size(all, part.target, part.most);
    for (uint32_t s0 = 0; s0 < a.seq.seqs; s0 += kCounters) {
        const uint32_t s = s0 + threadIdx.x;
        const int n = s < a.seq.seqs ? units_of(few_tiles(a, s), size) : 0;
        const int64_t before = sum_before(n, &all, waves);
        if (s < a.seq.seqs) {
            part.plan[2 * s] = static_cast<int32_t>(first + before);
            part.plan[2 * s + 1] = n;
        }
        first += all;
    }
}

// rows_kernel's: ends[s] the units up to sequence s's last, plan[2 s] the first of
// its units that are shares, plan[2 s + 1] the shares of a tile.
__global__ __launch_bounds__(kCounters) void rows_plan_kernel(PagedDev a, PagedPart part, int few) {
    __shared__ int64_t waves[kCounters / 64];
    int64_t mine = 0, all, units = 0, parts = 0;
    for (uint32_t s = threadIdx.x; s < a.seq.seqs; s += kCounters) {
        const RowWork w = row_work(a, s, few, static_cast<int>(part.rows));
        mine += static_cast<int64_t>(w.tiles) * w.steps;
    }
    sum_before(mine, &all, waves);
    const int size = rows_size(all, part.target);
    for (uint32_t s0 = 0; s0 < a.seq.seqs; s0 += kCounters) {
        const uint32_t s = s0 + threadIdx.x;
        RowWork w{};
        if (s < a.seq.seqs) w = row_work(a, s, few, static_cast<int>(part.rows));
        const int n = shares_of(w, size);
        const int64_t own = static_cast<int64_t>(w.tiles) * n, shares = n > 1 ? own : 0;
        const int64_t end = units + own + sum_before(own, &all, waves);
        units += all;
        const int64_t at = parts + sum_before(shares, &all, waves);
        parts += all;
        if (s < a.seq.seqs) {
            part.ends[s] = static_cast<int32_t>(min(end, static_cast<int64_t>(0x7fffffff)));   // more where starts do not ascend
            part.plan[2 * s] = static_cast<int32_t>(at);
            part.plan[2 * s + 1] = n;
        }
    }
}

// Staged's tiles from pages, or (PAGED false) from packed rows, a side at a time
// by the four waves of a group.  16-bit rows go from memory to LDS without
// registers; a wave's 1,024 bytes lie in one page.
template <int CT, int D, bool PAGED>
struct PageStage : Staged<CT, D> {
    using L = Staged<CT, D>;
    using L::kRow, L::kPieces, L::kKeyBytes, L::kCopies, L::kCopyRows, L::kCopyStep, L::turn, L::key_at, L::value_at, L::code_slot;
    static constexpr int kHeld = CT == PKV_FP8 ? D / 64 : 1;   // 16 codes a register
    struct Side {
        u32x4 codes[kHeld];                                    // 8-bit codes on their way
        uint32_t scale;
    };

    // A side's copies (16 bits): LDS place of the wave's part, and the lane's offset from the first row that it copies a
    // piece of.  turn() of the row is the same for all of a lane's copies.
    struct Copies {
        uint32_t to, off, stride;
    };
    template <bool VALUES>
    __device__ static Copies copies(const PagedDev& a, uint32_t t) {
        const uint32_t lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64), row = kCopyRows * wave + lane / kPieces;
        Copies c;
        c.stride = 2 * static_cast<uint32_t>(VALUES ? a.v_slot : a.k_slot);
        c.to = (VALUES ? kKeyBytes : 0) + kCopyRows * wave * kRow;
        c.off = lane / kPieces * c.stride + (lane % kPieces ^ turn(row, VALUES)) * 16;
        return c;
    }
    // Where the rows that copy x takes of the tile at `slot` start: of the head's pages (rows: the head's packed row 0).
    __device__ static const uint8_t* copy_from(const PagedDev& a, const uint8_t* side, const uint8_t* rows, uint64_t head,
                                               int words, int slot, int last, uint32_t stride, int x, uint32_t wave) {
        const int r = kCopyStep * x + kCopyRows * static_cast<int>(wave);
        if constexpr (PAGED) {
            const int start = piece_start(slot, r / 16, last);
            return side + 2 * piece_at(a, words, r / 16, start, head) + r % 16 * stride;
        } else {
            return rows + static_cast<uint64_t>(slot + r) * stride;
        }
    }
    // Start a side of a tile on its way to the tile at `lds`.  head: elements to the head's first page; rows: the head's
    // packed row 0 (PAGED false); slots past `last` read the last one.  t: the thread in its group.
    template <bool VALUES>
    __device__ static void fetch(Side& s, const Copies& c, const PagedDev& a, uint32_t lds, const uint8_t* rows,
                                 uint64_t head, int words, int slot, int last, uint32_t t) {
        const uint32_t lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
        const uint8_t* from = VALUES ? a.v : a.k;
        if constexpr (CT == PKV_FP8) {
            const int start = piece_start(slot, wave, last);
            const uint64_t e = piece_at(a, words, wave, start, head) +
                               static_cast<uint32_t>(min(static_cast<int>(code_slot(t) - 16 * wave), last - start)) * D;
            const uint32_t b = t % 4;
            for (int x = 0; x < kHeld; ++x) s.codes[x] = *reinterpret_cast<const u32x4*>(from + e + D / 4 * b + 16 * x);
            s.scale = (VALUES ? a.vs : a.ks)[e / 32 + (D == 128 ? b : b / 2)];
        } else {
            const int row = kCopyRows * static_cast<int>(wave) + static_cast<int>(lane / kPieces);
            for (int x = 0; x < kCopies; ++x) {
                const uint8_t* at = copy_from(a, from, rows, head, words, slot, last, c.stride, x, wave);
                // the piece may start in front of the tile's part, and the row lie in front of copy_from's
                const int r = kCopyStep * x + row, first = PAGED ? piece_start(slot, r / 16, last) + r % 16 : slot + r;
                const int32_t back = (min(slot + r, last) - first) * static_cast<int32_t>(c.stride);
                copy_row_to_lds(__builtin_amdgcn_readfirstlane(lds + c.to + kCopyStep * kRow * x), at + c.off + static_cast<int64_t>(back));
            }
        }
    }
    // What fetch started, into LDS (a barrier follows).
    template <bool VALUES>
    __device__ static void land(const Side& s, uint8_t* lds, uint32_t t) {
        if constexpr (CT == PKV_FP8) {
            const uint32_t row = code_slot(t), b = t % 4;
            for (int w = 0; w < D / 32; ++w) {
                const uint32_t lo = s.codes[w / 2][w % 2 * 2], hi = s.codes[w / 2][w % 2 * 2 + 1], piece = b * (D / 32) + w;
                *reinterpret_cast<u32x4*>(lds + (VALUES ? value_at(row, piece) : key_at(row, piece))) =
                    expand8(lo, hi, block_scale(s.scale));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else {
            copies_done();
        }
    }
    // Infinities and NaN among a staged tile's values to 0, by the group's 256 threads; true if this one had any.
    __device__ static bool clean(uint8_t* lds, uint32_t t) {
        bool odd = false;
        for (uint32_t x = t; x < kKeyBytes / 16; x += 256) {
            u32x4* p = reinterpret_cast<u32x4*>(lds + kKeyBytes) + x;
            u32x4 w = *p;
            bool any = false;
            for (int y = 0; y < 4; ++y) {
                const uint32_t z = w[y];
                any |= nonfinite2<mat_type(CT)>(z);
                w[y] = finite_or_0<mat_type(CT)>(z);
            }
            if (any) *p = w;
            odd |= any;
        }
        return odd;
    }
};

// copy_to_lds among products, free to pass LDS reads: between two meetings
// nothing reads what a copy overwrites.
__device__ inline void start_copy(uint32_t to, const uint8_t* from, uint32_t offset) {
    uint32_t m0;
    to = __builtin_amdgcn_readfirstlane(to);
    from = uniform(from);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "s"(to), "v"(offset), "s"(from));
}

// The waves of a workgroup meet; nothing moves across, no copy is waited for.
__device__ inline void meet() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Rows in tiles of 256 (KS 1), 32 a wave, against tiles of 64 slots staged
// through LDS in two buffers:
//   S^T = K Q^T (32x32 tiles; a lane holds one query row and half of each
//   piece's slots), softmax in registers, O^T += V^T P^T with the rounded
//   weights straight from those registers.
// The workgroup's waves are two groups of four, one of each on a SIMD, that take
// turns: while one has the matrix cores, O of the tile before and S of the next,
// the other has the vector units for its softmax, and they meet between.  For
// prompts of 8,192, 5,920 and 4,278 rows of 32 query heads of 128 that takes 841
// to 905 us, card by card (1,170 to 1,090 TFLOP/s; 1,250 for one of 16,384 rows; a
// library's square product reaches 1,330): the matrix cores are busy 62 % of the cycles, the tiles' LDS
// reads conflict in 0.1 %, and a workgroup's start and end, 9 us that nothing
// hides since one fills a CU's registers, take most of the rest.  Two workgroups
// of four waves each, which meet nobody, took 1,023 (matrix cores 44 %, vector
// units 47 %, one after the other); the turns alone made it 910, and copies by
// both groups among the products, with the largest logit looked for only where
// the weights' sums pass what one may be, the rest.
// Weights are rounded once to the type of the products (f16 queries over 8-bit
// codes: two bf16 terms), while their sum is that of the unrounded ones.
// KS 2, 4: 128, 64 rows; the groups take the slots' tiles in turn, at 4 also two
// waves of a group the halves of a tile, for calls whose larger row tiles would
// not fill the chip.
//
// A weight 0 times an infinity or NaN would be NaN in rows that do not see the
// slot.  The loop does not look for those: an output that is not finite sends
// the workgroup through it again, with infinities and NaN taken out of the
// staged values and each added afterwards to the rows that see it.  Where the
// sums of finite values are not finite either, a third time with smaller
// weights (kDown).
constexpr int rows_of_tile(int ks) { return 256 / ks; }

// The order of V operands of two reads and K operands of one, PRODUCTS products
// each, in pairs: the reads run kAhead operands ahead of the products (left to
// itself the compiler reads an operand, waits for it and multiplies).
constexpr int kAhead = 4;
constexpr int reads_of(int v, int k, int from, int to) {
    int n = 0;
    for (int i = from; i < (to < v + k ? to : v + k); ++i) n += i < v ? 2 : 1;
    return n;
}
template <int V, int K, int PRODUCTS, int AT = -kAhead>
__device__ inline void reads_ahead() {
    static_assert((V + K) % 2 == 0 && kAhead % 2 == 0, "pairs of operands");
    constexpr int reads = reads_of(V, K, AT < 0 ? 0 : AT + kAhead, AT < 0 ? kAhead : AT + kAhead + 2);
    if constexpr (AT >= 0) __builtin_amdgcn_sched_group_barrier(0x008, 2 * PRODUCTS, 0);
    if constexpr (reads > 0) __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
    constexpr int next = AT < 0 ? 0 : AT + 2;
    if constexpr (next < V + K) reads_ahead<V, K, PRODUCTS, next>();
}
template <int CT, int QT, int D, bool PAGED, int KS>
__global__ __launch_bounds__(512, 2) void rows_kernel(PagedDev a, PagedPart part, int few) {
    using T = typename Elem<QT>::T;
    using St = PageStage<CT, D, PAGED>;
    constexpr int MT = mat_type(CT), kU = KS == 4 ? 1 : 2, kO = D / 32;   // kU: 32-slot pieces a wave takes of a tile
    constexpr int NP = query_terms(CT, QT), kRowTile = rows_of_tile(KS);
    constexpr bool kTurns = KS > 1;                               // a group has tiles of its own
    constexpr int kRing = kTurns ? 2 : 3;                         // tiles in LDS, of a group or of both: keys, then values
    __shared__ __align__(16) uint8_t lds[(kTurns ? 2 : 1) * kRing * St::kBytes];
    const uint32_t work_blocks = a.heads * part.units;
    if (blockIdx.x >= work_blocks) return clear_rows<QT, D, 512>(a, blockIdx.x - work_blocks);
    const uint32_t lane = threadIdx.x % 64, wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = lane % 32, half = lane / 32, group = wave_id / 4, gt = threadIdx.x % 256;
    const uint32_t wave = KS == 1 ? wave_id : wave_id % (8 / KS);         // its 32 rows
    const int share = KS == 4 ? static_cast<int>(wave_id / 2 % 2) * 32 : 0;   // its slots of a tile: share .. + 32 kU
    // heads fastest, so that a head's workgroups share an XCD's L2 where the heads are a multiple of 8
    const uint32_t h = blockIdx.x % a.heads;
    RowUnit rt;
    const uint32_t u = blockIdx.x / a.heads;
    if (!(part.counted ? look_up_rows(a, part.plan, part.ends, u, few, kRowTile, lane, &rt)
                       : find_rows(a, u, few, kRowTile, part.target, lane, &rt)))
        return;
    rt = {__builtin_amdgcn_readfirstlane(rt.seq), __builtin_amdgcn_readfirstlane(rt.tile),
          __builtin_amdgcn_readfirstlane(rt.share), __builtin_amdgcn_readfirstlane(rt.shares),
          __builtin_amdgcn_readfirstlane(rt.part)};
    if (part.target && h == 0 && rt.tile == 0 && rt.share == 0 && threadIdx.x == 0 && !part.counted) {
        part.plan[2 * rt.seq] = rt.part;
        part.plan[2 * rt.seq + 1] = rt.shares;
    }
    const Seq sq = seq_of_all(a.seq, rt.seq, a.max_rows);
    const int R = sq.rows * static_cast<int>(a.group), r0 = rt.tile * kRowTile, G = static_cast<int>(a.group);
    const int last = min(r0 + kRowTile, R) - 1;
    const int pos0 = sq.first + __builtin_amdgcn_readfirstlane(r0 / G), pos1 = sq.first + __builtin_amdgcn_readfirstlane(last / G);
    const Tiles tl = uniform(tiles_of(a, pos0, pos1, St::kSlots));
    const int per = __builtin_amdgcn_readfirstlane((tl.count + rt.shares - 1) / rt.shares);
    const int t0 = rt.share * per, t1 = min(t0 + per, tl.count);
    // the group's tiles: t0 + first, + step, ..; as many steps for both
    constexpr int kEvery = kTurns ? 2 : 1;
    const int first = t0 + (kTurns ? static_cast<int>(group) : 0), steps = max(t1 - t0 + kEvery - 1, 0) / kEvery;
    auto tile = [&](int i) { return first + kEvery * i; };
    auto slot_of = [&](int i) { return tl.slot(tile(i), St::kSlots); };

    const int w0 = r0 + 32 * static_cast<int>(wave), w1 = min(w0 + 31, last), r = w0 + static_cast<int>(n);
    const bool real = r <= last;
    const int qi = (real ? r : last) / G, pos = real ? sq.first + qi : -1;
    // of the wave's rows (w0 > last: none)
    const int wpos0 = sq.first + __builtin_amdgcn_readfirstlane(w0 / G), wpos1 = sq.first + __builtin_amdgcn_readfirstlane(w1 / G);
    const Tiles wt = uniform(tiles_of(a, wpos0, w0 <= last ? wpos1 : -1, 1));
    Query<CT, QT, D> q;
    q.load(reinterpret_cast<const T*>(a.q) + static_cast<uint64_t>(sq.row0 + qi) * a.q_row +
               (h * a.group + (real ? r : last) % G) * a.q_head,
           real, half);

    const uint64_t head = h * a.k_head;
    const int32_t* table = PAGED ? a.seq.tables + rt.seq * a.seq.table : nullptr;
    const uint8_t* kp = PAGED ? nullptr : a.k + 2 * (static_cast<uint64_t>(sq.row0) * a.k_slot + head);
    const uint8_t* vp = PAGED ? nullptr : a.v + 2 * (static_cast<uint64_t>(sq.row0) * a.v_slot + h * a.v_head);

    uint8_t* const mine = lds + (kTurns ? group * kRing * St::kBytes : 0);
    // the keys and values that a group brings: of tiles of its own both
    const bool keys_mine = kTurns || group == 0, values_mine = kTurns || group == 1;
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte*)mine)), w4 = wave_id % 4;
    // places of the ring (the values' count from kKeyBytes before them)
    auto key_place = [](int ring) { return static_cast<uint32_t>(ring) * St::kKeyBytes; };
    auto value_place = [](int ring) { return static_cast<uint32_t>(kRing - 1 + ring) * St::kKeyBytes; };
    auto behind = [](int ring) { return ring + 1 == kRing ? 0 : ring + 1; };
    auto before = [](int ring) { return ring ? ring - 1 : kRing - 1; };
    float base = kInf, l = 0.0f;
    f32x16 o[kO], sc[kU];
    u32x4 pt[NP][2 * kU];
    typename St::Side ks, vs;
    const typename St::Copies kc = St::template copies<false>(a, gt), vc = St::template copies<true>(a, gt);
    // LDS addresses of the lane's operands in the first place: keys of slot n, values as Staged::values16 reads them
    constexpr int kX = D / 16;
    uint32_t key_read[kX], value_read[kO][2];
    for (int x = 0; x < kX; ++x) key_read[x] = at + share * St::kRow + St::key_at(n, 2 * x + half);
    for (int e = 0; e < kO; ++e)
        for (int y = 0; y < 2; ++y) {
            const uint32_t s = lane % 16, row = lane / 32 * 4 + s / 4 + 8 * y;
            value_read[e][y] = at + share * St::kRow + value_place(0) +
                               St::value_at(row, 4 * e + lane / 16 % 2 * 2 + s % 4 / 2) + s % 2 * 8;
        }
    // the words of step i's pages (past the last tile: the last's again, unused)
    auto pages = [&](int i) {
        if constexpr (!PAGED) return 0;
        else return read_pages<4>(a.seq, table, tl.slot(min(tile(i), t1 - 1), St::kSlots), tl.high - 1, lane);
    };
    auto there = [&](int i) { return tile(i) < t1; };
    auto fetch_keys = [&](int i, int ring, int words) {
        if (keys_mine && there(i))
            St::template fetch<false>(ks, kc, a, at + key_place(ring), kp, head, words, slot_of(i), tl.high - 1, gt);
    };
    auto fetch_values = [&](int i, int ring, int words) {
        if (values_mine && there(i))
            St::template fetch<true>(vs, vc, a, at + value_place(ring), vp, head, words, slot_of(i), tl.high - 1, gt);
    };
    auto land_keys = [&](int i, int ring) {
        if (keys_mine && there(i)) St::template land<false>(ks, mine + key_place(ring), gt);
    };
    auto land_values = [&](int i, int ring) {
        if (values_mine && there(i)) St::template land<true>(vs, mine + value_place(ring), gt);
    };
    // some row of the wave sees some of step i's tile
    auto sees = [&](int i) {
        if (!there(i)) return false;
        const int slot = slot_of(i) + share;
        return slot < wt.high && (slot + 32 * kU > wt.low || static_cast<uint32_t>(slot) < a.sinks);
    };
    float lift = kLift<MT>;
    // logits that the rows do not see to -inf; none: 16-slot pieces of the tile on no page
    auto hide = [&](int i) __attribute__((always_inline)) {
        const int slot = slot_of(i) + share;
        if (all_visible(a, wpos0, wpos1, slot, slot + 32 * kU - 1)) return;
        const int off = pos - slot - 4 * static_cast<int>(half);   // less the register's place: how far back
        if (static_cast<uint32_t>(slot) >= a.sinks) {
            for (int p = 0; p < kU; ++p)
                for (int x = 0; x < 16; ++x)
                    if (!in_reach(a, off, 32 * p + row32(x, 0))) sc[p][x] = -kInf;
        } else {
            for (int p = 0; p < kU; ++p)
                for (int x = 0; x < 16; ++x)
                    if (!visible(a, pos, slot + 32 * p + row32(x, half))) sc[p][x] = -kInf;
        }
    };
    auto hide_missing = [&](uint32_t none) __attribute__((always_inline)) {
        if (PAGED && none)
            for (int p = 0; p < kU; ++p)
                for (int x = 0; x < 16; ++x)
                    if (none >> (share / 16 + 2 * p + x / 8) & 1) sc[p][x] = -kInf;
    };
    // the base lowered by the largest of the logits
    auto lower = [&]() __attribute__((always_inline)) {
        float top = sc[0][0];
        for (int p = 0; p < kU; ++p)
            for (int x = 0; x < 16; ++x) top = fmaxf(top, sc[p][x]);
        top = across32(top, larger);
        if (__any(__builtin_fmaf(top, a.scale2, base) > lift + kLag<MT>)) {
            const float low = lower_base(a, lift, base, top), f = joined(low, base);
            if (low < base) {
                l *= f;
                for (int e = 0; e < kO; ++e) o[e] *= f;
                base = low;
            }
        }
    };
    // weights in the logits' place, and their sums: no weight is above its piece's
    auto weights = [&](float (&sum)[kU]) __attribute__((always_inline)) {
        const float from = base == kInf ? 0.0f : base;
        for (int p = 0; p < kU; ++p) {
            sum[p] = 0.0f;
            for (int x = 0; x < 16; ++x) {
                sc[p][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[p][x], a.scale2, from));
                sum[p] += sc[p][x];
            }
        }
    };
    auto pack = [&](const float (&sum)[kU]) __attribute__((always_inline)) {
        for (int p = 0; p < kU; ++p) {
            l += sum[p];
            for (int y = 0; y < 2; ++y) {
                float w[8];
                for (int x = 0; x < 8; ++x) w[x] = sc[p][8 * y + x];
                for (int k = 0; k < NP; ++k)
                    pt[k][2 * p + y] = u32x4{pack_term<MT>(w[0], w[1]), pack_term<MT>(w[2], w[3]),
                                             pack_term<MT>(w[4], w[5]), pack_term<MT>(w[6], w[7])};
            }
        }
    };
    auto softmax = [&](int i, uint32_t none) __attribute__((always_inline)) {
        float sum[kU];
        hide(i);
        hide_missing(none);
        lower();
        weights(sum);
        pack(sum);
    };
    // O += the values of the tile at `values` weighed, S = the logits of the one at `keys`; among the products copy(0),
    // copy(1), .. start what is copied meanwhile.
    auto products = [&](auto weighs, auto scores, uint32_t values, uint32_t keys, auto copy) __attribute__((always_inline)) {
        constexpr bool W = decltype(weighs)::value, S = decltype(scores)::value;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* Values;
        typedef const __attribute__((address_space(3))) u32x4* Keys;
        int next = 0;
        if constexpr (W) {
            for (int y = 0; y < 2 * kU; ++y) {
                for (int e = 0; e < kO; ++e) {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Values)(value_read[e][0] + (values + 16 * y * St::kRow)));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Values)(value_read[e][1] + (values + 16 * y * St::kRow)));
                    const u32x2 v0 = __builtin_bit_cast(u32x2, lo), v1 = __builtin_bit_cast(u32x2, hi);
                    for (int k = NP - 1; k >= 0; --k) o[e] = mma32<MT>(u32x4{v0[0], v0[1], v1[0], v1[1]}, pt[k][y], o[e]);
                }
                copy(next++);
            }
        }
        if constexpr (S) {
            for (int p = 0; p < kU; ++p) sc[p] = f32x16{};
            for (int x = 0; x < kX; ++x) {
                for (int p = 0; p < kU; ++p) {
                    const u32x4 k = *(Keys)(key_read[x] + (keys + 32 * p * St::kRow));
                    for (int y = NP - 1; y >= 0; --y) sc[p] = mma32<MT>(k, q.q[y][x], sc[p]);
                }
                if (kU == 1 || x % 2) copy(next++);
            }
        }
        reads_ahead<W ? 2 * kU * kO : 0, S ? kU * kX : 0, NP>();
    };
    using Yes = std::true_type;
    using No = std::false_type;
    auto no_copy = [](int) {};
    static_assert(2 * kU + kX / (kU == 1 ? 1 : 2) >= (kTurns ? 2 : 1) * St::kCopies, "every copy has its place");

    // Step i of a group, its tile at place `ring`: values of i - 1 and logits of i; meet; softmax of i; meet.  The second
    // group is a meeting behind.  From the products to the end of the softmax keys of i + 1 are on their way, and values of
    // i; of shared tiles the first group brings the keys, the second values of i + 1.  What a copy overwrites was last
    // read in front of the last meeting: keys of i - 1 (shared: i - 2), values of i - 2.
    int words = 0, next = 0;
    bool have = false;           // weights of the step before
    auto step = [&](int i, int ring) __attribute__((always_inline)) {
        const uint32_t none = PAGED ? no_page<4>(a.seq, words) : 0;
        const bool now = sees(i);
        fetch_keys(i + 1, behind(ring), next);
        if (kTurns) fetch_values(i, ring, words);
        else fetch_values(i + 1, behind(ring), next);
        __builtin_amdgcn_s_setprio(1);
        if (have) products(Yes(), No(), before(ring) * St::kKeyBytes, 0, no_copy);
        if (now) products(No(), Yes(), 0, key_place(ring), no_copy);
        have = now;
        __builtin_amdgcn_s_setprio(0);
        meet();
        const int ahead = pages(i + 2);
        if (have) softmax(i, none);
        land_keys(i + 1, behind(ring));
        if (kTurns) land_values(i, ring);
        else land_values(i + 1, behind(ring));
        words = next;
        next = ahead;
        meet();
    };
    // The same for a step in the middle: its tile and the next are whole, every row of the wave sees all of it and of the
    // one before, and its place is known.
    auto middle = [&](int i, auto place) __attribute__((always_inline)) {
        constexpr int kHere = decltype(place)::value, kNext = (kHere + 1) % kRing, kBefore = (kHere + kRing - 1) % kRing;
        const uint32_t none = PAGED ? no_page<4>(a.seq, words) : 0;
        const int slot = slot_of(i);
        if constexpr (CT == PKV_FP8) {
            fetch_keys(i + 1, kNext, next);
            if (kTurns) fetch_values(i, kHere, words);
            else fetch_values(i + 1, kNext, next);
        }
        // of shared tiles a group's side of the next one
        const typename St::Copies& c = !kTurns && group ? vc : kc;
        const uint32_t to = at + c.to + (!kTurns && group ? (kRing - 1 + kNext) * St::kKeyBytes : kNext * St::kKeyBytes);
        __builtin_amdgcn_s_setprio(1);
        products(Yes(), Yes(), kBefore * St::kKeyBytes, kHere * St::kKeyBytes, [&](int x) __attribute__((always_inline)) {
            if constexpr (CT != PKV_FP8) {
                const int y = x % St::kCopies;
                if (x < St::kCopies)
                    start_copy(to + y * St::kCopyStep * St::kRow,
                               St::copy_from(a, !kTurns && group ? a.v : a.k, !kTurns && group ? vp : kp, head, next,
                                             slot + kEvery * St::kSlots, tl.high - 1, c.stride, y, w4), c.off);
                else if (kTurns && x < 2 * St::kCopies)
                    start_copy(at + vc.to + (kRing - 1 + kHere) * St::kKeyBytes + y * St::kCopyStep * St::kRow,
                               St::copy_from(a, a.v, vp, head, words, slot, tl.high - 1, vc.stride, y, w4), vc.off);
            }
        });
        __builtin_amdgcn_s_setprio(0);
        meet();
        const int ahead = pages(i + 2);
        // weights by the base as it is; where their sums pass what one weight may be, from the logits again
        float sum[kU];
        hide_missing(none);
        weights(sum);
        constexpr float kMost = kPower<static_cast<int>(kLift<MT> + kLag<MT>)>;
        if (__builtin_expect(__any(!(sum[0] <= kMost && sum[kU - 1] <= kMost) || base == kInf), 0)) {
            products(No(), Yes(), 0, kHere * St::kKeyBytes, no_copy);
            hide_missing(none);
            lower();
            weights(sum);
        }
        pack(sum);
        land_keys(i + 1, kNext);
        if (kTurns) land_values(i, kHere);
        else land_values(i + 1, kNext);
        words = next;
        next = ahead;
        meet();
    };
    for (int e = 0; e < kO; ++e) o[e] = f32x16{};
    if (steps > 0) {
        // middle steps, as many at a time as there are places: tiles of the list whose slots all rows see, the one before
        // too, and whose next one is whole and there
        const int list = tl.second - tl.first;     // tile t of the list, behind the first ones, starts at slot 64 (t + list)
        int lo = tl.first, hi = min((wpos0 + 1) / St::kSlots, tl.high / St::kSlots - kEvery) - list;
        if (a.window)
            lo = max(lo, static_cast<int>(max(static_cast<int64_t>(pos1) - a.reach + St::kSlots, static_cast<int64_t>(0)) /
                                          St::kSlots) - list);
        hi = min(hi, t1 - kEvery);
        const int from = __builtin_amdgcn_readfirstlane(max(lo - first + kEvery - 1, 0) / kEvery + 1);
        const int middles = __builtin_amdgcn_readfirstlane(
            w0 <= last && wpos0 >= 0 ? max(hi - first + kEvery - 1, 0) / kEvery - from : 0);   // may be negative
        int i = 0, ring = (kRing - from % kRing) % kRing;      // the first of the middle in the first place
        words = pages(0);
        next = pages(1);
        fetch_keys(0, ring, words);
        land_keys(0, ring);
        if (!kTurns) {
            fetch_values(0, ring, words);
            land_values(0, ring);
        }
        // the query is there: else the compiler waits for it at its every use, and for the copies under way with it
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
        meet();
        if (group) meet();
        auto steps_to = [&](int end) {
            for (; i < end; ++i) {
                step(i, ring);
                ring = behind(ring);
            }
        };
        steps_to(min(from, steps));
        if (middles >= kRing)
            for (const int to = from + middles / kRing * kRing; i < to; i += kRing) {
                middle(i, std::integral_constant<int, 0>());
                middle(i + 1, std::integral_constant<int, 1>());
                if constexpr (kRing == 3) middle(i + 2, std::integral_constant<int, 2>());
            }
        steps_to(steps);
        if (have) products(Yes(), No(), before(ring) * St::kKeyBytes, 0, no_copy);
        if (!group) meet();
    }
    bool odd = false;
    for (int e = 0; e < kO; ++e)
        for (int x = 0; x < 16; ++x) odd |= (__float_as_uint(o[e][x]) & 0x7f800000u) == 0x7f800000u;
    if (__builtin_expect(__syncthreads_or(odd && real), 0)) {
        // both sides of step i's tile in the first place, by all
        auto stage = [&](int i, int words) {
            __syncthreads();
            fetch_keys(i, 0, words);
            fetch_values(i, 0, words);
            land_keys(i, 0);
            land_values(i, 0);
            __syncthreads();
        };
        auto cleaned = [&](int i) { return keys_mine && there(i) && St::clean(mine + value_place(0), gt); };
        for (int pass = 1; pass < 3; ++pass) {
            base = kInf;
            l = 0.0f;
            for (int e = 0; e < kO; ++e) o[e] = f32x16{};
#pragma unroll 1
            for (int i = 0; i < steps; ++i) {
                const int words = pages(i);
                stage(i, words);
                cleaned(i);
                __syncthreads();
                if (sees(i)) {
                    products(No(), Yes(), 0, 0, no_copy);
                    softmax(i, PAGED ? no_page<4>(a.seq, words) : 0);
                    products(Yes(), No(), 0, 0, no_copy);
                }
            }
            odd = false;
            for (int e = 0; e < kO; ++e)
                for (int x = 0; x < 16; ++x) odd |= (__float_as_uint(o[e][x]) & 0x7f800000u) == 0x7f800000u;
            // with the values finite, from a NaN among the logits, as the weights' sum, or past the type's end
            odd &= !__builtin_isnan(across32(l, [](float x, float y) { return x + y; }));
            if (!kDown<MT> || pass == 2 || !__syncthreads_or(odd && real)) break;
            lift -= kDown<MT>;
        }
        // not scaled down: that could make a weight 0
        const float from = base == kInf ? 0.0f : base + (kLift<MT> - lift);
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {
            const int words = pages(i);
            const uint32_t none = PAGED ? no_page<4>(a.seq, words) : 0;
            stage(i, words);
            if (!__syncthreads_or(cleaned(i))) continue;
            stage(i, words);
            if (!there(i)) continue;
#pragma unroll 1
            for (int j = share; j < share + 32 * kU; ++j) {
                const bool see = visible(a, pos, slot_of(i) + j) && !(none >> j / 16 & 1);
                if (!__any(see)) continue;
                uint32_t hf = half;
                asm volatile("" : "+v"(hf));   // this rare loop's addresses are not kept over the main one
                float dot = 0.0f;
                for (int x = 0; x < Query<CT, QT, D>::kRegs; ++x) {
                    const u32x4 k = *reinterpret_cast<const u32x4*>(mine + St::key_at(j, 2 * x + hf));
                    for (int w = 0; w < 4; ++w)
                        for (int y = 0; y < Query<CT, QT, D>::kTerms; ++y) {
                            const uint32_t kw = k[w], qw = q.q[y][x][w];
                            dot += dot_word<MT>(kw, qw);
                        }
                }
                dot += __shfl_xor(dot, 32);
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(dot, a.scale2, from));
                for (int e = 0; e < kO; ++e)
                    for (int x = 0; x < 16; ++x) {
                        const float v = St::value(mine + value_place(0), j, 32 * e + row32(x, hf));
                        if (see && (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[e][x] += p * v;
                    }
            }
        }
        __syncthreads();
    }
    l += __shfl_xor(l, 32);
    constexpr int kShared = KS == 1 ? 0 : KS == 2 ? 1 : 2;   // outputs are 2^-kShared as large from here on
    if constexpr (KS > 1) {
        // the other shares of the slots join the first: [share][row block][o, base, l][lane]
        constexpr int kBlocks = 8 / KS, kBlock = (16 * kO + 2) * 64;
        float* to = reinterpret_cast<float*>(lds) + wave * kBlock + lane;
        const uint32_t part_of = wave_id / kBlocks;
        __syncthreads();
        if (part_of) {
            float* x = to + (part_of - 1) * kBlocks * kBlock;
            for (int e = 0; e < 16 * kO; ++e) x[e * 64] = o[e / 16][e % 16];
            x[16 * kO * 64] = base;
            x[(16 * kO + 1) * 64] = l;
        }
        __syncthreads();
        if (part_of) return;
        float low = base;
        for (int s = 0; s < KS - 1; ++s) low = fminf(low, to[s * kBlocks * kBlock + 16 * kO * 64]);
        const float f = joined(low, base);
        l *= f;
        for (int e = 0; e < kO; ++e) o[e] *= f * kPower<-kShared>;
        for (int s = 0; s < KS - 1; ++s) {
            const float* x = to + s * kBlocks * kBlock;
            const float f2 = joined(low, x[16 * kO * 64]);
            l += x[(16 * kO + 1) * 64] * f2;
            for (int e = 0; e < 16 * kO; ++e) o[e / 16][e % 16] += x[e * 64] * (f2 * kPower<-kShared>);
        }
        base = low;
    }
    if (rt.shares > 1) {
        if (!real) return;
        const uint64_t to = (static_cast<uint64_t>(h) * part.parts + rt.part + rt.share) * kRowTile + (r - r0);
        for (int e = 0; e < kO; ++e)
            for (int x = 0; x < 4; ++x)
                *reinterpret_cast<f32x4*>(part.o + to * D + 32 * e + 8 * x + 4 * half) =
                    f32x4{o[e][4 * x], o[e][4 * x + 1], o[e][4 * x + 2], o[e][4 * x + 3]} * kPower<kShared - kPartDown>;
        if (half == 0) {
            part.ml[2 * to] = base;
            part.ml[2 * to + 1] = l;
        }
        return;
    }
    // through LDS, so that rows are written whole: the wave's 32 rows in 16-byte pieces at piece ^ row
    constexpr int kPieces = D / 8;
    uint8_t* mine_out = lds + (KS == 1 ? 32 * 2 * D : (16 * kO + 2) * 256) * wave;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l * kPower<kShared>;
    const uint32_t qh = h * a.group + static_cast<uint32_t>((real ? r : last) % G);
    for (int e = 0; e < kO; ++e)
        for (int x = 0; x < 4; ++x) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 y;
            for (int k = 0; k < 4; ++k) y[k] = static_cast<T>(l == 0.0f ? 0.0f : o[e][4 * x + k] * inv);
            *reinterpret_cast<T4*>(mine_out + n * 2 * D + ((4 * e + x) ^ n % kPieces) * 16 + half * 8) = y;
        }
    const uint64_t to = static_cast<uint64_t>(sq.row0 + qi) * a.o_row + qh * a.o_head;
    for (int x = 0; x < kPieces / 2; ++x) {
        const uint32_t row = x * (64 / kPieces) + lane / kPieces, piece = lane % kPieces;
        const u32x4 y = *reinterpret_cast<const u32x4*>(mine_out + row * 2 * D + (piece ^ row % kPieces) * 16);
        const uint64_t where = __shfl(static_cast<unsigned long long>(to), static_cast<int>(row));
        if (w0 + static_cast<int>(row) <= last)
            *reinterpret_cast<u32x4*>(reinterpret_cast<T*>(a.out) + where + 8 * piece) = y;
    }
    if (real && half == 0 && a.lse) a.lse[static_cast<uint64_t>(qh) * a.seq.rows + sq.row0 + qi] = lse_of(base, l);
}

// rows_kernel's shares joined: 16 rows a workgroup, 16 lanes a row, which read its
// shares' bases and sums at once and D / 16 channels each.  A row's chain of reads
// (its sequence, the plan, the bases, the outputs) is what bounds this, so that
// four rows a wave side by side are what counts (11,200 rows of 8 heads of 128:
// 23.7 us with a wave a row, one row after the other).
constexpr uint32_t kJoinRows = 16;
template <int QT, int D>
__global__ __launch_bounds__(256) void join_rows_kernel(PagedDev a, PagedPart part, int few) {
    using T = typename Elem<QT>::T;
    constexpr int V = D / 16;
    typedef T Out __attribute__((ext_vector_type(V)));
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 16;
    const uint32_t all = a.seq.rows * a.group, h = blockIdx.x % a.heads, b = blockIdx.x / a.heads * kJoinRows + 4 * wave;
    int s = -1, mine = -1;
    Seq q{}, sq{};
    for (uint32_t y = 0; y < 4 && b + y < all; ++y) {   // rows of one sequence but where it ends
        const int row = static_cast<int>((b + y) / a.group);
        if (s < 0 || row >= q.row0 + q.rows) {
            s = __builtin_amdgcn_readfirstlane(seq_of_row(a.seq, row, lane));
            if (s >= 0) q = seq_of_all(a.seq, s, a.max_rows);
        }
        if (lane / 16 == y) { mine = s; sq = q; }
    }
    const uint32_t x = b + lane / 16;
    const int row = static_cast<int>(x / a.group);
    int shares = 0;
    uint64_t at = 0;
    if (mine >= 0 && row < sq.row0 + sq.rows && static_cast<int64_t>(sq.rows) * a.group > few) {
        const int r = (row - sq.row0) * static_cast<int>(a.group) + static_cast<int>(x % a.group);
        const int first = part.plan[2 * mine], n = part.plan[2 * mine + 1], tile = r / static_cast<int>(part.rows);
        // starts that do not ascend may have more units than the launch, and no plan for the last
        if (n > 1 && first >= 0 && first + (tile + 1ll) * n <= static_cast<int64_t>(part.parts)) {
            shares = n;
            at = (static_cast<uint64_t>(h) * part.parts + first + static_cast<uint64_t>(tile) * n) * part.rows +
                 static_cast<uint64_t>(r - tile * static_cast<int>(part.rows));
        }
    }
    if (!__any(shares)) return;
    const float* ml = part.ml + 2 * at;
    const uint64_t step = 2ull * part.rows;
    float low = kInf;
    for (int y = static_cast<int>(i); y < shares; y += 16) low = fminf(low, ml[step * y]);
    for (int o = 8; o; o >>= 1) low = fminf(low, __shfl_xor(low, o));
    float sum = 0.0f;
    f32x4 acc[V / 4] = {};
    for (int c = 0; c < shares; c += 16) {
        const int y = c + static_cast<int>(i), n = min(16, shares - c);
        const float f = y < shares ? joined(low, ml[step * y]) : 0.0f;
        if (y < shares) sum += ml[step * y + 1] * f;
        for (int k = 0; k < n; ++k) {
            const float w = __shfl(f, static_cast<int>(lane / 16 * 16) + k) * kPower<-kJoinDown>;
            const float* from = part.o + (at + static_cast<uint64_t>(part.rows) * (c + k)) * D + V * i;
            for (int e = 0; e < V / 4; ++e) acc[e] += reinterpret_cast<const f32x4*>(from)[e] * w;
        }
    }
    for (int o = 8; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (!shares) return;
    const uint32_t qh = h * a.group + x % a.group;
    const float div = sum * kPower<-kPartDown - kJoinDown>;
    Out y;
    for (int e = 0; e < V; ++e) y[e] = static_cast<T>(sum == 0.0f ? 0.0f : acc[e / 4][e % 4] / div);
    *reinterpret_cast<Out*>(reinterpret_cast<T*>(a.out) + static_cast<uint64_t>(row) * a.o_row + qh * a.o_head + V * i) = y;
    if (i == 0 && a.lse) a.lse[static_cast<uint64_t>(qh) * a.seq.rows + row] = lse_of(low, sum);
}

uint32_t clears(const PagedDev& a) { return a.clear && a.seq.starts ? kClear : 0; }

uint64_t round256(uint64_t x) { return (x + 255) & ~255ull; }

// The launches of a call and its workspace.
struct Plan {
    bool few, many;                // sequences of few rows are looked for; of more
    bool wide;                     // decode_kernel: whole sequences, more waves each
    uint32_t units, target, most, rows;   // units a head at most, aimed at (most: if long), rows of one
    uint64_t ml, plan;             // offsets in the workspace (partial outputs first)
    int ks;                        // rows_kernel: 256 / ks rows a tile
    uint32_t row_units, row_target, parts;   // units a head at most, shares aimed at (0: none), room for
    uint64_t rows_ml, rows_plan, bytes;      // the two kernels follow each other in the same workspace; all of it
    bool counted;                  // by the plan kernels
};
Plan plan_of(const PagedDev& a, uint32_t dim, int cache_dtype) {
    Plan p{};
    const uint64_t most = static_cast<uint64_t>(a.max_rows) * a.group;
    p.few = a.seq.paged && (!a.seq.each || most <= kFew);
    p.many = !a.seq.paged || most > kFew;
    p.counted = a.seq.seqs > kCounted;
    // tiles of `step` slots that `rows` rows can see: all, or the window, the rows before the last and the sinks, rounded
    // to tiles apart
    auto tiles_for = [&](uint64_t rows, uint64_t step) {
        uint64_t slots = a.seq.max_len;
        if (a.window)
            slots = std::min<uint64_t>(slots, static_cast<uint64_t>(a.window) + std::min<uint64_t>(a.max_rows, rows) +
                                                  a.sinks + 4 * step);
        return (slots + step - 1) / step;
    };
    if (p.few) {
        p.rows = static_cast<uint32_t>(std::min<uint64_t>(kFew, most));
        // what fits at once, less half a unit a sequence for those that are not whole
        auto aim = [&](uint32_t all) {
            const uint32_t fit = all / a.heads;
            return std::max(fit > a.seq.seqs / 2 ? fit - a.seq.seqs / 2 : 1, std::max(fit / 4, 1u));
        };
        p.target = aim(fitting_units(dim, cache_dtype));
        const uint64_t tiles = tiles_for(kFew, kStep);
        p.wide = static_cast<uint64_t>(a.seq.seqs) * a.heads <= 256 && tiles <= 4ull * wide_waves(dim, cache_dtype);
        if (p.wide) p.target = 1;
        p.most = p.wide ? 1 : std::max(p.target, aim(kMostUnits));
        if (tiles * a.seq.seqs < static_cast<uint64_t>(kMany) * p.most) p.most = p.target;   // never as long
        const uint64_t each = p.wide ? 1 : std::max<uint64_t>(1, (tiles + kLeast - 1) / kLeast);
        p.units = static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(a.seq.seqs) + p.most, a.seq.seqs * each));
        const uint64_t rows = static_cast<uint64_t>(a.heads) * p.units * p.rows;
        p.ml = round256(rows * dim * 4);
        p.plan = p.ml + round256(rows * 8);
        p.bytes = p.plan + round256(8ull * a.seq.seqs);
    }
    if (p.many) {
        // The least time, in tenths of a step of shared tiles (KS 1; 2 and 4 take two tiles a step): the steps of a CU's
        // workgroups, one after the other, and about six steps' time for the start and end of each.
        uint64_t least = ~0ull, tiles = 0;
        for (int ks = 1; ks <= 4; ks *= 2) {
            const uint64_t rt = rows_of_tile(ks);
            const uint64_t n = std::min((static_cast<uint64_t>(a.seq.rows) * a.group + rt - 1) / rt + a.seq.seqs,
                                        a.seq.seqs * ((most + rt - 1) / rt));
            const uint64_t steps = (tiles_for(rt, 64) + (ks > 1 ? 1 : 0)) / (ks > 1 ? 2 : 1);
            const uint64_t rounds = (a.heads * n + 255) / 256;
            const uint64_t cost = rounds * (steps + 6) * (ks == 4 ? 8 : ks == 2 ? 12 : 10);
            if (cost < least) {
                least = cost;
                p.ks = ks;
                tiles = n;
            }
        }
        // Shares, where a call has less than three row tiles a CU: of a CU's work and more, of half of that where there
        // are more tiles than CUs (20 sequences of 600 to 6,000 slots with chunks of up to 512 rows: 267 us without).
        const uint64_t groups = a.heads * tiles;
        p.row_target = groups < 768 && tiles_for(rows_of_tile(p.ks), 64) >= 2 * kLeastSteps
                           ? static_cast<uint32_t>(((groups > 256 ? 512 : 256) + a.heads - 1) / a.heads) : 0;
        p.parts = p.row_target;
        p.row_units = static_cast<uint32_t>(tiles) + p.row_target;
        if (p.row_target || p.counted) {
            const uint64_t rows = static_cast<uint64_t>(a.heads) * p.parts * rows_of_tile(p.ks);
            p.rows_ml = round256(rows * dim * 4);
            p.rows_plan = p.rows_ml + round256(rows * 8);
            p.bytes = std::max(p.bytes, p.rows_plan + round256((p.counted ? 12ull : 8ull) * a.seq.seqs));
        }
    }
    return p;
}

uint32_t join_blocks(const PagedDev& a) { return (a.seq.rows * a.group + kJoinRows - 1) / kJoinRows; }

template <int CT, int QT, int D, bool PAGED>
int attend_typed(const PagedDev& a, uint8_t* ws, hipStream_t st) {
    const Plan p = plan_of(a, D, CT);
    if constexpr (PAGED)
        if (p.few) {
            const PagedPart part{reinterpret_cast<float*>(ws), reinterpret_cast<float*>(ws + p.ml),
                                 reinterpret_cast<int32_t*>(ws + p.plan), p.units, p.target, p.rows, p.units, p.most, nullptr,
                                 p.counted};
            if (p.counted) few_plan_kernel<<<1, kCounters, 0, st>>>(a, part);
            const uint32_t grid = a.heads * p.units + clears(a);
            constexpr int kWide = wide_waves(D, CT);
            if (p.wide) decode_kernel<CT, QT, D, kWide><<<grid, 64 * kWide, 0, st>>>(a, part);
            else decode_kernel<CT, QT, D, 4><<<grid, 256, 0, st>>>(a, part);
            if (p.units > a.seq.seqs) join_kernel<QT, D><<<a.seq.seqs * a.heads * p.rows, 256, 0, st>>>(a, part);
        }
    if (p.many) {
        const PagedPart part{reinterpret_cast<float*>(ws), reinterpret_cast<float*>(ws + p.rows_ml),
                             reinterpret_cast<int32_t*>(ws + p.rows_plan), p.row_units, p.row_target,
                             static_cast<uint32_t>(rows_of_tile(p.ks)), p.parts, 0,
                             reinterpret_cast<int32_t*>(ws + p.rows_plan) + 2ull * a.seq.seqs, p.counted};
        const int few = PAGED && p.few ? kFew : 0;
        if (p.counted) rows_plan_kernel<<<1, kCounters, 0, st>>>(a, part, few);
        const uint32_t grid = a.heads * p.row_units + (p.few ? 0 : clears(a));
        if (p.ks == 4) rows_kernel<CT, QT, D, PAGED, 4><<<grid, 512, 0, st>>>(a, part, few);
        else if (p.ks == 2) rows_kernel<CT, QT, D, PAGED, 2><<<grid, 512, 0, st>>>(a, part, few);
        else rows_kernel<CT, QT, D, PAGED, 1><<<grid, 512, 0, st>>>(a, part, few);
        if (p.row_target) join_rows_kernel<QT, D><<<a.heads * join_blocks(a), 256, 0, st>>>(a, part, few);
    }
    return hipGetLastError();
}
template <int CT, int QT, bool PAGED>
int attend_dim(const PagedDev& a, uint32_t dim, uint8_t* ws, hipStream_t st) {
    return dim == 64 ? attend_typed<CT, QT, 64, PAGED>(a, ws, st) : attend_typed<CT, QT, 128, PAGED>(a, ws, st);
}

template <int CT, int QT, int D>
int rows_typed(const PagedRowsDev& r, bool store, hipStream_t st) {
    // four workgroups a CU where there are heads enough (64 single rows of 8 heads of 128: 7.8 us with all heads in one)
    const uint32_t chunks = (r.seq.rows + kChunk - 1) / kChunk * r.layers;
    uint32_t heads = r.heads;
    while (heads > 1 && 2ull * chunks * ((r.heads + heads - 1) / heads) < 1024) heads = (heads + 1) / 2;
    const dim3 grid(chunks, 2, (r.heads + heads - 1) / heads);
    if (store) paged_store_kernel<CT, QT, D><<<grid, 256, 0, st>>>(r, heads);
    else paged_load_kernel<CT, QT, D><<<grid, 256, 0, st>>>(r, heads);
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

// The launches of attend_typed: threads along x stay below 2^32.
bool paged_fits(const PagedDev& a, uint32_t dim, int cache_dtype) {
    const uint64_t most = static_cast<uint64_t>(a.heads) * (static_cast<uint64_t>(a.seq.rows) * a.group / 64 + a.seq.seqs);
    if (most >= 1u << 28) return false;     // what plan_of counts in 32 bits
    const Plan p = plan_of(a, dim, cache_dtype);
    uint64_t blocks = 0;
    if (p.few)
        blocks = std::max(static_cast<uint64_t>(a.heads) * p.units, static_cast<uint64_t>(a.seq.seqs) * a.heads * p.rows);
    if (p.many) {
        blocks = std::max(blocks, static_cast<uint64_t>(a.heads) * p.row_units);
        if (p.row_target) blocks = std::max(blocks, static_cast<uint64_t>(a.heads) * join_blocks(a));
    }
    return blocks < (1u << 23) - kClear;     // workgroups of up to 512 threads
}

uint64_t paged_workspace(const PagedDev& a, uint32_t dim, int cache_dtype) { return plan_of(a, dim, cache_dtype).bytes; }

int launch_paged(const PagedDev& a, uint32_t dim, int cache_dtype, int dtype, uint8_t* ws, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (!a.seq.paged)
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
