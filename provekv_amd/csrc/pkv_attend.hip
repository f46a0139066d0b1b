// pkv_attend.hip -- kernels over live KV caches: attention with a sliding
// window and always-visible first slots, the 4-bit cache's store and load, and
// eviction by accumulated weight.  gfx950.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "pkv_attend.h"

namespace pkv {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_huge_valf();

template <int DT> struct Elem;
template <> struct Elem<PKV_F32> { using T = float; };
template <> struct Elem<PKV_BF16> { using T = __bf16; };
template <> struct Elem<PKV_F16> { using T = _Float16; };

// Scale byte b of a 4-bit block as the conversions' operand: 2^(b - 127) (they
// read the exponent field alone, so 0 is 2^-127 and 255 makes NaN).
__device__ inline float block_scale(uint32_t b) { return __uint_as_float(b << 23); }

// Elements d0, d0 + 1 of row `row` (element offset) as f32.
template <int CT>
__device__ inline f32x2 load2(const uint8_t* p, const uint8_t* sc, uint64_t row, uint32_t d0) {
    if constexpr (CT == PKV_FP4) {
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(p[(row + d0) / 2], block_scale(sc[(row + d0) / 32]), 0);
    } else {
        const auto* e = reinterpret_cast<const typename Elem<CT>::T*>(p) + row + d0;
        return f32x2{static_cast<float>(e[0]), static_cast<float>(e[1])};
    }
}

struct Span {
    int len, rows, first;   // slots, query rows, slot of row 0 (may be negative)
};
__device__ inline Span span(const AttendDev& a, uint32_t c) {
    Span s;
    s.len = min(max(a.lens[c], 0), static_cast<int>(a.max_len));
    s.rows = a.q_lens ? min(max(a.q_lens[c], 0), static_cast<int>(a.nq)) : static_cast<int>(a.nq);
    s.first = s.len - s.rows;
    return s;
}
__device__ inline bool visible(const AttendDev& a, int pos, int j) {
    return j <= pos && (!a.window || static_cast<uint32_t>(pos - j) < a.window || static_cast<uint32_t>(j) < a.sinks);
}

__device__ inline float wave_sum(float x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// One workgroup per (row, head, copy), four waves over every fourth visible
// slot, each with its own running maximum and sum.
template <int CT, int QT, int D>
__global__ __launch_bounds__(256) void attend_kernel(AttendDev a) {
    using T = typename Elem<QT>::T;
    const uint32_t r = blockIdx.x, h = blockIdx.y, c = blockIdx.z;
    const uint32_t i = r / a.group, g = r % a.group, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const Span s = span(a, c);
    if (static_cast<int>(i) >= s.rows) return;
    const int pos = s.first + static_cast<int>(i);
    __shared__ float sq[D], so[4][D], sm[4], sl[4];
    const T* q = reinterpret_cast<const T*>(a.q) + c * a.q_copy + i * a.q_row + (h * a.group + g) * a.q_head;
    if (threadIdx.x < D) sq[threadIdx.x] = static_cast<float>(q[threadIdx.x]);
    __syncthreads();
    const uint64_t base = c * a.kv.copy + h * a.kv.head;
    const uint32_t d0 = 2 * lane;
    const float q0 = d0 < D ? sq[d0] : 0.0f, q1 = d0 < D ? sq[d0 + 1] : 0.0f;
    float m = -kInf, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j = wave; j <= pos; j += 4) {
        if (!visible(a, pos, j)) continue;
        const uint64_t row = base + static_cast<uint64_t>(j) * a.kv.slot;
        float t = 0.0f;
        if (d0 < D) {
            const f32x2 k = load2<CT>(a.kv.k, a.kv.ks, row, d0);
            t = q0 * k[0] + q1 * k[1];
        }
        t = wave_sum(t) * a.scale2;
        const float mn = fmaxf(m, t), mu = mn == -kInf ? 0.0f : mn;
        const float p = exp2f(t - mu), f = exp2f(m - mu);
        l = l * f + p;
        if (d0 < D) {
            const f32x2 v = load2<CT>(a.kv.v, a.kv.vs, row, d0);
            o0 = o0 * f + p * v[0];
            o1 = o1 * f + p * v[1];
        }
        m = mn;
    }
    if (lane == 0) { sm[wave] = m; sl[wave] = l; }
    if (d0 < D) { so[wave][d0] = o0; so[wave][d0 + 1] = o1; }
    __syncthreads();
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), mu = top == -kInf ? 0.0f : top;
    float sum = 0.0f, f[4];
    for (int w = 0; w < 4; ++w) {
        f[w] = exp2f(sm[w] - mu);
        sum += sl[w] * f[w];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (threadIdx.x < D) {
        float o = 0.0f;
        for (int w = 0; w < 4; ++w) o += so[w][threadIdx.x] * f[w];
        T* out = reinterpret_cast<T*>(a.out) + c * a.o_copy + i * a.o_row + (h * a.group + g) * a.o_head;
        out[threadIdx.x] = static_cast<T>(sum == 0.0f ? 0.0f : o * inv);
    }
    if (threadIdx.x == 0) {
        if (a.lse) {
            const uint64_t hq = static_cast<uint64_t>(c) * a.heads * a.group + h * a.group + g;
            a.lse[hq * a.nq + i] = sum == 0.0f ? -kInf : (mu + log2f(sum)) * kLn2;
        }
        if (a.stats) {
            float* st = a.stats + 2 * ((static_cast<uint64_t>(c) * a.heads + h) * a.nq * a.group + r);
            st[0] = mu;
            st[1] = inv;
        }
    }
}

// One thread per slot: its weights over every row, in row order.
template <int CT, int QT, int D>
__global__ __launch_bounds__(256) void weights_kernel(AttendDev a) {
    using T = typename Elem<QT>::T;
    const uint32_t h = blockIdx.y, c = blockIdx.z;
    const int j = blockIdx.x * 256 + threadIdx.x;
    const Span s = span(a, c);
    if (j >= s.len) return;
    const uint64_t row = c * a.kv.copy + h * a.kv.head + static_cast<uint64_t>(j) * a.kv.slot;
    float k[D];
    for (int d = 0; d < D; d += 2) {
        const f32x2 x = load2<CT>(a.kv.k, a.kv.ks, row, d);
        k[d] = x[0];
        k[d + 1] = x[1];
    }
    const float* st = a.stats + 2 * (static_cast<uint64_t>(c) * a.heads + h) * a.nq * a.group;
    float sum = 0.0f;
    for (uint32_t i = 0; i < static_cast<uint32_t>(s.rows); ++i) {
        if (!visible(a, s.first + static_cast<int>(i), j)) continue;
        for (uint32_t g = 0; g < a.group; ++g) {
            const T* q = reinterpret_cast<const T*>(a.q) + c * a.q_copy + i * a.q_row + (h * a.group + g) * a.q_head;
            float t = 0.0f;
            for (int d = 0; d < D; ++d) t += static_cast<float>(q[d]) * k[d];
            const float* x = st + 2 * (i * a.group + g);
            sum += exp2f(t * a.scale2 - x[0]) * x[1];
        }
    }
    a.weights[c * a.w_copy + h * a.w_head + j] += sum;
}

// ------------------------------------------------------------ the 4-bit cache
struct Row {
    uint64_t src, dst;   // element offsets in the rows' tensor and in the cache
    bool there;
};
// Row `r` of all (copy, layer, head, i), i fastest.
__device__ inline Row row_of(const RowsDev& a, uint64_t r) {
    const uint32_t i = r % a.rows;
    r /= a.rows;
    const uint32_t h = r % a.heads;
    r /= a.heads;
    const uint32_t l = r % a.layers, c = r / a.layers;
    const int count = a.counts ? min(max(a.counts[c], 0), static_cast<int>(a.rows)) : static_cast<int>(a.rows);
    const int64_t slot = static_cast<int64_t>(a.first[c]) + i;
    Row o;
    o.there = static_cast<int>(i) < count && slot >= 0 && slot < a.slots;
    o.src = c * a.copy + l * a.layer + h * a.head + i * a.row;
    o.dst = c * a.kv.copy + l * a.kv.layer + h * a.kv.head + (o.there ? slot : 0) * a.kv.slot;
    return o;
}

// Exponent byte of a block: the smallest e with top <= 7 * 2^e, kept in -125 ..
// 125 (2^-125 so that half a step, 2^-126, is a normal number; 2^125 so that 6
// steps stay finite), 255 when the block holds an infinity or NaN.  top's bits,
// sign off.
__device__ inline uint32_t block_exponent(uint32_t top) {
    if (top >= 0x7f800000u) return 255;
    const int e = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(min(max(e, 2), 252));
}

// Eight values a thread, four threads a block.  Both sides of the same row are
// blockIdx.y.
template <int QT, int D>
__global__ __launch_bounds__(256) void fp4_store_kernel(RowsDev a, uint64_t total) {
    using T = typename Elem<QT>::T;
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint64_t r = t / (D / 8);
    const uint32_t d = t % (D / 8) * 8;
    const bool live = r < total;
    const Row o = row_of(a, live ? r : 0);
    const uint8_t* src = blockIdx.y ? a.values : a.keys;
    if (!src) return;
    float x[8];
    uint32_t top = 0;
    for (int e = 0; e < 8; ++e) {
        x[e] = static_cast<float>(reinterpret_cast<const T*>(src)[o.src + d + e]);
        top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
    const uint32_t b = block_exponent(top);
    uint32_t codes = 0;
    if (b != 255) {
        const float s = block_scale(b);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], s, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], s, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], s, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], s, 3);
    }
    if (!live || !o.there) return;
    uint8_t* dst = const_cast<uint8_t*>(blockIdx.y ? a.kv.v : a.kv.k);
    uint8_t* dsc = const_cast<uint8_t*>(blockIdx.y ? a.kv.vs : a.kv.ks);
    reinterpret_cast<uint32_t*>(dst)[(o.dst + d) / 8] = codes;
    if (d % 32 == 0) dsc[(o.dst + d) / 32] = static_cast<uint8_t>(b);
}

template <int QT, int D>
__global__ __launch_bounds__(256) void fp4_load_kernel(RowsDev a, uint64_t total) {
    using T = typename Elem<QT>::T;
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint64_t r = t / (D / 8);
    if (r >= total || !(blockIdx.y ? a.values : a.keys)) return;
    const uint32_t d = t % (D / 8) * 8;
    const Row o = row_of(a, r);
    const uint8_t* src = blockIdx.y ? a.kv.v : a.kv.k;
    const uint8_t* ssc = blockIdx.y ? a.kv.vs : a.kv.ks;
    T* dst = reinterpret_cast<T*>(blockIdx.y ? a.values : a.keys) + o.src + d;
    for (int e = 0; e < 8; e += 2) {
        const f32x2 x = o.there ? load2<PKV_FP4>(src, ssc, o.dst, d + e) : f32x2{0.0f, 0.0f};
        dst[e] = static_cast<T>(x[0]);
        dst[e + 1] = static_cast<T>(x[1]);
    }
}

// ------------------------------------------------------------ eviction
// Order of keeping: a larger key is kept first.  A NaN sorts as -inf, -0 as 0.
__device__ inline uint32_t weight_key(float w) {
    if (!(w == w)) w = -kInf;
    if (w == 0.0f) w = 0.0f;
    const uint32_t u = __float_as_uint(w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelect = 1024;   // threads of select_kernel

// Inclusive prefix sum over the workgroup, in thread order.
__device__ inline uint32_t block_scan(uint32_t x, uint32_t* tmp) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= static_cast<uint32_t>(o)) x += y;
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) x += tmp[w];
    return x;
}

// One workgroup per (head, layer, copy): the budget's border among the middle
// slots by four passes over 8 bits of the key, then the kept slots in order.
__global__ __launch_bounds__(kSelect) void select_kernel(EvictDev a) {
    const uint32_t h = blockIdx.x % a.heads, cl = blockIdx.x / a.heads, l = cl % a.layers, c = cl / a.layers;
    const uint32_t n = min(max(a.lens[c], 0), static_cast<int>(a.slots));
    const float* w = a.w + c * a.ws[0] + l * a.ws[1] + h * a.ws[2];
    float* wo = a.w_out + c * a.os[0] + l * a.os[1] + h * a.os[2];
    int32_t* kept = a.kept + static_cast<uint64_t>(blockIdx.x) * a.budget;
    const uint32_t keep = min(n, a.budget), t = threadIdx.x;
    __shared__ uint32_t hist[256], tmp[16], found[2];
    if (l == 0 && h == 0 && t == 0) a.new_lens[c] = static_cast<int32_t>(keep);
    if (n <= a.budget) {
        for (uint32_t j = t; j < a.budget; j += kSelect) kept[j] = j < n ? static_cast<int32_t>(j) : -1;
    } else {
        const uint32_t lo = a.sinks, hi = n - a.recent;
        uint32_t want = a.budget - a.sinks - a.recent;   // of the middle; < hi - lo
        uint32_t prefix = 0, mask = 0;
        // the key of the want-th largest: its bits from the top, 8 at a time
        for (int shift = 24; shift >= 0 && want; shift -= 8) {
            if (t < 256) hist[t] = 0;
            __syncthreads();
            for (uint32_t j = lo + t; j < hi; j += kSelect) {
                const uint32_t k = weight_key(w[j]);
                if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255], 1u);
            }
            __syncthreads();
            if (t == 0) {
                uint32_t above = 0;
                int b = 255;
                while (above + hist[b] < want) above += hist[b--];
                found[0] = b;
                found[1] = above;
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= 255u << shift;
            want -= found[1];
            __syncthreads();
        }
        // kept: protected slots, keys above the border, and the first `want` at it
        const bool any = mask != 0;
        uint32_t done = 0, ties = 0;
        for (uint32_t j0 = 0; j0 < n; j0 += kSelect) {
            const uint32_t j = j0 + t;
            const bool in = j < n, mid = in && j >= lo && j < hi;
            const uint32_t k = mid ? weight_key(w[j]) : 0;
            const bool tie = mid && any && k == prefix;
            const uint32_t before = block_scan(tie, tmp);
            if (t == kSelect - 1) found[0] = before;
            const bool take = in && (!mid || (any && (k > prefix || (tie && ties + before <= want))));
            const uint32_t at = block_scan(take, tmp);
            if (t == kSelect - 1) found[1] = at;
            if (take) kept[done + at - 1] = static_cast<int32_t>(j);
            __syncthreads();
            ties += found[0];
            done += found[1];
            __syncthreads();
        }
    }
    // the kept slots' weights, in steps: every read of a step comes before its
    // writes, and a later step's sources lie behind everything written
    __syncthreads();
    __threadfence_block();
    for (uint32_t j0 = 0; j0 < keep; j0 += kSelect) {
        const uint32_t j = j0 + t;
        const float x = j < keep ? w[kept[j]] : 0.0f;
        __syncthreads();
        if (j < keep) wo[j] = x;
        __syncthreads();
    }
    for (uint32_t j = keep + t; j < a.into_slots; j += kSelect) wo[j] = 0.0f;
}

template <int DT>
__device__ inline uint64_t elem_byte(uint64_t e) { return DT == PKV_FP4 ? e / 2 : DT == PKV_F32 ? e * 4 : e * 2; }

// Kept rows to their new slots, one workgroup per (head, layer, copy) and side
// (blockIdx.y), pieces of 16 bytes; in place by the same order as the weights.
template <int DT, int D>
__global__ __launch_bounds__(256) void move_kernel(EvictDev a) {
    constexpr uint32_t kBytes = DT == PKV_FP4 ? D / 2 : DT == PKV_F32 ? D * 4 : D * 2;
    constexpr uint32_t kLanes = kBytes / 16, kRows = 256 / kLanes;
    const uint32_t h = blockIdx.x % a.heads, cl = blockIdx.x / a.heads, l = cl % a.layers, c = cl / a.layers;
    const uint32_t n = min(max(a.lens[c], 0), static_cast<int>(a.slots)), keep = min(n, a.budget);
    const int32_t* kept = a.kept + static_cast<uint64_t>(blockIdx.x) * a.budget;
    const uint8_t* src = blockIdx.y ? a.kv.v : a.kv.k;
    uint8_t* dst = const_cast<uint8_t*>(blockIdx.y ? a.into.v : a.into.k);
    const uint8_t* ssc = blockIdx.y ? a.kv.vs : a.kv.ks;
    uint8_t* dsc = const_cast<uint8_t*>(blockIdx.y ? a.into.vs : a.into.ks);
    const uint64_t from = c * a.kv.copy + l * a.kv.layer + h * a.kv.head;
    const uint64_t to = c * a.into.copy + l * a.into.layer + h * a.into.head;
    const uint32_t sub = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
    for (uint32_t j0 = 0; j0 < keep; j0 += kRows) {
        const uint32_t j = j0 + row;
        const bool in = j < keep;
        uint4 x{};
        uint32_t sc = 0;
        if (in) {
            const uint64_t e = from + static_cast<uint64_t>(kept[j]) * a.kv.slot;
            x = *reinterpret_cast<const uint4*>(src + elem_byte<DT>(e) + 16 * sub);
            if constexpr (DT == PKV_FP4) {
                if (sub == 0)
                    sc = D == 64 ? *reinterpret_cast<const uint16_t*>(ssc + e / 32)
                                 : *reinterpret_cast<const uint32_t*>(ssc + e / 32);
            }
        }
        __syncthreads();
        if (in) {
            const uint64_t e = to + static_cast<uint64_t>(j) * a.into.slot;
            *reinterpret_cast<uint4*>(dst + elem_byte<DT>(e) + 16 * sub) = x;
            if constexpr (DT == PKV_FP4) {
                if (sub == 0) {
                    if constexpr (D == 64) *reinterpret_cast<uint16_t*>(dsc + e / 32) = static_cast<uint16_t>(sc);
                    else *reinterpret_cast<uint32_t*>(dsc + e / 32) = sc;
                }
            }
        }
        __syncthreads();
    }
}

template <int CT, int QT, int D>
int attend_typed(AttendDev a, uint8_t* ws, hipStream_t st) {
    a.stats = a.weights ? reinterpret_cast<float*>(ws) : nullptr;
    attend_kernel<CT, QT, D><<<dim3(a.nq * a.group, a.heads, a.copies), 256, 0, st>>>(a);
    if (a.weights)
        weights_kernel<CT, QT, D><<<dim3((a.max_len + 255) / 256, a.heads, a.copies), 256, 0, st>>>(a);
    return hipGetLastError();
}

template <int CT, int QT>
int attend_dim(const AttendDev& a, uint32_t dim, uint8_t* ws, hipStream_t st) {
    return dim == 64 ? attend_typed<CT, QT, 64>(a, ws, st) : attend_typed<CT, QT, 128>(a, ws, st);
}

}  // namespace

uint64_t attend_workspace(const AttendDev& a, uint32_t, int, int) {
    return 8ull * a.copies * a.heads * a.nq * a.group;
}

int launch_attend(const AttendDev& a, uint32_t dim, int cache_dtype, int dtype, uint8_t* ws, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (cache_dtype == PKV_F32) return attend_dim<PKV_F32, PKV_F32>(a, dim, ws, st);
    if (cache_dtype == PKV_BF16) return attend_dim<PKV_BF16, PKV_BF16>(a, dim, ws, st);
    if (cache_dtype == PKV_F16) return attend_dim<PKV_F16, PKV_F16>(a, dim, ws, st);
    if (dtype == PKV_F32) return attend_dim<PKV_FP4, PKV_F32>(a, dim, ws, st);
    if (dtype == PKV_BF16) return attend_dim<PKV_FP4, PKV_BF16>(a, dim, ws, st);
    return attend_dim<PKV_FP4, PKV_F16>(a, dim, ws, st);
}

#define PKV_ROWS_LAUNCH(kernel)                                                                          \
    hipStream_t st = static_cast<hipStream_t>(stream);                                                   \
    const uint64_t total = static_cast<uint64_t>(r.copies) * r.layers * r.heads * r.rows;                \
    const uint64_t wg = (total * (dim / 8) + 255) / 256;                                                 \
    if (wg > 0x7fffffffull) return hipErrorInvalidValue;                                                 \
    const dim3 grid(static_cast<uint32_t>(wg), 2);                                                       \
    if (dim == 64) {                                                                                     \
        if (dtype == PKV_F32) kernel<PKV_F32, 64><<<grid, 256, 0, st>>>(r, total);                       \
        else if (dtype == PKV_BF16) kernel<PKV_BF16, 64><<<grid, 256, 0, st>>>(r, total);                \
        else kernel<PKV_F16, 64><<<grid, 256, 0, st>>>(r, total);                                        \
    } else {                                                                                             \
        if (dtype == PKV_F32) kernel<PKV_F32, 128><<<grid, 256, 0, st>>>(r, total);                      \
        else if (dtype == PKV_BF16) kernel<PKV_BF16, 128><<<grid, 256, 0, st>>>(r, total);               \
        else kernel<PKV_F16, 128><<<grid, 256, 0, st>>>(r, total);                                       \
    }                                                                                                    \
    return hipGetLastError();

int launch_fp4_store(const RowsDev& r, uint32_t dim, int dtype, void* stream) { PKV_ROWS_LAUNCH(fp4_store_kernel) }
int launch_fp4_load(const RowsDev& r, uint32_t dim, int dtype, void* stream) { PKV_ROWS_LAUNCH(fp4_load_kernel) }

template <int DT>
static void move_dim(const EvictDev& e, uint32_t dim, dim3 grid, hipStream_t st) {
    if (dim == 64) move_kernel<DT, 64><<<grid, 256, 0, st>>>(e);
    else move_kernel<DT, 128><<<grid, 256, 0, st>>>(e);
}

int launch_evict(const EvictDev& e, uint32_t dim, int dtype, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    const uint32_t sets = e.copies * e.layers * e.heads;
    select_kernel<<<sets, kSelect, 0, st>>>(e);
    const dim3 grid(sets, 2);
    if (dtype == PKV_F32) move_dim<PKV_F32>(e, dim, grid, st);
    else if (dtype == PKV_BF16) move_dim<PKV_BF16>(e, dim, grid, st);
    else if (dtype == PKV_F16) move_dim<PKV_F16>(e, dim, grid, st);
    else move_dim<PKV_FP4>(e, dim, grid, st);
    return hipGetLastError();
}

}  // namespace pkv
