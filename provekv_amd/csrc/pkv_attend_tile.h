// pkv_attend_tile.h -- what the attention kernels share on the device: matrix
// operands, the softmax's running base, the slots that rows see, and tiles of
// slots in LDS.  Included by pkv_attend.hip (contiguous caches) and
// pkv_paged.hip (pages, packed prompts).
//
// A is a call's arguments: window, sinks, reach (the window, or 2^31 for none)
// and scale2 (scale * log2 e) are read.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/pkv_codec.h"

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

// Scale byte b of a block of codes as the conversions' operand: 2^(b - 127) (they
// read the exponent field alone, so 0 is 2^-127 and 255 makes NaN).
__device__ inline float block_scale(uint32_t b) { return __uint_as_float(b << 23); }

// The row at `pos` sees slot j (reach: the window, or 2^31 for none).
template <class A>
__device__ inline bool in_reach(const A& a, int pos, int j) { return static_cast<uint32_t>(pos - j) < a.reach; }
template <class A>
__device__ inline bool visible(const A& a, int pos, int j) {
    return in_reach(a, pos, j) | ((j <= pos) & (static_cast<uint32_t>(j) < a.sinks));   // no branches
}

// x combined with the lane 32 or 16 away, by lane swaps (a shuffle goes through LDS).
template <class F>
__device__ inline float across32(float x, F f) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <class F>
__device__ inline float across16(float x, F f) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float larger(float a, float b) { return fmaxf(a, b); }

__device__ inline float wave_sum(float x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Type of the matrix products over a cache: its own, bf16 for 4- and 8-bit
// codes (every code times its scale is exact in bf16).
constexpr bool coded(int ct) { return ct == PKV_FP4 || ct == PKV_FP8; }
constexpr int mat_type(int ct) { return coded(ct) ? PKV_BF16 : ct; }
// A query of QT over codes is the sum of this many bf16 terms (exact: 8 bits
// each), any other query is its own single term.
constexpr int query_terms(int ct, int qt) { return !coded(ct) ? 1 : qt == PKV_F32 ? 3 : qt == PKV_F16 ? 2 : 1; }

template <int MT>
__device__ inline f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (MT == PKV_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// (a, b) rounded to the matrix type, and what the rounding left of each.
template <int MT>
__device__ inline uint32_t pack_term(float& a, float& b) {
    if constexpr (MT == PKV_BF16) {
        const bf16x2 h = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
        a -= static_cast<float>(h[0]);
        b -= static_cast<float>(h[1]);
        return __builtin_bit_cast(uint32_t, h);
    } else {
        const f16x2 h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
        a -= static_cast<float>(h[0]);
        b -= static_cast<float>(h[1]);
        return __builtin_bit_cast(uint32_t, h);
    }
}

// The same for a query's values: what an infinity or NaN leaves is 0, so that
// the terms' products sum to what the value's own would.
__device__ inline uint32_t pack_query_term(float& a, float& b) {
    const uint32_t h = pack_term<PKV_BF16>(a, b);
    if ((h & 0x7f80u) == 0x7f80u) a = 0.0f;
    if ((h >> 16 & 0x7f80u) == 0x7f80u) b = 0.0f;
    return h;
}

// Two 16-bit values that hold an infinity or NaN.
template <int MT>
__device__ inline bool nonfinite2(uint32_t x) {
    constexpr uint32_t e = MT == PKV_BF16 ? 0x7f80u : 0x7c00u;
    return (x & e) == e || (x >> 16 & e) == e;
}

// One word's part of a dot product.
template <int MT>
__device__ inline float dot_word(uint32_t a, uint32_t b) {
    if constexpr (MT == PKV_F32) return __uint_as_float(a) * __uint_as_float(b);
    using T2 = typename std::conditional<MT == PKV_BF16, bf16x2, f16x2>::type;
    const T2 x = __builtin_bit_cast(T2, a), y = __builtin_bit_cast(T2, b);
    return static_cast<float>(x[0]) * static_cast<float>(y[0]) + static_cast<float>(x[1]) * static_cast<float>(y[1]);
}

// Infinities and NaN of the two cleared.
template <int MT>
__device__ inline uint32_t finite_or_0(uint32_t x) {
    constexpr uint32_t e = MT == PKV_BF16 ? 0x7f80u : 0x7c00u;
    if ((x & e) == e) x &= 0xffff0000u;
    if ((x >> 16 & e) == e) x &= 0x0000ffffu;
    return x;
}

// Softmax weights are held as 2^(s * scale2 + base), base = kLift - (largest
// logit) * scale2 when it was last set: the largest logit may since have grown
// by up to 2^kLag, so that sums are rescaled seldom.  +inf before the first
// logit.  A share's base goes with its sums, as it was used.
//
// f16 ends at 2^-24, so that weights up to 1 would lose all below 2^-25, and a
// long cache's sum with them.  Weights up to 2^(11 + 4) use its top instead:
// full precision down to 2^-25 of the largest, the end at 2^-36.
template <int MT> constexpr float kLag = MT == PKV_F16 ? 4.0f : 8.0f;
template <int MT> constexpr float kLift = MT == PKV_F16 ? 11.0f : 0.0f;
// Weighted values are summed before they are divided, and the sum can pass the
// end of f32 (and bf16) where the mean does not.  The output is then not finite,
// and the pass that looks for infinities among the values scales the weights by
// 2^-kDown, the lag over 2^30 slots and more (decode_kernel), or a further one
// does (rows_kernel); f16 values are far from it.  Shares' outputs are stored
// 2^-kPartDown as large and joined 2^-kJoinDown, by as many shares as there can be.
template <int MT> constexpr int kDown = MT == PKV_F16 ? 0 : 40;
constexpr int kPartDown = 2;            // decode_kernel's four waves
constexpr int kJoinDown = 10;           // shares of a row: up to 2^10 (768 of contiguous caches, 1,024 of pages)
constexpr float power(int x) { return x < 0 ? 0.5f * power(x + 1) : x ? 2.0f * power(x - 1) : 1.0f; }
template <int X> constexpr float kPower = power(X);   // 2^X
// The base with a row's logits up to `top` seen as well.
template <class A>
__device__ inline float lower_base(const A& a, float lift, float base, float top) {
    return fminf(base, __builtin_fmaf(-top, a.scale2, lift));
}
// Of the weights with `base` when they join those of a lower one.
__device__ inline float joined(float low, float base) { return base == low ? 1.0f : exp2f(low - base); }
// Log of the sum of exponentials, and a row's (base, factor): weight = 2^(s *
// scale2 + base) * factor.  An empty row: -inf, 0.
__device__ inline float lse_of(float base, float sum) {   // exponents by themselves: sums of one lift or another
    if (sum == 0.0f) return -kInf;
    const float e = static_cast<float>(__builtin_amdgcn_frexp_expf(sum));
    return (log2f(__builtin_amdgcn_frexp_mantf(sum)) + (e - base)) * kLn2;
}
__device__ inline void stats_of(float base, float sum, float* stats) {
    stats[0] = sum == 0.0f ? 0.0f : base;
    stats[1] = sum == 0.0f ? 0.0f : 1.0f / sum;
}

// The slots that the rows of a tile see, as tiles of `step` slots: [0, first)
// with the always-visible slots, then [second, second + count - first).
struct Tiles {
    int first, second, count;
    int low, high;          // rows see slots < a.sinks (with a window) and low .. high - 1
    __device__ int slot(int t, int step) const { return (t < first ? t : second + t - first) * step; }
};
template <class A>
__device__ inline Tiles tiles_of(const A& a, int pos0, int pos1, int step) {
    Tiles t;
    t.high = max(pos1 + 1, 0);
    t.low = a.window ? static_cast<int>(max(static_cast<int64_t>(pos0) - a.window + 1, static_cast<int64_t>(0))) : 0;
    const int sink = static_cast<int>(min(static_cast<uint32_t>(min(t.low, t.high)), a.sinks));
    t.first = (sink + step - 1) / step;
    t.second = max(t.first, t.low / step);
    t.count = t.first + max((t.high + step - 1) / step - t.second, 0);
    return t;
}
// Every row between pos0 and pos1 sees all of lo .. hi.
template <class A>
__device__ inline bool all_visible(const A& a, int pos0, int pos1, int lo, int hi) {
    return hi <= pos0 && (in_reach(a, pos1, lo) || static_cast<uint32_t>(hi) < a.sinks);
}
// Some row of the tile list's rows sees slot j.
template <class A>
__device__ inline bool any_visible(const A& a, const Tiles& t, int j) {
    return j < t.high && (j >= t.low || static_cast<uint32_t>(j) < a.sinks);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int MT>
__device__ inline f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (MT == PKV_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}
// Row of a 32x32 result that register r of lane half `half` holds.
__device__ constexpr int row32(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

// The query of one row as matrix operands, a lane half its half of every 16
// channels (f32: of every 8), 16 bytes a register.
template <int CT, int QT, int D>
struct Query {
    using T = typename Elem<QT>::T;
    static constexpr int kTerms = query_terms(CT, QT);
    static constexpr int kRegs = CT == PKV_F32 ? D / 8 : D / 16;
    u32x4 q[kTerms][kRegs];
    __device__ void load(const T* p, bool real, uint32_t half) {
        for (int s = 0; s < kRegs; ++s) {
            const uint32_t d = CT == PKV_F32 ? 8 * s + 4 * half : 16 * s + 8 * half;
            if constexpr (kTerms == 1) {
                q[0][s] = real ? *reinterpret_cast<const u32x4*>(p + d) : u32x4{};
            } else {
                for (int w = 0; w < 4; ++w) {
                    float x = real ? static_cast<float>(p[d + 2 * w]) : 0.0f;
                    float y = real ? static_cast<float>(p[d + 2 * w + 1]) : 0.0f;
                    for (int n = 0; n < kTerms; ++n) q[n][s][w] = pack_query_term(x, y);
                }
            }
        }
    }
};

// 16 bytes a lane from global memory straight to LDS (lane i at `to` + 16 i; to
// is uniform), nothing held in registers on the way.  Done when the wave waits
// (copies_done): the compiler, which would wait at the next LDS read of any
// kind, does not see them.  M0 is put back, since the compiler may hold a value there.
__device__ inline void copy_to_lds(uint32_t to, const uint8_t* from, uint32_t offset) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "s"(to), "v"(offset), "s"(from)
                 : "memory");
}
// The same from an address of each lane's own.
__device__ inline void copy_row_to_lds(uint32_t to, const uint8_t* from) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "s"(to), "v"(from)
                 : "memory");
}
__device__ inline void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

typedef __attribute__((address_space(3))) uint8_t LdsByte;

// A tile of slots in LDS: keys [slot][D], then values [slot][D], codes as bf16,
// in 16-byte pieces at piece ^ turn(slot) so that no read meets a bank
// conflict: an operand of the first product is one piece of 32 slots, one of
// the second 4 slots x 16 channels, transposed by the read itself
// (ds_read_tr16_b64; f32: 32 channels of a slot, no transposition).  f32 keys
// meet two lanes a bank: their products take four times longer than the read.
template <int CT, int D>
struct Staged {
    static constexpr int kSlots = CT == PKV_F32 ? 32 : 64;
    static constexpr int kRow = CT == PKV_F32 ? D * 4 : D * 2, kPieces = kRow / 16;
    static constexpr int kKeyBytes = kSlots * kRow, kBytes = 2 * kKeyBytes;
    static constexpr int kCopies = kKeyBytes / 4096;            // wave-wide copies of 1,024 bytes, a side
    static constexpr int kCopyRows = 1024 / kRow, kCopyStep = 4 * kCopyRows;

    __device__ static uint32_t turn(uint32_t slot, bool values) {
        if constexpr (CT == PKV_F32) return values ? slot / 4 % 2 * 8 : slot % 8;
        else if constexpr (D == 128) return slot % 4 * 4 + slot / 4 % 4;
        else return slot / 2 % 2 * 4 + slot / 4 % 4;
    }
    __device__ static uint32_t key_at(uint32_t slot, uint32_t piece) {
        return slot * kRow + (piece ^ turn(slot, false)) * 16;
    }
    __device__ static uint32_t value_at(uint32_t slot, uint32_t piece) {
        return kKeyBytes + slot * kRow + (piece ^ turn(slot, true)) * 16;
    }
    // The slot that thread t's codes belong to, 16 a wave: 16 lanes write 16 different places of the banks.
    __device__ static uint32_t code_slot(uint32_t t) {
        const uint32_t i = t % 64;
        return t / 64 * 16 + (D == 128 ? i / 16 + i / 4 % 4 * 4 : i / 4 % 2 + i / 8 % 2 * 4 + i / 16 % 2 * 2 + i / 32 * 8);
    }
    // Operand of O^T += V^T P^T for channels 32 e .. and 16 slots from `slot` on: a lane's channel 32 e + lane % 32,
    // the slots of row32 in its half of them.
    __device__ static u32x4 values16(const uint8_t* lds, uint32_t slot, uint32_t e, uint32_t lane) {
        const uint32_t s = lane % 16, piece = 4 * e + lane / 16 % 2 * 2 + s % 4 / 2;
        const uint32_t row = slot + lane / 32 * 4 + s / 4;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* Ptr;
        const LdsByte* p = (const LdsByte*)lds;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(p + value_at(row, piece) + s % 2 * 8));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(p + value_at(row + 8, piece) + s % 2 * 8));
        const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
        return u32x4{x[0], x[1], y[0], y[1]};
    }
    __device__ static uint32_t value32_at(uint32_t slot, uint32_t d) { return value_at(slot, d / 4) + d % 4 * 4; }
    // A staged value.
    __device__ static float value(const uint8_t* lds, uint32_t slot, uint32_t d) {
        if constexpr (CT == PKV_F32) return *reinterpret_cast<const float*>(lds + value32_at(slot, d));
        else return static_cast<float>(
            reinterpret_cast<const typename Elem<mat_type(CT)>::T*>(lds + value_at(slot, d / 8))[d % 8]);
    }
    // Infinities and NaN among a staged tile's values to 0; true if this thread had any.
    __device__ static bool clean(uint8_t* lds) {
        bool odd = false;
        for (uint32_t x = threadIdx.x; x < kKeyBytes / 16; x += 256) {
            u32x4* p = reinterpret_cast<u32x4*>(lds + kKeyBytes) + x;
            u32x4 w = *p;
            bool any = false;
            for (int y = 0; y < 4; ++y) {
                if constexpr (CT == PKV_F32) {
                    if ((w[y] & 0x7f800000u) == 0x7f800000u) {
                        w[y] = 0;
                        any = true;
                    }
                } else {
                    any |= nonfinite2<mat_type(CT)>(w[y]);
                    w[y] = finite_or_0<mat_type(CT)>(w[y]);
                }
            }
            if (any) *p = w;
            odd |= any;
        }
        return odd;
    }
};

// S^T of 32 slots (piece u of a staged tile) and 32 query rows.
template <int CT, int QT, int D>
__device__ inline f32x16 logits32(const uint8_t* lds, int u, const Query<CT, QT, D>& q, uint32_t lane) {
    constexpr int MT = mat_type(CT);
    f32x16 s = {};
    for (int x = 0; x < Query<CT, QT, D>::kRegs; ++x) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(lds + Staged<CT, D>::key_at(32 * u + lane % 32, 2 * x + lane / 32));
        if constexpr (CT == PKV_F32) {
            for (int e = 0; e < 4; ++e)
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[e]), __uint_as_float(q.q[0][x][e]), s, 0, 0, 0);
        } else {
            for (int n = Query<CT, QT, D>::kTerms - 1; n >= 0; --n) s = mma32<MT>(k, q.q[n][x], s);
        }
    }
    return s;
}

// Query rows (rows x group of one KV head) of a workgroup whose waves share
// every tile's slots `ks` ways.
constexpr uint32_t row_tile(int ks) { return 128u / ks; }

}  // namespace
}  // namespace pkv
