// pkv_attend.hip -- kernels over live KV caches: attention with a sliding
// window and always-visible first slots, the 4-bit cache's store and load, and
// eviction by accumulated weight.  gfx950.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

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
// The row at `pos` sees slot j (reach: the window, or 2^31 for none).
__device__ inline bool in_reach(const AttendDev& a, int pos, int j) { return static_cast<uint32_t>(pos - j) < a.reach; }
__device__ inline bool visible(const AttendDev& a, int pos, int j) {
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

// ------------------------------------------------------------ few rows: split over the slots
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Type of the matrix products over a cache: its own, bf16 for 4-bit codes
// (every code times its scale is exact in bf16).
constexpr int mat_type(int ct) { return ct == PKV_FP4 ? PKV_BF16 : ct; }
// A query of QT over 4-bit codes is the sum of this many bf16 terms (exact: 8
// bits each), any other query is its own single term.
constexpr int query_terms(int ct, int qt) { return ct != PKV_FP4 ? 1 : qt == PKV_F32 ? 3 : qt == PKV_F16 ? 2 : 1; }

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
constexpr int kJoinDown = 10;           // shares of a row: up to 768
constexpr float power(int x) { return x < 0 ? 0.5f * power(x + 1) : x ? 2.0f * power(x - 1) : 1.0f; }
template <int X> constexpr float kPower = power(X);   // 2^X
// The base with a row's logits up to `top` seen as well.
__device__ inline float lower_base(const AttendDev& a, float lift, float base, float top) {
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
__device__ inline Tiles tiles_of(const AttendDev& a, int pos0, int pos1, int step) {
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
__device__ inline bool all_visible(const AttendDev& a, int pos0, int pos1, int lo, int hi) {
    return hi <= pos0 && (in_reach(a, pos1, lo) || static_cast<uint32_t>(hi) < a.sinks);
}
// Some row of the tile list's rows sees slot j.
__device__ inline bool any_visible(const AttendDev& a, const Tiles& t, int j) {
    return j < t.high && (j >= t.low || static_cast<uint32_t>(j) < a.sinks);
}

// Up to 16 query rows (rows x group of one KV head) against a share of the
// slots, the whole product on the matrix cores with nothing staged in LDS:
//   S^T = K Q^T   A = 16 slots (lane % 16) x 8 channels a lane group (lane /
//                 16); B = 16 rows (lane % 16).  Any order of the channels will
//                 do as long as q has the same, so a lane reads 16 bytes of a
//                 row.  Result: row lane % 16, slots 4 (lane / 16) + r.
//   O^T = V^T P^T A wants, for one channel a lane, the slots its lane group
//                 has in S^T: the softmax's registers are B as they are.  Lane
//                 i of a group reads channels 8i .. of its 4 (x 2) slots and
//                 v_perm gathers each channel across them; channel order
//                 along M is free again, so O^T tile e holds channels 8m + e.
// Bound by the cache's bytes: 32 slots cost a wave 8 + 16 matrix instructions at
// head_dim 128 against 16 KB of bf16.  Weights go into the second product as
// two terms of a 16-bit type (f32 queries over 4-bit codes: three), which the
// bytes hide.  Measured: 4 x 32,768 slots of 8 heads of 128, four query heads
// each, bf16: 104 us, 5.0 TB/s (114 with the loads in front of their own tile's
// work instead of the one before); 8 x 930 slots of 32 heads of 64, f32: 23 us,
// 5.4 TB/s; the former in 4 bits: 29 us, 4.7 TB/s, where unpacking (a
// conversion per two channels and a permute per four) takes about as long as
// the bytes.  Tried and worse: offsets of whole tiles kept in registers and
// scale bytes of neighbouring slots in one read (4 bits: 34 us, more registers
// and one wave a SIMD less at head_dim 64).
template <int CT, int D>
struct SlotTile {
    static constexpr int kSub = CT == PKV_F32 ? 1 : 2;        // 16-slot pieces
    static constexpr int kStep = 16 * kSub;
    static constexpr int kKRegs = CT == PKV_FP4 ? 1 : CT == PKV_F32 ? D / 16 : D / 32;   // 16-byte reads of a key
    static constexpr int kVRegs = CT == PKV_F32 ? D / 64 : 1;
    static constexpr int kPer = CT == PKV_F32 ? 4 : D / 16;   // channels of a value that a lane reads at once
    u32x4 k[kSub][kKRegs];
    u32x4 v[kSub][4][kVRegs];
    uint32_t ks[kSub], vs[kSub][4];

    __device__ static uint32_t bytes(uint32_t e) { return CT == PKV_FP4 ? e / 2 : CT == PKV_F32 ? e * 4 : e * 2; }

    // kp, vp, ksp, vsp: slot 0 of the head.  Slots past `last` read the last one.
    __device__ void load(const uint8_t* kp, const uint8_t* vp, const uint8_t* ksp, const uint8_t* vsp, uint64_t stride,
                         int slot, int last, uint32_t lane) {
        const uint32_t i = lane % 16, g = lane / 16;
        const uint64_t base = static_cast<uint64_t>(slot) * stride;
        const uint8_t* kt = kp + (CT == PKV_FP4 ? base / 2 : CT == PKV_F32 ? base * 4 : base * 2);
        const uint8_t* vt = vp + (CT == PKV_FP4 ? base / 2 : CT == PKV_F32 ? base * 4 : base * 2);
        const uint32_t st = static_cast<uint32_t>(stride);
        const int room = last - slot;      // >= 0
        for (int t = 0; t < kSub; ++t) {
            const uint32_t e = static_cast<uint32_t>(min(16 * t + static_cast<int>(i), room)) * st;
            const uint8_t* p = kt + bytes(e);
            if constexpr (CT == PKV_FP4) {
                if constexpr (D == 128) k[t][0] = *reinterpret_cast<const u32x4*>(p + 16 * g);
                else {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(p + 8 * g);
                    k[t][0] = u32x4{x[0], x[1], 0, 0};
                }
                ks[t] = (ksp + base / 32)[e / 32 + (D == 128 ? g : g / 2)];
            } else {
                for (int s = 0; s < kKRegs; ++s) k[t][s] = *reinterpret_cast<const u32x4*>(p + 64 * s + 16 * g);
            }
        }
        for (int t = 0; t < kSub; ++t)
            for (int j = 0; j < 4; ++j) {
                const uint32_t e = static_cast<uint32_t>(min(16 * t + 4 * static_cast<int>(g) + j, room)) * st;
                const uint8_t* p = vt + bytes(e);
                if constexpr (CT == PKV_FP4) {
                    if constexpr (D == 128) v[t][j][0][0] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
                    else v[t][j][0][0] = *reinterpret_cast<const uint16_t*>(p + 2 * i);
                    vs[t][j] = (vsp + base / 32)[e / 32 + (D == 128 ? i / 4 : i / 8)];
                } else if constexpr (CT == PKV_F32) {
                    for (int q = 0; q < kVRegs; ++q)
                        v[t][j][q] = *reinterpret_cast<const u32x4*>(p + 256 * q + 16 * i);
                } else if constexpr (D == 128) {
                    v[t][j][0] = *reinterpret_cast<const u32x4*>(p + 16 * i);
                } else {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(p + 8 * i);
                    v[t][j][0] = u32x4{x[0], x[1], 0, 0};
                }
            }
    }
    // 4-bit codes to bf16: eight channels of dword `w` under scale byte b.
    __device__ static u32x4 expand(uint32_t w, uint32_t b) {
        const float s = block_scale(b);
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3))};
    }
    __device__ void expand_values() {
        if constexpr (CT == PKV_FP4)
            for (int t = 0; t < kSub; ++t)
                for (int j = 0; j < 4; ++j) v[t][j][0] = expand(v[t][j][0][0], vs[t][j]);
    }
    // Infinities and NaN among slot j of piece t's values to 0; true if the lane had any.
    __device__ bool clean(int t, int j) {
        bool odd = false;
        for (int q = 0; q < kVRegs; ++q)
            for (int w = 0; w < 4; ++w) {
                uint32_t y = v[t][j][q][w];
                if constexpr (CT == PKV_F32) y = (y & 0x7f800000u) == 0x7f800000u ? 0 : y;
                else if (w < kPer / 2) y = finite_or_0<mat_type(CT)>(y);
                odd |= y != v[t][j][q][w];
                v[t][j][q][w] = y;
            }
        return odd;
    }
    // The value that output register (e, r) of lane group g meets, of the row whose bytes are at `p` (scales `sp`).
    __device__ static float value(const uint8_t* p, const uint8_t* sp, int e, int r, uint32_t g) {
        const uint32_t d = out_channel(e, r, g);
        if constexpr (CT == PKV_F32) return reinterpret_cast<const float*>(p)[d];
        else if constexpr (CT == PKV_FP4)
            return __uint_as_float(expand(p[d / 2] >> d % 2 * 4, sp[d / 32])[0] << 16);
        else return static_cast<float>(reinterpret_cast<const typename Elem<CT>::T*>(p)[d]);
    }
    __device__ static uint32_t out_channel(int e, int r, uint32_t g) {
        return CT == PKV_F32 ? 64 * (e / 4) + 4 * (4 * g + r) + e % 4 : kPer * (4 * g + r) + e;
    }
    // The channel that word `word` of step `s` of a lane's keys starts at (two channels a word, 16-bit types).
    __device__ static uint32_t channel(int s, uint32_t g) {
        return CT == PKV_FP4 ? (D / 4) * g + 8 * s : CT == PKV_F32 ? 16 * s + 4 * g : 32 * s + 8 * g;
    }
};

struct Partial {
    float* o;        // [copy][kv head][split][rows][D]
    float* ml;       // [copy][kv head][split][rows][2]: base, sum of the weights
    float* logits;   // [copy][kv head][rows x group][ld], unscaled (few rows)
    uint32_t splits, ld, rows;
};

template <int CT, int QT, int D, bool LOGITS>
__global__ __launch_bounds__(256, 2) void decode_kernel(AttendDev a, Partial part) {
    using T = typename Elem<QT>::T;
    using Tile = SlotTile<CT, D>;
    constexpr int MT = mat_type(CT), NQ = query_terms(CT, QT), NP = QT == PKV_F32 ? 3 : 2, kSub = Tile::kSub;
    constexpr int kQ = CT == PKV_F32 ? D / 16 : D / 32;          // query registers (16 bytes) per term
    constexpr int kO = D / 16;                                   // 16-channel tiles of the output
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t split = blockIdx.x % part.splits, ch = blockIdx.x / part.splits, c = ch / a.heads, h = ch % a.heads;
    const uint32_t row = lane % 16, g = lane / 16;
    const Span sp = span(a, c);
    const int R = sp.rows * static_cast<int>(a.group);
    const int pos1 = sp.first + sp.rows - 1;
    const bool real = static_cast<int>(row) < R;
    const int qi = row / a.group, pos = real ? sp.first + qi : -1;
    const Tiles tl = tiles_of(a, sp.first, sp.rows ? pos1 : -1, Tile::kStep);
    const int per = (tl.count + part.splits - 1) / part.splits;
    const int t0 = split * per, t1 = min(t0 + per, tl.count);

    const T* qp = reinterpret_cast<const T*>(a.q) + c * a.q_copy + (real ? qi : 0) * a.q_row +
                  (h * a.group + (real ? row % a.group : 0)) * a.q_head;
    u32x4 q[NQ][kQ];
    for (int s = 0; s < kQ; ++s) {
        const uint32_t d = Tile::channel(s, g);
        if constexpr (CT == PKV_F32) {
            q[0][s] = real ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{};
        } else if constexpr (NQ == 1) {
            q[0][s] = real ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{};
        } else {
            for (int w = 0; w < 4; ++w) {
                float x = real ? static_cast<float>(qp[d + 2 * w]) : 0.0f;
                float y = real ? static_cast<float>(qp[d + 2 * w + 1]) : 0.0f;
                for (int n = 0; n < NQ; ++n) q[n][s][w] = pack_query_term(x, y);
            }
        }
    }

    const uint64_t head = c * a.kv.copy + h * a.kv.head;
    const uint64_t byte = CT == PKV_FP4 ? head / 2 : CT == PKV_F32 ? head * 4 : head * 2;
    const uint8_t *kp = a.kv.k + byte, *vp = a.kv.v + byte;
    const uint8_t *ksp = CT == PKV_FP4 ? a.kv.ks + head / 32 : nullptr;
    const uint8_t *vsp = CT == PKV_FP4 ? a.kv.vs + head / 32 : nullptr;

    float base = kInf, l = 0.0f;
    f32x4 o[kO] = {};
    auto fetch = [&](Tile& x, int t) {   // past the last tile: the last again, unused
        x.load(kp, vp, ksp, vsp, a.kv.slot, tl.slot(min(t, t1 - 1), Tile::kStep), tl.high - 1, lane);
    };
    auto work = [&](Tile& x, int t, auto again) {
        constexpr bool CLEAN = decltype(again)::value;   // infinities and NaN of the values by themselves
        const int slot = tl.slot(t, Tile::kStep);
        // logits
        f32x4 sc[kSub] = {};
        for (int u = 0; u < kSub; ++u)
            for (int s = 0; s < kQ; ++s) {
                if constexpr (CT == PKV_F32) {
                    for (int e = 0; e < 4; ++e)
                        sc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[u][s][e]),
                                                                     __uint_as_float(q[0][s][e]), sc[u], 0, 0, 0);
                } else {
                    const u32x4 ka = CT == PKV_FP4 ? Tile::expand(x.k[u][0][s], x.ks[u]) : x.k[u][s];
                    for (int n = NQ - 1; n >= 0; --n) sc[u] = mma16<MT>(ka, q[n][s], sc[u]);
                }
            }
        const bool full = all_visible(a, sp.first, pos1, slot, slot + Tile::kStep - 1);
        if (LOGITS && !CLEAN && real)
            for (int u = 0; u < kSub; ++u)
                *reinterpret_cast<f32x4*>(part.logits + (static_cast<uint64_t>(ch) * a.nq * a.group + row) * part.ld +
                                          slot + 16 * u + 4 * g) = sc[u];
        x.expand_values();
        if (!full) {
            for (int u = 0; u < kSub; ++u)
                for (int j = 0; j < 4; ++j) {
                    const int key = slot + 16 * u + 4 * static_cast<int>(g) + j;
                    if (!visible(a, pos, key)) sc[u][j] = -kInf;
                    if (!any_visible(a, tl, key))
                        for (int n = 0; n < Tile::kVRegs; ++n) x.v[u][j][n] = u32x4{};
                }
        }
        bool odd[kSub][4] = {};
        if constexpr (CLEAN)
            for (int u = 0; u < kSub; ++u)
                for (int j = 0; j < 4; ++j) odd[u][j] = x.clean(u, j);
        float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
        for (int u = 1; u < kSub; ++u)
            top = fmaxf(top, fmaxf(fmaxf(sc[u][0], sc[u][1]), fmaxf(sc[u][2], sc[u][3])));
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
        float p[kSub][4];
        for (int u = 0; u < kSub; ++u)
            for (int j = 0; j < 4; ++j) {
                p[u][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][j], a.scale2, from));
                if constexpr (CLEAN) p[u][j] *= kPower<-kDown<MT>>;
                l += p[u][j];
            }
        // weighted values
        if constexpr (CT == PKV_F32) {
            for (int j = 0; j < 4; ++j)
                for (int n = 0; n < Tile::kVRegs; ++n)
                    for (int e = 0; e < 4; ++e)
                        o[4 * n + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[0][j][n][e]), p[0][j],
                                                                            o[4 * n + e], 0, 0, 0);
        } else {
            float r[kSub][4];
            for (int u = 0; u < kSub; ++u)
                for (int j = 0; j < 4; ++j) r[u][j] = p[u][j];
            u32x4 pt[NP];
            for (int n = 0; n < NP; ++n)
                pt[n] = u32x4{pack_term<MT>(r[0][0], r[0][1]), pack_term<MT>(r[0][2], r[0][3]),
                              pack_term<MT>(r[1][0], r[1][1]), pack_term<MT>(r[1][2], r[1][3])};
            for (int e = 0; e < kO; ++e) {
                const uint32_t sel = e % 2 ? 0x07060302u : 0x05040100u;
                const u32x4 va = {__builtin_amdgcn_perm(x.v[0][1][0][e / 2], x.v[0][0][0][e / 2], sel),
                                  __builtin_amdgcn_perm(x.v[0][3][0][e / 2], x.v[0][2][0][e / 2], sel),
                                  __builtin_amdgcn_perm(x.v[1][1][0][e / 2], x.v[1][0][0][e / 2], sel),
                                  __builtin_amdgcn_perm(x.v[1][3][0][e / 2], x.v[1][2][0][e / 2], sel)};
                for (int n = NP - 1; n >= 0; --n) o[e] = mma16<MT>(va, pt[n], o[e]);
            }
        }
        if constexpr (CLEAN)
            for (int u = 0; u < kSub; ++u)
                for (int j = 0; j < 4; ++j) {
                    const uint64_t has = __ballot(odd[u][j]);
#pragma unroll 1
                    for (uint32_t g2 = 0; g2 < 4; ++g2) {
                        if (!(has >> 16 * g2 & 0xffff)) continue;
                        const int key = slot + 16 * u + 4 * static_cast<int>(g2) + j;
                        const bool sees = real && visible(a, pos, key);
                        // not scaled down: that could make it 0
                        const float w = __shfl(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][j], a.scale2, from)),
                                               static_cast<int>(16 * g2 + row));
                        const uint64_t at = static_cast<uint64_t>(key) * a.kv.slot;
                        const uint8_t* vr = vp + (CT == PKV_FP4 ? at / 2 : CT == PKV_F32 ? at * 4 : at * 2);
                        for (int e = 0; e < kO; ++e)
                            for (int r = 0; r < 4; ++r) {
                                const float v = Tile::value(vr, CT == PKV_FP4 ? vsp + at / 32 : nullptr, e, r, g);
                                if (sees && (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[e][r] += w * v;
                            }
                    }
                }
    };
    // two tiles in turn: one is on its way while the other is worked on
    const int first = t0 + static_cast<int>(wave);
    if (first < t1) {
        Tile even, odd;
        fetch(even, first);
        for (int t = first; t < t1; t += 8) {
            fetch(odd, t + 4);
            work(even, t, std::false_type());
            if (t + 4 >= t1) break;
            fetch(even, t + 8);
            work(odd, t + 4, std::false_type());
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
            for (int t = first; t < t1; t += 4) {
                fetch(even, t);
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

    // the four waves' shares joined
    __shared__ float so[4][16][D + 4], sb[4][16], sl[4][16];
    for (int r = 0; r < 4; ++r)
        for (int e = 0; e < kO; ++e) {
            so[wave][row][Tile::out_channel(e, r, g)] = o[e][r];
        }
    if (g == 0) { sb[wave][row] = base; sl[wave][row] = l; }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < static_cast<uint32_t>(R) * (D / 4); x += 256) {
        const uint32_t r = x / (D / 4), d = x % (D / 4) * 4;
        const float low = fminf(fminf(sb[0][r], sb[1][r]), fminf(sb[2][r], sb[3][r]));
        float sum = 0.0f;
        f32x4 acc = {};
        for (int w = 0; w < 4; ++w) {
            const float f = joined(low, sb[w][r]);
            sum += sl[w][r] * f;
            acc += *reinterpret_cast<const f32x4*>(&so[w][r][d]) * (f * kPower<-kPartDown>);
        }
        const uint64_t at = (static_cast<uint64_t>(ch) * part.splits + split) * part.rows + r;
        *reinterpret_cast<f32x4*>(part.o + at * D + d) = acc;
        if (d == 0) {
            part.ml[2 * at] = low;
            part.ml[2 * at + 1] = sum;
        }
    }
}

// The splits of a row joined: the lowest base and the sum under it (a share
// without a logit has the sum 0, or NaN from NaN logits).
__device__ inline void join_splits(const float* ml, uint32_t splits, uint32_t rows, uint32_t lane, float* base,
                                   float* sum) {
    const uint64_t step = 2ull * rows;
    float low = kInf;
    for (uint32_t s = lane; s < splits; s += 64) low = fminf(low, ml[step * s]);
    for (int x = 32; x; x >>= 1) low = fminf(low, __shfl_xor(low, x));
    float l = 0.0f;
    for (uint32_t s = lane; s < splits; s += 64) l += ml[step * s + 1] * joined(low, ml[step * s]);
    *sum = wave_sum(l);
    *base = low;
}

// The splits' shares joined, a workgroup a row: every wave the row's base
// and sum, then 1024 / D shares at a time, 4 channels a thread.  With
// weights of few rows, then, a workgroup's rows of softmax statistics against
// the stored logits, four slots a thread.  blockIdx.x < outs: rows of all
// copies x heads; else 1,024 slots.
template <int QT, int D>
__global__ __launch_bounds__(256) void join_kernel(AttendDev a, Partial part, uint32_t outs) {
    using T = typename Elem<QT>::T;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, all = a.nq * a.group;
    if (blockIdx.x < outs) {
        const uint32_t r = blockIdx.x % all, ch = blockIdx.x / all, c = ch / a.heads, h = ch % a.heads;
        const uint32_t i = r / a.group, g = r % a.group;
        if (static_cast<int>(i) >= span(a, c).rows) return;
        const uint64_t at = static_cast<uint64_t>(ch) * part.splits * part.rows + r;
        constexpr uint32_t kLanes = D / 4, kShares = 256 / kLanes;
        const uint32_t first = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
        float base, sum;
        join_splits(part.ml + 2 * at, part.splits, part.rows, lane, &base, &sum);
        f32x4 o = {};
        for (uint32_t s = first; s < part.splits; s += kShares) {
            const uint64_t x = at + static_cast<uint64_t>(part.rows) * s;
            const float f = joined(base, part.ml[2 * x]) * kPower<-kJoinDown>;
            o += *reinterpret_cast<const f32x4*>(part.o + x * D + d) * f;
        }
        __shared__ f32x4 so[256];
        so[threadIdx.x] = o;
        __syncthreads();
        if (first == 0) {
            for (uint32_t s = 1; s < kShares; ++s) o += so[threadIdx.x + s * kLanes];
            T* out = reinterpret_cast<T*>(a.out) + c * a.o_copy + i * a.o_row + (h * a.group + g) * a.o_head;
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 y;
            const float div = sum * kPower<-kPartDown - kJoinDown>;
            for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(sum == 0.0f ? 0.0f : o[e] / div);
            *reinterpret_cast<T4*>(out + d) = y;
        }
        if (threadIdx.x == 0) {
            if (a.lse)
                a.lse[(static_cast<uint64_t>(c) * a.heads * a.group + h * a.group + g) * a.nq + i] = lse_of(base, sum);
            if (a.stats) stats_of(base, sum, a.stats + 2 * (static_cast<uint64_t>(ch) * all + r));
        }
        return;
    }
    const uint32_t chunks = (a.max_len + 1023) / 1024;
    const uint32_t x = blockIdx.x - outs, chunk = x % chunks, ch = x / chunks, c = ch / a.heads, h = ch % a.heads;
    const Span sp = span(a, c);
    const int j0 = chunk * 1024, rows = sp.rows * static_cast<int>(a.group);
    const Tiles tl = tiles_of(a, sp.first, sp.rows ? sp.first + sp.rows - 1 : -1, 1);
    if (j0 >= tl.high || (j0 + 1023 < tl.low && static_cast<uint32_t>(j0) >= a.sinks)) return;
    __shared__ float st[16][2];
    for (int r = wave; r < rows; r += 4) {
        float base, sum;
        join_splits(part.ml + 2 * (static_cast<uint64_t>(ch) * part.splits * part.rows + r), part.splits, part.rows,
                    lane, &base, &sum);
        if (lane == 0) stats_of(base, sum, st[r]);
    }
    __syncthreads();
    const int j = j0 + 4 * static_cast<int>(threadIdx.x);
    if (j >= tl.high) return;
    float w[4] = {};
    for (int r = 0; r < rows; ++r) {
        const int pos = sp.first + r / static_cast<int>(a.group);
        // reads up to three logits that no tile wrote: unused
        const f32x4 s = *reinterpret_cast<const f32x4*>(part.logits + (static_cast<uint64_t>(ch) * all + r) * part.ld + j);
        for (int e = 0; e < 4; ++e)
            if (visible(a, pos, j + e) && st[r][1] != 0.0f)
                w[e] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.scale2, st[r][0])) * st[r][1];
    }
    float* out = a.weights + c * a.w_copy + h * a.w_head + j;
    for (int e = 0; e < 4; ++e)
        if (any_visible(a, tl, j + e)) out[e] += w[e];
}

// ------------------------------------------------------------ many rows: tiles of rows through LDS
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

// A tile of slots in LDS: keys [slot][D], then values [slot][D], 4-bit codes
// as bf16, in 16-byte pieces at piece ^ turn(slot) so that no read meets a bank
// conflict: an operand of the first product is one piece of 32 slots, one of
// the second 4 slots x 16 channels, transposed by the read itself
// (ds_read_tr16_b64; f32: 32 channels of a slot, no transposition).  f32 keys
// meet two lanes a bank: their products take four times longer than the read.
// 16- and 32-bit rows go from memory to LDS without registers; a lane reads
// the piece that its place holds.
template <int CT, int D>
struct Stage {
    static constexpr int kSlots = CT == PKV_F32 ? 32 : 64;
    static constexpr int kRow = CT == PKV_F32 ? D * 4 : D * 2, kPieces = kRow / 16;
    static constexpr int kKeyBytes = kSlots * kRow, kBytes = 2 * kKeyBytes;
    static constexpr int kCopies = kKeyBytes / 4096;            // wave-wide copies of 1,024 bytes, a side
    static constexpr int kCopyRows = 1024 / kRow, kCopyStep = 4 * kCopyRows;
    u32x4 k, v;                                                 // 4-bit codes on their way
    uint32_t ks, vs;

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
    // The slot that thread t's 4-bit codes belong to, 16 a wave: 16 lanes write 16 different places of the banks.
    __device__ static uint32_t code_slot(uint32_t t) {
        const uint32_t i = t % 64;
        return t / 64 * 16 + (D == 128 ? i / 16 + i / 4 % 4 * 4 : i / 4 % 2 + i / 8 % 2 * 4 + i / 16 % 2 * 2 + i / 32 * 8);
    }

    // Start a tile on its way.  kp, vp, ksp, vsp: slot 0 of the head; slots past `last` read the last one.
    __device__ void fetch(uint32_t lds, const uint8_t* kp, const uint8_t* vp, const uint8_t* ksp, const uint8_t* vsp,
                          uint64_t stride, int slot, int last) {
        const uint64_t base = static_cast<uint64_t>(slot) * stride;
        const uint32_t st = static_cast<uint32_t>(stride);
        const int room = last - slot;
        if constexpr (CT == PKV_FP4) {
            const uint32_t t = threadIdx.x, b = t % 4;
            const uint32_t e = static_cast<uint32_t>(min(static_cast<int>(code_slot(t)), room)) * st;
            const uint8_t *kt = kp + base / 2 + e / 2, *vt = vp + base / 2 + e / 2;
            if constexpr (D == 128) {
                k = *reinterpret_cast<const u32x4*>(kt + 16 * b);
                v = *reinterpret_cast<const u32x4*>(vt + 16 * b);
            } else {
                const u32x2 x = *reinterpret_cast<const u32x2*>(kt + 8 * b), y = *reinterpret_cast<const u32x2*>(vt + 8 * b);
                k = u32x4{x[0], x[1], 0, 0};
                v = u32x4{y[0], y[1], 0, 0};
            }
            const uint64_t sb = base / 32 + e / 32 + (D == 128 ? b : b / 2);
            ks = ksp[sb];
            vs = vsp[sb];
        } else {
            constexpr uint32_t kSize = CT == PKV_F32 ? 4 : 2;
            const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
            // turn() of the row is the same for all of a lane's copies
            const uint32_t row = kCopyRows * wave + lane / kPieces, piece = lane % kPieces;
            const uint32_t kc = (piece ^ turn(row, false)) * 16, vc = (piece ^ turn(row, true)) * 16;
            const uint8_t *kt = kp + base * kSize, *vt = vp + base * kSize;
            for (int x = 0; x < kCopies; ++x) {
                const uint32_t e = min(kCopyStep * x + static_cast<int>(row), room) * st * kSize;
                const uint32_t to = lds + (kCopyStep * x + kCopyRows * wave) * kRow;
                copy_to_lds(to, kt, e + kc);
                copy_to_lds(to + kKeyBytes, vt, e + vc);
            }
        }
    }
    // What fetch started, into LDS (a barrier follows).
    __device__ void land(uint8_t* lds) {
        if constexpr (CT == PKV_FP4) {
            const uint32_t t = threadIdx.x, row = code_slot(t), b = t % 4;
            for (int w = 0; w < D / 32; ++w) {
                *reinterpret_cast<u32x4*>(lds + key_at(row, b * (D / 32) + w)) = SlotTile<CT, D>::expand(k[w], ks);
                *reinterpret_cast<u32x4*>(lds + value_at(row, b * (D / 32) + w)) = SlotTile<CT, D>::expand(v[w], vs);
            }
        } else {
            copies_done();
        }
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
        const u32x4 k = *reinterpret_cast<const u32x4*>(lds + Stage<CT, D>::key_at(32 * u + lane % 32, 2 * x + lane / 32));
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

// Query rows in tiles of 128, 32 a wave, against tiles of 64 slots (f32: 32)
// staged through LDS in two buffers, one barrier a tile:
//   S^T = K Q^T (32x32 tiles; a lane holds one query row and half of each
//   piece's slots), softmax in registers, O^T += V^T P^T with the rounded
//   weights straight from those registers.
// Weights of a 16-bit call are rounded once to its type, while their sum is that
// of the unrounded ones: a weight is off by up to half a step, so the output by
// up to half a step of sum w |v| beside its own rounding -- twice that rounding
// where one slot has nearly all the weight (measured at 64 rows on 2,048 slots
// of 128, logits of deviation 4: 1.2 half steps of sum w |v| in bf16 against
// 0.98 of decode_kernel's, 0.9 in f16 for both), 1.01 to 1.4 times in the mean
// square.  A second term costs half as much matrix work again, and a sum of the
// rounded weights for the output's divisor (0.97 half steps, the mean square of
// even weights as before) 2.5 % of a prompt's time.  Over 4-bit codes weights
// are as many bf16 terms as the query, one for bf16 queries.
// Bound at head_dim 128 by the matrix cores (a tile is 32 matrix instructions of
// 32 cycles a wave) together with the softmax beside them (32 exponentials of
// 16 cycles, about 160 other vector instructions).  Measured: 8,192 causal rows
// of 32 query heads of 128, bf16: 555 us, 990 TFLOP/s, where a library's square
// product of 8,192 reaches 1,216; a tile takes a workgroup 2.0 us alone on a CU
// and 2.2 beside another, so that calls with few workgroups are bound by that
// latency.  With tiles held in registers on their way to LDS it took 1.93 ms:
// what no longer fitted was reloaded behind the prefetch.
// KS 2: a workgroup has 64 rows and two waves share a tile's slots (1.1 us a
// tile), for calls whose 128-row tiles would not fill the chip.
//
// A weight 0 times an infinity or NaN would be NaN in rows that do not see the
// slot.  The loop does not look for those: an output that is not finite sends
// the workgroup through it again, with infinities and NaN taken out of the
// staged values and each added afterwards to the rows that see it.  Where the
// sums of finite values are not finite either, a third time with smaller
// weights (kDown).
template <int CT, int QT, int D, int KS>
__global__ __launch_bounds__(256, (query_terms(CT, QT) * D >= 256 ? 1 : 2)) void rows_kernel(AttendDev a, Partial part,
                                                                                        uint32_t row_tiles) {
    __shared__ __align__(16) uint8_t lds[2 * Stage<CT, D>::kBytes];
    using T = typename Elem<QT>::T;
    using St = Stage<CT, D>;
    constexpr int MT = mat_type(CT), kU = St::kSlots / 32 / KS, kO = D / 32;   // kU: 32-slot pieces a wave takes of a tile
    constexpr int NP = CT == PKV_FP4 ? query_terms(CT, QT) : 1;
    constexpr uint32_t kRowTile = row_tile(KS);
    const uint32_t lane = threadIdx.x % 64, wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = lane % 32, half = lane / 32;
    const uint32_t wave = wave_id % (4 / KS);                     // its 32 rows
    const int share = static_cast<int>(wave_id / (4 / KS)) * 32 * kU;   // its slots of a tile: share .. + 32 kU
    // heads fastest, so that a head's workgroups share an XCD's L2 where the heads are a multiple of 8; row tiles
    // from the last, whose rows see most
    const uint32_t heads = a.copies * a.heads;
    const uint32_t ch = blockIdx.x % heads, c = ch / a.heads, h = ch % a.heads;
    const uint32_t split = blockIdx.x / heads % part.splits, tile = row_tiles - 1 - blockIdx.x / heads / part.splits;
    const Span sp = span(a, c);
    const int R = sp.rows * static_cast<int>(a.group), r0 = static_cast<int>(tile * kRowTile), G = static_cast<int>(a.group);
    if (r0 >= R) return;
    const int last = min(r0 + static_cast<int>(kRowTile), R) - 1;
    const int pos0 = sp.first + r0 / G, pos1 = sp.first + last / G;
    const Tiles tl = tiles_of(a, pos0, pos1, St::kSlots);
    const int per = (tl.count + static_cast<int>(part.splits) - 1) / static_cast<int>(part.splits);
    const int t0 = static_cast<int>(split) * per, t1 = min(t0 + per, tl.count);

    const int w0 = r0 + 32 * static_cast<int>(wave), w1 = min(w0 + 31, last), r = w0 + static_cast<int>(n);
    const bool real = r <= last;
    const int qi = (real ? r : last) / G, pos = real ? sp.first + qi : -1;
    const int wpos0 = sp.first + w0 / G, wpos1 = sp.first + w1 / G;   // of the wave's rows (w0 > last: none)
    const Tiles wt = tiles_of(a, wpos0, w0 <= last ? wpos1 : -1, 1);
    Query<CT, QT, D> q;
    q.load(reinterpret_cast<const T*>(a.q) + c * a.q_copy + qi * a.q_row + (h * a.group + (real ? r : last) % G) * a.q_head,
           real, half);

    const uint64_t head = c * a.kv.copy + h * a.kv.head;
    const uint64_t byte = CT == PKV_FP4 ? head / 2 : CT == PKV_F32 ? head * 4 : head * 2;
    const uint8_t *kp = a.kv.k + byte, *vp = a.kv.v + byte;
    const uint8_t *ksp = CT == PKV_FP4 ? a.kv.ks + head / 32 : nullptr;
    const uint8_t *vsp = CT == PKV_FP4 ? a.kv.vs + head / 32 : nullptr;

    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte*)lds));
    float base, l;
    f32x16 o[kO];
    St st;
    auto fetch = [&](int t) {
        st.fetch(at + ((t - t0) & 1) * St::kBytes, kp, vp, ksp, vsp, a.kv.slot, tl.slot(t, St::kSlots), tl.high - 1);
    };
    // no row of the wave sees any of the tile
    auto skip = [&](int slot) {
        return slot + share >= wt.high ||
               (slot + share + 32 * kU <= wt.low && static_cast<uint32_t>(slot + share) >= a.sinks);
    };
    float lift = kLift<MT>;
    for (int pass = 0;; ++pass) {
        base = kInf;
        l = 0.0f;
        for (int e = 0; e < kO; ++e) o[e] = f32x16{};
        if (t0 < t1) {
            fetch(t0);
            st.land(lds);
        }
        __syncthreads();
        for (int t = t0; t < t1; ++t) {
            uint8_t* buf = lds + ((t - t0) & 1) * St::kBytes;
            if (t + 1 < t1) fetch(t + 1);
            const int slot = tl.slot(t, St::kSlots);
            if (__builtin_expect(pass, 0)) {
                St::clean(buf);
                __syncthreads();
            }
            if (!skip(slot)) {
                f32x16 sc[kU];
                const int mine = slot + share;
                for (int u = 0; u < kU; ++u) sc[u] = logits32<CT, QT, D>(buf + share * St::kRow, u, q, lane);
                if (!all_visible(a, wpos0, wpos1, mine, mine + 32 * kU - 1)) {
                    const int off = pos - mine - 4 * static_cast<int>(half);   // less the register's place: how far back
                    if (static_cast<uint32_t>(mine) >= a.sinks) {
                        for (int u = 0; u < kU; ++u)
                            for (int x = 0; x < 16; ++x)
                                if (!in_reach(a, off, 32 * u + row32(x, 0))) sc[u][x] = -kInf;
                    } else {
                        for (int u = 0; u < kU; ++u)
                            for (int x = 0; x < 16; ++x)
                                if (!visible(a, pos, mine + 32 * u + row32(x, half))) sc[u][x] = -kInf;
                    }
                }
                float top = sc[0][0];
                for (int u = 0; u < kU; ++u)
                    for (int x = 0; x < 16; ++x) top = fmaxf(top, sc[u][x]);
                top = across32(top, larger);
                if (__any(__builtin_fmaf(top, a.scale2, base) > lift + kLag<MT>)) {
                    const float low = lower_base(a, lift, base, top), f = joined(low, base);
                    if (low < base) {
                        l *= f;
                        for (int e = 0; e < kO; ++e) o[e] *= f;
                        base = low;
                    }
                }
                const float from = base == kInf ? 0.0f : base;
                for (int u = 0; u < kU; ++u)
                    for (int x = 0; x < 16; ++x) {
                        sc[u][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][x], a.scale2, from));
                        l += sc[u][x];
                    }
                // ahead of the other workgroup's softmax while the matrix cores have work: 573 -> 565 us (8,192 rows)
                __builtin_amdgcn_s_setprio(1);
                for (int u = 0; u < kU; ++u) {
                    if constexpr (CT == PKV_F32) {
                        for (int x = 0; x < 16; ++x)
                            for (int e = 0; e < kO; ++e)
                                o[e] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                                    *reinterpret_cast<const float*>(
                                        buf + St::value32_at(32 * u + row32(x, half), 32 * e + n)),
                                    sc[u][x], o[e], 0, 0, 0);
                    } else {
                        for (int y = 0; y < 2; ++y) {
                            float p[8];
                            for (int x = 0; x < 8; ++x) p[x] = sc[u][8 * y + x];
                            u32x4 pt[NP];
                            for (int k = 0; k < NP; ++k)
                                pt[k] = u32x4{pack_term<MT>(p[0], p[1]), pack_term<MT>(p[2], p[3]),
                                              pack_term<MT>(p[4], p[5]), pack_term<MT>(p[6], p[7])};
                            for (int e = 0; e < kO; ++e) {
                                const u32x4 v = St::values16(buf + share * St::kRow, 32 * u + 16 * y, e, lane);
                                for (int k = NP - 1; k >= 0; --k) o[e] = mma32<MT>(v, pt[k], o[e]);
                            }
                        }
                    }
                }
            }
            __builtin_amdgcn_s_setprio(0);
            if (t + 1 < t1) st.land(lds + ((t + 1 - t0) & 1) * St::kBytes);
            __syncthreads();
        }
        if (pass < 2) {
            bool odd = false;
            for (int e = 0; e < kO; ++e)
                for (int x = 0; x < 16; ++x) odd |= (__float_as_uint(o[e][x]) & 0x7f800000u) == 0x7f800000u;
            // with the values finite, from a NaN among the logits, as the weights' sum, or past the type's end
            if (pass) odd &= !__builtin_isnan(across32(l, [](float x, float y) { return x + y; }));
            const bool again = __syncthreads_or(odd && real);
            if (!pass && !again) break;
            if (!pass) continue;
            if (again && kDown<MT>) {
                lift -= kDown<MT>;
                continue;
            }
        }
        // not scaled down: that could make a weight 0
        const float from = base == kInf ? 0.0f : base + (kLift<MT> - lift);
#pragma unroll 1
        for (int t = t0; t < t1; ++t) {
            const int slot = tl.slot(t, St::kSlots);
            uint8_t* buf = lds + ((t - t0) & 1) * St::kBytes;
            fetch(t);
            st.land(buf);
            __syncthreads();
            if (!__syncthreads_or(St::clean(buf))) continue;
            fetch(t);
            st.land(buf);
            __syncthreads();
#pragma unroll 1
            for (int j = share; j < share + 32 * kU; ++j) {
                const bool sees = visible(a, pos, slot + j);
                if (!__any(sees)) continue;
                uint32_t hf = half;
                asm volatile("" : "+v"(hf));   // this rare loop's addresses are not kept over the main one
                float dot = 0.0f;
                for (int x = 0; x < Query<CT, QT, D>::kRegs; ++x) {
                    const u32x4 k = *reinterpret_cast<const u32x4*>(buf + St::key_at(j, 2 * x + hf));
                    for (int w = 0; w < 4; ++w)
                        for (int y = 0; y < Query<CT, QT, D>::kTerms; ++y) dot += dot_word<MT>(k[w], q.q[y][x][w]);
                }
                dot += __shfl_xor(dot, 32);
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(dot, a.scale2, from));
                for (int e = 0; e < kO; ++e)
                    for (int x = 0; x < 16; ++x) {
                        const float v = St::value(buf, j, 32 * e + row32(x, hf));
                        if (sees && (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[e][x] += p * v;
                    }
            }
            __syncthreads();
        }
        break;
    }
    l += __shfl_xor(l, 32);
    constexpr int kShared = KS > 1 ? 1 : 0;   // outputs are 2^-kShared as large from here on
    if constexpr (KS > 1) {
        // the other share of the slots joins the first: [row block][o, base, l][lane]
        float* to = reinterpret_cast<float*>(lds) + wave * (16 * kO + 2) * 64 + lane;
        if (share) {
            for (int x = 0; x < 16 * kO; ++x) to[x * 64] = o[x / 16][x % 16];
            to[16 * kO * 64] = base;
            to[(16 * kO + 1) * 64] = l;
        }
        __syncthreads();
        if (share) return;
        const float base2 = to[16 * kO * 64], low = fminf(base, base2);
        const float f = joined(low, base), f2 = joined(low, base2);
        const float of = f * kPower<-kShared>, of2 = f2 * kPower<-kShared>;
        base = low;
        l = l * f + to[(16 * kO + 1) * 64] * f2;
        for (int x = 0; x < 16 * kO; ++x) o[x / 16][x % 16] = o[x / 16][x % 16] * of + to[x * 64] * of2;
    }
    if (!real) return;
    const uint64_t all = static_cast<uint64_t>(a.nq) * a.group;
    if (part.splits > 1) {
        const uint64_t at = (static_cast<uint64_t>(ch) * part.splits + split) * part.rows + r;
        for (int e = 0; e < kO; ++e)
            for (int x = 0; x < 4; ++x)
                *reinterpret_cast<f32x4*>(part.o + at * D + 32 * e + 8 * x + 4 * half) =
                    f32x4{o[e][4 * x], o[e][4 * x + 1], o[e][4 * x + 2], o[e][4 * x + 3]} * kPower<kShared - kPartDown>;
        if (half == 0) {
            part.ml[2 * at] = base;
            part.ml[2 * at + 1] = l;
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l * kPower<kShared>;
    const uint32_t g = static_cast<uint32_t>(r % G);
    T* out = reinterpret_cast<T*>(a.out) + c * a.o_copy + qi * a.o_row + (h * a.group + g) * a.o_head;
    for (int e = 0; e < kO; ++e)
        for (int x = 0; x < 4; ++x) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 y;
            for (int k = 0; k < 4; ++k) y[k] = static_cast<T>(l == 0.0f ? 0.0f : o[e][4 * x + k] * inv);
            *reinterpret_cast<T4*>(out + 32 * e + 8 * x + 4 * half) = y;
        }
    if (half == 0) {
        if (a.lse)
            a.lse[(static_cast<uint64_t>(c) * a.heads * a.group + h * a.group + g) * a.nq + qi] = lse_of(base, l);
        if (a.stats) stats_of(base, l, a.stats + 2 * (ch * all + r));
    }
    return;
}

// rows_kernel's shares joined: D / 4 lanes a row, this many rows a workgroup.
constexpr uint32_t join_rows(uint32_t dim) { return 1024 / dim; }
template <int QT, int D>
__global__ __launch_bounds__(256) void join_rows_kernel(AttendDev a, Partial part) {
    using T = typename Elem<QT>::T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr uint32_t kLanes = D / 4, kRows = join_rows(D);
    const uint32_t all = a.nq * a.group, blocks = (all + kRows - 1) / kRows, ch = blockIdx.x / blocks;
    const uint32_t r = blockIdx.x % blocks * kRows + threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
    const uint32_t c = ch / a.heads, h = ch % a.heads, i = r / a.group, g = r % a.group;
    if (static_cast<int>(i) >= span(a, c).rows || r >= all) return;
    const uint64_t at = static_cast<uint64_t>(ch) * part.splits * part.rows + r;
    float base = kInf, sum = 0.0f;
    for (uint32_t s = 0; s < part.splits; ++s)
        base = fminf(base, part.ml[2 * (at + static_cast<uint64_t>(part.rows) * s)]);
    f32x4 o = {};
    for (uint32_t s = 0; s < part.splits; ++s) {
        const uint64_t x = at + static_cast<uint64_t>(part.rows) * s;
        const float f = joined(base, part.ml[2 * x]);
        sum += part.ml[2 * x + 1] * f;
        o += *reinterpret_cast<const f32x4*>(part.o + x * D + d) * (f * kPower<-kJoinDown>);
    }
    T4 y;
    const float div = sum * kPower<-kPartDown - kJoinDown>;
    for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(sum == 0.0f ? 0.0f : o[e] / div);
    *reinterpret_cast<T4*>(reinterpret_cast<T*>(a.out) + c * a.o_copy + i * a.o_row + (h * a.group + g) * a.o_head + d) = y;
    if (d == 0) {
        if (a.lse)
            a.lse[(static_cast<uint64_t>(c) * a.heads * a.group + h * a.group + g) * a.nq + i] = lse_of(base, sum);
        if (a.stats) stats_of(base, sum, a.stats + 2 * (static_cast<uint64_t>(ch) * all + r));
    }
}

// left[0 .. N) = the half of left[0 .. 2N) that the lane keeps (upper: the
// second) and the lane across's share of it.
template <int CTRL, int N>
__device__ inline void hand_over(float (&left)[16], bool upper) {
    for (int x = 0; x < N; ++x) {
        const float keep = upper ? left[x + N] : left[x], give = upper ? left[x] : left[x + N];
        left[x] = keep + __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(give), CTRL, 15, 15, true));
    }
}

// Accumulated weights of many rows: 32 slots a wave, its keys held in registers
// as the S^T operand, all rows that can see them streamed through LDS (four
// waves share them) 64 at a time (queries of more than one term: 32), straight
// from memory while the rows before are worked on; every slot belongs to one
// wave, so sums have one order.  S^T, one multiply-add, one exponential and one
// more multiply-add a logit: half of rows_kernel's matrix work, its softmax
// work without maximum and rounding.  Measured: 3 x 701 rows of 24 query heads of
// 64, window 1,024, f16: 26 us (89 with rows read when they were needed, 48 with
// half as many shares), of which those vector instructions are about 6: bound by
// the latency of a step (copies drained and a barrier every 64 rows, about five
// steps a workgroup).
//
// With few blocks of slots their rows are cut into shares as well (splits > 1),
// whose sums go to `shares` [split][copy][kv head][ld] for add_weights_kernel.
struct Shares {
    float* sums;
    uint32_t splits, ld;
};
template <int CT, int QT, int D>
__global__ __launch_bounds__(256, 2) void weights_kernel(AttendDev a, Shares shares) {
    using T = typename Elem<QT>::T;
    using Q = Query<CT, QT, D>;
    using St = Stage<CT, D>;
    constexpr int MT = mat_type(CT), kPieces = St::kPieces, kTerms = Q::kTerms;
    constexpr int kRows = kTerms == 1 ? 64 : 32, kU = kRows / 32;
    constexpr uint32_t kTermBytes = kRows * St::kRow;
    __shared__ __align__(16) uint8_t lds[2][kTerms * kTermBytes];
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = lane % 32, half = lane / 32, heads = a.copies * a.heads;
    const uint32_t ch = blockIdx.x % heads, c = ch / a.heads, h = ch % a.heads;
    const uint32_t split = blockIdx.x / heads % shares.splits;
    const Span sp = span(a, c);
    // the grid's blocks are those that some row sees, the first ones and those of the window, of this copy's length
    const Tiles tl = tiles_of(a, sp.first, sp.rows ? sp.first + sp.rows - 1 : -1, 128);
    const int block = static_cast<int>(blockIdx.x / heads / shares.splits);
    if (block >= tl.count) return;
    const int G = static_cast<int>(a.group), b0 = tl.slot(block, 128), s0 = b0 + 32 * static_cast<int>(wave);
    const int high = tl.high;
    // rows i0 .. i1 see something of b0 .. b0 + 127
    const int i0 = max(b0 - sp.first, 0);
    const int64_t reach = !a.window || static_cast<uint32_t>(b0) < a.sinks
                              ? sp.rows - 1
                              : static_cast<int64_t>(b0) + 126 + a.window - sp.first;
    const int i1 = static_cast<int>(min(reach, static_cast<int64_t>(sp.rows - 1)));
    if (i0 > i1) return;
    const int per = ((i1 - i0 + 1) * G + kRows * static_cast<int>(shares.splits) - 1) / (kRows * static_cast<int>(shares.splits)) * kRows;
    const int r0 = i0 * G + static_cast<int>(split) * per, r1 = min(r0 + per, i1 * G + G);   // may be none

    // the wave's keys as operand A: slot n, channels as Query
    u32x4 k[Q::kRegs];
    {
        const uint64_t e = c * a.kv.copy + h * a.kv.head + static_cast<uint64_t>(min(s0 + static_cast<int>(n), high - 1)) * a.kv.slot;
        if constexpr (CT == PKV_FP4) {
            for (int s = 0; s < Q::kRegs; ++s) {
                const uint64_t x = e + 16 * s + 8 * half;
                k[s] = SlotTile<CT, D>::expand(*reinterpret_cast<const uint32_t*>(a.kv.k + x / 2), a.kv.ks[x / 32]);
            }
        } else {
            const uint8_t* p = a.kv.k + e * (CT == PKV_F32 ? 4 : 2);
            for (int s = 0; s < Q::kRegs; ++s) k[s] = *reinterpret_cast<const u32x4*>(p + 32 * s + 16 * half);
        }
    }
    const uint64_t all = static_cast<uint64_t>(a.nq) * a.group;
    const T* qp = reinterpret_cast<const T*>(a.q) + c * a.q_copy + static_cast<uint64_t>(h) * a.group * a.q_head;
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte*)&lds[0][0]));
    // Rows that this thread fetches a piece of: (row, head of the group) and where it is; a step of kRows rows without
    // dividing or multiplying again.
    struct At {
        int i, g;
        const T* p;
    };
    const int adv_i = kRows / G, adv_g = kRows % G;
    const int64_t adv = static_cast<int64_t>(adv_i) * a.q_row + static_cast<int64_t>(adv_g) * a.q_head;
    const int64_t wrap = static_cast<int64_t>(a.q_row) - static_cast<int64_t>(G) * a.q_head;
    auto step = [&](At x) {
        x.i += adv_i;
        x.g += adv_g;
        x.p += adv;
        if (x.g >= G) {
            x.g -= G;
            ++x.i;
            x.p += wrap;
        }
        return x;
    };
    const T* last_row = qp + static_cast<uint64_t>(i1) * a.q_row + static_cast<uint64_t>(G - 1) * a.q_head;
    constexpr int kCopies = kRows * St::kRow / 4096, kStep = St::kCopyStep;
    const uint32_t mine = kTerms == 1 ? St::kCopyRows * wave + lane / kPieces : threadIdx.x / kPieces;
    constexpr int kMoves = kTerms == 1 ? kCopies : kRows * kPieces / 256, kMoveStep = kTerms == 1 ? kStep : 256 / kPieces;
    At here[kMoves];
    for (int x = 0; x < kMoves; ++x) {
        const int row = static_cast<int>(mine) + kMoveStep * x;
        const int i = (r0 + row) / G, g = (r0 + row) % G;
        here[x] = At{i, g, qp + static_cast<uint64_t>(i) * a.q_row + static_cast<uint64_t>(g) * a.q_head};
    }
    u32x4 w[kTerms == 1 ? 1 : kMoves];      // a multi-term query on its way (f16: 8 values; f32: the first half)
    u32x4 w2[QT == PKV_F32 && kTerms > 1 ? kMoves : 1];
    auto fetch = [&](uint32_t b) {
        const uint32_t piece = (kTerms == 1 ? lane : threadIdx.x) % kPieces;
        for (int x = 0; x < kMoves; ++x) {
            const T* p = here[x].i <= i1 ? here[x].p : last_row;
            if constexpr (kTerms == 1) {
                const uint32_t row = mine + kStep * x;
                copy_row_to_lds(at + b * kTermBytes + (kStep * x + St::kCopyRows * wave) * St::kRow,
                                reinterpret_cast<const uint8_t*>(p) + (piece ^ St::turn(row, false)) * 16);
            } else {
                w[x] = reinterpret_cast<const u32x4*>(p + 8 * piece)[0];
                if constexpr (QT == PKV_F32) w2[x] = reinterpret_cast<const u32x4*>(p + 8 * piece)[1];
            }
            here[x] = step(here[x]);
        }
    };
    auto land = [&](uint32_t b) {
        if constexpr (kTerms == 1) {
            copies_done();
        } else {
            for (int x = 0; x < kMoves; ++x) {
                const uint32_t row = mine + kMoveStep * x, to = St::key_at(row, threadIdx.x % kPieces);
                u32x4 y[kTerms];
                for (int e = 0; e < 4; ++e) {
                    float f0, f1;
                    if constexpr (QT == PKV_F32) {
                        f0 = __uint_as_float(e < 2 ? w[x][2 * e] : w2[x][2 * e - 4]);
                        f1 = __uint_as_float(e < 2 ? w[x][2 * e + 1] : w2[x][2 * e - 3]);
                    } else {
                        const uint32_t word = w[x][e];   // not bit_cast of the element itself: that reads element 0
                        const f16x2 f = __builtin_bit_cast(f16x2, word);
                        f0 = static_cast<float>(f[0]);
                        f1 = static_cast<float>(f[1]);
                    }
                    for (int z = 0; z < kTerms; ++z) y[z][e] = pack_query_term(f0, f1);
                }
                for (int z = 0; z < kTerms; ++z) *reinterpret_cast<u32x4*>(lds[b] + z * kTermBytes + to) = y[z];
            }
        }
    };
    float sum[16] = {};
    typedef float f32x2u __attribute__((ext_vector_type(2)));
    const f32x2u* stats = reinterpret_cast<const f32x2u*>(a.stats) + ch * all;
    f32x2u next[kU], now[kU];
    if (r0 < r1) {
        fetch(0);
        for (int u = 0; u < kU; ++u) next[u] = stats[min(r0 + 32 * u + static_cast<int>(n), r1 - 1)];
        land(0);
    }
    __syncthreads();
    uint32_t b = 0;
    At top = {r0 / G, r0 % G, qp};           // of row r
    for (int r = r0; r < r1; r += kRows, b ^= 1) {
        for (int u = 0; u < kU; ++u) now[u] = next[u];
        if (r + kRows < r1) {
            fetch(b ^ 1);
            for (int u = 0; u < kU; ++u) next[u] = stats[min(r + kRows + 32 * u + static_cast<int>(n), r1 - 1)];
        }
        for (int u = 0; u < kU; ++u) {
            const int ru = r + 32 * u;
            if (ru >= r1) break;
            // positions of the piece's rows, from below and above
            const int pa = sp.first + top.i + (kU > 1 && u ? 32 / G : 0), pb = sp.first + top.i + (32 * u + 31 + G) / G;
            // none of them sees any of the wave's slots
            if (pb < s0 || (pa > s0 + 31 && !in_reach(a, pa, s0 + 31) && static_cast<uint32_t>(s0) >= a.sinks)) continue;
            f32x16 s = {};
            for (int x = 0; x < Q::kRegs; ++x)
                for (int z = kTerms - 1; z >= 0; --z) {
                    const u32x4 y = *reinterpret_cast<const u32x4*>(lds[b] + z * kTermBytes +
                                                                    St::key_at(32 * u + n, 2 * x + half));
                    if constexpr (CT == PKV_F32) {
                        for (int e = 0; e < 4; ++e)
                            s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[x][e]), __uint_as_float(y[e]), s,
                                                                     0, 0, 0);
                    } else {
                        s = mma32<MT>(k[x], y, s);
                    }
                }
            const float mc = now[u][0], inv = now[u][1];
            if (ru + 32 <= r1 && all_visible(a, pa, pb, s0, s0 + 31)) {
                for (int x = 0; x < 16; ++x)
                    sum[x] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[x], a.scale2, mc)), inv, sum[x]);
            } else {
                const int pos = sp.first + (ru + static_cast<int>(n)) / G;
                const bool in = (ru + static_cast<int>(n) < r1) & (inv != 0.0f);
                const bool sink = static_cast<uint32_t>(s0) < a.sinks;
                const int off = in ? pos - s0 - 4 * static_cast<int>(half) : -1;   // less the register's place: how far back
                for (int x = 0; x < 16; ++x) {
                    const float more = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[x], a.scale2, mc)), inv, sum[x]);
                    bool see = in_reach(a, off, row32(x, 0));
                    if (sink) see = in & visible(a, pos, s0 + row32(x, half));
                    sum[x] = see ? more : sum[x];
                }
            }
        }
        top = step(top);
        if (r + kRows < r1) land(b ^ 1);
        __syncthreads();
    }
    // Register n % 16 summed over the half's 32 lanes: each step hands half of the registers to the lane across and
    // keeps the other half, 16 to 1 over 16 lanes, then the other 16.
    float left[16];
    for (int x = 0; x < 16; ++x) left[x] = sum[x];
    hand_over<0x140, 8>(left, n & 8);        // row_mirror
    hand_over<0x141, 4>(left, n & 4);        // row_half_mirror
    hand_over<0x1b, 2>(left, n & 2);         // quad_perm 3 2 1 0
    hand_over<0xb1, 1>(left, n & 1);         // quad_perm 1 0 3 2
    const float total = across16(left[0], [](float x, float y) { return x + y; });
    const int j = s0 + row32(static_cast<int>(n), half);
    if (n >= 16 || !any_visible(a, tl, j)) return;
    if (shares.splits == 1) a.weights[c * a.w_copy + h * a.w_head + j] += total;
    else shares.sums[(static_cast<uint64_t>(split) * heads + ch) * shares.ld + j] = total;
}

// The shares of every slot that some row sees, in their order.
__global__ __launch_bounds__(256) void add_weights_kernel(AttendDev a, Shares shares, uint32_t blocks) {
    const uint32_t heads = a.copies * a.heads, ch = blockIdx.x / blocks, c = ch / a.heads, h = ch % a.heads;
    const int j = static_cast<int>(blockIdx.x % blocks * 256 + threadIdx.x);
    const Span sp = span(a, c);
    if (!sp.rows || !any_visible(a, tiles_of(a, sp.first, sp.first + sp.rows - 1, 1), j)) return;
    float sum = 0.0f;
    for (uint32_t s = 0; s < shares.splits; ++s) sum += shares.sums[(static_cast<uint64_t>(s) * heads + ch) * shares.ld + j];
    a.weights[c * a.w_copy + h * a.w_head + j] += sum;
}

// ------------------------------------------------------------ the 4-bit cache
struct Row {
    uint64_t src, dst;   // element offsets in the rows' tensor and in the cache
    bool there;
};
// Row `r` of all (copy, layer, head, i), i fastest.
__device__ inline Row row_of(const RowsDev& a, uint32_t r) {
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

// Pieces of the rows, in line, one a thread and step; both sides of the rows
// are blockIdx.y.  A store's piece is 8 values (4 threads a block, whose codes
// are one word), a load's 16 bytes of the tensor it writes (f32: 4 values; with
// 8 its 16-byte writes leave gaps between lanes: 147 us instead of 110 for the
// 200 MB of a 24-layer pool's 1,024 tokens).  Bound by the rows' bytes.
template <int QT, bool STORE> constexpr int kPiece = QT == PKV_F32 && !STORE ? 4 : 8;

template <int QT, int D>
__global__ __launch_bounds__(256) void fp4_store_kernel(RowsDev a, uint64_t pieces) {
    using T = typename Elem<QT>::T;
    constexpr int V = kPiece<QT, true>;
    typedef T Vec __attribute__((ext_vector_type(V)));
    const uint8_t* src = blockIdx.y ? a.values : a.keys;
    if (!src) return;
    uint8_t* dst = const_cast<uint8_t*>(blockIdx.y ? a.kv.v : a.kv.k);
    uint8_t* dsc = const_cast<uint8_t*>(blockIdx.y ? a.kv.vs : a.kv.ks);
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * 256;
    // `pieces` is a multiple of a block's, so that a block's threads leave together
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; t < pieces; t += step) {
        const Row o = row_of(a, static_cast<uint32_t>(t / (D / V)));
        const uint32_t d = t % (D / V) * V;
        const Vec in = *reinterpret_cast<const Vec*>(reinterpret_cast<const T*>(src) + o.src + d);
        float x[V];
        uint32_t top = 0;
        for (int e = 0; e < V; ++e) {
            x[e] = static_cast<float>(in[e]);
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
        if (!o.there) continue;
        reinterpret_cast<uint32_t*>(dst)[(o.dst + d) / 8] = codes;
        if (d % 32 == 0) dsc[(o.dst + d) / 32] = static_cast<uint8_t>(b);
    }
}

template <int QT, int D>
__global__ __launch_bounds__(256) void fp4_load_kernel(RowsDev a, uint64_t pieces) {
    using T = typename Elem<QT>::T;
    constexpr int V = kPiece<QT, false>;
    typedef T Vec __attribute__((ext_vector_type(V)));
    uint8_t* dst = blockIdx.y ? a.values : a.keys;
    if (!dst) return;
    const uint8_t* src = blockIdx.y ? a.kv.v : a.kv.k;
    const uint8_t* ssc = blockIdx.y ? a.kv.vs : a.kv.ks;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * 256;
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; t < pieces; t += step) {
        const Row o = row_of(a, static_cast<uint32_t>(t / (D / V)));
        const uint32_t d = t % (D / V) * V;
        uint32_t codes;                      // a row without a slot reads slot 0, and is 0
        if constexpr (V == 8) codes = reinterpret_cast<const uint32_t*>(src)[(o.dst + d) / 8];
        else codes = reinterpret_cast<const uint16_t*>(src)[(o.dst + d) / 4];
        const float s = block_scale(ssc[(o.dst + d) / 32]);
        f32x2 x[4];
        x[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0);
        x[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1);
        x[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2);
        x[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
        Vec y;
        for (int e = 0; e < V; ++e) y[e] = static_cast<T>(o.there ? x[e / 2][e % 2] : 0.0f);
        *reinterpret_cast<Vec*>(reinterpret_cast<T*>(dst) + o.src + d) = y;
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

constexpr int kSelect = 1024, kWaves = kSelect / 64;   // threads of select_kernel
constexpr int kHeld = 32;                              // weights a lane holds: 32,768 a workgroup

// The bin that holds the want-th largest key and how many lie above it, by the
// first wave: four bins a lane, counted from the top.
__device__ inline void find_bin(const uint32_t* hist, uint32_t want, uint32_t* found) {
    const uint32_t lane = threadIdx.x;
    uint32_t h[4], s = 0;
    for (int x = 0; x < 4; ++x) s += h[x] = hist[4 * lane + x];
    uint32_t up = s;                                   // of this lane's bins and all above
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_down(up, o);
        if (lane + o < 64) up += y;
    }
    uint32_t above = up - s;
    if (above < want && want <= up) {
        int x = 3;
        while (above + h[x] < want) above += h[x--];
        found[0] = 4 * lane + x;
        found[1] = above;
    }
}

// One workgroup per (head, layer, copy): the border among the middle slots by
// four passes over 8 bits of the key, then the kept slots in order.  Each wave
// has a run of slots, so that two counts a wave place every slot; up to 32,768
// slots are read once and held in registers.  A bin has 16 counts, by lane: the
// high bytes of weights are nearly all the same, and 64 lanes adding to one
// word would take their turns.  Bound by its instructions: six passes over 32
// weights a lane.  64 heads of 32,768 slots: 45 us (65 with one count a bin),
// 256 heads of 1,024: 10 us (43 with a serial search of the bins).
__global__ __launch_bounds__(kSelect) void select_kernel(EvictDev a) {
    const uint32_t h = blockIdx.x % a.heads, cl = blockIdx.x / a.heads, l = cl % a.layers, c = cl / a.layers;
    const uint32_t n = min(max(a.lens[c], 0), static_cast<int>(a.slots));
    const float* w = a.w + c * a.ws[0] + l * a.ws[1] + h * a.ws[2];
    float* wo = a.w_out + c * a.os[0] + l * a.os[1] + h * a.os[2];
    int32_t* kept = a.kept + static_cast<uint64_t>(blockIdx.x) * a.budget;
    const uint32_t keep = min(n, a.budget), t = threadIdx.x, lane = t % 64, wave = t / 64;
    constexpr uint32_t kCopies = 16;
    __shared__ __align__(16) uint32_t hist[256 * kCopies];
    __shared__ uint32_t total[256], sures[kWaves], ties[kWaves], found[2];
    static_assert(256 * kCopies == 4 * kSelect, "four counts a thread");
    if (l == 0 && h == 0 && t == 0) a.new_lens[c] = static_cast<int32_t>(keep);
    // the wave's slots: `run` from `from` on, 64 a step
    const uint32_t run = (n + kSelect - 1) / kSelect * 64, from = wave * run, to = min(from + run, n);
    const bool held = n <= kSelect * kHeld, all = n <= a.budget;
    const uint32_t lo = all ? 0 : a.sinks, hi = all ? 0 : n - a.recent;
    // the key of a middle slot; 0, below every weight's, for the others: they
    // only add to the lowest bin, behind everything that is looked for
    auto key_of = [&](uint32_t j, float x) { return j >= lo && j < hi ? weight_key(x) : 0u; };
    float mine[kHeld];
    uint32_t key[kHeld];
    if (held)
#pragma unroll
        for (int x = 0; x < kHeld; ++x) {
            const uint32_t j = from + 64 * x + lane;
            mine[x] = j < to ? w[j] : 0.0f;
            key[x] = j < to ? key_of(j, mine[x]) : 0;
        }
    // f(slot, weight, key, there) for every step of the wave's slots
    auto each = [&](auto f) {
        if (held) {
#pragma unroll
            for (int x = 0; x < kHeld; ++x) {
                if (from + 64 * x >= to) break;
                f(from + 64 * x + lane, mine[x], key[x], from + 64 * x + lane < to);
            }
        } else {
            for (uint32_t j0 = from; j0 < to; j0 += 64) {
                const bool in = j0 + lane < to;
                const float x = in ? w[j0 + lane] : 0.0f;
                f(j0 + lane, x, in ? key_of(j0 + lane, x) : 0, in);
            }
        }
    };
    uint32_t want = all ? 0 : a.budget - a.sinks - a.recent;   // of the middle; < hi - lo
    uint32_t prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0 && want; shift -= 8) {
        *reinterpret_cast<u32x4*>(&hist[4 * t]) = u32x4{};
        __syncthreads();
        each([&](uint32_t, float, uint32_t k, bool) {
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift & 255) * kCopies + lane % kCopies], 1u);
        });
        __syncthreads();
        const u32x4 four = *reinterpret_cast<const u32x4*>(&hist[4 * t]);
        uint32_t sum = four[0] + four[1] + four[2] + four[3];
        sum += __shfl_xor(sum, 1);
        sum += __shfl_xor(sum, 2);
        if (t % 4 == 0) total[t / 4] = sum;
        __syncthreads();
        if (wave == 0) find_bin(total, want, found);
        __syncthreads();
        prefix |= found[0] << shift;
        mask |= 255u << shift;
        want -= found[1];
    }
    // kept: protected slots and keys above the border (sure), and the first `want` at it
    const uint32_t above = mask ? prefix : ~0u;
    auto sure = [&](uint32_t j, uint32_t k, bool in) { return k > above || (in && (j < lo || j >= hi)); };
    auto tie = [&](uint32_t k) { return mask && k == prefix; };
    uint32_t ns = 0, nt = 0;
    each([&](uint32_t j, float, uint32_t k, bool in) {
        ns += __popcll(__ballot(sure(j, k, in)));
        nt += __popcll(__ballot(tie(k)));
    });
    if (lane == 0) { sures[wave] = ns; ties[wave] = nt; }
    __syncthreads();
    ns = nt = 0;
    for (uint32_t x = 0; x < wave; ++x) { ns += sures[x]; nt += ties[x]; }
    const uint64_t below = (1ull << lane) - 1;
    // held weights are all read by now: their places may be written
    each([&](uint32_t j, float x, uint32_t k, bool in) {
        const bool s = sure(j, k, in), e = tie(k);
        const uint64_t bs = __ballot(s), be = __ballot(e);
        const uint32_t ps = ns + __popcll(bs & below), pe = nt + __popcll(be & below);
        if (s || (e && pe < want)) {
            const uint32_t at = ps + min(pe, want);
            kept[at] = static_cast<int32_t>(j);
            if (held) wo[at] = x;
        }
        ns += __popcll(bs);
        nt += __popcll(be);
    });
    for (uint32_t j = keep + t; j < a.budget; j += kSelect) kept[j] = -1;
    if (!held) {
        // in steps: every read of a step comes before its writes, and a later step's sources lie behind them
        __syncthreads();
        for (uint32_t j0 = 0; j0 < keep; j0 += kSelect) {
            const uint32_t j = j0 + t;
            const float x = j < keep ? w[kept[j]] : 0.0f;
            __syncthreads();
            if (j < keep) wo[j] = x;
            __syncthreads();
        }
    }
    for (uint32_t j = keep + t; j < a.into_slots; j += kSelect) wo[j] = 0.0f;
}

template <int DT>
__device__ inline uint64_t elem_byte(uint64_t e) { return DT == PKV_FP4 ? e / 2 : DT == PKV_F32 ? e * 4 : e * 2; }

// Kept rows to their new slots, in pieces of 16 bytes, four rows' at a time
// (4-bit caches: the scale bytes with the first piece).
//   into other memory  a workgroup takes kBatch rows of one side of a (copy,
//                      layer, head); bound by the rows' bytes (8,192 of 32,768
//                      rows of 64 heads of 128, bf16: 107 us, 5.0 TB/s)
//   in place           a workgroup takes a column of at most 64 bytes of all
//                      rows, in order: a step's rows are read before it writes
//                      (a barrier), and rows read later lie behind everything
//                      it writes, so the next step's reads are already under
//                      way; columns do not meet.
template <int DT, int D, bool IN_PLACE>
struct Move {
    static constexpr uint32_t kBytes = DT == PKV_FP4 ? D / 2 : DT == PKV_F32 ? D * 4 : D * 2;
    static constexpr uint32_t kPieces = IN_PLACE && kBytes > 64 ? 4 : kBytes / 16, kColumns = kBytes / 16 / kPieces;
    static constexpr uint32_t kHold = IN_PLACE ? 8 : 4, kStep = 256 / kPieces, kBatch = kStep * kHold;
    u32x4 x[kHold];
    uint32_t s[DT == PKV_FP4 ? kHold : 1];
    // rows j0 + row, + kStep, .. below `keep`
    __device__ void read(const EvictDev& a, const uint8_t* src, const uint8_t* scales, uint64_t from, const int32_t* kept,
                         uint32_t j0, uint32_t keep, uint32_t piece) {
#pragma unroll
        for (uint32_t k = 0; k < kHold; ++k) {
            const uint32_t j = j0 + k * kStep;
            const uint64_t e = from + static_cast<uint64_t>(j < keep ? kept[j] : 0) * a.kv.slot;   // slot 0: read, not written
            x[k] = *reinterpret_cast<const u32x4*>(src + elem_byte<DT>(e) + 16 * piece);
            if constexpr (DT == PKV_FP4)
                s[k] = D == 64 ? *reinterpret_cast<const uint16_t*>(scales + e / 32)
                               : *reinterpret_cast<const uint32_t*>(scales + e / 32);
        }
    }
    __device__ void write(const EvictDev& a, uint8_t* dst, uint8_t* scales, uint64_t to, uint32_t j0, uint32_t keep,
                          uint32_t piece) const {
#pragma unroll
        for (uint32_t k = 0; k < kHold; ++k) {
            const uint32_t j = j0 + k * kStep;
            if (j >= keep) continue;
            const uint64_t e = to + static_cast<uint64_t>(j) * a.into.slot;
            *reinterpret_cast<u32x4*>(dst + elem_byte<DT>(e) + 16 * piece) = x[k];
            if constexpr (DT == PKV_FP4)
                if (piece == 0) {
                    if constexpr (D == 64) *reinterpret_cast<uint16_t*>(scales + e / 32) = static_cast<uint16_t>(s[k]);
                    else *reinterpret_cast<uint32_t*>(scales + e / 32) = s[k];
                }
        }
    }
};

template <int DT, int D, bool IN_PLACE>
__global__ __launch_bounds__(256) void move_kernel(EvictDev a, uint32_t batches) {
    using M = Move<DT, D, IN_PLACE>;
    const uint32_t per = IN_PLACE ? M::kColumns : batches, part = blockIdx.x % per, set = blockIdx.x / per / 2;
    const bool values = blockIdx.x / per % 2;
    const uint32_t h = set % a.heads, cl = set / a.heads, l = cl % a.layers, c = cl / a.layers;
    const uint32_t n = min(max(a.lens[c], 0), static_cast<int>(a.slots)), keep = min(n, a.budget);
    const int32_t* kept = a.kept + static_cast<uint64_t>(set) * a.budget;
    const uint8_t *src = values ? a.kv.v : a.kv.k, *ssc = values ? a.kv.vs : a.kv.ks;
    uint8_t *dst = const_cast<uint8_t*>(values ? a.into.v : a.into.k);
    uint8_t* dsc = const_cast<uint8_t*>(values ? a.into.vs : a.into.ks);
    const uint64_t from = c * a.kv.copy + l * a.kv.layer + h * a.kv.head;
    const uint64_t to = c * a.into.copy + l * a.into.layer + h * a.into.head;
    const uint32_t row = threadIdx.x / M::kPieces, piece = threadIdx.x % M::kPieces + (IN_PLACE ? part * M::kPieces : 0);
    if constexpr (!IN_PLACE) {
        M m;
        m.read(a, src, ssc, from, kept, part * M::kBatch + row, keep, piece);
        m.write(a, dst, dsc, to, part * M::kBatch + row, keep, piece);
    } else {
        if (n <= a.budget) return;             // every slot stays where it is
        M m, next;
        m.read(a, src, ssc, from, kept, row, keep, piece);
        for (uint32_t j0 = 0; j0 < keep; j0 += M::kBatch) {
            next.read(a, src, ssc, from, kept, j0 + M::kBatch + row, keep, piece);
            __builtin_amdgcn_s_waitcnt(0);     // this step's rows have been read ..
            __syncthreads();                   // .. by every wave
            m.write(a, dst, dsc, to, j0 + row, keep, piece);
            m = next;
        }
    }
}

uint64_t round256(uint64_t x) { return (x + 255) & ~255ull; }

constexpr uint32_t kDecodeRows = 16;   // rows x group that decode_kernel takes

// How a call is cut: row tiles (one of at most 16 rows, or tiles of 128 or 64)
// times `splits` shares of the slots, so that the chip is full while a share has
// work for its waves.
struct Plan {
    uint32_t row_tiles, splits, rows, ld;
    int ks;                              // rows_kernel: shares of a tile's slots among a workgroup's waves
    uint32_t w_blocks, w_splits, w_ld;   // weights_kernel: blocks of slots, shares of the rows
    uint64_t ml, logits, stats, shares, bytes;   // offsets in the workspace (partial outputs first), all of it
};
constexpr uint64_t kHalf = 6;
constexpr uint32_t kMaxShares = 64;     // of many rows
constexpr uint32_t kJoinRows = 4096;    // rows of all heads up to which a workgroup joins one
Plan plan_of(const AttendDev& a, uint32_t dim, int cache_dtype) {
    Plan p{};
    const uint64_t all = static_cast<uint64_t>(a.nq) * a.group, heads = static_cast<uint64_t>(a.copies) * a.heads;
    const bool few = all <= kDecodeRows;
    const uint32_t step = (few ? 32 : 64) / (cache_dtype == PKV_F32 ? 2 : 1);
    // tiles of slots that a tile of `rows` rows can see: all, or the window, the rows before its last and the sinks, each up
    // to a tile more
    auto tiles_for = [&](uint32_t rows) {
        uint64_t most = a.max_len;
        if (a.window)
            most = std::min<uint64_t>(most, static_cast<uint64_t>(a.window) + std::min<uint64_t>(a.nq, rows) + a.sinks + 2 * step);
        return (most + step - 1) / step;
    };
    p.ks = 1;
    if (few) {
        // 768 workgroups are three a CU; every wave of a share has a tile
        p.row_tiles = 1;
        p.rows = static_cast<uint32_t>(all);
        p.splits = static_cast<uint32_t>(std::max<uint64_t>(
            1, std::min<uint64_t>((768 + heads - 1) / heads, tiles_for(kDecodeRows) / 4)));
    } else {
        // The least time, in tenths of the 2 us that a tile takes a workgroup of 128 rows (64 rows: kHalf): as many
        // workgroups as fit run at the speed of one, and a share costs four tiles' time for its start and end, and the
        // passage of its outputs through memory.
        const uint64_t fit = 256 * (dim == 64 && cache_dtype != PKV_FP4 ? 3 : 2);
        uint64_t least = ~0ull;
        for (int ks = 1; ks <= (cache_dtype == PKV_F32 ? 1 : 2); ++ks) {
            const uint32_t rt = row_tile(ks), row_tiles = static_cast<uint32_t>((all + rt - 1) / rt);
            const uint64_t groups = heads * row_tiles, tiles = tiles_for(rt);
            for (uint32_t n = 1; n <= kMaxShares && (n == 1 || n * 4 <= tiles); ++n) {
                const uint64_t rounds = (groups * n + fit - 1) / fit;
                const uint64_t cost = rounds * ((tiles + n - 1) / n + (n == 1 ? 2 : 4)) * (ks == 1 ? 10 : kHalf) +
                                      (n == 1 ? 0 : heads * all * dim * 8 * n / 800000);
                if (cost < least) {
                    least = cost;
                    p.splits = n;
                    p.ks = ks;
                    p.row_tiles = row_tiles;
                    p.rows = row_tiles * rt;
                }
            }
        }
    }
    const bool parts = few || p.splits > 1;
    p.ld = few && a.weights ? (a.max_len + 31) / 32 * 32 + 4 : 0;
    p.ml = parts ? round256(heads * p.splits * p.rows * dim * 4) : 0;
    p.logits = p.ml + (parts ? round256(heads * p.splits * p.rows * 8) : 0);
    p.stats = p.logits + round256(4 * heads * all * p.ld);
    p.shares = p.stats + (!few && a.weights ? round256(8 * heads * all) : 0);
    p.w_splits = 1;
    p.w_ld = (a.max_len + 127) / 128 * 128;
    if (!few && a.weights) {
        // blocks of 128 slots that some row sees, one more for the window's first; eight workgroups a CU, since they see
        // very different numbers of rows, of at least 256 rows each
        p.w_blocks = p.w_ld / 128;
        if (a.window)
            p.w_blocks = static_cast<uint32_t>(std::min<uint64_t>(
                p.w_blocks, (static_cast<uint64_t>(a.window) + a.nq + 126) / 128 + 1 + (static_cast<uint64_t>(a.sinks) + 127) / 128));
        p.w_splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(2048 / (p.w_blocks * heads), all / 256)));
    }
    p.bytes = p.shares + (p.w_splits > 1 ? round256(4ull * heads * p.w_splits * p.w_ld) : 0);
    return p;
}

template <int CT, int QT, int D>
int attend_typed(AttendDev a, uint8_t* ws, hipStream_t st) {
    const Plan p = plan_of(a, D, CT);
    const Partial part{reinterpret_cast<float*>(ws), reinterpret_cast<float*>(ws + p.ml),
                       reinterpret_cast<float*>(ws + p.logits), p.splits, p.ld, p.rows};
    const uint32_t heads = a.copies * a.heads, outs = heads * a.nq * a.group;
    if (a.nq * a.group <= kDecodeRows) {
        if (a.weights) decode_kernel<CT, QT, D, true><<<heads * p.splits, 256, 0, st>>>(a, part);
        else decode_kernel<CT, QT, D, false><<<heads * p.splits, 256, 0, st>>>(a, part);
        const uint32_t chunks = a.weights ? (a.max_len + 1023) / 1024 * heads : 0;
        join_kernel<QT, D><<<outs + chunks, 256, 0, st>>>(a, part, outs);
        return hipGetLastError();
    }
    a.stats = a.weights ? reinterpret_cast<float*>(ws + p.stats) : nullptr;
    if constexpr (CT != PKV_F32) {
        if (p.ks == 2) rows_kernel<CT, QT, D, 2><<<heads * p.row_tiles * p.splits, 256, 0, st>>>(a, part, p.row_tiles);
    }
    if (p.ks == 1) rows_kernel<CT, QT, D, 1><<<heads * p.row_tiles * p.splits, 256, 0, st>>>(a, part, p.row_tiles);
    // a workgroup a row reads its shares side by side, D / 4 lanes a row one after the other; whole calls on 32,768
    // slots: 1,024 rows 42 us against 61, 4,096 rows 93 and 93, 8,192 rows (16,384 slots) 93 against 87
    constexpr uint32_t kJoin = join_rows(D);
    if (p.splits > 1 && outs <= kJoinRows) join_kernel<QT, D><<<outs, 256, 0, st>>>(a, part, outs);
    else if (p.splits > 1) join_rows_kernel<QT, D><<<(a.nq * a.group + kJoin - 1) / kJoin * heads, 256, 0, st>>>(a, part);
    if (a.weights) {
        const Shares shares{reinterpret_cast<float*>(ws + p.shares), p.w_splits, p.w_ld};
        weights_kernel<CT, QT, D><<<p.w_blocks * heads * p.w_splits, 256, 0, st>>>(a, shares);
        const uint32_t blocks = (a.max_len + 255) / 256;
        if (p.w_splits > 1) add_weights_kernel<<<blocks * heads, 256, 0, st>>>(a, shares, blocks);
    }
    return hipGetLastError();
}

template <int CT, int QT>
int attend_dim(const AttendDev& a, uint32_t dim, uint8_t* ws, hipStream_t st) {
    return dim == 64 ? attend_typed<CT, QT, 64>(a, ws, st) : attend_typed<CT, QT, 128>(a, ws, st);
}

}  // namespace

// The launches of attend_typed: threads along x stay below 2^32.
bool attend_fits(const AttendDev& a, uint32_t dim, int cache_dtype) {
    const Plan p = plan_of(a, dim, cache_dtype);
    const uint64_t heads = static_cast<uint64_t>(a.copies) * a.heads, all = static_cast<uint64_t>(a.nq) * a.group;
    uint64_t most = heads * p.splits * p.row_tiles;
    if (all <= kDecodeRows) {
        most = std::max<uint64_t>(most, heads * all + (a.weights ? heads * ((a.max_len + 1023ull) / 1024) : 0));
    } else {
        const uint64_t join = join_rows(dim);
        if (p.splits > 1) most = std::max(most, heads * (heads * all <= kJoinRows ? all : (all + join - 1) / join));
        if (a.weights) most = std::max(most, heads * p.w_blocks * p.w_splits);
        if (p.w_splits > 1) most = std::max<uint64_t>(most, heads * ((a.max_len + 255ull) / 256));
    }
    return most < 1u << 24;
}

uint64_t attend_workspace(const AttendDev& a, uint32_t dim, int cache_dtype, int) {
    return plan_of(a, dim, cache_dtype).bytes;
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

template <int QT, int D>
static int rows_typed(const RowsDev& r, bool store, hipStream_t st) {
    const uint64_t pieces = static_cast<uint64_t>(r.copies) * r.layers * r.heads * r.rows *
                            (D / (store ? kPiece<QT, true> : kPiece<QT, false>));
    // one piece a thread up to 2^20 workgroups a side
    const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>((pieces + 255) / 256, 1u << 20)), 2);
    if (store) fp4_store_kernel<QT, D><<<grid, 256, 0, st>>>(r, pieces);
    else fp4_load_kernel<QT, D><<<grid, 256, 0, st>>>(r, pieces);
    return hipGetLastError();
}
static int launch_rows(const RowsDev& r, uint32_t dim, int dtype, bool store, hipStream_t st) {
    if (dtype == PKV_F32) return dim == 64 ? rows_typed<PKV_F32, 64>(r, store, st) : rows_typed<PKV_F32, 128>(r, store, st);
    if (dtype == PKV_BF16) return dim == 64 ? rows_typed<PKV_BF16, 64>(r, store, st) : rows_typed<PKV_BF16, 128>(r, store, st);
    return dim == 64 ? rows_typed<PKV_F16, 64>(r, store, st) : rows_typed<PKV_F16, 128>(r, store, st);
}
int launch_fp4_store(const RowsDev& r, uint32_t dim, int dtype, void* stream) {
    return launch_rows(r, dim, dtype, true, static_cast<hipStream_t>(stream));
}
int launch_fp4_load(const RowsDev& r, uint32_t dim, int dtype, void* stream) {
    return launch_rows(r, dim, dtype, false, static_cast<hipStream_t>(stream));
}

// Workgroups that move a call's rows: for each side of a (copy, layer, head) a
// column of all rows in place, else kBatch rows.
template <int DT>
static uint64_t move_blocks(const EvictDev& e, uint32_t dim) {
    const uint64_t sides = 2ull * e.copies * e.layers * e.heads;
    if (e.in_place) return sides * (dim == 64 ? Move<DT, 64, true>::kColumns : Move<DT, 128, true>::kColumns);
    const uint32_t rows = dim == 64 ? Move<DT, 64, false>::kBatch : Move<DT, 128, false>::kBatch;
    return sides * ((std::min(e.budget, e.slots) + rows - 1) / rows);
}
static uint64_t move_blocks(const EvictDev& e, uint32_t dim, int dtype) {
    if (dtype == PKV_F32) return move_blocks<PKV_F32>(e, dim);
    if (dtype == PKV_FP4) return move_blocks<PKV_FP4>(e, dim);
    return move_blocks<PKV_BF16>(e, dim);   // f16 rows are as long
}

template <int DT, int D>
static int move_typed(const EvictDev& e, hipStream_t st) {
    const uint32_t grid = static_cast<uint32_t>(move_blocks<DT>(e, D));
    if (e.in_place) move_kernel<DT, D, true><<<grid, 256, 0, st>>>(e, 0);
    else move_kernel<DT, D, false><<<grid, 256, 0, st>>>(e, grid / (2 * e.copies * e.layers * e.heads));
    return hipGetLastError();
}

// The launches of launch_evict: threads along x stay below 2^32 (select_kernel: 1,024 threads a set).
bool evict_fits(const EvictDev& e, uint32_t dim, int dtype) {
    const uint64_t sets = static_cast<uint64_t>(e.copies) * e.layers * e.heads;
    return sets < 1u << 22 && move_blocks(e, dim, dtype) < 1u << 24;
}

int launch_evict(const EvictDev& e, uint32_t dim, int dtype, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    select_kernel<<<e.copies * e.layers * e.heads, kSelect, 0, st>>>(e);
    if (dtype == PKV_F32) return dim == 64 ? move_typed<PKV_F32, 64>(e, st) : move_typed<PKV_F32, 128>(e, st);
    if (dtype == PKV_BF16) return dim == 64 ? move_typed<PKV_BF16, 64>(e, st) : move_typed<PKV_BF16, 128>(e, st);
    if (dtype == PKV_F16) return dim == 64 ? move_typed<PKV_F16, 64>(e, st) : move_typed<PKV_F16, 128>(e, st);
    return dim == 64 ? move_typed<PKV_FP4, 64>(e, st) : move_typed<PKV_FP4, 128>(e, st);
}

}  // namespace pkv
