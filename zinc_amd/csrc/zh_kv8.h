// zh_kv8.h — the 8-bit KV cache's formats and how a kernel finds a batch's rows
// (zh_kv8.hip, zh_kv8_attn.hip).
//
// A block (16 tokens of a page, one head) holds codes and a scale s; a value is
// code * s. Scales are powers of two: a value over its scale is then exact, only
// the code's rounding counts, and a block whose scale rises is rounded again by a
// shift, which an e4m3 code outlives unchanged unless it falls below 2^-6, and an
// i8 code within half a step of the new scale: after any number of rises a value is
// less than one step of the last scale off (halves of s, s/2, s/4, ...). Against a
// scale that makes the block's largest value the largest code, the step is up to
// twice as long.
#pragma once
#include <type_traits>

#include "zh_device.h"
#include "zh_internal.h"
#include "zh_kv.h"

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(4))) uint32_t const_u32;  // what no kernel writes while it runs

constexpr int KV8_LOW = -64, KV8_HIGH = 64;  // exponents of the scales
constexpr int KV8_NAN = 1 << 20;             // the exponent of a block whose scale is NaN

static inline bool kv8_type_ok(uint32_t t) { return t == ZH_I8 || t == ZH_E4M3; }
// The shape and the ranges of the caches, tables and rows of a batch; n_rows: rows
// of the call.
bool kv8_batch_ok(const zh_kv8_batch *kv, uint32_t n_rows);

// The bits of a scale in [2^-64, 2^64] (positive).
ZH_DEV bool kv8_scale_ok(uint32_t bits) { return bits - 0x1F800000u <= 0x5F800000u - 0x1F800000u; }

// The least e for which x <= largest * 2^e (exactly: 448 = 7/8 2^9, 127 = 127/128
// 2^7), KV8_LOW at least, KV8_NAN past KV8_HIGH. x: the largest of some magnitudes, and
// `sum` their sum, which is no number (or too large) if one of them is none, where the
// largest would not tell.
template <uint32_t F, typename T>
ZH_DEV int kv8_exp(T x, T sum) {
    int e;
    T m;
    if constexpr (sizeof(T) == 8) {
        e = __builtin_amdgcn_frexp_exp(x);
        m = __builtin_amdgcn_frexp_mant(x);
    } else {
        e = __builtin_amdgcn_frexp_expf(x);
        m = __builtin_amdgcn_frexp_mantf(x);
    }
    e = F == ZH_I8 ? e - 7 + (m > (T)0.9921875) : e - 9 + (m > (T)0.875);
    if (x == 0) e = KV8_LOW;
    if (!(sum < (T)INFINITY)) e = KV8_NAN;
    return e > KV8_HIGH ? KV8_NAN : max(e, KV8_LOW);
}
// The largest of each team's (L lanes, 8 or 16) and of the wave's values, by lane
// exchanges within rows of 16.
template <int L>
ZH_DEV int team_max(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
    return L == 16 ? max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false)) : v;
}
ZH_DEV int wave_max(int v) {
    v = team_max<16>(v);
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
// The sum over teams of L lanes (8 or 16) in 64 bits.
template <int CTRL>
ZH_DEV double dpp_add64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int L>
ZH_DEV double team_sum64(double v) {
    v = dpp_add64<0x141>(dpp_add64<0x4E>(dpp_add64<0xB1>(v)));
    return L == 16 ? dpp_add64<0x140>(v) : v;
}
ZH_DEV float kv8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four codes of values over their scale, rounded to nearest, ties to even.
template <uint32_t F>
ZH_DEV uint32_t kv8_encode(const float (&v)[4]) {
    if (F == ZH_I8) return pack4((int)rintf(v[0]), (int)rintf(v[1]), (int)rintf(v[2]), (int)rintf(v[3]));
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
}
// In 64 bits (a value that 32 bits round to the middle of two codes is not taken
// for it): from 2^(e - 1) on e4m3 goes in steps of 2^(e - 4), and in 2^-9 at least.
template <uint32_t F>
ZH_DEV uint32_t kv8_encode(const double (&v)[4]) {
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (F == ZH_I8) {
            r[i] = (float)__builtin_rint(v[i]);
        } else {
            const int s = max(__builtin_amdgcn_frexp_exp(v[i]), -5) - 4;
            r[i] = (float)__builtin_amdgcn_ldexp(__builtin_rint(__builtin_amdgcn_ldexp(v[i], -s)), s);
        }
    }
    return kv8_encode<F>(r);
}
// The numbers of four codes.
template <uint32_t F>
ZH_DEV void kv8_decode(uint32_t c, float (&v)[4]) {
    if (F == ZH_I8) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (float)((int)(c << (24 - 8 * i)) >> 24);
    } else {
        v[0] = __builtin_amdgcn_cvt_f32_fp8(c, 0);
        v[1] = __builtin_amdgcn_cvt_f32_fp8(c, 1);
        v[2] = __builtin_amdgcn_cvt_f32_fp8(c, 2);
        v[3] = __builtin_amdgcn_cvt_f32_fp8(c, 3);
    }
}

// Which rows of a call are a sequence's: rows [row, row + n) at positions
// [pos, pos + n) (the rows that have a place), of the sequence's `len` tokens.
struct Kv8Seq {
    uint32_t row, n, pos, len;
};
ZH_DEV Kv8Seq kv8_seq(const uint32_t *row_start, const uint32_t *seq_lens, uint32_t s, uint32_t n_rows, uint32_t &bad) {
    Kv8Seq x;
    x.len = seq_lens[s];
    if (!row_start) {
        x.row = s;
        x.n = x.len && s < n_rows ? 1u : 0u;
    } else {
        const uint32_t a = row_start[s], b = row_start[s + 1];
        if (a > b || b > n_rows) bad = 1;
        x.row = min(a, n_rows);
        x.n = b > a ? min(b, n_rows) - x.row : 0u;
        if (x.n > x.len) {  // (the first ones stand before the sequence's begin)
            bad = 1;
            x.row += x.n - x.len;
            x.n = x.len;
        }
    }
    x.pos = x.len - x.n;
    return x;
}
// Sums over the lanes up to each one (row shifts, then the rows' totals passed on).
ZH_DEV uint32_t wave_scan(uint32_t v) {
    auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    typedef std::integral_constant<int, 0xF> all;
    step(std::integral_constant<int, 0x111>{}, all{});  // row_shr 1, 2, 4, 8
    step(std::integral_constant<int, 0x112>{}, all{});
    step(std::integral_constant<int, 0x114>{}, all{});
    step(std::integral_constant<int, 0x118>{}, all{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast 15 to rows 1 and 3
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast 31 to rows 2 and 3
    return v;
}
ZH_DEV uint32_t wave_total(uint32_t v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Item `u` of those that the sequences have (n(s) each, in order): its sequence, and u
// counted from the sequence's first. Every wave by itself, 64 sequences at a time;
// false: there are fewer.
template <typename C>
ZH_DEV bool kv8_find(uint32_t n_seq, uint32_t u, C count, uint32_t &s, uint32_t &item) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t s0 = 0; s0 < n_seq; s0 += 64) {
        const uint32_t n = s0 + lane < n_seq ? count(s0 + lane) : 0u, sum = wave_scan(n);
        const uint64_t past = __builtin_amdgcn_ballot_w64(sum > u);
        if (past) {
            const uint32_t k = __builtin_ctzll(past);
            item = u - (__builtin_amdgcn_readlane(sum, k) - __builtin_amdgcn_readlane(n, k));
            s = s0 + k;
            return true;
        }
        u -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}
