// zh_kv8_attn.hip — causal paged attention of a batch over a cache held in 8 bits
// (zh_flash_attn_kv8).
//
// For row i of sequence s and query head h of kv head k, over the tokens t that it
// may see, with codes Kc, Vc and block scales a_t, b_t:
//   out = sum_t w_t Vc[t] / sum_t w_t / b_t,  w_t = 2^(x_t + log2 b_t - m),
//   x_t = log2 e scale a_t q . Kc[t]
// The scales never meet the codes: a_t multiplies a score, b_t goes into the weight,
// whose reference m is the largest x_t + log2 b_t. Weights of products with V are
// then relative to the largest contribution whatever the blocks' scales are, and fit
// fp16. Codes become fp16 exactly (i8 as its value times 2^-10).
#include <math.h>

#include <atomic>
#include <type_traits>

#include "zh_kv8.h"

namespace {

constexpr int W = 4;         // waves of a streaming workgroup
constexpr uint32_t NJ = 2;   // pages of a wave's step
constexpr uint32_t CUT = 64;  // tokens of a unit, of which a streaming workgroup takes whole ones

struct Kv8Attn {
    const uint8_t *q;
    uint8_t *out;
    uint64_t q_row, out_row;  // bytes between rows
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const uint32_t *tables, *row_start, *seq_lens;
    float *part, *stat;  // a part's unnormalised sums; maximum (base 2) and sum of weights
    uint32_t *err;
    uint32_t n_seq, stride, cache_tokens, nh, nkv, G, n_rows, max_rows, max_len;
    uint32_t few;             // rows of a sequence and kv head that are streamed; more go through LDS tiles
    uint32_t rt, tiles;       // rows of a streamed tile, tiles of a sequence at most
    uint32_t groups, least;   // streaming workgroups of a kv head, units of each at least (0: one takes one tile)
    float *tpart, *tstat;     // parts of LDS tiles
    uint32_t tslots;          // workgroups that a kv head's LDS tiles are dealt out to (0: one a tile)
    float scale;              // |attn_scale| log2 e = scale * 2^scale_exp, with attn_scale's sign
    int32_t scale_exp;
};

// A uniform value, which the compiler does not take for one behind a division.
ZH_DEV uint32_t scalar(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// A value that the compiler knows nothing of, so that it stays the one base of addresses.
ZH_DEV uint32_t opaque(uint32_t v) {
    asm("" : "+v"(v));
    return v;
}

// A sequence's rows: [row, row + n), row i over the tokens below lim(i).
struct AttnSeq {
    uint32_t s, row, n, all, len, cut;  // all: rows before the cut at max_rows; len, cut at `cut`
    ZH_DEVM uint32_t lim(uint32_t i) const {
        const uint32_t after = all - 1 - i;
        return len > after ? min(len - after, cut) : 0u;
    }
};
ZH_DEV AttnSeq attn_seq(const Kv8Attn &a, uint32_t s, bool &bad) {
    AttnSeq x;
    uint32_t first = s, end = min(s + 1, a.n_rows);
    const const_u32 *row_start = (const const_u32 *)a.row_start, *lens = (const const_u32 *)a.seq_lens;
    if (row_start) {
        first = row_start[s];
        end = row_start[s + 1];
        if (first > end || end > a.n_rows) bad = true;
        end = min(end, a.n_rows);
    }
    x.s = s;
    x.len = lens[s];
    x.row = first;
    x.all = end > first ? end - first : 0u;
    x.n = min(x.all, a.max_rows);
    x.cut = min(x.len, a.max_len);
    if (x.all > a.max_rows || (x.all && x.len > a.max_len) || (a.row_start && x.all > x.len)) bad = true;
    return x;
}

// What takes the products of a row's q, scaled by 2^-e, times a block's scale to
// base-2 scores. 2^-120 at least: products lie below 2^32, so every weight is 1 there, as
// without the bound, and no score that is masked (-inf) meets a factor of 0. A score
// past the range of 32 bits makes its row NaN.
ZH_DEV float score_factor(float c, float scale) { return fmaxf(c * scale, 0x1p-120f); }

// V's scales may lie 2^128 apart, and exp2 gives 0 below 2^-126. A weight that small adds
// nothing to the products with V, but its share w_t / b_t, in a block of a small scale, may
// be most of the sum. So where parts are joined, or sums moved to a reference far above,
// they are multiplied by 2^d in two factors (Shift); and blocks of scales below 2^-24 or
// above 2^8 (none of a cache of ordinary values) are marked, for their tokens' shares to be
// taken without b: streamed rows, by going over the scores again (far_sum: code in the loop
// cost rows of f32 in tiles of 32 5 to 10%), LDS tiles in a branch that adds what fell out
// (0.5%). Between the two scales nothing that counts is lost: of a share w_t / b_t with w_t
// below 2^-126, b_t 2^-24, it is 2^-102; the sum is 2^-60 at least (a weight of 2^4 or more
// over 2^64), so tokens lose it 2^-42 each at most.
constexpr uint32_t LOW = (127 - 24) << 23, HIGH = (127 + 8) << 23;
struct Shift {
    float a, b;
    ZH_DEVM explicit Shift(float d) {
        const float e = fmaxf(d, -126.f);
        a = __builtin_amdgcn_exp2f(e);
        b = __builtin_amdgcn_exp2f(d - e);
    }
    ZH_DEVM float both() const { return a * b; }
};
ZH_DEV float lost_share(float a, float iv) {  // what the weight's product with iv has not
    return a < -126.f ? __builtin_amdgcn_exp2f(a + 64.f) * (iv * 0x1p-64f) - __builtin_amdgcn_exp2f(a) * iv : 0.f;
}

// A block's scales as the kernels take them: the scores' factor, the weights'
// exponent and what takes a weight to its share of the sum; `ok` false: it reads as NaN
// (and the others are harmless).
template <uint32_t F>
struct Block {
    float ks, lv, iv;
    bool ok, apart;
    ZH_DEVM static constexpr float unit() { return F == ZH_I8 ? 0x1p-10f : 1.f; }  // (the fp16 codes' of 1)
    ZH_DEVM void set(uint32_t k, uint32_t v) {
        ok = kv8_scale_ok(k) && kv8_scale_ok(v);
        const uint32_t kb = ok ? k : 0x3F800000u, vb = ok ? v : 0x3F800000u;
        apart = vb - LOW > HIGH - LOW;
        // (exact for powers of two; for others the exponent's fraction is within 2^-21)
        const float mant = __uint_as_float((vb & 0x7FFFFFu) | 0x3F800000u);
        ks = __uint_as_float(kb) * (1.f / unit());
        lv = (float)((int)(vb >> 23) - 127) + __builtin_amdgcn_logf(mant);
        iv = __builtin_amdgcn_rcpf(mant) * __uint_as_float((254u - (vb >> 23)) << 23) * unit();
    }
};

// ---- codes to fp16 (i8: the code plus 128 is an fp16 subnormal's bits, 2^-24 each)
ZH_DEV half2v i8_pair(uint32_t biased, uint32_t sel) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0u, biased, sel)) * (_Float16)16384.f - (_Float16)0.125f;
}
// eight codes of a row
template <uint32_t F>
ZH_DEV half8 row8(uint32_t lo, uint32_t hi) {
    half2v h[4];
    if (F == ZH_I8) {
        lo ^= 0x80808080u;
        hi ^= 0x80808080u;
        h[0] = i8_pair(lo, 0x0C010C00u);
        h[1] = i8_pair(lo, 0x0C030C02u);
        h[2] = i8_pair(hi, 0x0C010C00u);
        h[3] = i8_pair(hi, 0x0C030C02u);
    } else {
        h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
        h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
        h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    }
    return half8{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
}
// the codes of dims n and n + 1 (n even, of a dword) of tokens a and b: (a, b) of n, (a, b) of n + 1
template <uint32_t F>
ZH_DEV void pair2(uint32_t a, uint32_t b, int n, half2v &x, half2v &y) {
    if (F == ZH_I8) {  // (a and b biased)
        const uint32_t sel = n % 4 == 0 ? 0x0C040C00u : 0x0C060C02u;
        x = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(b, a, sel)) * (_Float16)16384.f - (_Float16)0.125f;
        y = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(b, a, sel + 0x00010001u)) * (_Float16)16384.f - (_Float16)0.125f;
    } else {
        const uint32_t p = __builtin_amdgcn_perm(b, a, n % 4 == 0 ? 0x05010400u : 0x07030602u);
        x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(p, 1.0f, false);
        y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(p, 1.0f, true);
    }
}

// (a load that goes by the L2s, where no other workgroup reads the same)
template <bool ONCE, typename V>
ZH_DEV V ld_once(const V *p) {
    return ONCE ? __builtin_nontemporal_load(p) : *p;
}
ZH_DEV void ld8(const float *p, float (&v)[8]) {
    const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
ZH_DEV void ld8(const _Float16 *p, float (&v)[8]) {
    const half8 a = *(const half8 *)p;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)a[e];
}
template <typename T>
ZH_DEV void st_out(const Kv8Attn &a, uint32_t row, uint32_t h, uint32_t d, uint32_t hd, const f32x4 &v) {
    T *op = (T *)(a.out + row * a.out_row) + (size_t)h * hd + d;
    if constexpr (sizeof(T) == 4) *(f32x4 *)op = v;
    else *(half4 *)op = half4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
}

// What sequence s has for the streaming workgroups: row tiles, and units of tokens of
// each (one at least, for rows without tokens).
struct UnitSeq {
    uint32_t tiles, units;
};
ZH_DEV UnitSeq unit_seq(const Kv8Attn &a, uint32_t s, bool &bad) {
    const AttnSeq x = attn_seq(a, s, bad);
    const uint64_t n = (uint64_t)x.n * a.G;
    UnitSeq u = {0, 1};
    if (n && n <= a.few) {
        u.tiles = ((uint32_t)n + a.rt - 1) / a.rt;
        u.units = max((x.lim(x.n - 1) + CUT - 1) / CUT, 1u);
    }
    return u;
}

// How the units of the streamed sequences are dealt out to the workgroups of a kv
// head. Shares of q units, whatever sequences they are of, so that ragged lengths even
// out; or, where no more workgroups than there are take parts of at most q units that
// each lie in one sequence, those: sequences of one length (16 of 4096 tokens 27 us; in
// shares, whose second sequence begins with loads that nothing hides, 32). Every wave by
// itself.
struct Share {
    uint32_t q, total;
    bool parts;
    // the workgroups (parts) or units of a sequence
    ZH_DEVM uint32_t items(const UnitSeq &u) const { return u.tiles * (parts ? (u.units + q - 1) / q : u.units); }
};
// u0: the lane's sequence (of the first 64)
ZH_DEV Share share(const Kv8Attn &a, const UnitSeq &u0, bool &bad) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t n = u0.tiles * u0.units;
    for (uint32_t s = lane + 64; s < a.n_seq; s += 64) {
        const UnitSeq u = unit_seq(a, s, bad);
        n += u.tiles * u.units;
    }
    Share x;
    x.total = wave_total(n);
    x.q = max((x.total + a.groups - 1) / a.groups, a.least);
    x.parts = true;
    n = x.items(u0);
    for (uint32_t s = lane + 64; s < a.n_seq; s += 64) n += x.items(unit_seq(a, s, bad));
    x.parts = wave_total(n) <= a.groups;
    return x;
}
ZH_DEV UnitSeq first_units(const Kv8Attn &a, bool &bad) {
    const uint32_t lane = threadIdx.x & 63;
    return lane < a.n_seq ? unit_seq(a, lane, bad) : UnitSeq{0, 1};
}

// A share of units of one kv head: in each sequence that it reaches into, up to 16 RT
// rows over some of its tokens. A sequence that lies in one share is finished there;
// of the others, each share leaves its unnormalised sum, maximum and sum of weights for
// k_kv8_join: in slot 0 of the workgroup if it begins inside the sequence, else in slot
// 1, so that a workgroup needs two however many sequences there are. Each wave takes
// steps of NJ pages by itself, K and V straight from the cache into registers (no
// LDS, no barrier before the end), the next step's K requested when the scores are
// done and its V after the products with this one's:
//   S^T = K q^T (tokens x rows): lane (li = lane % 16, lg = lane / 16) reads 16
//   codes of token li, dims 64 u + 16 lg .., which are two fragments (the dims'
//   order within a product is free, q's fragments follow it), and holds the scores
//   of tokens 4 lg + r of row li;
//   O^T += V^T P^T, k = (token 4 lg + r of a page, then of the next): lane li reads
//   dims HD/16 li .. of its 4 tokens, and pairs of tokens are put side by side by byte
//   permutes before they become fp16; column li of output tile n is dim HD/16 li + n.
// NP pieces of q (scaled by a power of two to a maximum in [2^14, 2^15)) as sums of
// fp16 values, 2 of the weights: 22 bits of each.
// Bound by HBM where the sequences are long (64 of 16384 tokens, 8 kv heads of 128: 315 us,
// 6.4 TB/s), by 8 to 10 us of start, last steps and the waves' joining where not (48 ragged
// ones to 4096 tokens, f32 i8: 41 us, 4.9 TB/s; 16 of 4096 25 us, 5.1); 24 sequences of 20
// rows at 3000 tokens, head_dim 64, 4 kv heads, 16 us: three steps in every wave, behind a
// start of some five loads that depend on one another and the finding of its share; vector
// instructions in 61% of the cycles, on 32 row slots.
template <int HD, int NP, int RT, uint32_t F, typename T>
__global__ __launch_bounds__(64 * W, RT == 1 || HD == 64 ? 3 : 2) void k_kv8_attn(Kv8Attn a) {
    constexpr uint32_t KB = 16 * NJ;
    constexpr int U = HD / 64, ND = HD / 16, VD = ND / 4;  // 16-code pieces of a K row, dims and dwords of V per lane
    constexpr int LD = HD + 4, NQ = sizeof(T) == 2 ? 1 : NP, PV = 2;
    constexpr uint32_t ROWS = 16 * RT;
    __shared__ __align__(16) float so[W * 16 * LD];
    __shared__ float sm[W * 16], sl[W * 16];
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t li = lane % 16, lg = lane / 16, koff = li * HD + 16 * lg, voff = 4 * lg * HD + ND * li;
    // (kv heads fastest: with 8 of them every head's K and V stay in one XCD's L2)
    const uint32_t kvh = blockIdx.x % a.nkv, group = blockIdx.x / a.nkv;
    // the sequence and row tile, the unit in it, units to take from there
    uint32_t s = group / a.tiles, tile = group % a.tiles, unit = 0, left = ~0u;
    bool bad = false;
    if (a.least) {
        const UnitSeq u0 = first_units(a, bad);
        const Share x = share(a, u0, bad);
        if (__builtin_amdgcn_ballot_w64(bad) && blockIdx.x == 0 && tid == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
        auto count = [&](uint32_t i) { return x.items(i < 64 ? u0 : unit_seq(a, i, bad)); };
        uint32_t item;
        if (!kv8_find(a.n_seq, x.parts ? group : group * x.q, count, s, item)) return;
        const UnitSeq u = unit_seq(a, s, bad);
        const uint32_t p = x.parts ? (u.units + x.q - 1) / x.q : u.units;
        tile = item / p;
        unit = item % p;
        left = x.q;
        if (x.parts) {  // (all of a length)
            const uint32_t c = (u.units + p - 1) / p;
            unit *= c;
            left = u.units > unit ? min(c, u.units - unit) : 0u;
        }
    } else {
        attn_seq(a, s, bad);
        if (bad && kvh == 0 && tile == 0 && tid == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
    }
    // (made scalars before the loop, or, with 32 rows, in it: the other way round 16 rows
    // of f32 spill 5 registers, 32 spill 14, and 48 ragged sequences take 56 us for 46.5)
    auto scalars = [&]() __attribute__((always_inline)) {
        s = scalar(s);
        tile = RT == 1 ? 0u : scalar(tile);  // (16 rows: one tile)
        unit = scalar(unit);
        left = scalar(left);
    };
    if (RT == 1) scalars();
    while (true) {
        if (RT > 1) scalars();
        if (!left || s >= a.n_seq) break;
        bad = false;
        const AttnSeq seq = attn_seq(a, s, bad);
        bad = false;
        const uint32_t all_rows = seq.n * a.G, row0 = RT == 1 ? 0u : tile * ROWS;
        if (row0 >= all_rows || all_rows > a.few) {  // (none, or no streamed ones)
            if (!a.least) return;
            s++;
            continue;
        }
        const uint32_t nrow = min(ROWS, all_rows - row0);
        // the tokens that some row of the sequence sees, of the tile, and those that all of
        // the tile see
        const uint32_t far = scalar(seq.lim(seq.n - 1)), end = RT == 1 ? far : scalar(seq.lim((row0 + nrow - 1) / a.G));
        const uint32_t every = scalar(seq.lim(row0 / a.G));
        const uint32_t units = max((far + CUT - 1) / CUT, 1u);
        const uint32_t take = min(left, units - unit), t0 = min(unit * CUT, end), t1 = min(t0 + take * CUT, end);
        const bool direct = take == units;
        const uint32_t slot = unit ? 0u : 1u;
        left = a.least ? left - take : 0u;
        unit = 0;
        // (where the next one begins, if there is one)
        const bool last = RT == 1 || row0 + ROWS >= all_rows;
        tile = last ? 0u : tile + 1;
        s += last;
        const uint32_t nstep = t1 > t0 ? (t1 - t0 + KB - 1) / KB : 0u;
        const uint8_t *kh = a.kc + (size_t)kvh * a.cache_tokens * HD, *vh = a.vc + (size_t)kvh * a.cache_tokens * HD;
        const const_u32 *tab = (const const_u32 *)(a.tables + (size_t)seq.s * a.stride);
        const const_u32 *ksc = (const const_u32 *)(a.ks + kvh), *vsc = (const const_u32 *)(a.vs + kvh);
        // a step's pages (clamped to the last of the part), looked up a step ahead by
        // scalar loads, whose wait does not wait for K and V
        struct Step {
            uint32_t tk, pg[NJ];
        };
        auto step = [&](uint32_t st) __attribute__((always_inline)) {
            Step x;
            x.tk = t0 + st * KB;
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) {
                x.pg[j] = tab[min(x.tk / 16 + j, (t1 - 1) / 16)];
                if (x.pg[j] >= a.cache_tokens / 16) {
                    bad = true;
                    x.pg[j] = 0;
                }
            }
            return x;
        };
        u32x4 kr[NJ][U];
        uint32_t vr[NJ][4][VD];
        auto load_k = [&](const Step &x) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) {
                const uint8_t *p = kh + (size_t)x.pg[j] * (16 * HD) + koff;
#pragma unroll
                for (int u = 0; u < U; u++) kr[j][u] = ld_once<RT == 1>((const u32x4 *)(p + 64 * u));
            }
        };
        auto load_v = [&](const Step &x) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) {
                const uint8_t *p = vh + (size_t)x.pg[j] * (16 * HD) + voff;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (VD == 2) *(u32x2 *)vr[j][r] = ld_once<RT == 1>((const u32x2 *)(p + r * HD));
                    else vr[j][r][0] = ld_once<RT == 1>((const uint32_t *)(p + r * HD));
                }
            }
        };
        uint32_t ksb[NJ], vsb[NJ];  // this step's scales
        auto load_s = [&](const Step &x) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) {
                ksb[j] = ksc[(size_t)x.pg[j] * a.nkv];
                vsb[j] = vsc[(size_t)x.pg[j] * a.nkv];
            }
        };
        Step x = {}, nx = {};
        if (wave < nstep) {
            x = step(wave);
            load_k(x);
            load_v(x);
            load_s(x);
            if (wave + W < nstep) nx = step(wave + W);
        }
        // the rows' q as operand fragments: dims 64 u + 16 lg + 8 h .. (the scale's sign in them)
        auto load_q = [&](int rt, half8 (&qf)[NQ][2 * U], float &cf, uint32_t &lim) __attribute__((always_inline)) {
            const uint32_t r = row0 + min(16 * rt + li, nrow - 1), i = r / a.G;
            lim = min(seq.lim(i), t1);
            const T *qp = (const T *)(a.q + (uint64_t)(seq.row + i) * a.q_row) + (size_t)(kvh * a.G + r % a.G) * HD + 16 * lg;
            float v[2 * U][8], mx = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * U; k++) {
                ld8(qp + 64 * (k / 2) + 8 * (k % 2), v[k]);
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(v[k][e]));
            }
            int e = 0;  // q is scaled by 2^-e
            if (NQ > 1) {
                mx = xor32_max(xor16_max(mx));
                const uint32_t E = __float_as_uint(mx) >> 23;
                if (E < 255) e = (int)E - 141;  // (E == 0, subnormal or zero rows: a smaller maximum)
            }
            const float sign = copysignf(1.f, a.scale);
#pragma unroll
            for (int k = 0; k < 2 * U; k++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float y = (NQ > 1 ? ldexpf(v[k][i], -e) : v[k][i]) * sign;
#pragma unroll
                    for (int p = 0; p < NQ; p++) {
                        qf[p][k][i] = (_Float16)y;
                        y -= (float)qf[p][k][i];
                    }
                }
            cf = fabsf(ldexpf(a.scale, a.scale_exp + e));
        };
        half8 qf[RT][NQ][2 * U];
        float cf[RT];  // products to base-2 scores, but for the block's scale
        uint32_t lim[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) load_q(rt, qf[rt], cf[rt], lim[rt]);
        floatx4 o[RT][ND];
        float m[RT], l[RT];  // the row's reference (every lg alike), this lane's share of its sum
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            m[rt] = -INFINITY;
            l[rt] = 0.f;
#pragma unroll
            for (int n = 0; n < ND; n++) o[rt][n] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
        bool far_apart = false;  // (some block's scale of V is)
        // the weights and products of step x; `more`: the next step's loads on the way.
        // (The last step is code of its own: a load that may not be there would make
        // the compiler wait for V before the scores.)
        auto work = [&](auto more) __attribute__((always_inline)) {
            Block<F> b[NJ];
            bool ok = true;
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) {
                b[j].set(scalar(ksb[j]), scalar(vsb[j]));
                ok = ok && b[j].ok;
                far_apart = far_apart || b[j].apart;
            }
            floatx4 d[RT][NJ];
#pragma unroll
            for (uint32_t j = 0; j < NJ; j++) {
                half8 kf[2 * U];
#pragma unroll
                for (int k = 0; k < 2 * U; k++)
                    kf[k] = row8<F>(kr[j][k / 2][2 * (k % 2)], kr[j][k / 2][2 * (k % 2) + 1]);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    d[rt][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int p = NQ - 1; p >= 0; p--)
#pragma unroll
                        for (int k = 0; k < 2 * U; k++)
                            d[rt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k], qf[rt][p][k], d[rt][j], 0, 0, 0);
                }
            }
            if constexpr (more) {
                load_k(nx);
                load_s(nx);
            }
            const bool whole = ok && x.tk + KB <= min(every, t1);
            half8 pf[RT][PV][NJ / 2];
            float f[RT];
            if (!whole) {
                // V of tokens past the part: zero (0 times what the cache holds there may be NaN)
#pragma unroll
                for (uint32_t j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int y = 0; y < VD; y++) vr[j][r][y] = x.tk + 16 * j + 4 * lg + r >= t1 ? 0u : vr[j][r][y];
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                float sc[NJ][4], mb = -INFINITY;
#pragma unroll
                for (uint32_t j = 0; j < NJ; j++) {
                    const float ck = score_factor(cf[rt], b[j].ks);
#pragma unroll
                    for (int r = 0; r < 4; r++) sc[j][r] = fmaf(d[rt][j][r], ck, b[j].lv);
                }
                if (!whole) {
#pragma unroll
                    for (uint32_t j = 0; j < NJ; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const bool out = x.tk + 16 * j + 4 * lg + r >= lim[rt];
                            sc[j][r] = out ? -INFINITY : b[j].ok ? sc[j][r] : NAN;
                        }
                }
#pragma unroll
                for (uint32_t j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) mb = fmaxf(mb, sc[j][r]);
                mb = xor32_max(xor16_max(mb));
                // (the largest weight is 2^14: what fp16's subnormals lose of the others is 2^-39 of
                // it; scores of 2^24 on have steps of 2 and more, and no room for 14 exactly)
                const float mn = fmaxf(m[rt], fabsf(mb) < 0x1p24f ? mb - 14.f : mb), ms = mn == -INFINITY ? 0.f : mn;
                f[rt] = __builtin_amdgcn_exp2f(m[rt] - ms);  // (m = -inf: 0)
                m[rt] = mn;
                float ls = 0.f;
#pragma unroll
                for (uint32_t j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float p = __builtin_amdgcn_exp2f(sc[j][r] - ms);
                        ls = fmaf(p, b[j].iv, ls);
#pragma unroll
                        for (int k = 0; k < PV; k++) {
                            pf[rt][k][j / 2][4 * (j % 2) + r] = (_Float16)p;
                            p -= (float)pf[rt][k][j / 2][4 * (j % 2) + r];
                        }
                    }
                l[rt] = fmaf(l[rt], f[rt], ls);
            }
            if (F == ZH_I8) {
#pragma unroll
                for (uint32_t j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int y = 0; y < VD; y++) vr[j][r][y] ^= 0x80808080u;
            }
#pragma unroll
            for (int n = 0; n < ND; n += 2) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        o[rt][n][r] *= f[rt];
                        o[rt][n + 1][r] *= f[rt];
                    }
#pragma unroll
                for (uint32_t jj = 0; jj < NJ / 2; jj++) {
                    half2v e[2][4];  // dims n and n + 1: token pairs of the two pages
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        pair2<F>(vr[2 * jj + i / 2][2 * (i % 2)][n / 4], vr[2 * jj + i / 2][2 * (i % 2) + 1][n / 4], n, e[0][i],
                                 e[1][i]);
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const half8 vf = {e[y][0].x, e[y][0].y, e[y][1].x, e[y][1].y, e[y][2].x, e[y][2].y, e[y][3].x, e[y][3].y};
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int p = PV - 1; p >= 0; p--)
                                o[rt][n + y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt][p][jj], o[rt][n + y], 0, 0, 0);
                    }
                }
            }
            if constexpr (more) load_v(nx);
        };
        if (wave < nstep) {
            for (uint32_t st = wave + W; st < nstep; st += W) {
                const Step nn = st + W < nstep ? step(st + W) : nx;
                work(std::true_type{});
                x = nx;
                nx = nn;
            }
            work(std::false_type{});
        }
        if (bad && lane == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
        // a lane's share of a row's sum again, from the scores without V's scales
        auto far_sum = [&](int rt, float m) __attribute__((always_inline)) {
            half8 qf[NQ][2 * U];
            float cf, sum = 0.f;
            uint32_t lim;
            load_q(rt, qf, cf, lim);
            const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll 1
            for (uint32_t tk = t0 + KB * wave, j = 0; tk < t1; tk += j ? KB * W - 16 * (NJ - 1) : 16, j ^= 1) {
                const uint32_t pg = scalar(tab[tk / 16]), page = pg < a.cache_tokens / 16 ? pg : 0u;
                const uint8_t *at = kh + (size_t)page * (16 * HD) + koff;
                Block<F> b;
                b.set(scalar(ksc[(size_t)page * a.nkv]), scalar(vsc[(size_t)page * a.nkv]));
                half8 kf[2 * U];
#pragma unroll
                for (int k = 0; k < 2 * U; k++) {
                    const u32x2 c = *(const u32x2 *)(at + 64 * (k / 2) + 8 * (k % 2));
                    kf[k] = row8<F>(c.x, c.y);
                }
                floatx4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = NQ - 1; p >= 0; p--)
#pragma unroll
                    for (int k = 0; k < 2 * U; k++) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k], qf[p][k], d, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float s = fmaf(d[r], score_factor(cf, b.ks), b.lv) - ms - b.lv;
                    sum += tk + 4 * lg + r >= lim ? 0.f : __builtin_amdgcn_exp2f(s) * b.unit();
                }
            }
            return sum;
        };
        // ---- join the waves; lane li, lg: row li, dims ND (4 lg + r) + n
        if (far_apart)  // (uniform per wave)
#pragma unroll 1
            for (int rt = 0; rt < RT; rt++) {
                const float sum = far_sum(rt, m[RT == 1 ? 0 : rt ? RT - 1 : 0]);
                if (RT == 1 || rt == 0) l[0] = sum;
                else l[RT - 1] = sum;
            }
        const size_t p0 = ((size_t)blockIdx.x * 2 + slot) * ROWS;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            __syncthreads();  // (the words below have been read)
            const float ls = xor32_sum(xor16_sum(l[rt]));
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int n = 0; n < ND; n += 4)
                    *(f32x4 *)(so + (wave * 16 + li) * LD + ND * (4 * lg + r) + n) =
                        f32x4{o[rt][n][r], o[rt][n + 1][r], o[rt][n + 2][r], o[rt][n + 3][r]};
            if (lg == 0) {
                sm[wave * 16 + li] = m[rt];
                sl[wave * 16 + li] = ls;
            }
            __syncthreads();
            for (uint32_t i = tid; i < 16 * (HD / 4); i += 64 * W) {
                const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
                if (16 * rt + r >= nrow) break;
                const uint32_t R = row0 + 16 * rt + r, qi = R / a.G, h = kvh * a.G + R % a.G;
                float M = sm[r], low = M, L = 0.f;
                f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 1; k < W; k++) {
                    M = fmaxf(M, sm[k * 16 + r]);
                    low = fminf(low, sm[k * 16 + r]);
                }
                const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
                for (int k = 0; k < W; k++) {
                    const float fk = __builtin_amdgcn_exp2f(sm[k * 16 + r] - Ms);
                    const f32x4 v = *(const f32x4 *)(so + (k * 16 + r) * LD + d);
                    O.x = fmaf(v.x, fk, O.x);
                    O.y = fmaf(v.y, fk, O.y);
                    O.z = fmaf(v.z, fk, O.z);
                    O.w = fmaf(v.w, fk, O.w);
                    L = fmaf(sl[k * 16 + r], fk, L);
                }
                if (__builtin_amdgcn_ballot_w64(low - Ms < -126.f)) {
                    L = 0.f;
#pragma unroll
                    for (int k = 0; k < W; k++) {
                        const Shift to(sm[k * 16 + r] - Ms);
                        L = fmaf(sl[k * 16 + r] * to.a, to.b, L);
                    }
                }
                if (direct) {
                    const f32x4 v = seq.lim(qi) ? f32x4{O.x / L, O.y / L, O.z / L, O.w / L} : f32x4{0.f, 0.f, 0.f, 0.f};
                    st_out<T>(a, seq.row + qi, h, d, HD, v);
                } else {
                    const size_t pr = p0 + 16 * rt + r;
                    *(f32x4 *)(a.part + pr * HD + d) = O;
                    if (d == 0) {
                        a.stat[2 * pr] = M;
                        a.stat[2 * pr + 1] = L;
                    }
                }
            }
        }
    }
}

// Many rows: a workgroup takes 256 of them (rows of a kv head in the order query,
// head), each wave 32, over K and V that pass through LDS once for all of them, in
// stages of 64 tokens, as fp16: every thread converts its pieces on the way there, so
// a code becomes fp16 once a workgroup and not once a wave.
//   S^T = K q^T by v_mfma_f32_32x32x16_f16: lane (i = lane % 32, h = lane / 32)
//   holds tokens 8 (r / 4) + 4 h + r % 4 of row i in register r: registers 0 .. 7 are
//   one page's, 8 .. 15 the next one's, each with its block's scales; registers
//   8 s .. 8 s + 7 are the weights' operand of the s-th 16-token product
//   O^T += V^T P^T. V stays row-major in LDS, its transposed fragments come from
//   ds_read_b64_tr_b16. Rows are padded, K's by 16 bytes, V's by 64: 16 rows' reads of
//   one 16-byte piece hit every bank once, the transposing reads (64 bytes of 8 rows)
//   every bank twice, and all of a lane's fragments lie at constant offsets from one
//   address (swizzled pieces took 24 registers of addresses, and 12 others to scratch,
//   whose reloads wait for the loads on the way).
// The products of the next 32 tokens' scores run while the current ones' weights
// are computed. Weights are in two pieces, as where rows are streamed: in one, f16 results
// were 2.7e-4 off where their rounding alone is 2.1e-4 (4096 rows then 730 us for 960). 4096
// rows after 8192 tokens, 32 heads of 128 in f16, 687 GFLOP (1030 with the second piece) in
// 955 to 1000 us: the matrix units are busy for 50% of the cycles, vector instructions for
// 59%, and the clock falls under both. The reference moves only when a score passes it by
// 2^8 (the weights then reach 2^12 in fp16 at most), so the output is rarely rescaled. A
// wave stops at the last token that one of its rows sees.
constexpr int TW = 8;                          // waves of a workgroup
constexpr uint32_t TILE = 32 * TW;             // its rows
constexpr uint32_t TK = 64, TS = 3;            // tokens of a stage, stages in LDS
template <int HD>
constexpr uint32_t t_krow() { return 2 * HD + 16; }
template <int HD>
constexpr uint32_t t_vrow() { return 2 * HD + 64; }
template <int HD>
constexpr uint32_t t_lds() { return TS * TK * (t_krow<HD>() + t_vrow<HD>()) + TS * 64; }

typedef float f32x16 __attribute__((ext_vector_type(16)));

// The LDS tiles of sequence s and the stages of its longest one.
struct TileSeq {
    uint32_t tiles, stages;
};
ZH_DEV TileSeq tile_seq(const Kv8Attn &a, uint32_t rows, uint32_t s) {
    bool bad = false;
    const AttnSeq x = attn_seq(a, s, bad);
    const uint64_t n = (uint64_t)x.n * a.G;
    TileSeq t = {0, 1};
    if (n > a.few) {
        t.tiles = (uint32_t)((n + rows - 1) / rows);
        t.stages = max((x.lim(x.n - 1) + TK - 1) / TK, 1u);
    }
    return t;
}
// The most stages of a workgroup where tiles are cut: about the least for which no more
// workgroups than there are take all parts, so that the tiles of a long context are cut
// into more parts than those of a short one. Every wave by itself. t0: the lane's
// sequence's tiles (of the first 64).
ZH_DEV uint32_t tile_share(const Kv8Attn &a, uint32_t rows, const TileSeq &t0) {
    if (!a.tslots) return 1u << 30;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t n = t0.tiles * t0.stages;
    for (uint32_t s = lane + 64; s < a.n_seq; s += 64) {
        const TileSeq t = tile_seq(a, rows, s);
        n += t.tiles * t.stages;
    }
    uint32_t q = max((wave_total(n) + a.tslots - 1) / a.tslots, 4u);
    while (q < 1u << 24) {  // (a part a tile always fits)
        n = t0.tiles * ((t0.stages + q - 1) / q);
        for (uint32_t s = lane + 64; s < a.n_seq; s += 64) {
            const TileSeq t = tile_seq(a, rows, s);
            n += t.tiles * ((t.stages + q - 1) / q);
        }
        if (wave_total(n) <= a.tslots) break;
        q += (q + 7) / 8;
    }
    return q;
}
// A workgroup's part of a tile.
struct TileJob {
    AttnSeq seq;
    uint32_t tile, part, c;  // parts of c stages
};
ZH_DEV TileSeq first_seqs(const Kv8Attn &a, uint32_t rows) {
    const uint32_t lane = threadIdx.x & 63;
    return lane < a.n_seq ? tile_seq(a, rows, lane) : TileSeq{0, 1};
}
// Workgroup `u` of a kv head: sequences in order, of each the last tiles (which see the
// most tokens) first, of each tile the parts.
ZH_DEV bool tile_job(const Kv8Attn &a, uint32_t rows, uint32_t u, TileJob &j) {
    const TileSeq t0 = first_seqs(a, rows);
    const uint32_t q = tile_share(a, rows, t0);
    auto count = [&](uint32_t i) {
        const TileSeq t = i < 64 ? t0 : tile_seq(a, rows, i);
        return t.tiles * ((t.stages + q - 1) / q);
    };
    uint32_t s, item;
    if (!kv8_find(a.n_seq, u, count, s, item)) return false;
    s = scalar(s);
    bool bad = false;
    j.seq = attn_seq(a, s, bad);
    const TileSeq t = tile_seq(a, rows, s);
    const uint32_t p = (t.stages + q - 1) / q;
    j.c = scalar((t.stages + p - 1) / p);
    j.tile = scalar(t.tiles - 1 - item / p);
    j.part = scalar(item % p);
    return true;
}

template <int HD, int NP, uint32_t F, typename T>
__global__ __launch_bounds__(64 * TW, 2) void k_kv8_tile(Kv8Attn a) {
    constexpr int KS = HD / 16, DT = HD / 32;        // k-steps of the scores, 32-dim tiles of the output
    constexpr int PW = 2;                            // pieces of the weights
    constexpr uint32_t KROW = t_krow<HD>(), VROW = t_vrow<HD>(), KST = TK * KROW, VST = TK * VROW;  // of a row, a stage
    constexpr uint32_t ROWS = TILE, NT = 64 * TW;
    constexpr uint32_t CPR = HD / 16, PC = TK * CPR;  // 16-code pieces of a row and of a stage's K (or V)
    constexpr uint32_t NPC = 2 * PC / NT;             // a thread's pieces
    extern __shared__ __align__(16) uint8_t lds[];
    typedef __fp16 tr4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) tr4 lds_tr4;
    float *const scl = (float *)(lds + TS * (KST + VST));  // [stage][page]: Block's ks, lv, iv; 0 not ok, 2 apart, 1 else
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t i32 = lane % 32, h = lane / 32;
    // (kv heads fastest: with 8 of them every head's K and V stay in one XCD's L2)
    const uint32_t kvh = blockIdx.x % a.nkv;
    if (!a.few && blockIdx.x == 0) {  // (no streamed rows: their launch would report these)
        bool wrong = false;
        for (uint32_t i = tid; i < a.n_seq; i += NT) attn_seq(a, i, wrong);
        if (wrong) atomicOr(a.err, ZH_DEVERR_KV_ROW);
    }
    TileJob job;
    if (!tile_job(a, ROWS, blockIdx.x / a.nkv, job)) return;
    const AttnSeq &seq = job.seq;
    const uint32_t rows = seq.n * a.G, r0 = job.tile * ROWS, w0 = r0 + wave * 32;
    const uint32_t end = scalar(seq.lim((min(r0 + ROWS, rows) - 1) / a.G)), t0 = job.part * job.c * TK;
    if (job.part && t0 >= end) return;  // (rows without tokens: part 0 writes their zeros)
    const uint32_t t1 = min(t0 + job.c * TK, end), nst = t1 > t0 ? (t1 - t0 + TK - 1) / TK : 0u;
    // the wave's rows: the stages that it takes, the tokens that all of them see
    const bool mine = w0 < rows;
    const uint32_t wend = mine ? min(scalar(seq.lim((min(w0 + 32, rows) - 1) / a.G)), t1) : 0u;
    const uint32_t wst = wend > t0 ? (wend - t0 + TK - 1) / TK : 0u, every = mine ? min(scalar(seq.lim(w0 / a.G)), t1) : 0u;
    const uint32_t row = min(w0 + i32, rows - 1), qi = row / a.G, lim = min(seq.lim(qi), t1);
    // ---- a thread's pieces of a stage: 16 codes of a token each, of K or V (HD 64) or of both
    const uint8_t *kh = a.kc + (size_t)kvh * a.cache_tokens * HD, *vh = a.vc + (size_t)kvh * a.cache_tokens * HD;
    const uint32_t *tab = a.tables + (size_t)seq.s * a.stride;
    bool bad = false;
    const uint32_t trow = tid % PC / CPR, col = tid % CPR;  // the token of the stage, 16 dims of it
    const bool isk = NPC == 2 || tid < PC, scales = isk && col == 0 && trow % 16 == 0;
    // (one address of each kind in a register: the ring's other slots lie at immediate
    // offsets from it, which reach 64 KiB)
    const uint32_t kput = opaque(isk ? trow * KROW + col * 32 : TS * KST + trow * VROW + col * 32);
    const uint32_t vput = opaque(TS * KST + trow * VROW + col * 32), sput = opaque(TS * (KST + VST) + trow);
    struct Raw {
        u32x4 x[NPC];
        uint32_t k, v;  // scales (of the threads that have a page's first piece of K)
    };
    uint32_t pg;
    auto look = [&](uint32_t st) __attribute__((always_inline)) { pg = tab[min((t0 + st * TK + trow) / 16, (t1 - 1) / 16)]; };
    auto fetch = [&](Raw &r) __attribute__((always_inline)) {
        if (pg >= a.cache_tokens / 16) {
            bad = true;
            pg = 0;
        }
        const size_t at = ((size_t)pg * 16 + trow % 16) * HD + col * 16;
        r.x[0] = *(const u32x4 *)((isk ? kh : vh) + at);
        if (NPC == 2) r.x[NPC - 1] = *(const u32x4 *)(vh + at);
        if (scales) {
            r.k = ((const uint32_t *)a.ks)[(size_t)pg * a.nkv + kvh];
            r.v = ((const uint32_t *)a.vs)[(size_t)pg * a.nkv + kvh];
        }
    };
    auto put = [&](uint32_t st, const Raw &r) __attribute__((always_inline)) {
        const uint32_t slot = st % TS;
#pragma unroll
        for (uint32_t i = 0; i < NPC; i++) {
            u32x4 x = r.x[i];
            // V past the part: zero (0 times what the cache holds there may be NaN)
            if ((NPC == 2 ? i : !isk) && t0 + st * TK + trow >= t1) x = u32x4{0, 0, 0, 0};
            uint8_t *to = lds + (i ? vput + slot * VST : kput + (isk ? slot * KST : slot * VST));
            *(half8 *)to = row8<F>(x.x, x.y);
            *(half8 *)(to + 16) = row8<F>(x.z, x.w);
        }
        if (scales) {
            Block<F> b;
            b.set(r.k, r.v);
            *(f32x4 *)(lds + sput + slot * 64) = f32x4{b.ks, b.lv, b.iv, !b.ok ? 0.f : b.apart ? 2.f : 1.f};
        }
    };
    Raw raw;
    if (nst) {
        Raw raw1;
        look(0);
        fetch(raw);
        look(1);
        fetch(raw1);
        look(2);
        put(0, raw);
        if (nst > 1) put(1, raw1);
        fetch(raw);
        look(3);
    }
    // ---- the row's q: dims 16 k + 8 h ..
    half8 qf[NP][KS];
    float cf;  // products to base-2 scores, but for the block's scale
    {
        const T *qp = (const T *)(a.q + (uint64_t)(seq.row + qi) * a.q_row) + (size_t)(kvh * a.G + row % a.G) * HD + 8 * h;
        float v[KS][8], mx = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            ld8(qp + 16 * k, v[k]);
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(v[k][e]));
        }
        int qe = 0;  // q is scaled by 2^-qe
        if (NP > 1) {
            mx = xor32_max(mx);
            const uint32_t E = __float_as_uint(mx) >> 23;
            if (E < 255) qe = (int)E - 141;
        }
        // (the scale's sign goes into q: the largest product is the largest score)
        const float sign = copysignf(1.f, a.scale);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float x = (NP > 1 ? ldexpf(v[k][e], -qe) : v[k][e]) * sign;
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    qf[p][k][e] = (_Float16)x;
                    x -= (float)qf[p][k][e];
                }
            }
        cf = fabsf(ldexpf(a.scale, a.scale_exp + qe));
    }
    f32x16 o[DT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.f;
    // a lane's fragments in a stage: K's k-step k at kp + 32 k, V's 32-dim tile d at vp +
    // 64 d, of tokens 4 h .. +3, and of those 8 on
    const uint32_t l16 = lane % 16;
    const uint8_t *const kp = lds + i32 * KROW + 16 * h;
    const uint8_t *const vp = lds + opaque(TS * KST + (4 * h + l16 / 4) * VROW + 32 * (lane / 16 % 2) + 8 * (l16 % 4));
    f32x16 sc, sn;  // products of the current and the next 32 tokens
    half8 kf[KS];   // K fragments of the next ones
    struct Half {   // of 32 tokens' two pages: scores' factors, weights' exponents and shares
        float ck[2], lv[2], iv[2];
        bool ok;
        uint32_t apart;
    };
    Half hc, hn;
    // (two pieces of f32 leave no registers for V beside the scores' products, nor for
    // all of K ahead of them)
    constexpr bool LATE = NP == 2 && HD == 128;
    constexpr int AHEAD = LATE ? KS / 2 : KS;
    auto load_k = [&](uint32_t slot, uint32_t kt, int k0, int k1) __attribute__((always_inline)) {
#pragma unroll
        for (int k = k0; k < k1; k++) kf[k] = *(const half8 *)(kp + slot * KST + kt * 32 * KROW + 32 * k);
    };
    auto load_h = [&](Half &x, uint32_t slot, uint32_t kt) __attribute__((always_inline)) {
        float ok = 1.f;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const f32x4 b = *(const f32x4 *)(scl + (slot * 4 + 2 * kt + j) * 4);
            x.ck[j] = score_factor(cf, b.x);
            x.lv[j] = b.y;
            x.iv[j] = b.z;
            ok *= b.w;
        }
        const uint32_t all = __builtin_amdgcn_readfirstlane(__float_as_uint(ok));
        x.ok = all != 0;
        x.apart = all > 0x3F800000u;
    };
    // the reference, for scores up to mx: moved, and the sums with it, where one
    // passes it by 2^8
    auto refer = [&](float mx) __attribute__((always_inline)) {
        mx = xor32_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx);
            const Shift to(m - (mn == -INFINITY ? 0.f : mn));
            const float f = to.both();
            m = mn;
            l = l * to.a * to.b;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] *= f;
        }
    };
    auto largest = [&](const f32x16 &d, const Half &x) __attribute__((always_inline)) {
        float y = d[0], z = d[8];
#pragma unroll
        for (int r = 1; r < 8; r++) {
            y = fmaxf(y, d[r]);
            z = fmaxf(z, d[8 + r]);
        }
        return fmaxf(fmaf(y, x.ck[0], x.lv[0]), fmaf(z, x.ck[1], x.lv[1]));
    };
    // tokens from t on that the row does not see: no score; blocks that read as NaN
    // (their factors are harmless)
    auto mask = [&](uint32_t t, f32x16 &d, uint32_t slot, uint32_t kt) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const bool ok = scl[(slot * 4 + 2 * kt + j) * 4 + 3] != 0.f;
#pragma unroll
            for (int r = 8 * j; r < 8 * j + 8; r++)
                d[r] = t + 8 * (r / 4) + 4 * h + r % 4 >= lim ? -INFINITY : ok ? d[r] : NAN;
        }
    };
    lds_bar();
    if (wst) {
        load_k(0, 0, 0, KS);
        load_h(hc, 0, 0);
#pragma unroll
        for (int r = 0; r < 16; r++) sc[r] = 0.f;
#pragma unroll
        for (int p = NP - 1; p >= 0; p--)
#pragma unroll
            for (int k = 0; k < KS; k++) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k], qf[p][k], sc, 0, 0, 0);
        load_k(0, 1, 0, AHEAD);
        if (t0 + 32 > every || !hc.ok) mask(t0, sc, 0, 0);
        refer(largest(sc, hc));
    }
    constexpr int PAIRS = 8, EARLY = 6;  // weights in pairs; those taken beside the scores' products
    for (uint32_t s0 = 0; s0 < nst; s0 += TS)  // (the ring's slots unrolled: constant LDS offsets)
#pragma unroll
    for (uint32_t slot = 0; slot < TS; slot++) {
        const uint32_t st = s0 + slot;
        if (st >= nst) break;  // uniform
        lds_bar();
        auto next = [&]() __attribute__((always_inline)) {  // the stages ahead
            if (st + 2 < nst) put(st + 2, raw);
            if (st + 3 < nst) {
                fetch(raw);
                look(st + 4);
            }
        };
        if (st >= wst) {  // uniform per wave
            next();
            continue;
        }
        const uint32_t tk = t0 + st * TK;
#pragma unroll
        for (uint32_t kt = 0; kt < 2; kt++) {
            half8 pf[PW][2], vf[2][DT];
            const float ms = m == -INFINITY ? 0.f : m;
            float bl[2] = {hc.lv[0] + (4.f - ms), hc.lv[1] + (4.f - ms)};
            // where m's own rounding passes 1/4, the scores are rounded as it was before it is
            // taken from them
            const uint64_t far = __builtin_amdgcn_ballot_w64(fabsf(ms) >= 0x1p22f);
            if (far | hc.apart) {  // (one branch)
                if (far) {
#pragma unroll
                    for (int r = 0; r < 16; r++) sc[r] = fmaf(sc[r], hc.ck[r / 8], hc.lv[r / 8]) - ms;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        hc.ck[j] = 1.f;
                        bl[j] = 4.f;
                    }
                }
                if (hc.apart)
#pragma unroll
                    for (int r = 0; r < 16; r++) l += lost_share(fmaf(sc[r], hc.ck[r / 8], bl[r / 8]), hc.iv[r / 8]);
            }
            float mx = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r++) sn[r] = 0.f;
            auto weights = [&](int i) __attribute__((always_inline)) {  // 2 i and 2 i + 1
#pragma unroll
                for (int r = 2 * i; r < 2 * i + 2; r++) {
                    float p = __builtin_amdgcn_exp2f(fmaf(sc[r], hc.ck[r / 8], bl[r / 8]));
                    l = fmaf(p, hc.iv[r / 8], l);
#pragma unroll
                    for (int k = 0; k < PW; k++) {
                        pf[k][r / 8][r % 8] = (_Float16)p;
                        p -= (float)pf[k][r / 8][r % 8];
                    }
                }
            };
            auto load_v = [&](int s2) __attribute__((always_inline)) {
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const uint32_t at = slot * VST + (32 * kt + 16 * s2) * VROW + 64 * d;
                    const tr4 x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4 *)(vp + at));
                    const tr4 y = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4 *)(vp + at + 8 * VROW));
                    vf[s2][d] = half8{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3],
                                      (_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
                }
            };
            // three runs of products, each group of them (64 cycles) with vector
            // work that does not need it; the order is pinned by the barriers
            if (kt == 1) next();  // (their loads have had half a stage more)
            if (!LATE) load_v(0);
#pragma unroll
            for (int k = 0; k < KS; k++) {
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k], qf[p][k], sn, 0, 0, 0);
                if (LATE && k % 2 && k < KS / 2) load_k(kt == 0 ? slot : (slot + 1) % TS, 1 - kt, KS / 2 + k - 1, KS / 2 + k + 1);
#pragma unroll
                for (int i = EARLY * k / KS; i < EARLY * (k + 1) / KS; i++) weights(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            load_v(LATE ? 0 : 1);
            load_h(hn, kt == 0 ? slot : (slot + 1) % TS, 1 - kt);
#pragma unroll
            for (int d = 0; d < DT; d++) {
#pragma unroll
                for (int p = PW - 1; p >= 0; p--)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[0][d], pf[p][0], o[d], 0, 0, 0);
#pragma unroll
                for (int i = EARLY + (PAIRS - EARLY) * d / DT; i < EARLY + (PAIRS - EARLY) * (d + 1) / DT; i++) weights(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (LATE) load_v(1);
            load_k((slot + 1) % TS, kt, 0, AHEAD);
#pragma unroll
            for (int d = 0; d < DT; d++) {
#pragma unroll
                for (int p = PW - 1; p >= 0; p--)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[1][d], pf[p][1], o[d], 0, 0, 0);
                if (d == 0) mx = largest(sn, hn);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (kt == 0 || st + 1 < wst) {  // (after the wave's last tokens the products are of nothing)
                const uint32_t tn = tk + 32 * (kt + 1);
                if (tn + 32 > every || !hn.ok) {
                    mask(tn, sn, kt == 0 ? slot : (slot + 1) % TS, 1 - kt);
                    mx = largest(sn, hn);
                }
                refer(mx);
            }
            sc = sn;
            hc = hn;
        }
    }
    if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
    l = xor32_sum(l);
    if (w0 + i32 >= rows) return;
    if (end <= job.c * TK) {  // (one part)
        const bool none = seq.lim(qi) == 0;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
                if (!none) v = f32x4{o[d][4 * g] / l, o[d][4 * g + 1] / l, o[d][4 * g + 2] / l, o[d][4 * g + 3] / l};
                st_out<T>(a, seq.row + qi, kvh * a.G + row % a.G, 32 * d + 8 * g + 4 * h, HD, v);
            }
        return;
    }
    const size_t pr = (size_t)blockIdx.x * ROWS + (row - r0);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *(f32x4 *)(a.tpart + pr * HD + 32 * d + 8 * g + 4 * h) =
                f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (h == 0) {
        a.tstat[2 * pr] = m - 4.f;
        a.tstat[2 * pr + 1] = l;
    }
}

// (Launches of their own, 4.3 us for 16 sequences of 4096 tokens, a chain of four loads; 12 us
// for 777 rows of 28 heads on LDS tiles, 30 MB of parts: vector instructions in 91% of the
// cycles, most of them to find a tile's parts from the whole batch in every wave.)
// Joins the parts of a row: HD / 4 lanes, of 4 dims each, take the parts'
// statistics, as many at a time, then all of them the parts' sums, 8 loads of 16
// bytes in flight. Part p is row at(p) of part and stat.
template <int HD, typename A>
ZH_DEV f32x4 join_row(const float *part, const float *stat, uint32_t parts, A at) {
    constexpr uint32_t N = HD / 4, U = 8;
    const uint32_t lane = threadIdx.x & 63, l = lane % N;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t b = 0; b < parts; b += N) {
        const uint32_t n = min(N, parts - b);
        const float2 st = *(const float2 *)(stat + 2 * at(b + min(l, n - 1)));
        f32x4 v[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) v[u] = *(const f32x4 *)(part + at(b + min(u, n - 1)) * HD + 4 * l);
        float mx = st.x;
#pragma unroll
        for (uint32_t x = 1; x < N; x *= 2) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
        const float mn = fmaxf(M, mx), ms = mn == -INFINITY ? 0.f : mn;
        const Shift old(M - ms), own(st.x - ms);
        const float w = l < n ? own.both() : 0.f;
        float ls = l < n ? st.y * own.a * own.b : 0.f;
#pragma unroll
        for (uint32_t x = 1; x < N; x *= 2) ls += __shfl_xor(ls, x, 64);
        M = mn;
        L = fmaf(L * old.a, old.b, ls);
        O *= old.both();
        for (uint32_t p = 0; p < n; p += U) {
            if (p)
#pragma unroll
                for (uint32_t u = 0; u < U; u++) v[u] = *(const f32x4 *)(part + at(b + min(p + u, n - 1)) * HD + 4 * l);
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {  // (past the last part: its values again, weight 0)
                const float f = __shfl(w, lane - l + min(p + u, N - 1), 64);
                O.x = fmaf(v[u].x, p + u < n ? f : 0.f, O.x);
                O.y = fmaf(v[u].y, p + u < n ? f : 0.f, O.y);
                O.z = fmaf(v[u].z, p + u < n ? f : 0.f, O.z);
                O.w = fmaf(v[u].w, p + u < n ? f : 0.f, O.w);
            }
        }
    }
    return f32x4{O.x / L, O.y / L, O.z / L, O.w / L};
}

template <int HD, int RT, typename T>
__global__ __launch_bounds__(256) void k_kv8_join(Kv8Attn a) {
    constexpr uint32_t N = HD / 4, PER = 256 / N, ROWS = 16 * RT;  // rows of a workgroup, of a tile
    const uint32_t item = blockIdx.x / (ROWS / PER), r = blockIdx.x % (ROWS / PER) * PER + threadIdx.x / N;
    const uint32_t kvh = item % a.nkv, tile = item / a.nkv % a.tiles, s = item / a.nkv / a.tiles;
    bool bad = false;
    const uint32_t lane = threadIdx.x & 63;
    const AttnSeq seq = attn_seq(a, s, bad);
    const uint32_t all_rows = seq.n * a.G, row0 = tile * ROWS;
    if (row0 >= all_rows || all_rows > a.few) return;
    const uint32_t nrow = min(ROWS, all_rows - row0);
    if (r / (64 / N) * (64 / N) >= nrow) return;  // (uniform per wave)
    const UnitSeq u0 = first_units(a, bad);
    const Share x = share(a, u0, bad);
    uint32_t before = 0;
    for (uint32_t i = lane; i < s; i += 64) before += x.items(i < 64 ? u0 : unit_seq(a, i, bad));
    const uint32_t units = unit_seq(a, s, bad).units;
    uint32_t first, parts;
    if (x.parts) {  // (parts of one length: the last ones may be empty)
        const uint32_t p = (units + x.q - 1) / x.q, c = (units + p - 1) / p;
        first = wave_total(before) + tile * p;
        parts = (units + c - 1) / c;
    } else {
        const uint32_t u = wave_total(before) + tile * units;
        first = u / x.q;
        parts = (u + units - 1) / x.q - first + 1;
    }
    if (parts <= 1) return;
    const uint32_t R = min(r, nrow - 1), qi = (row0 + R) / a.G, h = kvh * a.G + (row0 + R) % a.G;
    // (the first part begins with the sequence, the others in it)
    auto at = [&](uint32_t p) { return ((size_t)((first + p) * a.nkv + kvh) * 2 + (p ? 0u : 1u)) * ROWS + R; };
    const f32x4 v = join_row<HD>(a.part, a.stat, parts, at);
    if (r < nrow) st_out<T>(a, seq.row + qi, h, threadIdx.x % N * 4, HD, seq.lim(qi) ? v : f32x4{0.f, 0.f, 0.f, 0.f});
}

template <int HD, typename T>
__global__ __launch_bounds__(256) void k_kv8_tile_join(Kv8Attn a) {
    constexpr uint32_t N = HD / 4, PER = 256 / N, ROWS = TILE;
    const uint32_t item = blockIdx.x / (ROWS / PER), r = blockIdx.x % (ROWS / PER) * PER + threadIdx.x / N;
    const uint32_t kvh = item % a.nkv, lane = threadIdx.x & 63;
    const TileSeq t0 = first_seqs(a, ROWS);
    const uint32_t q = tile_share(a, ROWS, t0);
    auto get = [&](uint32_t i) { return i < 64 ? t0 : tile_seq(a, ROWS, i); };
    uint32_t s, at_s, before = 0;
    if (!kv8_find(a.n_seq, item / a.nkv, [&](uint32_t i) { return get(i).tiles; }, s, at_s)) return;
    // the workgroups of the sequences before
    for (uint32_t i = lane; i < s; i += 64) before += get(i).tiles * ((get(i).stages + q - 1) / q);
    before = wave_total(before);
    bool bad = false;
    const AttnSeq seq = attn_seq(a, s, bad);
    const TileSeq t = tile_seq(a, ROWS, s);
    const uint32_t p = (t.stages + q - 1) / q, c = (t.stages + p - 1) / p * TK;
    const uint32_t r0 = (t.tiles - 1 - at_s) * ROWS, nrow = min(ROWS, seq.n * a.G - r0);
    const uint32_t parts = (seq.lim((r0 + nrow - 1) / a.G) + c - 1) / c;
    if (parts <= 1 || r / (64 / N) * (64 / N) >= nrow) return;  // (uniform per wave)
    const uint32_t R = r0 + min(r, nrow - 1), qi = R / a.G, h = kvh * a.G + R % a.G, first = before + at_s * p;
    auto at = [&](uint32_t i) { return ((size_t)(first + i) * a.nkv + kvh) * ROWS + (R - r0); };
    const f32x4 v = join_row<HD>(a.tpart, a.tstat, parts, at);
    if (r < nrow) st_out<T>(a, seq.row + qi, h, threadIdx.x % N * 4, HD, seq.lim(qi) ? v : f32x4{0.f, 0.f, 0.f, 0.f});
}

// How a call is cut (the same for every call of these sizes).
struct Kv8Plan {
    uint32_t rt, few, tiles, groups, least;    // streamed
    uint32_t items, tslots;                    // LDS tiles (items 0: none)
    uint64_t stat_off, tpart_off, tstat_off, bytes;  // of ws
};
constexpr uint32_t LEAST = 4;    // units of a share at least
// Rows of a sequence and kv head that are streamed, in tiles of 32 that each read K and V
// (through the L2s) again, where LDS tiles of 256 rows would be emptier than that costs.
// us streamed / on LDS tiles, head_dim 128, sequences of 2000 tokens: f16 36 rows of 16 30 /
// 52, 128 of 1 16 / 20, of 4 26 / 29, of 16 42 / 58, of 40 99 / 168, 192 of 1 20 / 24, of 4
// 34 / 32, of 16 59 / 69, of 40 140 / 178, 256 of 4 26 / 34, of 16 82 / 77; f32 128 of 16 54 /
// 66, of 40 116 / 188, 192 of 4 40 / 35, of 16 70 / 81, of 40 160 / 207; 100 of 500 f16 192
// rows 119 / 119, 256 154 / 131; one of 30000 f16 128 rows 46 / 46, 192 65 / 57, 256 72 / 64, f32
// 128 50 / 51, 256 81 / 74.
constexpr uint32_t FEW = 192;
// Sequences from which on the few rows of some are streamed in a launch of their own
// before the tiles of others; below, they take emptier tiles. us with / without, 512 rows
// after 2000 tokens and n decode rows at 1000, 2000, 4000 and 8000 tokens, f16: n = 0 60 / 58;
// 4 64, 64, 67, 85 / 64, 61, 74, 88; 8 67, 78, 72, 94 / 61, 76, 80, 117; 12 73, 89, 81, 110 / 77,
// 84, 126, 145; 15 75, 89, 118, 126 / 77, 84, 139, 190; f32 8 76, 88, 82, 106 / 67, 83, 89, 131; 15
// 85, 100, 133, 141 / 86, 93, 153, 203
constexpr uint32_t MIXED = 9;
constexpr uint32_t TILE_FIX = 5; // a tile launch's start and end, in stages

// Streaming workgroups of a CU, as many as its registers hold (head_dim 64, 32 rows, two
// for three: 48 sequences of 3000 tokens f16 42.5 us for 39.1, f32 46.6 for 41.2; 16 rows,
// four for three: no faster).
constexpr uint64_t kv8_slots(uint32_t rt, uint64_t hd) { return rt == 1 || hd == 64 ? 3 : 2; }
// The max_len up to which a workgroup takes a whole sequence and row tile: it goes through
// its tokens one step after the other, where shares are even, but begin anew, and wait for
// memory, in every sequence that they reach into, and are joined; and dealing out takes every
// workgroup, of the join's too, a pass over all sequences. The host knows the longest length
// only, so the rule lies between what batches of like lengths and what one long sequence among
// short ones would have it be. us whole / in shares, 8 kv heads, f16, n of a length | n - 1 of
// 200 tokens and one of it: head_dim 128, 16 of 1000 12.2 / 14.3, 1250 | 13.8 / 12.1; 64 of
// 2000 46 / 53 | 21 / 16; 200 of 4000 276 / 281 | 51 / 43; 600 of 6000 1149 / 1200, 10375 | 134 /
// 127; 800 of 13500 | 171 / 170, 27000 | 264 / 178; 1600 of 26000 | 344 / 452, 52000 | 540 / 453;
// head_dim 64, 64 of 1900 28 / 32, 1525 | 14 / 13, 3050 | 22 / 14; 200 of 3800 159 / 146, 3437 | 32
// / 28; 600 of 9000 855 / 910, 9062 | 82 / 72, 18125 | 130 / 72; 20 rows, head_dim 128, 16 of 1000
// 17.4 / 20.1 | 16.5 / 14.7, 2000 29 / 25 | 26 / 15; 64 of 2400 61 / 67 | 34 / 29, 3400 90 / 94 | 45
// / 30; 6400 of 300 and one of 30000, 1 kv head 313 / 790.
constexpr uint64_t kv8_one(uint32_t rt, uint64_t hd, uint64_t n_seq, uint64_t jobs, uint64_t cus) {
    const uint64_t even = rt == 2 ? 800 + 800 * jobs / cus : 1000 + (hd == 64 ? 450 : 500) * jobs / cus;
    return std::max(even, n_seq * jobs * rt * hd / 64000);
}
uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

bool kv8_plan(uint32_t cus, const zh_kv8_batch *kv, uint32_t nh, uint32_t n_rows, uint32_t max_rows, uint32_t max_len,
              Kv8Plan &p) {
    const uint64_t G = nh / kv->n_kv_heads, rows = max_rows * G, nkv = kv->n_kv_heads, hd = kv->head_dim;
    p = {};
    if (n_rows * G >= 1ull << 31) return false;
    p.rt = rows <= 16 ? 1 : 2;
    p.few = rows <= FEW ? (uint32_t)rows : kv->n_seq < MIXED ? 0 : FEW;
    p.tiles = ceil_div(p.few, 16 * p.rt);
    const uint64_t jobs = kv->n_seq * nkv * p.tiles, slots = kv8_slots(p.rt, hd) * cus;
    // one workgroup a sequence and row tile
    // (so many that the join would not fit a launch: always)
    const bool whole = jobs >= 1u << 20 || max_len <= kv8_one(p.rt, hd, kv->n_seq, jobs, cus);
    p.least = whole ? 0 : LEAST;
    const uint64_t units = kv->n_seq * (uint64_t)ceil_div(max_len, CUT) * p.tiles;
    p.groups = whole ? kv->n_seq * p.tiles
                     : (uint32_t)std::min<uint64_t>(std::max<uint64_t>(slots / nkv, 1), (units + LEAST - 1) / LEAST);
    if (units >= 1ull << 31 || p.groups * nkv >= 1ull << 23) return false;  // (a launch has fewer than 2^32 threads)
    const uint64_t parts = whole || !p.few ? 0 : 2ull * p.groups * nkv * 16 * p.rt;
    uint64_t tparts = 0;
    if (rows > p.few) {
        const uint64_t tr = TILE;
        // a sequence of n rows takes at most (n + tr - 1) / tr tiles, and n / (few + 1) sequences take any
        // (and all rows at least so many, which the parts are chosen for)
        const uint64_t seqs = std::min<uint64_t>(kv->n_seq, n_rows * G / (p.few + 1));
        const uint64_t items = (n_rows * G + seqs * (tr - 1)) / tr, tj = (n_rows * G + tr - 1) / tr * nkv;
        // the parts that fill 1 to 4 rounds of one workgroup per CU, by the rounds' stages
        const uint32_t top = ceil_div(max_len, 256);
        uint64_t best = ~0ull, slots = 0;
        for (uint64_t r = 1; r <= 4; r++) {
            const uint32_t fit = (uint32_t)(r * cus / tj), k = fit < 1 ? 1u : fit < top ? fit : top;
            const uint64_t cost = ceil_div(tj * k, cus) * (uint64_t)(ceil_div(ceil_div(max_len, k), TK) + TILE_FIX);
            if (cost < best) {
                best = cost;
                slots = k == 1 ? 0 : std::max<uint64_t>(items, ceil_div(tj * k, cus) * (uint64_t)cus / nkv);
            }
        }
        // (uncut, where the kernels' 32-bit sums of all sequences' stages could pass their
        // range, whatever row_start says)
        if (kv->n_seq * ((rows + tr - 1) / tr) * ceil_div(max_len, TK) >= 1ull << 30) slots = 0;
        p.items = (uint32_t)items;
        p.tslots = (uint32_t)slots;
        if (std::max(items, slots) * nkv >= 1ull << 22 || items * nkv * tr >= 1ull << 27) return false;
        tparts = slots * nkv * tr;
    }
    p.stat_off = parts * hd * 4;
    p.tpart_off = p.stat_off + parts * 8;
    p.tstat_off = p.tpart_off + tparts * hd * 4;
    p.bytes = p.tstat_off + tparts * 8;
    return true;
}

bool kv8_shape_ok(const zh_kv8_batch *kv, uint32_t nh, uint32_t n_rows, uint32_t max_rows, uint32_t max_len) {
    return kv8_batch_ok(kv, n_rows) && nh && nh % kv->n_kv_heads == 0 && n_rows && n_rows < 1u << 30 && max_rows &&
           max_rows <= n_rows && max_len && max_len <= 1u << 30;
}

}  // namespace

static zh_attn_rows with_strides(const zh_kv8_batch *kv, const zh_attn_rows *r) {
    zh_attn_rows x = *r;
    if (!x.q_stride) x.q_stride = x.n_heads * kv->head_dim;
    if (!x.out_stride) x.out_stride = x.n_heads * kv->head_dim;
    return x;
}

// The checks of zh_flash_attn_kv8, of host data only (exported for the tests; c may
// be null: no message then). cus: the device's CUs.
extern "C" int zh_check_attn_kv8(zh_ctx *c, const zh_kv8_batch *kv, const zh_attn_rows *rows, uint32_t cus) {
    const char *const who = "flash_attn_kv8";
    if (!rows || !kv8_shape_ok(kv, rows->n_heads, rows->n_rows, rows->max_rows, rows->max_len))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: caches, heads, rows or lengths", who);
    if (!kv8_type_ok(kv->type)) return zh_set_err(c, ZH_ERR_UNSUPPORTED_QUANT_TYPE, "%s: cache type %u", who, kv->type);
    const zh_attn_rows x = with_strides(kv, rows), *r = &x;
    if ((uint64_t)r->max_len > 16ull * kv->table_stride)
        return zh_set_err(c, ZH_ERR_CONTEXT_LENGTH_EXCEEDED, "%s: max_len %u in tables of %u pages", who, r->max_len,
                          kv->table_stride);
    if (r->type != ZH_F32 && r->type != ZH_F16)
        return zh_set_err(c, ZH_ERR_UNSUPPORTED_QUANT_TYPE, "%s: type %u", who, r->type);
    if (!isfinite(r->attn_scale)) return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: attn_scale", who);
    const uint64_t size = r->type == ZH_F32 ? 4 : 2, w = (uint64_t)r->n_heads * kv->head_dim, n = r->n_rows;
    if (w > 0xFFFFFFFFull || (n > 1 && (r->q_stride < w || r->out_stride < w)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: rows overlap", who);
    const uint64_t qb = ((n - 1) * r->q_stride + w) * size, ob = ((n - 1) * r->out_stride + w) * size;
    Kv8Plan p;
    if (!kv8_plan(cus, kv, r->n_heads, r->n_rows, r->max_rows, r->max_len, p))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: too large", who);
    if (!kv_in_range(r->q, r->q_off, qb) || !kv_in_range(r->out, r->out_off, ob) ||
        (p.bytes && !kv_in_range(r->ws, 0, p.bytes)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: range (ws: %llu bytes)", who, (unsigned long long)p.bytes);
    // out and ws: not what the call reads besides q
    const zh_buf *const read[] = {kv->k_cache, kv->v_cache, kv->k_scale, kv->v_scale, kv->tables, kv->row_start, kv->seq_lens};
    for (const zh_buf *b : read)
        if (b && (b->ptr == r->out->ptr || (p.bytes && b->ptr == r->ws->ptr)))
            return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: out or ws is an input", who);
    if (p.bytes && (r->ws->ptr == r->out->ptr || r->ws->ptr == r->q->ptr))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: ws holds q or out", who);
    if (r->q_off % 16 || r->out_off % 16 || (n > 1 && (r->q_stride * size % 16 || r->out_stride * size % 16)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: rows not 16-byte aligned", who);
    const bool same = r->q->ptr == r->out->ptr && r->q_off == r->out_off && (n == 1 || r->q_stride == r->out_stride);
    if (!same && kv_rows_overlap(r->q, r->q_off, qb, r->out, r->out_off, ob) &&
        !(r->q_stride == r->out_stride &&
          kv_columns_apart(r->out, r->out_off, r->q, r->q_off, r->q_stride, w, w, (uint32_t)size)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: out overlaps q", who);
    return ZH_OK;
}

// zh_flash_attn_kv8_ws of a device of `cus` CUs (exported for the tests): what kv8_plan
// asks for at most, over smaller calls too, so every term grows with the sizes.
extern "C" uint64_t zh_check_attn_kv8_ws(const zh_kv8_batch *kv, uint32_t n_heads, uint32_t n_rows, uint32_t max_rows,
                                         uint32_t max_len, uint32_t cus) {
    Kv8Plan p;
    if (!kv8_shape_ok(kv, n_heads, n_rows, max_rows, max_len) ||
        !kv8_plan(cus, kv, n_heads, n_rows, max_rows, max_len, p))
        return 0;
    const uint64_t nkv = kv->n_kv_heads, G = n_heads / nkv, rows = max_rows * G;
    // streamed: two parts of a tile's rows in each workgroup
    auto streamed = [&](uint64_t few, uint64_t tile, uint64_t slots) {
        const uint64_t units = kv->n_seq * (uint64_t)ceil_div(max_len, CUT) * ceil_div(few, tile);
        return 2 * std::min<uint64_t>(std::max<uint64_t>(slots / nkv, 1), (units + LEAST - 1) / LEAST) * nkv * tile;
    };
    uint64_t parts = streamed(std::min<uint64_t>(rows, 16), 16, kv8_slots(1, kv->head_dim) * cus);
    if (rows > 16) parts = std::max(parts, streamed(std::min<uint64_t>(rows, FEW), 32, kv8_slots(2, kv->head_dim) * cus));
    // LDS tiles: cut ones are at most two a CU before that
    if (rows > FEW && max_len > 256) {
        const uint64_t all = std::min<uint64_t>(n_rows * G, 2ull * cus / nkv * TILE), tj = ceil_div(all, TILE) * nkv;
        const uint64_t seqs = std::max(std::min<uint64_t>(kv->n_seq, MIXED - 1), std::min<uint64_t>(kv->n_seq, all / FEW));
        const uint64_t rounds = std::min<uint64_t>(4, ceil_div(tj * ceil_div(max_len, 256), cus));
        parts += std::max<uint64_t>((all + seqs * (TILE - 1)) / TILE, rounds * cus / nkv) * nkv * TILE;
    }
    return parts * (kv->head_dim * 4 + 8);
}

extern "C" uint64_t zh_flash_attn_kv8_ws(zh_ctx *c, const zh_kv8_batch *kv, uint32_t n_heads, uint32_t n_rows,
                                         uint32_t max_rows, uint32_t max_len) {
    return c ? zh_check_attn_kv8_ws(kv, n_heads, n_rows, max_rows, max_len, (uint32_t)c->cu_count) : 0;
}

template <int HD, int NP, int RT, uint32_t F, typename T>
static int attn_launch(zh_ctx *c, const Kv8Attn &a, const Kv8Plan &p) {
    hipLaunchKernelGGL((k_kv8_attn<HD, NP, RT, F, T>), dim3(p.groups * a.nkv), dim3(64 * W), 0, c->stream, a);
    ZH_LAUNCH_CHECK(c);
    if (p.least) {
        const uint32_t per = 256 / (HD / 4);
        hipLaunchKernelGGL((k_kv8_join<HD, RT, T>), dim3(a.n_seq * a.nkv * a.tiles * (16 * RT / per)), dim3(256), 0, c->stream, a);
        ZH_LAUNCH_CHECK(c);
    }
    return ZH_OK;
}

template <int HD, int NP, uint32_t F, typename T>
static int tile_launch(zh_ctx *c, const Kv8Attn &a, const Kv8Plan &p) {
    static std::atomic<bool> attr[64];  // by device
    if (c->device >= 64 || !attr[c->device].load(std::memory_order_relaxed)) {
        ZH_HIP(c, hipFuncSetAttribute((const void *)k_kv8_tile<HD, NP, F, T>,
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)t_lds<HD>()));
        if (c->device < 64) attr[c->device].store(true, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL((k_kv8_tile<HD, NP, F, T>), dim3((p.tslots ? p.tslots : p.items) * a.nkv), dim3(64 * TW), t_lds<HD>(), c->stream, a);
    ZH_LAUNCH_CHECK(c);
    if (p.tslots) {
        const uint32_t per = 256 / (HD / 4);
        hipLaunchKernelGGL((k_kv8_tile_join<HD, T>), dim3(p.items * a.nkv * (TILE / per)), dim3(256), 0, c->stream, a);
        ZH_LAUNCH_CHECK(c);
    }
    return ZH_OK;
}

template <int HD, int NP, uint32_t F, typename T>
static int attn_rt(zh_ctx *c, const Kv8Attn &a, const Kv8Plan &p) {
    const int rc = !p.few ? ZH_OK : p.rt == 1 ? attn_launch<HD, NP, 1, F, T>(c, a, p) : attn_launch<HD, NP, 2, F, T>(c, a, p);
    return rc || !p.items ? rc : tile_launch<HD, NP, F, T>(c, a, p);
}
template <int HD, uint32_t F>
static int attn_type(zh_ctx *c, const Kv8Attn &a, const Kv8Plan &p, uint32_t type) {
    return type == ZH_F32 ? attn_rt<HD, 2, F, float>(c, a, p) : attn_rt<HD, 1, F, _Float16>(c, a, p);
}

extern "C" int zh_flash_attn_kv8(zh_ctx *c, const zh_kv8_batch *kv, const zh_attn_rows *rows) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    const int rc = zh_check_attn_kv8(c, kv, rows, (uint32_t)c->cu_count);
    if (rc) return rc;
    const zh_attn_rows x = with_strides(kv, rows), *r = &x;
    zh_device_scope dev(c);
    Kv8Plan p;
    kv8_plan((uint32_t)c->cu_count, kv, r->n_heads, r->n_rows, r->max_rows, r->max_len, p);
    Kv8Attn a = {};
    const uint64_t size = r->type == ZH_F32 ? 4 : 2;
    a.q = (const uint8_t *)r->q->ptr + r->q_off;
    a.out = (uint8_t *)r->out->ptr + r->out_off;
    a.q_row = r->q_stride * size;
    a.out_row = r->out_stride * size;
    a.kc = (const uint8_t *)kv->k_cache->ptr;
    a.vc = (const uint8_t *)kv->v_cache->ptr;
    a.ks = (const float *)kv->k_scale->ptr;
    a.vs = (const float *)kv->v_scale->ptr;
    a.tables = (const uint32_t *)kv->tables->ptr;
    a.row_start = kv->row_start ? (const uint32_t *)kv->row_start->ptr : nullptr;
    a.seq_lens = (const uint32_t *)kv->seq_lens->ptr;
    a.part = p.bytes ? (float *)r->ws->ptr : nullptr;
    a.stat = p.bytes ? (float *)((char *)r->ws->ptr + p.stat_off) : nullptr;
    a.err = c->err_dev;
    a.n_seq = kv->n_seq;
    a.stride = kv->table_stride;
    a.cache_tokens = kv->cache_tokens;
    a.nh = r->n_heads;
    a.nkv = kv->n_kv_heads;
    a.G = a.nh / a.nkv;
    a.n_rows = r->n_rows;
    a.max_rows = r->max_rows;
    a.max_len = r->max_len;
    a.tpart = p.bytes ? (float *)((char *)r->ws->ptr + p.tpart_off) : nullptr;
    a.tstat = p.bytes ? (float *)((char *)r->ws->ptr + p.tstat_off) : nullptr;
    a.few = p.few;
    a.tslots = p.tslots;
    a.rt = 16 * p.rt;
    a.tiles = p.tiles;
    a.groups = p.groups;
    a.least = p.least;
    // (64 bits: a scale of any size times log2 e)
    const double scale = (double)(r->attn_scale != 0.f ? r->attn_scale : 1.0f / sqrtf((float)kv->head_dim)) *
                         1.44269504088896340736f;
    int scale_exp = 0;
    a.scale = (float)frexp(scale, &scale_exp);
    a.scale_exp = scale_exp;
    if (kv->head_dim == 128)
        return kv->type == ZH_I8 ? attn_type<128, ZH_I8>(c, a, p, r->type) : attn_type<128, ZH_E4M3>(c, a, p, r->type);
    return kv->type == ZH_I8 ? attn_type<64, ZH_I8>(c, a, p, r->type) : attn_type<64, ZH_E4M3>(c, a, p, r->type);
}
