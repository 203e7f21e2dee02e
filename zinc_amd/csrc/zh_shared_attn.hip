// zh_shared_attn.hip — paged decode attention of a batch of sequences whose
// first prefix_len tokens are shared (zh_flash_decode_shared).
//
// For sequence s and query head h of kv head k:
//   out = sum_t p_t V[t] / sum_t p_t,  p_t = exp(scale q . K[t] - m)
// over t < len[s]. The tokens below prefix_len have the same K and V for every
// sequence, so their products run once per kv head over the rows of all
// sequences (n_seq * G rows, G = heads per kv head); the tokens past it run per
// sequence. Both are cut along the tokens into parts, each of which leaves its
// unnormalised sum, running maximum and sum of weights; a second kernel joins a
// row's parts (log-sum-exp weights). One part: the first kernel writes the
// result itself.
#include <math.h>

#include <atomic>
#include <type_traits>

#include "zh_device.h"
#include "zh_internal.h"
#include "zh_kv.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(4))) uint32_t const_u32;  // what no kernel writes while it runs

constexpr uint32_t SA_ROWS = 16;  // rows of an MFMA tile
constexpr uint32_t SA_KB = 32;    // tokens of a wave's step
constexpr int W = 4;              // waves of a workgroup
// The host's choices (shared_plan), measured with 32 heads on 8, 64 own tokens a
// sequence, f16, prefix 1024 / 4096 / 16384:
//  * LDS tiles where the 16-row tiles' prefix tokens over the kv heads reach
//    sa_tile: below it one more reading of K and V through the L2s costs less
//    than the tiles' longer launch. us tiled / streamed, f16 at head_dim 128: 96
//    rows over 6144 tokens (294K) 21.0 / 19.9, 8192 (393K) 22.5 / 23.7, 128 over
//    8192 (524K) 24.5 / 27.3; f32 128 over 8192 30.2 / 27.6, 12288 (786K) 34.6 /
//    36.2; f16 at 64 128 over 4096 (262K) 13.2 / 12.4, 96 over 8192 14.2 / 15.4;
//    f32 at 64 128 over 6144 (393K) 16.3 / 15.2, 96 over 12288 (589K) 19.7 / 20.1;
//    none for 32 rows and fewer, which keep one wave of a workgroup busy: 32 rows,
//    f16 at 128, over 32768 tokens of 8 heads 32.0 / 29.0, 65536 of 8 51.7 / 47.6,
//    16384 of 32 47.5 / 50.1, 131072 of 4 52.7 / 82.5; f32 65536 of 8 80.9 / 50.4;
//    f16 at 64 over 65536 of 8 34.9 / 30.1;
//  * a prefix's parts: those that fill 1 to 4 rounds of one workgroup per CU best,
//    a round's start and end counted as SA_TILE_FIX stages, streamed SA_FIX steps
//    (180 sequences at 8192 in tiles 58.5 us, in the nearest number of parts 73.9;
//    streamed 48 rows at 12288 20.5, in the nearest number 27.5, 384 at 8192 68.3,
//    with one round 81.9; 16 sequences at 4096 f32 14.2, with two rounds 17.6);
//  * a whole context, prefix and own tokens, in one workgroup where there is at
//    most one per CU, the more of them the longer (sa_one tokens for few, twice
//    that for one per CU), a prefix past sa_one excepted. us whole / in parts, f16
//    at 128: 2 sequences at 512 tokens 7.6 / 8.5; 16 at 700 13.4 / 13.9, at 1000
//    18.4 / 15.3; 32 at 1000 22.4 / 26.1, of 1 to 1400 24.6 / 23.0, with a prefix
//    of 500 18.4 / 18.8, of 900 12.9 / 11.2; at 64: 8 at 760 7.2 / 7.8, 16 at
//    1500 14.4 / 13.0, 32 at 1400 16.1 / 19.4;
//  * workgroups per CU that the own tokens' parts are cut for: 8 (100 sequences
//    of 1 to 4000 167 us, 4: 197, 12: 164; 128 of up to 4000 after a tile launch
//    221, 251, 215; 64 of 4000 173, 163, 177; of 1000 49.8, 48.0, 49.8);
//  * a prefix's parts of at least 128 tokens, a step for each wave; of own tokens at
//    most one for each 256 begun, all of a length (300 tokens: two of 160; 16
//    sequences at 4096 of up to 300 own 15.9 us, one for each 128: 17.0), and for
//    each 512 after a tile launch, where a single own part of a sequence also joins
//    the prefix's (32 sequences of up to 512: 38 us, in two parts and a launch that
//    joins them 40.7; up to 1000 48.8, 45.9; 64 of up to 4000 139 us, in one part 171).
constexpr uint64_t sa_tile(uint32_t hd, bool f32) {
    return hd == 64 ? (f32 ? 560000 : 290000) : (f32 ? 750000 : 350000);
}
constexpr uint32_t sa_one(uint32_t hd) { return hd == 64 ? 768 : 512; }
constexpr uint32_t SA_OWN_PER = 8, SA_FIX = 3, SA_TILE_FIX = 5;

struct SharedArgs {
    const uint8_t *q;
    uint8_t *out;
    uint64_t q_row, out_row;  // bytes between rows
    const uint16_t *kc, *vc;
    const uint32_t *tables, *lens;
    float *part;   // [parts][n_seq * nh][hd]
    float *stat;   // [parts][n_seq * nh][2]: maximum (base 2), sum of weights
    uint32_t *err;
    uint32_t n_seq, stride, cache_tokens, nh, nkv, G, prefix, max_len;
    uint32_t n_pre, n_own;           // parts of the prefix and of a sequence's own tokens
    uint32_t pre_tiles, pre_blocks;  // row tiles per kv head, workgroups of the prefix
    uint32_t pre_len;                // tokens of a prefix part (a multiple of SA_KB)
    uint32_t own_len;                // tokens of a sequence's own part, at least
    uint32_t join;                   // the own parts' workgroups write the result (n_own == 1, the prefix's parts are there)
    float scale;        // |attn_scale| log2 e = scale * 2^scale_exp, with attn_scale's sign
    int32_t scale_exp;
};

// What takes the products of a row's q, scaled by 2^-e, to base-2 scores: the
// scale's magnitude times 2^e, kept in [2^-120, 2^80]. Products lie below 2^39 in
// steps of 2^-48 at least, so below that range every weight is 1 and above it all
// but a row's largest are 0, as without the bounds; within it no score is
// infinite, and none that is masked (-inf) meets a factor of 0.
ZH_DEV float score_factor(const SharedArgs &a, int e) {
    const float f = fabsf(ldexpf(a.scale, a.scale_exp + e));
    return f < 0x1p-120f ? 0x1p-120f : f > 0x1p80f ? 0x1p80f : f;  // (NaN stays)
}

// The sequence's length as the kernels take it: cut at max_len (the host has
// checked that the table holds that many tokens).
ZH_DEV uint32_t seq_len(const SharedArgs &a, uint32_t s) {
    return min(a.lens[s], a.max_len);
}

// 8 elements of a row (16-byte aligned) as floats.
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

template <bool ONCE, typename V>
ZH_DEV V ld_kv(const V *p) {
    return ONCE ? __builtin_nontemporal_load(p) : *p;
}

// What a workgroup of k_shared_attn does: rows row0 .. of one kv head (numbered
// s * G + g), tokens [t0, t1) through table row `tab`, after the tokens [0, first)
// through table row 0 (a sequence's whole context in one workgroup).
struct SharedPart {
    uint32_t part, row0, nrow, t0, t1, tab, first;
    bool pre, shares;  // a part of the prefix; of a sequence that has the prefix's parts too
};

// 16 rows of one kv head. Each wave takes steps of 32 tokens by itself, K and V
// straight from the cache into the matrix operands' registers (no LDS, no barrier
// before the end), the next step's K requested when the scores are done and its V
// after the products with this one's:
//   S^T = K q^T (tokens x rows): lane (li = lane % 16, lg = lane / 16) holds
//   tokens 16 j + 4 lg + r of row li, so that a row's maximum is in-lane plus
//   two lane exchanges, and its weights lie as the second product's operand
//   wants them: O^T += V^T P^T, k = (token 4 lg + r of tile 0, then of tile 1).
//   V's rows are read whole (lane li: dims HD/16 li ..), transposed by byte
//   permutes; column li of the output tile n is dim HD/16 li + n.
// NP pieces: q (scaled by a power of two to a maximum in [2^14, 2^15)) and P as
// sums of NP fp16 values; 2 keep 22 bits of each, of q's dims down to 2^-14 of the
// row's largest (below that they lie in fp16's subnormals: 2^-39 of the largest).
// The scale's and q's powers of two meet in score_factor, for queries and scales of
// any size.
// An f16 query is one piece; its weights take 2 too, which cost at most 2% here (48
// sequences of 1 to 4096 tokens 86.5 us against 85.9, 16 over 4096 15.1 / 14.8, 32 of
// 500 11.8 / 11.7) and leave the store's rounding as the only one to fp16.
// Bound by the reads: 3 workgroups of 4 waves a CU (168 registers), each wave's
// step 16 KB; 64 sequences of 4000 tokens (1.05 GB) 167 us, 6.3 TB/s, 48 of 1 to
// 4096 (400 MB) 79 us, 5 TB/s. Two or four row tiles a wave, or a workgroup on the
// same tokens, read less from the L2s but hold fewer steps in flight: 16
// sequences at 4096 20 and 29 us, 16.3 with one.
// ONCE: no other workgroup reads these K and V (loads that go by the L2s).
template <int HD, int NP, bool ONCE, typename T>
ZH_DEV void shared_part(const SharedArgs &a, const SharedPart &w, uint32_t kvh, float *lds) {
    constexpr int K4 = HD / 32, ND = HD / 16;  // k-steps of the scores, dims per lane and output tiles
    constexpr int LD = HD + 4, NQ = sizeof(T) == 2 ? 1 : NP;  // (an f16 query is one piece)
    float *const so = lds, *const sm = lds + W * SA_ROWS * LD, *const sl = sm + W * SA_ROWS;
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t li = lane % 16, lg = lane / 16;
    // steps start on a page; tokens outside their range are masked
    const uint32_t n0 = (w.first + SA_KB - 1) / SA_KB, ta = w.t0 & ~15u;
    const uint32_t nstep = n0 + (w.t1 > w.t0 ? (w.t1 - ta + SA_KB - 1) / SA_KB : 0u);
    const uint16_t *kh = a.kc + (size_t)kvh * a.cache_tokens * HD, *vh = a.vc + (size_t)kvh * a.cache_tokens * HD;
    bool bad = false;
    // a step's tokens [lo, hi) from tk on, and its two pages (the second clamped to the last of the range)
    struct Step {
        uint32_t tk, lo, hi, pg[2];
    };
    auto step = [&](uint32_t st) __attribute__((always_inline)) {
        Step x;
        const bool f = st < n0;
        x.tk = f ? st * SA_KB : ta + (st - n0) * SA_KB;
        x.lo = f ? 0u : w.t0;
        x.hi = f ? w.first : w.t1;
        // (scalar loads: a wait for them does not wait for K and V)
        const const_u32 *tb = (const const_u32 *)(a.tables + (f ? (size_t)0 : (size_t)w.tab * a.stride));
#pragma unroll
        for (int j = 0; j < 2; j++) {
            x.pg[j] = tb[min(x.tk / 16 + j, (x.hi - 1) / 16)];
            if (x.pg[j] >= a.cache_tokens / 16) {
                bad = true;
                x.pg[j] = 0;
            }
        }
        return x;
    };
    half8 kf[2][K4];
    uint32_t pv[2][4][ND / 2];
    auto load_k = [&](const Step &x) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint16_t *kp = kh + ((size_t)x.pg[j] * 16 + li) * HD + 8 * lg;
#pragma unroll
            for (int k4 = 0; k4 < K4; k4++) kf[j][k4] = ld_kv<ONCE>((const half8 *)(kp + 32 * k4));
        }
    };
    auto load_v = [&](const Step &x) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint16_t *vp = vh + ((size_t)x.pg[j] * 16 + 4 * lg) * HD + ND * li;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (ND == 8) *(u32x4 *)pv[j][r] = ld_kv<ONCE>((const u32x4 *)(vp + r * HD));
                else *(u32x2 *)pv[j][r] = ld_kv<ONCE>((const u32x2 *)(vp + r * HD));
            }
        }
    };
    Step x = {}, nx = {};  // this step and the next, whose pages are looked up one step ahead
    if (wave < nstep) {
        x = step(wave);
        load_k(x);
        load_v(x);
        if (wave + W < nstep) nx = step(wave + W);
    }
    // the row's q as operand fragments: dims 32 k4 + 8 lg ..
    half8 qf[NQ][K4];
    int e = 0;  // q is scaled by 2^-e
    {
        const uint32_t row = w.row0 + min(li, w.nrow - 1), rs = row / a.G, rh = kvh * a.G + row % a.G;
        const T *qp = (const T *)(a.q + rs * a.q_row) + (size_t)rh * HD + 8 * lg;
        float v[K4][8], mx = 0.f;
#pragma unroll
        for (int k4 = 0; k4 < K4; k4++) {
            ld8(qp + 32 * k4, v[k4]);
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(v[k4][e]));
        }
        if (NQ > 1) {
            mx = xor32_max(xor16_max(mx));
            const uint32_t E = __float_as_uint(mx) >> 23;
            if (E < 255) e = (int)E - 141;  // (E == 0, subnormal or zero rows: a smaller maximum)
        }
#pragma unroll
        for (int k4 = 0; k4 < K4; k4++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float y = NQ > 1 ? ldexpf(v[k4][i], -e) : v[k4][i];
#pragma unroll
                for (int p = 0; p < NQ; p++) {
                    qf[p][k4][i] = (_Float16)y;
                    y -= (float)qf[p][k4][i];
                }
            }
    }
    const float c = copysignf(score_factor(a, e), a.scale);
    floatx4 o[ND];
#pragma unroll
    for (int n = 0; n < ND; n++) o[n] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // the row's maximum (every lg alike), this lane's share of its sum
    // the weights and products of step x; `more`: the next step's loads on the way.
    // (The last step is code of its own: a load that may not be there would make
    // the compiler wait for V before the scores.)
    auto work = [&](auto more) __attribute__((always_inline)) {
        const bool whole = x.tk >= x.lo && x.tk + SA_KB <= x.hi;
        floatx4 d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int p = NQ - 1; p >= 0; p--)
#pragma unroll
            for (int k4 = 0; k4 < K4; k4++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    d[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[j][k4], qf[p][k4], d[j], 0, 0, 0);
        if constexpr (more) load_k(nx);
        float s[2][4], mb = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[j][r] = d[j][r] * c;
        if (!whole) {
            // a token outside the range: no score, and no V (0 times what the
            // cache holds there may be NaN)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t t = x.tk + 16 * j + 4 * lg + r;
                    const bool out = t < x.lo || t >= x.hi;
                    s[j][r] = out ? -INFINITY : s[j][r];
#pragma unroll
                    for (int y = 0; y < ND / 2; y++) pv[j][r][y] = out ? 0u : pv[j][r][y];
                }
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) mb = fmaxf(mb, s[j][r]);
        mb = xor32_max(xor16_max(mb));
        // (weights up to 2^8, away from fp16's subnormals)
        const float mn = fmaxf(m, mb - 8.f), ms = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m - ms);  // (m = -inf: 0)
        m = mn;
        half8 pf[NP];
        float ls = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float p = __builtin_amdgcn_exp2f(s[j][r] - ms);
                ls += p;
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    pf[k][4 * j + r] = (_Float16)p;
                    p -= (float)pf[k][4 * j + r];
                }
            }
        l = fmaf(l, f, ls);
#pragma unroll
        for (int n = 0; n < ND; n++) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; i++)  // tokens 2 i, 2 i + 1 of the operand: their halfs of dim n
                y[i] = __builtin_amdgcn_perm(pv[i >> 1][2 * (i & 1) + 1][n >> 1], pv[i >> 1][2 * (i & 1)][n >> 1],
                                             (n & 1) ? 0x07060302u : 0x05040100u);
            const u32x4 yv = {y[0], y[1], y[2], y[3]};
            const half8 vf = __builtin_bit_cast(half8, yv);
#pragma unroll
            for (int r = 0; r < 4; r++) o[n][r] *= f;
#pragma unroll
            for (int p = NP - 1; p >= 0; p--) o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[p], o[n], 0, 0, 0);
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
    // ---- join the waves; lane li, lg: row li, dims ND (4 lg + r) + n
    const bool direct = !w.pre && (a.join || a.n_pre + a.n_own == 1);
    l = xor32_sum(xor16_sum(l));
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int n = 0; n < ND; n += 4)
            *(f32x4 *)(so + (wave * SA_ROWS + li) * LD + ND * (4 * lg + r) + n) =
                f32x4{o[n][r], o[n + 1][r], o[n + 2][r], o[n + 3][r]};
    if (lg == 0) {
        sm[wave * SA_ROWS + li] = m;
        sl[wave * SA_ROWS + li] = l;
    }
    __syncthreads();
    for (uint32_t i = tid; i < w.nrow * (HD / 4); i += 64 * W) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4, R = w.row0 + r, s = R / a.G, h = kvh * a.G + R % a.G;
        float M = sm[r], L = 0.f;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 1; k < W; k++) M = fmaxf(M, sm[k * SA_ROWS + r]);
        const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float fk = __builtin_amdgcn_exp2f(sm[k * SA_ROWS + r] - Ms);
            const f32x4 v = *(const f32x4 *)(so + (k * SA_ROWS + r) * LD + d);
            O.x = fmaf(v.x, fk, O.x);
            O.y = fmaf(v.y, fk, O.y);
            O.z = fmaf(v.z, fk, O.z);
            O.w = fmaf(v.w, fk, O.w);
            L = fmaf(sl[k * SA_ROWS + r], fk, L);
        }
        if (!w.pre && a.join && a.n_pre) {
            // the row's parts of the prefix, 8 at a time
            const uint32_t np = w.shares ? a.n_pre : 0u, rows = a.n_seq * a.nh, row = s * a.nh + h;
            for (uint32_t p0 = 0; p0 < np; p0 += 8) {
                float2 st[8];
                f32x4 v[8];
#pragma unroll
                for (uint32_t u = 0; u < 8; u++) {  // (past the last part: its values again, weight 0)
                    const size_t pr = (size_t)min(p0 + u, np - 1) * rows + row;
                    st[u] = *(const float2 *)(a.stat + 2 * pr);
                    v[u] = *(const f32x4 *)(a.part + pr * HD + d);
                }
                float mn = M;
#pragma unroll
                for (uint32_t u = 0; u < 8; u++) mn = fmaxf(mn, st[u].x);
                const float mr = mn == -INFINITY ? 0.f : mn, old = __builtin_amdgcn_exp2f(M - mr);
                M = mn;
                O *= old;
                L *= old;
#pragma unroll
                for (uint32_t u = 0; u < 8; u++) {
                    const float f = p0 + u < np ? __builtin_amdgcn_exp2f(st[u].x - mr) : 0.f;
                    O.x = fmaf(v[u].x, f, O.x);
                    O.y = fmaf(v[u].y, f, O.y);
                    O.z = fmaf(v[u].z, f, O.z);
                    O.w = fmaf(v[u].w, f, O.w);
                    L = fmaf(st[u].y, f, L);
                }
            }
        }
        if (direct) {
            const f32x4 v = nstep || w.shares ? f32x4{O.x / L, O.y / L, O.z / L, O.w / L} : f32x4{0.f, 0.f, 0.f, 0.f};
            T *op = (T *)(a.out + s * a.out_row) + h * HD + d;
            if constexpr (sizeof(T) == 4) *(f32x4 *)op = v;
            else *(half4 *)op = half4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
        } else {
            const size_t pr = (size_t)w.part * a.n_seq * a.nh + (size_t)s * a.nh + h;
            *(f32x4 *)(a.part + pr * HD + d) = O;
            if (d == 0) {
                a.stat[2 * pr] = M;
                a.stat[2 * pr + 1] = L;
            }
        }
    }
}

// The tokens of a sequence that are its own (from `b` on; a sequence shorter than
// the prefix, or a call without parts of the prefix: all), in parts of `c`.
ZH_DEV uint32_t own_tokens(const SharedArgs &a, uint32_t len, uint32_t &b, uint32_t &c) {
    b = len < a.prefix || !a.n_pre ? 0u : a.prefix;
    const uint32_t least = (len - b + a.n_own - 1) / a.n_own;
    c = max(a.own_len, (least + SA_KB - 1) / SA_KB * SA_KB);
    return (len - b + c - 1) / c;  // parts
}

// The prefix's workgroups, then the sequences' own.
template <int HD, int NP, typename T>
__global__ __launch_bounds__(64 * W, 3) void k_shared_attn(SharedArgs a) {
    __shared__ __align__(16) float lds[W * SA_ROWS * (HD + 6)];
    const bool pre = blockIdx.x < a.pre_blocks;
    // (kv heads fastest: with 8 of them every head's K and V stay in one XCD's L2)
    const uint32_t job = pre ? blockIdx.x : blockIdx.x - a.pre_blocks, kvh = job % a.nkv;
    SharedPart w;
    w.first = 0;
    w.pre = pre;
    w.shares = false;
    if (pre) {
        const uint32_t tile = job / a.nkv % a.pre_tiles;
        w.part = job / a.nkv / a.pre_tiles;
        w.row0 = tile * SA_ROWS;
        w.nrow = min(SA_ROWS, a.n_seq * a.G - w.row0);
        w.tab = 0;
        w.t0 = w.part * a.pre_len;
        w.t1 = min(w.t0 + a.pre_len, a.prefix);
        shared_part<HD, NP, false, T>(a, w, kvh, lds);
    } else {
        const uint32_t s = job / a.nkv % a.n_seq, p = job / a.nkv / a.n_seq;
        w.part = a.n_pre + p;
        w.row0 = s * a.G;
        w.nrow = a.G;
        w.tab = s;
        const uint32_t len = seq_len(a, s);
        if (threadIdx.x == 0 && p == 0 && kvh == 0 && a.lens[s] > a.max_len) atomicOr(a.err, ZH_DEVERR_KV_ROW);
        uint32_t b, c;
        const uint32_t n = own_tokens(a, len, b, c);
        if (p >= n && a.n_pre + a.n_own > 1 && !a.join) return;  // (the join reads the parts there are)
        w.shares = a.n_pre && len >= a.prefix;
        w.t0 = b + p * c;
        w.t1 = min(w.t0 + c, len);
        if (!a.n_pre && a.prefix && len >= a.prefix) w.first = w.t0 = a.prefix;  // (one part: the whole context)
        shared_part<HD, NP, true, T>(a, w, kvh, lds);
    }
}

// Many rows (a workgroup: 8 or 4 waves of 32): K and V pass through LDS once for
// all of them, in stages of 64 tokens copied there three ahead without passing
// registers.
//   S^T = K q^T by v_mfma_f32_32x32x16_f16: lane (i = lane % 32, h = lane / 32)
//   holds tokens 8 (r / 4) + 4 h + r % 4 of row i in register r; registers
//   8 s .. 8 s + 7 are the weights' operand of the s-th 16-token product
//   O^T += V^T P^T. V stays row-major in LDS, its transposed fragments come from
//   ds_read_b64_tr_b16. 16-byte piece p of a row lies at p ^ st_swz(row), so that
//   16 rows' reads of one piece hit every bank once and the transposing reads
//   (4 pieces of 8 rows) every bank twice.
// The products of the next 32 tokens' scores run while the current ones' weights
// are computed. The reference maximum moves only when a score passes it by 2^8
// (the weights then reach 2^12 in fp16 at most), so the output is rarely rescaled.
// Bound by the matrix units: 2000 rows a kv head over 8192 tokens (34 GFLOP)
// 48 us, of which 6 before the first product, 6 for the parts' stores (33 MB)
// and 26 the products alone (1.3 PFLOP/s, a large library product's rate); the
// rest is the softmax (4), the copies and the LDS reads (4) where they do not
// hide. 4 waves of 64 rows, each K and V fragment for two products: 70 us (past
// 256 registers the accumulators move between the two register files).
// NP pieces as in k_shared_attn, but f16 weights in 1: their second products would
// take 106 us for 75 (64 sequences over 32768 tokens) and 100 for 72 (250 over 8192);
// the rounding adds to the store's, 2.8e-4 of the output's root mean square over 1550
// tokens for 2.07e-4.
constexpr uint32_t ST_KB = 64, ST_NS = 4;
template <int HD>
constexpr uint32_t st_lds() { return 2 * ST_NS * ST_KB * HD * 2; }

// Of 16 pieces a row: rows 4 apart differ in the low bits, rows 1 apart in the
// high ones; of 8 (two rows side by side in the banks) the same of row pairs.
template <uint32_t PPR>
ZH_DEV uint32_t st_swz(uint32_t row) {
    return PPR == 16 ? (row & 3) * 4 + (row / 4 & 3) : (row / 2 & 1) * 4 + (row / 4 & 3);
}

// 16 bytes per lane from base + off to LDS at the wave-uniform address + 16 lane.
ZH_DEV void dma16_s(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
                 : "memory", "m0");
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int HD, int NP, int NW, typename T>
__global__ __launch_bounds__(64 * NW, NP == 2 && HD == 128 && NW == 4 ? 1 : 2) void k_shared_tile(SharedArgs a) {
    constexpr int KS = HD / 16, DT = HD / 32;       // k-steps of the scores, 32-dim tiles of the output
    constexpr uint32_t ROWB = HD * 2, PPR = HD / 8;  // bytes and 16-byte pieces of a row
    constexpr uint32_t STAGE = ST_KB * ROWB, NI = 16 * ROWB / 1024;  // bytes of a stage, copies of a page
    extern __shared__ __align__(16) uint8_t lds[];
    typedef __fp16 tr4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) tr4 lds_tr4;
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t i32 = lane % 32, h = lane / 32;
    // (the row tiles of one part and kv head on one XCD: they read the same K and V)
    const uint32_t per = a.nkv * a.n_pre, tile = blockIdx.x / per, kvh = blockIdx.x % per % a.nkv;
    const uint32_t part = blockIdx.x % per / a.nkv;
    const uint32_t rows = a.n_seq * a.G, row0 = (tile * NW + wave) * 32;
    const bool mine = row0 < rows;  // (uniform per wave: it has rows)
    const uint32_t t0 = part * a.pre_len, t1 = min(t0 + a.pre_len, a.prefix);
    const uint32_t nst = (t1 - t0 + ST_KB - 1) / ST_KB;
    // ---- copies, 1 KB (1024 / ROWB rows) each: 4 waves a page of K and of V of a
    // stage; 8 waves a page of one of them
    const uint32_t lds0 = lds_addr(lds);
    uint32_t off[NI];
#pragma unroll
    for (uint32_t i = 0; i < NI; i++) {
        const uint32_t r = i * (64 / PPR) + lane / PPR;
        off[i] = r * ROWB + ((lane % PPR) ^ st_swz<PPR>(r)) * 16;
    }
    const uint8_t *kh = (const uint8_t *)(a.kc + (size_t)kvh * a.cache_tokens * HD);
    const uint8_t *vh = (const uint8_t *)(a.vc + (size_t)kvh * a.cache_tokens * HD);
    // the page that this wave copies of a stage, looked up (by a scalar load, which
    // the copies' order does not wait for) before the barrier ahead of its copy
    bool bad = false;
    auto page = [&](uint32_t st) __attribute__((always_inline)) {
        return ((const const_u32 *)a.tables)[min(t0 / 16 + st * 4 + wave % 4, (t1 - 1) / 16)];
    };
    auto issue = [&](uint32_t st, uint32_t pg) __attribute__((always_inline)) {
        if (pg >= a.cache_tokens / 16) {
            bad = true;
            pg = 0;
        }
        const uint64_t at = (uint64_t)pg * (16 * ROWB);
        const uint32_t to = lds0 + st % ST_NS * STAGE + wave % 4 * (16 * ROWB);
        if (NW == 4 || wave < 4) {
#pragma unroll
            for (uint32_t i = 0; i < NI; i++) dma16_s(kh + at, off[i], to + i * 1024);
        }
        if (NW == 4 || wave >= 4) {
#pragma unroll
            for (uint32_t i = 0; i < NI; i++) dma16_s(vh + at, off[i], to + ST_NS * STAGE + i * 1024);
        }
    };
    // waits until this wave's copies of V of stage st and K of stage st + 1 have
    // landed, those of the two stages after it issued (as far as there are any)
    auto landed = [&](uint32_t st) __attribute__((always_inline)) {
        if (NW == 4) {
            if (st + 2 < nst) wait_vm<3 * NI>();
            else if (st + 1 < nst) wait_vm<NI>();
            else wait_vm<0>();
        } else if (wave < 4) {
            if (st + 2 < nst) wait_vm<NI>();
            else wait_vm<0>();
        } else {
            if (st + 2 < nst) wait_vm<2 * NI>();
            else if (st + 1 < nst) wait_vm<NI>();
            else wait_vm<0>();
        }
    };
    // the first copies go out before the rows are read
    const uint32_t pg0 = page(0), pg1 = page(1), pg2 = page(2);
    uint32_t pg = page(3);
    issue(0, pg0);
    if (nst > 1) issue(1, pg1);
    if (nst > 2) issue(2, pg2);
    // ---- the row's q: dims 16 k + 8 h ..
    half8 qf[NP][KS];
    int qe = 0;  // q is scaled by 2^-qe
    {
        const uint32_t row = min(row0 + i32, rows - 1);
        const T *qp = (const T *)(a.q + row / a.G * a.q_row) + (size_t)(kvh * a.G + row % a.G) * HD + 8 * h;
        float v[KS][8], mx = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            ld8(qp + 16 * k, v[k]);
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(v[k][e]));
        }
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
    }
    const float c = score_factor(a, qe);  // raw scores to base 2
    f32x16 o[DT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.f;
    // fragment addresses in a stage (their k-step and 32-dim tile by exclusive or)
    const uint32_t ka = i32 * ROWB + ((h ^ st_swz<PPR>(i32)) * 16);
    const uint32_t l16 = lane % 16, vr = 4 * h + l16 / 4, vp = 2 * (lane / 16 % 2) + l16 % 4 / 2;
    const uint32_t va = vr * ROWB + ((vp ^ st_swz<PPR>(vr)) * 16) + 8 * (l16 % 2);
    const uint8_t *kp[KS], *vp0[DT], *vp1[DT];  // (the stage and the tokens in it: constant offsets)
#pragma unroll
    for (int k = 0; k < KS; k++) kp[k] = lds + (ka ^ (k * 32));
#pragma unroll
    for (int d = 0; d < DT; d++) {
        // tokens 4 h .. +3 and those 8 on (8 rows on, the piece's bit 1 flipped)
        vp0[d] = lds + ST_NS * STAGE + (va ^ (d * 64));
        vp1[d] = lds + ST_NS * STAGE + 8 * ROWB + (va ^ (d * 64) ^ 32);
    }
    f32x16 s, sn;  // scores of the current and the next 32 tokens (raw)
    half8 kf[KS];  // K fragments of the next ones
    auto load_k = [&](uint32_t slot, uint32_t kt) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < KS; k++) kf[k] = *(const half8 *)(kp[k] + slot * STAGE + kt * 32 * ROWB);
    };
    // the reference maximum, for scores up to mx: moved, and the sums with it,
    // where one passes it by 2^8
    auto refer = [&](float mx) __attribute__((always_inline)) {
        mx = xor32_max(mx) * c;
        if (__builtin_amdgcn_ballot_w64(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] *= f;
        }
    };
    auto largest = [&](const f32x16 &d) __attribute__((always_inline)) {
        float x = d[0];
#pragma unroll
        for (int r = 1; r < 16; r++) x = fmaxf(x, d[r]);
        return x;
    };
    // tokens past the part: no score
    auto mask = [&](uint32_t t, f32x16 &d) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 16; r++)
            if (t + 8 * (r / 4) + 4 * h + r % 4 >= t1) d[r] = -INFINITY;
    };
    if (nst > 2) wait_vm<(NW == 4 ? 5 : 2) * NI>();  // K of stage 0
    else wait_vm<0>();
    lds_bar();
    if (mine) {
        load_k(0, 0);
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.f;
#pragma unroll
        for (int p = NP - 1; p >= 0; p--)
#pragma unroll
            for (int k = 0; k < KS; k++) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k], qf[p][k], s, 0, 0, 0);
        load_k(0, 1);
        if (t0 + 32 > t1) mask(t0, s);
        refer(largest(s));
    }
    constexpr int PAIRS = 8, EARLY = 6;  // weights in pairs; those taken beside the scores' products
    for (uint32_t s0 = 0; s0 < nst; s0 += ST_NS)  // (the ring's slots unrolled: constant LDS offsets)
#pragma unroll
    for (uint32_t slot = 0; slot < ST_NS; slot++) {
        const uint32_t st = s0 + slot;
        if (st >= nst) break;  // uniform
        landed(st);
        lds_bar();
        if (st + 3 < nst) issue(st + 3, pg);
        const uint32_t tk = t0 + st * ST_KB;
        if (tk + ST_KB > t1) {  // V of the tokens past the part: zero (0 times NaN is NaN)
            for (uint32_t i = (t1 - tk) * ROWB + tid * 16; i < STAGE; i += 64 * NW * 16)
                *(u32x4 *)(lds + (ST_NS + slot) * STAGE + i) = u32x4{0, 0, 0, 0};
            lds_bar();
        }
        if (!mine) {
            pg = page(st + 4);
            continue;
        }
#pragma unroll
        for (uint32_t kt = 0; kt < 2; kt++) {
            half8 pf[NP][2], vf[2][DT];
            const float b = m == -INFINITY ? 0.f : 4.f - m;
            float mx = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r++) sn[r] = 0.f;
            auto weights = [&](int i) __attribute__((always_inline)) {  // 2 i and 2 i + 1
#pragma unroll
                for (int r = 2 * i; r < 2 * i + 2; r++) {
                    float p = __builtin_amdgcn_exp2f(fmaf(s[r], c, b));
                    l += p;
#pragma unroll
                    for (int k = 0; k < NP; k++) {
                        pf[k][r / 8][r % 8] = (_Float16)p;
                        p -= (float)pf[k][r / 8][r % 8];
                    }
                }
            };
            auto load_v = [&](int s2) __attribute__((always_inline)) {
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const uint32_t at = slot * STAGE + (32 * kt + 16 * s2) * ROWB;
                    const tr4 x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4 *)(vp0[d] + at));
                    const tr4 y = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4 *)(vp1[d] + at));
                    vf[s2][d] = half8{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3],
                                      (_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
                }
            };
            // three runs of products, each group of them (64 cycles) with vector
            // work that does not need it; the order is pinned by the barriers
            load_v(0);
#pragma unroll
            for (int k = 0; k < KS; k++) {
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k], qf[p][k], sn, 0, 0, 0);
#pragma unroll
                for (int i = EARLY * k / KS; i < EARLY * (k + 1) / KS; i++) weights(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            load_v(1);
#pragma unroll
            for (int d = 0; d < DT; d++) {
#pragma unroll
                for (int p = NP - 1; p >= 0; p--)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[0][d], pf[p][0], o[d], 0, 0, 0);
#pragma unroll
                for (int i = EARLY + (PAIRS - EARLY) * d / DT; i < EARLY + (PAIRS - EARLY) * (d + 1) / DT; i++) weights(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            load_k((slot + 1) % ST_NS, kt);
            if (kt == 1) pg = page(st + 4);
#pragma unroll
            for (int d = 0; d < DT; d++) {
#pragma unroll
                for (int p = NP - 1; p >= 0; p--)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[1][d], pf[p][1], o[d], 0, 0, 0);
                if (d == 0) mx = largest(sn);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (kt == 0 || st + 1 < nst) {  // (after the last tokens the scores are of nothing)
                const uint32_t tn = tk + 32 * (kt + 1);
                if (tn + 32 > t1) {
                    mask(tn, sn);
                    mx = largest(sn);
                }
                refer(mx);
            }
            s = sn;
        }
    }
    if (bad && lane == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
    const uint32_t row = row0 + i32;
    l = xor32_sum(l);
    if (row >= rows) return;
    const size_t pr = (size_t)part * a.n_seq * a.nh + (size_t)(row / a.G) * a.nh + kvh * a.G + row % a.G;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *(f32x4 *)(a.part + pr * HD + 32 * d + 8 * g + 4 * h) =
                f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (h == 0) {
        a.stat[2 * pr] = m - 4.f;
        a.stat[2 * pr + 1] = l;
    }
}

// (A launch of its own, 4 us for 35 parts of 512 rows: the workgroup that finishes
// a row last would have to take the parts from past the L2s, 1.6 us more.)
// Joins the parts of a row: HD / 4 lanes, of 4 dims each, take the parts'
// statistics, as many at a time, then all of them the parts' sums, 8 loads of 16
// bytes in flight.
template <int HD, typename T>
__global__ __launch_bounds__(256) void k_shared_join(SharedArgs a) {
    constexpr uint32_t N = HD / 4, U = 8;
    const uint32_t rows = a.n_seq * a.nh, lane = threadIdx.x & 63, l = lane % N;
    const uint32_t row = min(blockIdx.x * (256 / N) + threadIdx.x / N, rows - 1);  // (past the last: that row again)
    const uint32_t s = row / a.nh, len = seq_len(a, s);
    // (a sequence shorter than the prefix has no part in it)
    uint32_t first, c;
    const uint32_t p0 = len < a.prefix ? a.n_pre : 0u, p1 = a.n_pre + own_tokens(a, len, first, c);
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t b = p0; b < p1; b += N) {
        const uint32_t n = min(N, p1 - b);
        const float2 st = *(const float2 *)(a.stat + 2 * ((size_t)(b + min(l, n - 1)) * rows + row));
        float mx = st.x;
#pragma unroll
        for (uint32_t x = 1; x < N; x *= 2) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
        const float mn = fmaxf(M, mx), ms = mn == -INFINITY ? 0.f : mn;
        const float old = __builtin_amdgcn_exp2f(M - ms), w = l < n ? __builtin_amdgcn_exp2f(st.x - ms) : 0.f;
        float ls = l < n ? st.y * w : 0.f;
#pragma unroll
        for (uint32_t x = 1; x < N; x *= 2) ls += __shfl_xor(ls, x, 64);
        M = mn;
        L = fmaf(L, old, ls);
        O *= old;
        for (uint32_t p = 0; p < n; p += U) {
            f32x4 v[U];
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                v[u] = *(const f32x4 *)(a.part + ((size_t)(b + min(p + u, n - 1)) * rows + row) * HD + 4 * l);
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {  // (past the last part: its values again, weight 0)
                const float f = __shfl(w, lane - l + p + u, 64);
                O.x = fmaf(v[u].x, f, O.x);
                O.y = fmaf(v[u].y, f, O.y);
                O.z = fmaf(v[u].z, f, O.z);
                O.w = fmaf(v[u].w, f, O.w);
            }
        }
    }
    const f32x4 r = len ? f32x4{O.x / L, O.y / L, O.z / L, O.w / L} : f32x4{0.f, 0.f, 0.f, 0.f};
    T *op = (T *)(a.out + s * a.out_row) + row % a.nh * HD + 4 * l;
    if constexpr (sizeof(T) == 4) *(f32x4 *)op = r;
    else *(half4 *)op = half4{(_Float16)r.x, (_Float16)r.y, (_Float16)r.z, (_Float16)r.w};
}

// How a call is cut (the same for every call of these sizes).
struct SharedPlan {
    uint32_t n_pre, n_own, pre_tiles, pre_len, own_len, pre_blocks, blocks, tile;
    uint64_t stat_off, bytes;  // of ws
};

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// Whether the prefix of rows_kv rows a kv head goes through LDS tiles.
bool shared_tiled(uint64_t rows_kv, uint32_t nkv, uint32_t hd, uint32_t prefix, bool f32) {
    const uint64_t through = (rows_kv + SA_ROWS - 1) / SA_ROWS * prefix * nkv;
    return rows_kv > 2 * SA_ROWS && through >= sa_tile(hd, f32);
}

bool shared_plan(uint32_t cus, uint32_t n_seq, uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t prefix, uint32_t max_len,
                 bool f32, SharedPlan &p) {
    const uint32_t G = nh / nkv, own = max_len - prefix;
    const uint64_t rows_kv = (uint64_t)n_seq * G, jobs = (uint64_t)n_seq * nkv;
    p = {};
    const bool one = jobs <= cus && prefix <= sa_one(hd) && max_len <= sa_one(hd) + sa_one(hd) * jobs / cus;
    if (prefix && !one) {
        // rows of a prefix workgroup: 128 or 256 on LDS tiles, or 16 streamed
        p.tile = !shared_tiled(rows_kv, nkv, hd, prefix, f32) ? 0 : rows_kv > 128 ? 2 : 1;
        p.pre_tiles = ceil_div(rows_kv, p.tile ? 128u * p.tile : SA_ROWS);
        const uint64_t pj = (uint64_t)p.pre_tiles * nkv;
        // the parts that fill 1 to 4 rounds of one workgroup per CU, by the rounds'
        // stages (steps of all waves) and SA_FIX of their start and end
        const uint32_t fix = p.tile ? SA_TILE_FIX : SA_FIX;
        const uint32_t step = p.tile ? ST_KB : SA_KB, unit = p.tile ? ST_KB : W * SA_KB, most = ceil_div(prefix, 128);
        uint32_t n = 1;
        uint64_t best = ~0ull;
        for (uint64_t r = 1; r <= 4; r++) {
            const uint32_t fit = (uint32_t)(r * cus / pj), k = fit < 1 ? 1u : fit < most ? fit : most;
            const uint64_t cost = ceil_div(pj * k, cus) * (uint64_t)(ceil_div(ceil_div(prefix, k), unit) + fix);
            if (cost < best) {
                best = cost;
                n = k;
            }
        }
        p.pre_len = ceil_div(ceil_div(prefix, n), step) * step;
        p.n_pre = ceil_div(prefix, p.pre_len);
    }
    // a sequence's own tokens (all of them where the prefix has no parts)
    const uint32_t tokens = p.n_pre ? (own ? own : 1) : max_len;
    const uint32_t most = one ? 1 : ceil_div(tokens, p.tile ? 512 : 256);
    const uint32_t want = (uint32_t)(((uint64_t)SA_OWN_PER * cus + jobs / 2) / jobs);
    p.n_own = want < 1 ? 1u : want < most ? want : most;
    p.own_len = ceil_div(ceil_div(tokens, p.n_own), SA_KB) * SA_KB;
    const uint64_t pre = (uint64_t)p.n_pre * p.pre_tiles * nkv, all = pre + (uint64_t)p.n_own * n_seq * nkv;
    // (a launch has fewer than 2^32 threads: workgroups of up to 512, rows of 32 lanes)
    if (all >= 1ull << 23 || (uint64_t)n_seq * nh >= 1ull << 27) return false;
    p.pre_blocks = (uint32_t)pre;
    p.blocks = (uint32_t)all;
    const uint64_t parts = p.n_pre + p.n_own, rows = (uint64_t)n_seq * nh;
    p.stat_off = parts == 1 ? 0 : parts * rows * hd * 4;
    p.bytes = parts == 1 ? 0 : p.stat_off + parts * rows * 8;
    return true;
}

bool shared_shape_ok(const zh_kv_batch *kv, uint32_t nh, uint32_t prefix, uint32_t max_len) {
    return kv_batch_ok(kv) && (kv->head_dim == 64 || kv->head_dim == 128) && nh && nh % kv->n_kv_heads == 0 &&
           nh / kv->n_kv_heads <= SA_ROWS && max_len && max_len <= 1u << 30 && prefix <= max_len;
}

}  // namespace

// The rows with their strides (0: rows without gaps).
static zh_decode_rows with_strides(const zh_kv_batch *kv, const zh_decode_rows *r) {
    zh_decode_rows x = *r;
    if (!x.q_stride) x.q_stride = x.n_heads * kv->head_dim;
    if (!x.out_stride) x.out_stride = x.n_heads * kv->head_dim;
    return x;
}

// The checks of zh_flash_decode_shared, of host data only (exported for the
// tests; c may be null: no message then). cus: the device's CUs.
extern "C" int zh_check_decode_rows(zh_ctx *c, const zh_kv_batch *kv, const zh_decode_rows *rows, uint32_t cus) {
    if (!rows || !shared_shape_ok(kv, rows->n_heads, rows->prefix_len, rows->max_len))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: cache, heads, head_dim or lengths");
    const zh_decode_rows x = with_strides(kv, rows), *r = &x;
    if ((uint64_t)r->max_len > 16ull * kv->table_stride)
        return zh_set_err(c, ZH_ERR_CONTEXT_LENGTH_EXCEEDED, "flash_decode_shared: max_len %u in tables of %u pages",
                          r->max_len, kv->table_stride);
    if (r->type != ZH_F32 && r->type != ZH_F16)
        return zh_set_err(c, ZH_ERR_UNSUPPORTED_QUANT_TYPE, "flash_decode_shared: type %u", r->type);
    const uint64_t size = r->type == ZH_F32 ? 4 : 2, w = (uint64_t)r->n_heads * kv->head_dim, n = kv->n_seq;
    if (n > 1 && (r->q_stride < w || r->out_stride < w))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: rows overlap");
    const uint64_t qb = ((n - 1) * r->q_stride + w) * size, ob = ((n - 1) * r->out_stride + w) * size;
    SharedPlan p;
    if (!shared_plan(cus, kv->n_seq, r->n_heads, kv->n_kv_heads, kv->head_dim, r->prefix_len, r->max_len,
                     r->type == ZH_F32, p))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: too large");
    if (!kv_in_range(r->q, r->q_off, qb) || !kv_in_range(r->out, r->out_off, ob) || !kv_in_range(r->seq_lens, 0, 4 * n) ||
        (p.bytes && !kv_in_range(r->ws, 0, p.bytes)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: range (ws: %llu bytes)",
                          (unsigned long long)p.bytes);
    // out and ws: not what the call reads besides q
    const zh_buf *const read[] = {kv->k_cache, kv->v_cache, kv->tables, r->seq_lens};
    for (const zh_buf *b : read)
        if (b->ptr == r->out->ptr || (p.bytes && b->ptr == r->ws->ptr))
            return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: out or ws is an input");
    if (p.bytes && (r->ws->ptr == r->out->ptr || r->ws->ptr == r->q->ptr))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: ws holds q or out");
    if (r->q_off % 16 || r->out_off % 16 || (n > 1 && (r->q_stride * size % 16 || r->out_stride * size % 16)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: rows not 16-byte aligned");
    const bool same = r->q->ptr == r->out->ptr && r->q_off == r->out_off && (n == 1 || r->q_stride == r->out_stride);
    if (!same && kv_rows_overlap(r->q, r->q_off, qb, r->out, r->out_off, ob) &&
        !(r->q_stride == r->out_stride &&
          kv_columns_apart(r->out, r->out_off, r->q, r->q_off, r->q_stride, w, w, (uint32_t)size)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: out overlaps q");
    return ZH_OK;
}

// How a call of these sizes and type is cut: out = {rows of a prefix workgroup / 128
// where it goes through LDS tiles (0: streamed), parts of the prefix, parts of a
// sequence's own tokens, bytes of ws}. Exported for the tests.
extern "C" int zh_check_shared_plan(const zh_kv_batch *kv, uint32_t n_heads, uint32_t prefix_len, uint32_t max_len,
                                    uint32_t type, uint32_t cus, uint64_t *out) {
    SharedPlan p;
    if (!shared_shape_ok(kv, n_heads, prefix_len, max_len) ||
        !shared_plan(cus, kv->n_seq, n_heads, kv->n_kv_heads, kv->head_dim, prefix_len, max_len, type == ZH_F32, p))
        return ZH_ERR_INVALID_ARGUMENT;
    out[0] = p.tile;
    out[1] = p.n_pre;
    out[2] = p.n_own;
    out[3] = p.bytes;
    return ZH_OK;
}

// zh_flash_decode_shared_ws of a device of `cus` CUs (exported for the tests): an
// upper bound for every smaller n_seq, prefix_len and max_len and both types, since
// one call's bytes (shared_plan) fall and rise with each of them. Its rows of parts,
// n_seq (n_pre + n_own) of them per head, are
//  * own ones: n_own is 1 or at most SA_OWN_PER cus / (n_seq nkv) + 1/2, and at most
//    one per 256 tokens;
//  * the prefix's: n_pre is 1 or at most 4 cus / (nkv pre_tiles), where pre_tiles
//    holds n_seq heads / nkv rows in tiles of 16, 128 or 256, and at most one per 128
//    tokens.
extern "C" uint64_t zh_check_shared_ws(const zh_kv_batch *kv, uint32_t n_heads, uint32_t prefix_len, uint32_t max_len,
                                       uint32_t cus) {
    SharedPlan p;
    if (!shared_shape_ok(kv, n_heads, prefix_len, max_len)) return 0;
    const uint32_t nkv = kv->n_kv_heads, hd = kv->head_dim;
    const uint64_t n = kv->n_seq, rows_kv = n * (n_heads / nkv);
    if (!shared_plan(cus, kv->n_seq, n_heads, nkv, hd, prefix_len, max_len, false, p) ||
        !shared_plan(cus, kv->n_seq, n_heads, nkv, hd, prefix_len, max_len, true, p))
        return 0;
    const uint64_t own = std::min(n * ceil_div(max_len, 256),
                                  std::max<uint64_t>(n, (uint64_t)SA_OWN_PER * cus / nkv + n / 2 + 1));
    // (f16 takes the tiles first)
    const uint64_t tile = !shared_tiled(rows_kv, nkv, hd, prefix_len, false) ? SA_ROWS : rows_kv > 128 ? 256 : 128;
    const uint64_t pre =
        !prefix_len ? 0 : std::min(n * ceil_div(prefix_len, 128), std::max<uint64_t>(n, 4ull * cus * tile / n_heads));
    return std::max<uint64_t>(16, (own + pre) * n_heads * (4ull * hd + 8));
}

extern "C" uint64_t zh_flash_decode_shared_ws(zh_ctx *c, const zh_kv_batch *kv, uint32_t n_heads, uint32_t prefix_len,
                                              uint32_t max_len) {
    return c ? zh_check_shared_ws(kv, n_heads, prefix_len, max_len, (uint32_t)c->cu_count) : 0;
}

template <int HD, int NP, int NW, typename T>
static int tile_launch(zh_ctx *c, const SharedArgs &a, const SharedPlan &p) {
    static std::atomic<bool> attr[64];  // by device
    if (c->device >= 64 || !attr[c->device].load(std::memory_order_relaxed)) {
        ZH_HIP(c, hipFuncSetAttribute((const void *)k_shared_tile<HD, NP, NW, T>,
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)st_lds<HD>()));
        if (c->device < 64) attr[c->device].store(true, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL((k_shared_tile<HD, NP, NW, T>), dim3(p.pre_blocks), dim3(64 * NW), st_lds<HD>(), c->stream, a);
    ZH_LAUNCH_CHECK(c);
    return ZH_OK;
}

template <int HD, int NP, typename T>
static int shared_launch(zh_ctx *c, const SharedArgs &a, const SharedPlan &p) {
    SharedArgs b = a;
    uint32_t blocks = p.blocks;
    if (p.n_pre && p.tile) {
        const int rc = p.tile == 2 ? tile_launch<HD, NP, 8, T>(c, a, p) : tile_launch<HD, NP, 4, T>(c, a, p);
        if (rc) return rc;
        b.pre_blocks = 0;
        blocks -= p.pre_blocks;
        b.join = p.n_own == 1;
    }
    hipLaunchKernelGGL((k_shared_attn<HD, 2, T>), dim3(blocks), dim3(64 * W), 0, c->stream, b);
    ZH_LAUNCH_CHECK(c);
    if (a.n_pre + a.n_own > 1 && !b.join) {
        const uint32_t per = 256 / (HD / 4);  // rows of a workgroup
        hipLaunchKernelGGL((k_shared_join<HD, T>), dim3((a.n_seq * a.nh + per - 1) / per), dim3(256), 0, c->stream, a);
        ZH_LAUNCH_CHECK(c);
    }
    return ZH_OK;
}

extern "C" int zh_flash_decode_shared(zh_ctx *c, const zh_kv_batch *kv, const zh_decode_rows *rows) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    const int rc = zh_check_decode_rows(c, kv, rows, (uint32_t)c->cu_count);
    if (rc) return rc;
    const zh_decode_rows x = with_strides(kv, rows), *r = &x;
    zh_device_scope dev(c);
    SharedPlan p;
    shared_plan((uint32_t)c->cu_count, kv->n_seq, r->n_heads, kv->n_kv_heads, kv->head_dim, r->prefix_len, r->max_len,
                r->type == ZH_F32, p);
    SharedArgs a = {};
    const uint64_t size = r->type == ZH_F32 ? 4 : 2;
    a.q = (const uint8_t *)r->q->ptr + r->q_off;
    a.out = (uint8_t *)r->out->ptr + r->out_off;
    a.q_row = r->q_stride * size;
    a.out_row = r->out_stride * size;
    a.kc = (const uint16_t *)kv->k_cache->ptr;
    a.vc = (const uint16_t *)kv->v_cache->ptr;
    a.tables = (const uint32_t *)kv->tables->ptr;
    a.lens = (const uint32_t *)r->seq_lens->ptr;
    a.part = p.bytes ? (float *)r->ws->ptr : nullptr;
    a.stat = p.bytes ? (float *)((char *)r->ws->ptr + p.stat_off) : nullptr;
    a.err = c->err_dev;
    a.n_seq = kv->n_seq;
    a.stride = kv->table_stride;
    a.cache_tokens = kv->cache_tokens;
    a.nh = r->n_heads;
    a.nkv = kv->n_kv_heads;
    a.G = a.nh / a.nkv;
    a.prefix = r->prefix_len;
    a.max_len = r->max_len;
    a.n_pre = p.n_pre;
    a.n_own = p.n_own;
    a.pre_tiles = p.pre_tiles;
    a.pre_blocks = p.pre_blocks;
    a.pre_len = p.pre_len;
    a.own_len = p.own_len;
    // (64 bits: a scale of any size times log2 e)
    const double scale = (double)(r->attn_scale != 0.f ? r->attn_scale : 1.0f / sqrtf((float)kv->head_dim)) *
                         1.44269504088896340736f;
    int scale_exp = 0;
    a.scale = isfinite(scale) ? (float)frexp(scale, &scale_exp) : NAN;
    a.scale_exp = scale_exp;
    if (kv->head_dim == 128)
        return size == 4 ? shared_launch<128, 2, float>(c, a, p) : shared_launch<128, 1, _Float16>(c, a, p);
    return size == 4 ? shared_launch<64, 2, float>(c, a, p) : shared_launch<64, 1, _Float16>(c, a, p);
}
