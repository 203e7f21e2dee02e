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

#include "zh_device.h"
#include "zh_internal.h"
#include "zh_kv.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t SA_ROWS = 16;  // rows of a workgroup: one MFMA tile
constexpr uint32_t SA_KB = 32;    // tokens of a wave's step
constexpr int SA_W = 4;           // waves of a workgroup, each on its own steps

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
    float scale;
};

// The sequence's length as the kernels take it: cut at max_len (the host has
// checked that the table holds that many tokens).
ZH_DEV uint32_t seq_len(const SharedArgs &a, uint32_t s) {
    return min(a.lens[s], a.max_len);
}

template <typename T>
ZH_DEV float ld(const uint8_t *p, uint32_t i) {
    return sizeof(T) == 4 ? ((const float *)p)[i] : (float)((const _Float16 *)p)[i];
}

// One workgroup: 16 rows of one kv head over the tokens of one part. Each wave
// takes steps of 32 tokens by itself, K and V straight from the cache into the
// matrix operands' registers (no LDS, no barrier before the end):
//   S^T = K q^T (tokens x rows): lane (li = lane % 16, lg = lane / 16) holds
//   tokens 16 j + 4 lg + r of row li, so that a row's maximum is in-lane plus
//   two lane exchanges, and its weights lie as the second product's operand
//   wants them: O^T += V^T P^T, k = (token 4 lg + r of tile 0, then of tile 1).
//   V's rows are read whole (lane li: dims HD/16 li ..), transposed by byte
//   permutes; column li of the output tile n is dim HD/16 li + n.
// NP pieces: q (scaled by a power of two to a maximum in [1, 2)) and P as sums
// of NP fp16 values; 2 keep 22 bits of each.
template <int HD, int NP, typename T>
__global__ __launch_bounds__(64 * SA_W, 2) void k_shared_attn(SharedArgs a) {
    constexpr int K4 = HD / 32, ND = HD / 16;  // k-steps of the scores, dims per lane and output tiles
    __shared__ float so[SA_W][SA_ROWS][HD + 4];
    __shared__ float sm[SA_W][SA_ROWS], sl[SA_W][SA_ROWS];
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t li = lane % 16, lg = lane / 16;
    const bool pre = blockIdx.x < a.pre_blocks;
    // (kv heads fastest: with 8 of them every head's K and V stay in one XCD's L2)
    const uint32_t job = pre ? blockIdx.x : blockIdx.x - a.pre_blocks, kvh = job % a.nkv;
    uint32_t part, row0, nrow, t0, t1, tab;  // rows row0 .. (s * G + g), tokens [t0, t1) through table `tab`
    if (pre) {
        const uint32_t tile = job / a.nkv % a.pre_tiles;
        part = job / a.nkv / a.pre_tiles;
        row0 = tile * SA_ROWS;
        nrow = min(SA_ROWS, a.n_seq * a.G - row0);
        tab = 0;
        t0 = part * a.pre_len;
        t1 = min(t0 + a.pre_len, a.prefix);
    } else {
        const uint32_t s = job / a.nkv % a.n_seq, p = job / a.nkv / a.n_seq;
        part = a.n_pre + p;
        row0 = s * a.G;
        nrow = a.G;
        tab = s;
        const uint32_t len = seq_len(a, s);
        if (tid == 0 && p == 0 && kvh == 0 && a.lens[s] > a.max_len) atomicOr(a.err, ZH_DEVERR_KV_ROW);
        // a sequence shorter than the prefix: all of its tokens are its own
        const uint32_t b = len < a.prefix ? 0u : a.prefix, n = (len - b + a.n_own - 1) / a.n_own;
        const uint32_t c = (n + SA_KB - 1) / SA_KB * SA_KB;
        t0 = min(b + p * c, len);
        t1 = min(b + (p + 1) * c, len);
    }
    const uint32_t ta = t0 & ~15u;  // steps start on a page; tokens before t0 are masked
    const uint32_t nstep = t1 > t0 ? (t1 - ta + SA_KB - 1) / SA_KB : 0u;
    // the row's q as operand fragments: dims 32 k4 + 8 lg ..
    const uint32_t row = row0 + min(li, nrow - 1), rs = row / a.G, rh = kvh * a.G + row % a.G;
    half8 qf[NP][K4];
    float c = a.scale * 1.44269504088896340736f;  // scores in base 2
    {
        const uint8_t *qp = a.q + rs * a.q_row + (size_t)rh * HD * sizeof(T);
        float v[K4][8], mx = 0.f;
#pragma unroll
        for (int k4 = 0; k4 < K4; k4++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[k4][e] = ld<T>(qp, 32 * k4 + 8 * lg + e);
                mx = fmaxf(mx, fabsf(v[k4][e]));
            }
        float up = 1.f;
        if (NP > 1) {
            mx = xor32_max(xor16_max(mx));
            // 2^-E for a maximum in [2^E, 2^(E+1)) (not for zero, infinite or tiny rows)
            const uint32_t E = __float_as_uint(mx) >> 23;
            if (E >= 8 && E <= 246) {
                up = __uint_as_float((254u - E) << 23);
                c *= __uint_as_float(E << 23);
            }
        }
#pragma unroll
        for (int k4 = 0; k4 < K4; k4++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float x = v[k4][e] * up;
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    qf[p][k4][e] = (_Float16)x;
                    x -= (float)qf[p][k4][e];
                }
            }
    }
    floatx4 o[ND];
#pragma unroll
    for (int n = 0; n < ND; n++) o[n] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // the row's maximum (every lg alike), this lane's share of its sum
    const uint16_t *kh = a.kc + (size_t)kvh * a.cache_tokens * HD, *vh = a.vc + (size_t)kvh * a.cache_tokens * HD;
    const uint32_t *tb = a.tables + (size_t)tab * a.stride;
    bool bad = false;
    for (uint32_t st = wave; st < nstep; st += SA_W) {
        const uint32_t tk = ta + st * SA_KB;
        // the step's two pages (the second clamped to the part's last)
        uint32_t pg[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            pg[j] = tb[min(tk / 16 + j, (t1 - 1) / 16)];
            if (pg[j] >= a.cache_tokens / 16) {
                bad = true;
                pg[j] = 0;
            }
        }
        half8 kf[2][K4];
        uint32_t pv[2][4][ND / 2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint16_t *kp = kh + ((size_t)pg[j] * 16 + li) * HD + 8 * lg;
#pragma unroll
            for (int k4 = 0; k4 < K4; k4++) kf[j][k4] = *(const half8 *)(kp + 32 * k4);
            const uint16_t *vp = vh + ((size_t)pg[j] * 16 + 4 * lg) * HD + ND * li;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (ND == 8) *(u32x4 *)pv[j][r] = *(const u32x4 *)(vp + r * HD);
                else *(u32x2 *)pv[j][r] = *(const u32x2 *)(vp + r * HD);
            }
        }
        const bool whole = tk >= t0 && tk + SA_KB <= t1;
        float s[2][4], mb = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            floatx4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                for (int k4 = 0; k4 < K4; k4++)
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[j][k4], qf[p][k4], d, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[j][r] = d[r] * c;
                if (!whole) {
                    // a token outside the part: no score, and no V (0 times
                    // what the cache holds there may be NaN)
                    const uint32_t t = tk + 16 * j + 4 * lg + r;
                    if (t < t0 || t >= t1) {
                        s[j][r] = -INFINITY;
#pragma unroll
                        for (int w = 0; w < ND / 2; w++) pv[j][r][w] = 0u;
                    }
                }
                mb = fmaxf(mb, s[j][r]);
            }
        }
        mb = xor32_max(xor16_max(mb));
        const float mn = fmaxf(m, mb), ms = mn == -INFINITY ? 0.f : mn;
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
                p *= 256.f;  // (away from fp16's subnormals; taken back at the end)
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    pf[k][4 * j + r] = (_Float16)p;
                    p -= (float)pf[k][4 * j + r];
                }
            }
        l = fmaf(l, f, ls);
#pragma unroll
        for (int n = 0; n < ND; n++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++)  // tokens 2 i, 2 i + 1 of the operand: their halfs of dim n
                w[i] = __builtin_amdgcn_perm(pv[i >> 1][2 * (i & 1) + 1][n >> 1], pv[i >> 1][2 * (i & 1)][n >> 1],
                                             (n & 1) ? 0x07060302u : 0x05040100u);
            const u32x4 wv = {w[0], w[1], w[2], w[3]};
            const half8 vf = __builtin_bit_cast(half8, wv);
#pragma unroll
            for (int r = 0; r < 4; r++) o[n][r] *= f;
#pragma unroll
            for (int p = NP - 1; p >= 0; p--) o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[p], o[n], 0, 0, 0);
        }
    }
    if (bad && lane == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
    l = xor32_sum(xor16_sum(l));
    // ---- join the waves; lane li, lg: row li, dims ND (4 lg + r) + n
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int n = 0; n < ND; n++) so[wave][li][ND * (4 * lg + r) + n] = o[n][r];
    if (lg == 0) {
        sm[wave][li] = m;
        sl[wave][li] = l;
    }
    __syncthreads();
    const bool direct = a.n_pre + a.n_own == 1;
    for (uint32_t i = tid; i < nrow * HD; i += 64 * SA_W) {
        const uint32_t r = i / HD, d = i % HD, R = row0 + r, s = R / a.G, h = kvh * a.G + R % a.G;
        float M = sm[0][r], O = 0.f, L = 0.f;
#pragma unroll
        for (int w = 1; w < SA_W; w++) M = fmaxf(M, sm[w][r]);
        const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < SA_W; w++) {
            const float f = __builtin_amdgcn_exp2f(sm[w][r] - Ms);
            O = fmaf(so[w][r][d], f, O);
            L = fmaf(sl[w][r], f, L);
        }
        O *= 1.f / 256.f;
        if (direct) {
            const float v = t1 > t0 ? O / L : 0.f;
            uint8_t *op = a.out + s * a.out_row;
            if (sizeof(T) == 4) ((float *)op)[h * HD + d] = v;
            else ((_Float16 *)op)[h * HD + d] = (_Float16)v;
        } else {
            const size_t pr = (size_t)part * a.n_seq * a.nh + (size_t)s * a.nh + h;
            a.part[pr * HD + d] = O;
            if (d == 0) {
                a.stat[2 * pr] = M;
                a.stat[2 * pr + 1] = L;
            }
        }
    }
}

// Joins the parts of a row (one wave each).
template <int HD, typename T>
__global__ __launch_bounds__(64) void k_shared_join(SharedArgs a) {
    const uint32_t row = blockIdx.x, s = row / a.nh, lane = threadIdx.x;
    const uint32_t len = seq_len(a, s), rows = a.n_seq * a.nh;
    const uint32_t p0 = len < a.prefix ? a.n_pre : 0u;  // (such a sequence has no part in the prefix)
    constexpr int E = HD / 64;
    float M = -INFINITY, L = 0.f, O[E];
#pragma unroll
    for (int e = 0; e < E; e++) O[e] = 0.f;
    for (uint32_t p = p0; p < a.n_pre + a.n_own; p++) M = fmaxf(M, a.stat[2 * ((size_t)p * rows + row)]);
    const float Ms = M == -INFINITY ? 0.f : M;
    for (uint32_t p = p0; p < a.n_pre + a.n_own; p++) {
        const size_t pr = (size_t)p * rows + row;
        const float f = __builtin_amdgcn_exp2f(a.stat[2 * pr] - Ms);
        L = fmaf(a.stat[2 * pr + 1], f, L);
#pragma unroll
        for (int e = 0; e < E; e++) O[e] = fmaf(a.part[pr * HD + E * lane + e], f, O[e]);
    }
    uint8_t *op = a.out + s * a.out_row;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float v = len ? O[e] / L : 0.f;
        const uint32_t i = row % a.nh * HD + E * lane + e;
        if (sizeof(T) == 4) ((float *)op)[i] = v;
        else ((_Float16 *)op)[i] = (_Float16)v;
    }
}

// How a call is cut (the same for every call of these sizes).
struct SharedPlan {
    uint32_t n_pre, n_own, pre_tiles, pre_len, pre_blocks, blocks;
    uint64_t stat_off, bytes;  // of ws
};

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

bool shared_plan(uint32_t cus, uint32_t n_seq, uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t prefix, uint32_t max_len,
                 SharedPlan &p) {
    const uint32_t G = nh / nkv, own = max_len - prefix;
    p.pre_tiles = ceil_div((uint64_t)n_seq * G, SA_ROWS);
    // parts: two workgroups per CU, at least 128 tokens each
    auto cut = [&](uint64_t jobs, uint32_t tokens) {
        const uint32_t most = ceil_div(tokens, 128), want = ceil_div(2ull * cus, jobs);
        return want < most ? want : most;
    };
    p.n_pre = 0;
    p.pre_len = 0;
    if (prefix) {
        const uint32_t n = cut((uint64_t)p.pre_tiles * nkv, prefix);
        p.pre_len = ceil_div(ceil_div(prefix, n), SA_KB) * SA_KB;
        p.n_pre = ceil_div(prefix, p.pre_len);
    }
    p.n_own = own || !prefix ? cut((uint64_t)n_seq * nkv, own ? own : 1) : 1u;
    if (p.n_own == 0) p.n_own = 1;
    const uint64_t pre = (uint64_t)p.n_pre * p.pre_tiles * nkv, all = pre + (uint64_t)p.n_own * n_seq * nkv;
    if (all > 0x7FFFFFFFull || (uint64_t)n_seq * nh > 0x7FFFFFFFull) return false;
    p.pre_blocks = (uint32_t)pre;
    p.blocks = (uint32_t)all;
    const uint64_t parts = p.n_pre + p.n_own, rows = (uint64_t)n_seq * nh;
    p.stat_off = parts == 1 ? 0 : parts * rows * hd * 4;
    p.bytes = parts == 1 ? 0 : p.stat_off + parts * rows * 8;
    return true;
}

bool shared_shape_ok(const zh_kv_batch *kv, uint32_t nh, uint32_t prefix, uint32_t max_len) {
    return kv_batch_ok(kv) && (kv->head_dim == 64 || kv->head_dim == 128) && nh && nh % kv->n_kv_heads == 0 &&
           nh / kv->n_kv_heads <= SA_ROWS && max_len && prefix <= max_len;
}

}  // namespace

// The rows with their strides (0: rows without gaps).
static zh_decode_rows with_strides(const zh_kv_batch *kv, const zh_decode_rows *r) {
    zh_decode_rows x = *r;
    if (!x.q_stride) x.q_stride = x.n_heads * kv->head_dim;
    if (!x.out_stride) x.out_stride = x.n_heads * kv->head_dim;
    return x;
}

// The checks of zh_flash_decode_shared, of host data only; cus: the device's CUs.
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
    if (!shared_plan(cus, kv->n_seq, r->n_heads, kv->n_kv_heads, kv->head_dim, r->prefix_len, r->max_len, p))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: too large");
    if (!kv_in_range(r->q, r->q_off, qb) || !kv_in_range(r->out, r->out_off, ob) || !kv_in_range(r->seq_lens, 0, 4 * n) ||
        (p.bytes && !kv_in_range(r->ws, 0, p.bytes)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: range (ws: %llu bytes)",
                          (unsigned long long)p.bytes);
    if (r->q_off % 16 || r->out_off % 16 || (n > 1 && (r->q_stride * size % 16 || r->out_stride * size % 16)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: rows not 16-byte aligned");
    const bool same = r->q->ptr == r->out->ptr && r->q_off == r->out_off && (n == 1 || r->q_stride == r->out_stride);
    if (!same && kv_rows_overlap(r->q, r->q_off, qb, r->out, r->out_off, ob) &&
        !(r->q_stride == r->out_stride &&
          kv_columns_apart(r->out, r->out_off, r->q, r->q_off, r->q_stride, w, w, (uint32_t)size)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "flash_decode_shared: out overlaps q");
    return ZH_OK;
}

extern "C" uint64_t zh_flash_decode_shared_ws(zh_ctx *c, const zh_kv_batch *kv, uint32_t n_heads, uint32_t prefix_len,
                                              uint32_t max_len) {
    SharedPlan p;
    if (!c || !shared_shape_ok(kv, n_heads, prefix_len, max_len) ||
        !shared_plan((uint32_t)c->cu_count, kv->n_seq, n_heads, kv->n_kv_heads, kv->head_dim, prefix_len, max_len, p))
        return 0;
    return p.bytes ? p.bytes : 16;
}

template <int HD, int NP, typename T>
static int shared_launch(zh_ctx *c, const SharedArgs &a, const SharedPlan &p) {
    hipLaunchKernelGGL((k_shared_attn<HD, NP, T>), dim3(p.blocks), dim3(64 * SA_W), 0, c->stream, a);
    ZH_LAUNCH_CHECK(c);
    if (a.n_pre + a.n_own > 1) {
        hipLaunchKernelGGL((k_shared_join<HD, T>), dim3(a.n_seq * a.nh), dim3(64), 0, c->stream, a);
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
    shared_plan((uint32_t)c->cu_count, kv->n_seq, r->n_heads, kv->n_kv_heads, kv->head_dim, r->prefix_len, r->max_len, p);
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
    a.scale = r->attn_scale != 0.f ? r->attn_scale : 1.0f / sqrtf((float)kv->head_dim);
    if (kv->head_dim == 128)
        return size == 4 ? shared_launch<128, 2, float>(c, a, p) : shared_launch<128, 1, _Float16>(c, a, p);
    return size == 4 ? shared_launch<64, 2, float>(c, a, p) : shared_launch<64, 1, _Float16>(c, a, p);
}
