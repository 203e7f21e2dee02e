// zh_kv8.hip — a paged KV cache held in 8 bits: the fused q/k RMSNorm + RoPE +
// quantised KV write of a batch, and pages quantised, read back and copied.
#include <new>

#include "zh_kv8.h"

bool kv8_batch_ok(const zh_kv8_batch *kv, uint32_t n_rows) {
    if (!kv || !kv->n_seq || !kv->table_stride || !kv->cache_tokens || kv->cache_tokens % 16 || !kv->n_kv_heads ||
        kv->n_kv_heads > 65535 || (kv->head_dim != 64 && kv->head_dim != 128))
        return false;
    const uint64_t codes = (uint64_t)kv->n_kv_heads * kv->cache_tokens * kv->head_dim;
    const uint64_t scales = 4ull * kv->n_kv_heads * (kv->cache_tokens / 16);
    const zh_buf *const own[] = {kv->k_cache, kv->v_cache, kv->k_scale, kv->v_scale};
    for (int i = 0; i < 4; i++) {
        if (!kv_in_range(own[i], 0, i < 2 ? codes : scales)) return false;
        for (int j = 0; j < i; j++)
            if (own[i]->ptr == own[j]->ptr) return false;
    }
    const zh_buf *const in[] = {kv->tables, kv->seq_lens, kv->row_start};
    for (const zh_buf *b : in)
        for (const zh_buf *o : own)
            if (b && b->ptr == o->ptr) return false;
    return kv->tables && (uint64_t)kv->n_seq * kv->table_stride <= kv->tables->size / 4 &&
           kv_in_range(kv->seq_lens, 0, 4ull * kv->n_seq) &&
           (kv->row_start ? kv_in_range(kv->row_start, 0, 4ull * kv->n_seq + 4) : n_rows <= kv->n_seq);
}

// ---------------------------------------------------------------------------
// q/k RMSNorm + RoPE + quantised KV write. The arithmetic of q is the fp16
// cache's operator's (zh_kv.hip). k goes in 64 bits from the row to the code, its
// angle as a fraction of a turn with the product's own rounding put back: a code
// does not then depend on the order of 32-bit sums, and the same tokens leave the
// same cache whatever batch they came in. That is 30 operations of half rate for
// each element of k beside its loads, 2 us of the chip for 8192 rows of 8 heads.
//
// A workgroup that writes takes one page of one sequence and some heads of k or v:
// thread (slot, l) holds slot `slot` of the page and 8 dims, so the block's largest
// value is a reduction of exponents over the workgroup, and the page's old tokens,
// where the scale rises, are there to be rounded again. In a decode step one slot of
// 16 has a row; the others' threads wait, which costs nothing where latency counts.
// q's heads are workgroups of a row each, behind these in the same launch.
// ---------------------------------------------------------------------------
namespace {

struct Kv8Write {
    const uint8_t *q, *k, *v;
    uint8_t *q_out;
    uint64_t q_row, k_row, v_row, out_row;  // bytes between rows
    const float *qw, *kw, *inv_freq;
    uint8_t *kc, *vc;
    float *ks, *vs;
    const uint32_t *tables, *row_start, *seq_lens;
    uint32_t *err;
    uint32_t n_seq, stride, cache_tokens, nq, nkv, rd, n_rows;
    uint32_t hpb, groups;    // heads of a workgroup that writes, workgroups of a page's k (and of its v)
    uint32_t kv_blocks;      // workgroups that write
    uint32_t q_groups;       // workgroups of a row's q
    uint32_t unit0;          // pages (rows) before this launch's
    float eps;
};

ZH_DEV void ld4(const float *p, float (&v)[4]) {
    const f32x4 a = *(const f32x4 *)p;
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
ZH_DEV void ld4(const _Float16 *p, float (&v)[4]) {
    const half4 a = *(const half4 *)p;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (float)a[e];
}
ZH_DEV void st4(float *p, const float (&v)[4]) { *(f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]}; }
ZH_DEV void st4(_Float16 *p, const float (&v)[4]) {
    *(half4 *)p = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

// pos * f in turns, less whole ones. The product is rounded to 64 bits (as the
// angle is defined); what its own quotient by 2 pi loses is put back.
ZH_DEV double turns(uint32_t pos, float f) {
    const double hi = 0.15915494309189534561, lo = -9.8393383375912439e-18;  // 1 / (2 pi)
    const double a = (double)pos * (double)f, t = a * hi;
    return (t - __builtin_rint(t)) + __builtin_fma(a, lo, __builtin_fma(a, hi, -t));
}

// The dims of lane l of L: four from lo on and four from hi on, partners of each
// other in the rotation, or the passed-through ones in order.
ZH_DEV bool quads(uint32_t l, uint32_t rd, uint32_t &lo, uint32_t &hi) {
    const bool rot = 8 * l < rd;
    lo = rot ? 4 * l : 8 * l;
    hi = rot ? rd / 2 + 4 * l : 8 * l + 4;
    return rot;
}

template <int L>
ZH_DEV double team_sum64(double v) {
#pragma unroll
    for (int d = 1; d < L; d *= 2) v += __shfl_xor(v, d, 64);
    return v;
}

// Heads [h0, h0 + n) of k (or v) in the slots of one page.
template <typename TI, uint32_t F, int HD, bool K>
ZH_DEV void write_heads(const Kv8Write &a, const Kv8Seq &seq, uint32_t page, uint32_t phys, uint32_t h0, uint32_t n) {
    constexpr int L = HD / 8, NW = L / 4;  // lanes of a row, waves
    __shared__ int top[2][NW];
    const uint32_t tid = threadIdx.x, l = tid % L, slot = tid / L, pos = page * 16 + slot;
    const bool mine = pos >= seq.pos && pos < seq.len, begun = page * 16 >= seq.pos;
    uint32_t lo = 8 * l, hi = 8 * l + 4;
    bool rot = false;
    if (K) rot = quads(l, a.rd, lo, hi);
    const uint32_t row = seq.row + (mine ? pos - seq.pos : 0u);
    const TI *src = (const TI *)((K ? a.k : a.v) + row * (K ? a.k_row : a.v_row)) + (size_t)h0 * HD;
    uint8_t *dst = (K ? a.kc : a.vc) + ((size_t)h0 * a.cache_tokens + phys * 16 + slot) * HD;
    float *scale = (K ? a.ks : a.vs) + (size_t)phys * a.nkv + h0;
    float x0[4] = {}, x1[4] = {};
    if (mine) {
        ld4(src + lo, x0);
        ld4(src + hi, x1);
    }
    double co[4], sn[4];
    float w0[4] = {1.f, 1.f, 1.f, 1.f}, w1[4] = {1.f, 1.f, 1.f, 1.f};
    if constexpr (K) {
        if (rot && mine) {
            float f[4];
            ld4(a.inv_freq + 4 * l, f);
#pragma unroll
            for (int e = 0; e < 4; e++) sincospi(2.0 * turns(pos, f[e]), &sn[e], &co[e]);
        }
        if (a.kw) {
            ld4(a.kw + lo, w0);
            ld4(a.kw + hi, w1);
        }
    }
    for (uint32_t i = 0; i < n; i++, src += HD, dst += (size_t)a.cache_tokens * HD, scale++) {
        using V = typename std::conditional<K, double, float>::type;
        V y0[4], y1[4];
        const uint32_t old = __float_as_uint(*scale);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y0[e] = x0[e];
            y1[e] = x1[e];
        }
        if (mine && i + 1 < n) {
            ld4(src + HD + lo, x0);
            ld4(src + HD + hi, x1);
        }
        if constexpr (K) {
            if (a.kw) {  // (uniform; all lanes take part in the sum)
                double sq = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) sq = fma(y0[e], y0[e], fma(y1[e], y1[e], sq));
                const double ri = 1.0 / sqrt(team_sum64<L>(sq) / HD + (double)a.eps);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    y0[e] = w0[e] * (y0[e] * ri);
                    y1[e] = w1[e] * (y1[e] * ri);
                }
            }
            if (rot && mine)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const double p = y0[e], q = y1[e];
                    y0[e] = p * co[e] - q * sn[e];
                    y1[e] = p * sn[e] + q * co[e];
                }
        }
        int t = KV8_LOW;
        if (mine)
#pragma unroll
            for (int e = 0; e < 4; e++) t = max(t, max(kv8_exp<F>(y0[e]), kv8_exp<F>(y1[e])));
#pragma unroll
        for (int d = 1; d < 64; d *= 2) t = max(t, __shfl_xor(t, d, 64));
        if (tid % 64 == 0) top[i & 1][tid / 64] = t;
        __syncthreads();  // (one a head: the next but one writes these words after every thread has passed the next)
#pragma unroll
        for (int j = 0; j < NW; j++) t = max(t, top[i & 1][j]);
        // the block's scale: the larger of its own and the rows'
        float s = t == KV8_NAN || (!begun && !kv8_scale_ok(old)) ? NAN : kv8_pow2(t);
        if (!begun) s = s < __uint_as_float(old) ? __uint_as_float(old) : s;
        const float inv = 1.0f / s;
        if (mine) {
            uint32_t c0 = 0, c1 = 0;
            if (s == s) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    y0[e] *= inv;
                    y1[e] *= inv;
                }
                c0 = kv8_encode<F>(y0);
                c1 = kv8_encode<F>(y1);
            }
            *(uint32_t *)(dst + lo) = c0;
            *(uint32_t *)(dst + hi) = c1;
        } else if (begun) {
            *(uint32_t *)(dst + lo) = 0;
            *(uint32_t *)(dst + hi) = 0;
        } else if (s != __uint_as_float(old) && s == s) {
            const float f = __uint_as_float(old) * inv;
            float v[4];
            for (uint32_t d : {lo, hi}) {
                kv8_decode<F>(*(const uint32_t *)(dst + d), v);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] *= f;
                *(uint32_t *)(dst + d) = kv8_encode<F>(v);
            }
        }
        if (tid == 0) *scale = s;
    }
}

template <typename TI, typename TQ, uint32_t F, int HD>
__global__ __launch_bounds__(2 * HD) void k_kv8_write(Kv8Write a) {
    constexpr uint32_t L = HD / 8, NS = 16, T = 2 * HD;  // lanes of a head vector, vectors of a workgroup
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < a.kv_blocks) {
        const uint32_t per = 2 * a.groups, u = a.unit0 + blockIdx.x / per, g = blockIdx.x % per;
        if (blockIdx.x == 0 && a.unit0 == 0) {  // the rows' description, checked once
            uint32_t bad = 0;
            for (uint32_t s = tid; s < a.n_seq; s += T) {
                const Kv8Seq x = kv8_seq(a.row_start, a.seq_lens, s, a.n_rows, bad);
                if (x.n && (x.len - 1) / 16 >= a.stride) bad = 1;
            }
            if (bad) atomicOr(a.err, ZH_DEVERR_KV_ROW);
        }
        uint32_t s = u, page;
        Kv8Seq seq;
        if (!a.row_start) {
            uint32_t bad;
            if (u >= a.n_seq) return;
            seq = kv8_seq(nullptr, a.seq_lens, u, a.n_rows, bad);
            if (!seq.n) return;
            page = 0;
        } else {
            uint32_t bad;
            auto pages = [&](uint32_t i) {
                const Kv8Seq x = kv8_seq(a.row_start, a.seq_lens, i, a.n_rows, bad);
                return x.n ? (x.len - 1) / 16 - x.pos / 16 + 1 : 0u;
            };
            if (!kv8_find(a.n_seq, u, pages, s, page)) return;
            seq = kv8_seq(a.row_start, a.seq_lens, s, a.n_rows, bad);
        }
        page += seq.pos / 16;
        if (page >= a.stride) return;
        const uint32_t phys = a.tables[(size_t)s * a.stride + page];
        if (phys >= a.cache_tokens / 16) {
            if (tid == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
            return;
        }
        const uint32_t h0 = g % a.groups * a.hpb, n = min(a.hpb, a.nkv - h0);
        if (g < a.groups) write_heads<TI, F, HD, true>(a, seq, page, phys, h0, n);
        else write_heads<TI, F, HD, false>(a, seq, page, phys, h0, n);
        return;
    }
    // ---- q: NS heads of one row at a time
    __shared__ float2 cs[HD / 2];
    const uint32_t b = blockIdx.x - a.kv_blocks, t = a.unit0 + b / a.q_groups, l = tid % L;
    Kv8Seq seq;
    uint32_t pos = 0;
    if (!a.row_start) {
        uint32_t bad;
        seq = kv8_seq(nullptr, a.seq_lens, t, a.n_rows, bad);
        if (!seq.n) return;
        pos = seq.pos;
    } else {
        bool found = false;  // the sequence with row t
        for (uint32_t s0 = 0; s0 < a.n_seq && !found; s0 += 64) {
            uint32_t bad = 0;
            Kv8Seq x = {0, 0, 0, 0};
            if (s0 + tid % 64 < a.n_seq) x = kv8_seq(a.row_start, a.seq_lens, s0 + tid % 64, a.n_rows, bad);
            const uint64_t hit = __builtin_amdgcn_ballot_w64(t >= x.row && t - x.row < x.n);
            if (hit) {
                const uint32_t k = __builtin_ctzll(hit);
                pos = __builtin_amdgcn_readlane(x.pos, k) + (t - __builtin_amdgcn_readlane(x.row, k));
                found = true;
            }
        }
        if (!found) return;
    }
    uint32_t lo, hi;
    const bool rot = quads(l, a.rd, lo, hi);
    if (a.rd) {  // (uniform)
        for (uint32_t i = tid; i < a.rd / 2; i += T)
            sincospif(2.0f * (float)turns(pos, a.inv_freq[i]), &cs[i].y, &cs[i].x);
        __syncthreads();
    }
    float co[4] = {}, sn[4] = {}, w0[4] = {1.f, 1.f, 1.f, 1.f}, w1[4] = {1.f, 1.f, 1.f, 1.f};
    if (rot)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            co[e] = cs[4 * l + e].x;
            sn[e] = cs[4 * l + e].y;
        }
    if (a.qw) {
        ld4(a.qw + lo, w0);
        ld4(a.qw + hi, w1);
    }
    const uint8_t *src = a.q + t * a.q_row;
    uint8_t *out = a.q_out + t * a.out_row;
    for (uint32_t h0 = b % a.q_groups * NS; h0 < a.nq; h0 += a.q_groups * NS) {
        const uint32_t h = min(h0 + tid / L, a.nq - 1);
        float x[4], y[4];
        ld4((const TI *)src + h * HD + lo, x);
        ld4((const TI *)src + h * HD + hi, y);
        if (a.qw) {
            float sq = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) sq = fmaf(x[e], x[e], fmaf(y[e], y[e], sq));
            const float ri = 1.0f / sqrtf(team_sum_dpp<L>(sq) / (float)HD + a.eps);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = w0[e] * (x[e] * ri);
                y[e] = w1[e] * (y[e] * ri);
            }
        }
        if (rot)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p = x[e], q = y[e];
                x[e] = p * co[e] - q * sn[e];
                y[e] = p * sn[e] + q * co[e];
            }
        if (h0 + tid / L >= a.nq) continue;
        st4((TQ *)out + h * HD + lo, x);
        st4((TQ *)out + h * HD + hi, y);
    }
}

}  // namespace

// The checks of zh_qk_norm_rope_kv8_write_batched, of host data only (exported
// for the tests; c may be null: no message then).
extern "C" int zh_check_kv8_rows(zh_ctx *c, const zh_kv8_batch *kv, const zh_qkv_rows *rows) {
    const char *who = "qk_norm_rope_kv8 batch";
    if (!rows || !kv8_batch_ok(kv, rows->n_rows))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: caches, tables or rows of the batch", who);
    if (!kv8_type_ok(kv->type)) return zh_set_err(c, ZH_ERR_UNSUPPORTED_QUANT_TYPE, "%s: cache type %u", who, kv->type);
    if (rows->seq || rows->pos)
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: seq and pos come from the batch", who);
    const zh_qkv_rows x = kv_with_strides(rows, kv->n_kv_heads, kv->head_dim), *r = &x;
    const zh_buf *const written[] = {kv->k_cache, kv->v_cache, kv->k_scale, kv->v_scale};
    const zh_buf *const read[] = {kv->tables, kv->row_start, kv->seq_lens};
    const int rc = kv_check_rows(c, who, r, kv->n_kv_heads, kv->head_dim, written, 4, read, 3);
    if (rc || r->n_rows == 0) return rc;
    if (r->rope_dim % 8) return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: rope_dim %u", who, r->rope_dim);
    const uint64_t si = r->type == ZH_F32 ? 4 : 2, so = r->q_out_type == ZH_F32 ? 4 : 2;
    if ((r->q_off | r->k_off | r->v_off | r->q_out_off) % 16 ||
        (r->n_rows > 1 && ((r->q_stride * si) | (r->k_stride * si) | (r->v_stride * si) | (r->q_out_stride * so)) % 16))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: rows not 16-byte aligned", who);
    return ZH_OK;
}

template <typename TI, typename TQ, uint32_t F, int HD>
static int kv8_write_launch(zh_ctx *c, const Kv8Write &a, uint64_t units) {
    // the pages and rows that a launch of fewer than 2^32 threads takes
    const uint64_t per = 2ull * a.groups + a.q_groups, most = std::max<uint64_t>((1ull << 23) / per, 1);
    for (uint64_t u0 = 0; u0 < units || u0 < a.n_rows; u0 += most) {
        Kv8Write b = a;
        b.unit0 = (uint32_t)u0;
        const uint64_t n = u0 < units ? std::min(units - u0, most) : 0, r = u0 < a.n_rows ? std::min(a.n_rows - u0, most) : 0;
        b.kv_blocks = (uint32_t)(n * 2 * a.groups);
        hipLaunchKernelGGL((k_kv8_write<TI, TQ, F, HD>), dim3((uint32_t)(b.kv_blocks + r * a.q_groups)), dim3(2 * HD), 0,
                           c->stream, b);
        ZH_LAUNCH_CHECK(c);
    }
    return ZH_OK;
}

template <typename TI, typename TQ>
static int kv8_write_type(zh_ctx *c, const Kv8Write &a, uint64_t units, uint32_t type, uint32_t hd) {
    if (type == ZH_I8)
        return hd == 128 ? kv8_write_launch<TI, TQ, ZH_I8, 128>(c, a, units) : kv8_write_launch<TI, TQ, ZH_I8, 64>(c, a, units);
    return hd == 128 ? kv8_write_launch<TI, TQ, ZH_E4M3, 128>(c, a, units) : kv8_write_launch<TI, TQ, ZH_E4M3, 64>(c, a, units);
}

extern "C" int zh_qk_norm_rope_kv8_write_batched(zh_ctx *c, const zh_kv8_batch *kv, const zh_qkv_rows *rows) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    const int rc = zh_check_kv8_rows(c, kv, rows);
    if (rc || rows->n_rows == 0) return rc;
    const zh_qkv_rows x = kv_with_strides(rows, kv->n_kv_heads, kv->head_dim), *r = &x;
    zh_device_scope dev(c);
    const uint32_t si = r->type == ZH_F32 ? 4 : 2, so = r->q_out_type == ZH_F32 ? 4 : 2;
    Kv8Write a = {};
    a.q = (const uint8_t *)r->q->ptr + r->q_off;
    a.k = (const uint8_t *)r->k->ptr + r->k_off;
    a.v = (const uint8_t *)r->v->ptr + r->v_off;
    a.q_out = (uint8_t *)r->q_out->ptr + r->q_out_off;
    a.q_row = (uint64_t)r->q_stride * si;
    a.k_row = (uint64_t)r->k_stride * si;
    a.v_row = (uint64_t)r->v_stride * si;
    a.out_row = (uint64_t)r->q_out_stride * so;
    a.qw = r->q_norm_w ? (const float *)r->q_norm_w->ptr : nullptr;
    a.kw = r->k_norm_w ? (const float *)r->k_norm_w->ptr : nullptr;
    a.inv_freq = r->rope_dim ? (const float *)r->inv_freq->ptr : nullptr;
    a.kc = (uint8_t *)kv->k_cache->ptr;
    a.vc = (uint8_t *)kv->v_cache->ptr;
    a.ks = (float *)kv->k_scale->ptr;
    a.vs = (float *)kv->v_scale->ptr;
    a.tables = (const uint32_t *)kv->tables->ptr;
    a.row_start = kv->row_start ? (const uint32_t *)kv->row_start->ptr : nullptr;
    a.seq_lens = (const uint32_t *)kv->seq_lens->ptr;
    a.err = c->err_dev;
    a.n_seq = kv->n_seq;
    a.stride = kv->table_stride;
    a.cache_tokens = kv->cache_tokens;
    a.nq = r->n_q_heads;
    a.nkv = kv->n_kv_heads;
    a.rd = r->rope_dim;
    a.n_rows = r->n_rows;
    a.eps = r->eps;
    // pages that rows reach: a sequence of n rows at most (n + 30) / 16, and n
    const uint64_t units = a.row_start ? std::min<uint64_t>((a.n_rows + 30ull * a.n_seq) / 16, a.n_rows) : a.n_rows;
    a.hpb = 1;
    a.groups = (a.nkv + a.hpb - 1) / a.hpb;
    a.q_groups = (a.nq + 15) / 16;
    if (si == 4)
        return so == 4 ? kv8_write_type<float, float>(c, a, units, kv->type, kv->head_dim)
                       : kv8_write_type<float, _Float16>(c, a, units, kv->type, kv->head_dim);
    return so == 4 ? kv8_write_type<_Float16, float>(c, a, units, kv->type, kv->head_dim)
                   : kv8_write_type<_Float16, _Float16>(c, a, units, kv->type, kv->head_dim);
}

// ---------------------------------------------------------------------------
// Pages quantised (pack), read back (unpack) and copied. A wave takes one page of
// one cache and head, all of it in registers: the block's largest value is a
// reduction over the wave, no LDS and no barrier. Bound by HBM.
// ---------------------------------------------------------------------------
namespace {

// NC caches and NP pages (numbers of type P) per launch, in 4 KB of arguments.
template <typename P, uint32_t NC, uint32_t NP>
struct Kv8PageArgs {
    typedef P Page;
    static constexpr uint32_t caches = NC, n = NP;
    const uint8_t *src[NC];
    uint8_t *dst[NC];
    const float *src_scale[NC];
    float *dst_scale[NC];
    uint64_t src_tokens, dst_tokens;
    uint32_t n_pages, nkv;
    uint32_t last;  // tokens of page n_pages - 1
    P pages[NP][2];  // source, destination
};

template <uint32_t F, int HD, typename A>
__global__ __launch_bounds__(256) void k_kv8_pack(A a) {
    constexpr int N = 16 * HD / 512;  // 16-byte pieces of a lane
    const uint32_t p = blockIdx.x * 4 + threadIdx.x / 64, h = blockIdx.y, c = blockIdx.z, lane = threadIdx.x % 64;
    if (p >= a.n_pages) return;
    const u32x4 *s = (const u32x4 *)(a.src[c] + (h * a.src_tokens + (uint64_t)a.pages[p][0] * 16) * (2 * HD));
    u32x2 *d = (u32x2 *)(a.dst[c] + (h * a.dst_tokens + (uint64_t)a.pages[p][1] * 16) * HD);
    half8 x[N];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = __builtin_bit_cast(half8, __builtin_nontemporal_load(s + 64 * i + lane));
    if (p == a.n_pages - 1) {
#pragma unroll
        for (int i = 0; i < N; i++)
            if ((64 * i + lane) * 8 / HD >= a.last) x[i] = half8{};
    }
    int t = KV8_LOW;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) t = max(t, kv8_exp<F>((float)x[i][e]));
#pragma unroll
    for (int k = 1; k < 64; k *= 2) t = max(t, __shfl_xor(t, k, 64));
    const bool nan = t == KV8_NAN;
    const float inv = nan ? 0.f : kv8_pow2(-t);
#pragma unroll
    for (int i = 0; i < N; i++) {
        float v0[4], v1[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v0[e] = nan ? 0.f : (float)x[i][e] * inv;
            v1[e] = nan ? 0.f : (float)x[i][e + 4] * inv;
        }
        __builtin_nontemporal_store(u32x2{kv8_encode<F>(v0), kv8_encode<F>(v1)}, d + 64 * i + lane);
    }
    if (lane == 0) a.dst_scale[c][(uint64_t)a.pages[p][1] * a.nkv + h] = nan ? NAN : kv8_pow2(t);
}

template <uint32_t F, int HD, typename A>
__global__ __launch_bounds__(256) void k_kv8_unpack(A a) {
    constexpr int N = 16 * HD / 512;  // 8-byte pieces of a lane
    const uint32_t p = blockIdx.x * 4 + threadIdx.x / 64, h = blockIdx.y, c = blockIdx.z, lane = threadIdx.x % 64;
    if (p >= a.n_pages) return;
    const u32x2 *s = (const u32x2 *)(a.src[c] + (h * a.src_tokens + (uint64_t)a.pages[p][0] * 16) * HD);
    u32x4 *d = (u32x4 *)(a.dst[c] + (h * a.dst_tokens + (uint64_t)a.pages[p][1] * 16) * (2 * HD));
    float scale = a.src_scale[c][(uint64_t)a.pages[p][0] * a.nkv + h];
    u32x2 x[N];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = __builtin_nontemporal_load(s + 64 * i + lane);
    scale = kv8_scale_ok(__float_as_uint(scale)) ? scale : NAN;
#pragma unroll
    for (int i = 0; i < N; i++) {
        float v0[4], v1[4];
        kv8_decode<F>(x[i].x, v0);
        kv8_decode<F>(x[i].y, v1);
        half8 y;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e] = (_Float16)(v0[e] * scale);
            y[e + 4] = (_Float16)(v1[e] * scale);
        }
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, y), d + 64 * i + lane);
    }
}

// The scales of copied pages (their codes go as half as many fp16 dims do).
template <typename A>
__global__ __launch_bounds__(256) void k_kv8_scales(A a) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t p = (uint32_t)(i / a.nkv), h = (uint32_t)(i % a.nkv), c = blockIdx.z;
    if (p >= a.n_pages) return;
    a.dst_scale[c][(uint64_t)a.pages[p][1] * a.nkv + h] = a.src_scale[c][(uint64_t)a.pages[p][0] * a.nkv + h];
}

enum class Pages { pack, unpack, scales };

// What a call's launches take: the caches' addresses (NULL: not there).
struct Kv8Move {
    void *const *dst;
    const void *const *src;
    void *const *dst_scale;
    const void *const *src_scale;
    uint32_t n_caches, dst_tokens, src_tokens, nkv, hd, type;
    const uint32_t *dst_pages, *src_pages;
    uint32_t n_pages, last;
};

template <Pages OP, uint32_t F, int HD, typename A>
int kv8_page_launches(zh_ctx *c, const Kv8Move &m) {
    static_assert(sizeof(A) <= 4096, "kernel arguments");
    A a = {};
    a.src_tokens = m.src_tokens;
    a.dst_tokens = m.dst_tokens;
    a.nkv = m.nkv;
    for (uint32_t c0 = 0; c0 < m.n_caches; c0 += A::caches) {
        const uint32_t nc = std::min(m.n_caches - c0, A::caches);
        for (uint32_t i = 0; i < nc; i++) {
            if (m.src) a.src[i] = (const uint8_t *)m.src[c0 + i];
            if (m.dst) a.dst[i] = (uint8_t *)m.dst[c0 + i];
            if (m.src_scale) a.src_scale[i] = (const float *)m.src_scale[c0 + i];
            if (m.dst_scale) a.dst_scale[i] = (float *)m.dst_scale[c0 + i];
        }
        for (uint32_t p0 = 0; p0 < m.n_pages; p0 += A::n) {
            a.n_pages = std::min(m.n_pages - p0, A::n);
            a.last = p0 + a.n_pages == m.n_pages ? m.last : 16u;
            for (uint32_t i = 0; i < a.n_pages; i++) {
                a.pages[i][0] = (typename A::Page)m.src_pages[p0 + i];
                a.pages[i][1] = (typename A::Page)m.dst_pages[p0 + i];
            }
            const dim3 grid((a.n_pages + 3) / 4, m.nkv, nc);
            if constexpr (OP == Pages::pack)
                hipLaunchKernelGGL((k_kv8_pack<F, HD, A>), grid, dim3(256), 0, c->stream, a);
            else if constexpr (OP == Pages::unpack)
                hipLaunchKernelGGL((k_kv8_unpack<F, HD, A>), grid, dim3(256), 0, c->stream, a);
            else
                hipLaunchKernelGGL((k_kv8_scales<A>), dim3((uint32_t)(((uint64_t)a.n_pages * m.nkv + 255) / 256), 1, nc),
                                   dim3(256), 0, c->stream, a);
            ZH_LAUNCH_CHECK(c);
        }
    }
    return ZH_OK;
}

// The lists that fit the call in few launches; few pages take short arguments,
// which the host writes sooner.
template <Pages OP, uint32_t F, int HD>
int kv8_pages_list(zh_ctx *c, const Kv8Move &m) {
    if (m.n_pages <= 16) return kv8_page_launches<OP, F, HD, Kv8PageArgs<uint32_t, 64, 16>>(c, m);
    if (m.dst_tokens > 16u << 16 || m.src_tokens > 16u << 16)  // (page numbers past 16 bits)
        return kv8_page_launches<OP, F, HD, Kv8PageArgs<uint32_t, 32, 370>>(c, m);
    return kv8_page_launches<OP, F, HD, Kv8PageArgs<uint16_t, 32, 750>>(c, m);
}
template <Pages OP>
int kv8_pages(zh_ctx *c, const Kv8Move &m) {
    if (m.type == ZH_I8)
        return m.hd == 128 ? kv8_pages_list<OP, ZH_I8, 128>(c, m) : kv8_pages_list<OP, ZH_I8, 64>(c, m);
    return m.hd == 128 ? kv8_pages_list<OP, ZH_E4M3, 128>(c, m) : kv8_pages_list<OP, ZH_E4M3, 64>(c, m);
}

bool kv8_caches_ok(const zh_kv8_caches *s) {
    if (!s || !s->caches || !s->scales || s->n_caches == 0 || s->n_caches > KC_MAX || s->n_kv_heads == 0 ||
        s->n_kv_heads > 65535 || (s->head_dim != 64 && s->head_dim != 128) || s->cache_tokens == 0 || s->cache_tokens % 16)
        return false;
    for (uint32_t i = 0; i < s->n_caches; i++)
        if (!kv_in_range(s->caches[i], 0, (uint64_t)s->n_kv_heads * s->cache_tokens * s->head_dim) ||
            !kv_in_range(s->scales[i], 0, 4ull * s->n_kv_heads * (s->cache_tokens / 16)))
            return false;
    return true;
}

// Buffers by address, in a small hash table (comparing every pair would take longer
// than a call's pages).
struct BufTab {
    const void *p[4 * KC_MAX];
    uint16_t tab[8 * KC_MAX] = {};
    uint32_t n = 0;
    bool add(const zh_buf *b) {  // false: it is there
        uint32_t i = (uint32_t)(((uint64_t)(uintptr_t)b->ptr * 0x9E3779B97F4A7C15ull) >> 53);
        while (tab[i]) {
            if (p[tab[i] - 1] == b->ptr) return false;
            i = (i + 1) % (8 * KC_MAX);
        }
        p[n] = b->ptr;
        tab[i] = (uint16_t)++n;
        return true;
    }
};

}  // namespace

// The checks of the three, of host data only (exported for the tests; c may be
// null: no message then). op 0: pack (dst8, src16), 1: unpack (dst16, src8), 2: copy
// (dst8, src8).
extern "C" int zh_check_kv8_pages(zh_ctx *c, uint32_t op, const zh_kv8_caches *dst8, const zh_kv8_caches *src8,
                                  const zh_kv_caches *half, const uint32_t *dst_pages, const uint32_t *src_pages,
                                  uint32_t n_pages) {
    const char *const who = op == 0 ? "kv8_pack_pages" : op == 1 ? "kv8_unpack_pages" : "kv8_copy_pages";
    const zh_kv8_caches *s8 = op == 0 ? dst8 : src8;
    if (!kv8_caches_ok(s8) || (op == 2 ? !kv8_caches_ok(dst8) : !kv_caches_ok(half)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: cache sets", who);
    if (!kv8_type_ok(s8->type)) return zh_set_err(c, ZH_ERR_UNSUPPORTED_QUANT_TYPE, "%s: cache type %u", who, s8->type);
    const uint32_t n = s8->n_caches;
    const bool alike = op == 2 ? dst8->n_caches == n && dst8->n_kv_heads == s8->n_kv_heads &&
                                     dst8->head_dim == s8->head_dim && dst8->type == s8->type
                               : half->n_caches == n && half->n_kv_heads == s8->n_kv_heads && half->head_dim == s8->head_dim;
    if (!alike) return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: sets of other shapes", who);
    if (n_pages && (!dst_pages || !src_pages))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: no page numbers", who);
    // one set copied within itself, or every buffer in one place
    bool alias = op == 2 && dst8->cache_tokens == src8->cache_tokens;
    for (uint32_t i = 0; i < n && alias; i++)
        alias = dst8->caches[i]->ptr == src8->caches[i]->ptr && dst8->scales[i]->ptr == src8->scales[i]->ptr;
    BufTab tab;
    bool once = true;
    for (uint32_t i = 0; i < n; i++) {
        once = once && tab.add(s8->caches[i]) && tab.add(s8->scales[i]);
        if (op == 2) once = once && (alias || (tab.add(dst8->caches[i]) && tab.add(dst8->scales[i])));
        else once = once && tab.add(half->caches[i]);
    }
    if (!once) return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "%s: a buffer in two places", who);
    const uint32_t dp = (op == 1 ? half->cache_tokens : dst8->cache_tokens) / 16;
    const uint32_t sp = (op == 0 ? half->cache_tokens : src8->cache_tokens) / 16;
    return kv_check_pages(c, who, dst_pages, src_pages, n_pages, dp, sp, alias);
}

namespace {
struct Ptrs {
    void *p[KC_MAX];
    Ptrs(zh_buf *const *b, uint32_t n) {
        for (uint32_t i = 0; i < n; i++) p[i] = b[i]->ptr;
    }
};
}  // namespace

extern "C" int zh_kv8_pack_pages(zh_ctx *c, const zh_kv8_caches *dst, const zh_kv_caches *src, const uint32_t *dst_pages,
                                 const uint32_t *src_pages, uint32_t n_tokens) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    const uint32_t n = n_tokens / 16 + (n_tokens % 16 != 0);
    const int rc = zh_check_kv8_pages(c, 0, dst, nullptr, src, dst_pages, src_pages, n);
    if (rc || !n) return rc;
    zh_device_scope dev(c);
    const Ptrs d(dst->caches, dst->n_caches), ds(dst->scales, dst->n_caches), s(src->caches, dst->n_caches);
    const Kv8Move m = {d.p, s.p, ds.p, nullptr, dst->n_caches, dst->cache_tokens, src->cache_tokens, dst->n_kv_heads,
                       dst->head_dim, dst->type, dst_pages, src_pages, n, n_tokens - 16 * (n - 1)};
    return kv8_pages<Pages::pack>(c, m);
}

extern "C" int zh_kv8_unpack_pages(zh_ctx *c, const zh_kv_caches *dst, const zh_kv8_caches *src, const uint32_t *dst_pages,
                                   const uint32_t *src_pages, uint32_t n_pages) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    const int rc = zh_check_kv8_pages(c, 1, nullptr, src, dst, dst_pages, src_pages, n_pages);
    if (rc || !n_pages) return rc;
    zh_device_scope dev(c);
    const Ptrs d(dst->caches, src->n_caches), s(src->caches, src->n_caches), ss(src->scales, src->n_caches);
    const Kv8Move m = {d.p, s.p, nullptr, ss.p, src->n_caches, dst->cache_tokens, src->cache_tokens, src->n_kv_heads,
                       src->head_dim, src->type, dst_pages, src_pages, n_pages, 16};
    return kv8_pages<Pages::unpack>(c, m);
}

extern "C" int zh_kv8_copy_pages(zh_ctx *c, const zh_kv8_caches *dst, const zh_kv8_caches *src, const uint32_t *dst_pages,
                                 const uint32_t *src_pages, uint32_t n_pages) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    int rc = zh_check_kv8_pages(c, 2, dst, src, nullptr, dst_pages, src_pages, n_pages);
    if (rc || !n_pages) return rc;
    zh_device_scope dev(c);
    const uint32_t n = src->n_caches;
    const Ptrs d(dst->caches, n), s(src->caches, n), ds(dst->scales, n), ss(src->scales, n);
    rc = zhk_kv_copy(c, n, d.p, s.p, dst->cache_tokens, src->cache_tokens, src->n_kv_heads, src->head_dim / 2, dst_pages,
                     src_pages, n_pages);
    if (rc) return rc;
    const Kv8Move m = {nullptr, nullptr, ds.p, ss.p, n, dst->cache_tokens, src->cache_tokens, src->n_kv_heads,
                       src->head_dim, src->type, dst_pages, src_pages, n_pages, 16};
    return kv8_pages_list<Pages::scales, ZH_I8, 64>(c, m);
}
