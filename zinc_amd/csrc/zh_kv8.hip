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
// does not then depend on the order of 32-bit sums, and tokens written in the same steps
// leave the same cache whichever form takes them and whatever else is in their calls. (In
// other steps the scales are the same at the end, not every code: see zh_kv8.h.) That is some
// 30 operations for each element of k beside its loads, 6 us of all vector units for 8192
// rows of 8 heads.
//
// Two forms. Sequences with several rows: a workgroup takes one page of one sequence
// and some heads of q, k or v: thread (slot, l) holds slot `slot` of the page and 8
// dims, the angles of its four pairs are taken once for all its heads, a block's largest
// value is a reduction over the workgroup, and the page's old tokens, where the scale
// rises, are there to be rounded again. One row a sequence (a decode step): 16 head
// vectors of a row a workgroup, each on 16 (8) lanes, which reach for the page's other
// slots themselves where the scale rises; in the first form 15 of 16 threads would idle
// (250 rows of 8 heads 12.8 us, 5.3 so).
// 8192 rows of 32 + 16 heads of 128 in f16 (100 MB read, 84 written) 44 us, 4.2 TB/s: vector
// instructions issue in 86% of the cycles, and waves wait for 43% of theirs. A decode step of
// 61 sequences 4.7 us: a chain of loads, length, page, scale and rows, and a launch.
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
    uint32_t q_heads, kv_heads;    // heads of a workgroup
    uint32_t q_groups, kv_groups;  // workgroups of a page's (a row's) q, of its k (and of its v)
    uint32_t unit0;           // pages (rows) before this launch's
    float eps;
};

// four elements as they are, and as floats
template <typename T>
struct Quad {
    typedef T V __attribute__((ext_vector_type(4)));
    V v;
    ZH_DEVM void load(const T *p) { v = *(const V *)p; }
    ZH_DEVM void load_once(const T *p) { v = __builtin_nontemporal_load((const V *)p); }
    template <typename S>
    ZH_DEVM void get(S (&x)[4]) const {
        x[0] = (S)v.x;
        x[1] = (S)v.y;
        x[2] = (S)v.z;
        x[3] = (S)v.w;
    }
};
template <typename T>
ZH_DEV void ld4(const T *p, float (&x)[4]) {
    Quad<T> q;
    q.load(p);
    q.get(x);
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

enum class Part { q, k, v };

// Normalises and rotates the two quads of a lane's dims of one head (k: in 64 bits).
template <typename V, int L>
ZH_DEV void turned(V (&x)[4], V (&y)[4], bool norm, const float (&w0)[4], const float (&w1)[4], float eps, bool rot,
                   const V (&co)[4], const V (&sn)[4]) {
    if (norm) {  // (uniform; all lanes take part in the sum)
        V sq = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) sq = fma(x[e], x[e], fma(y[e], y[e], sq));
        V ri;
        if constexpr (sizeof(V) == 8) ri = 1.0 / sqrt(team_sum64<L>(sq) / (8 * L) + (double)eps);
        else ri = 1.0f / sqrtf(team_sum_dpp<L>(sq) / (float)(8 * L) + eps);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] = w0[e] * (x[e] * ri);
            y[e] = w1[e] * (y[e] * ri);
        }
    }
    if (rot)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const V p = x[e], q = y[e];
            x[e] = p * co[e] - q * sn[e];
            y[e] = p * sn[e] + q * co[e];
        }
}

// The larger of a block's own scale (its bits; begun: it has none) and 2^t.
ZH_DEV float block_scale(int t, uint32_t own, bool begun) {
    if (t == KV8_NAN || (!begun && !kv8_scale_ok(own))) return NAN;
    const float s = kv8_pow2(t);
    return !begun && s < __uint_as_float(own) ? __uint_as_float(own) : s;
}
// The largest magnitude of two quads as kv8_exp takes it.
template <uint32_t F, typename V>
ZH_DEV int quads_exp(const V (&x)[4], const V (&y)[4]) {
    V most = 0, sum = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const V p = x[e] < 0 ? -x[e] : x[e], q = y[e] < 0 ? -y[e] : y[e];
        most = fmax(most, fmax(p, q));
        sum += p + q;
    }
    return kv8_exp<F>(most, sum);
}
template <uint32_t F, typename V>
ZH_DEV uint32_t code4(V (&x)[4], float s, float inv) {
    if (s != s) return 0;
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] *= inv;
    return kv8_encode<F>(x);
}
template <uint32_t F>
ZH_DEV uint32_t recode(uint32_t c, float f) {
    float v[4];
    kv8_decode<F>(c, v);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= f;
    return kv8_encode<F>(v);
}

// Heads [h0, h0 + n) of q, k or v in the slots of one page (phys; q: of its tokens), B
// at a time: the next ones' loads are on the way while these are worked on (a lane's
// loads are 8 bytes an fp16 head: with one head on the way 20 waves of a CU have 20 KB
// in flight, a quarter of what HBM takes to stay busy), and one barrier serves B
// reductions. The rows go by the caches, which keep what is read next, q_out and the
// codes (8192 rows 46.0 us for 44.5; those gone by too, 43.4).
template <typename TI, typename TQ, uint32_t F, int HD, Part P>
ZH_DEV void page_heads(const Kv8Write &a, const Kv8Seq &seq, uint32_t page, uint32_t phys, uint32_t h0, uint32_t n) {
    constexpr int L = HD / 8, NW = L / 4, B = P == Part::k ? 2 : 4;  // lanes of a row, waves
    using V = typename std::conditional<P == Part::k, double, float>::type;
    __shared__ int top[2][B][NW];
    const uint32_t tid = threadIdx.x, l = tid % L, slot = tid / L, pos = page * 16 + slot;
    const bool mine = pos >= seq.pos && pos < seq.len, begun = page * 16 >= seq.pos;
    uint32_t lo = 8 * l, hi = 8 * l + 4;
    bool rot = false;
    if (P != Part::v) rot = quads(l, a.rd, lo, hi);
    const uint32_t row = seq.row + (mine ? pos - seq.pos : 0u);
    const uint8_t *base = P == Part::q ? a.q + row * a.q_row : P == Part::k ? a.k + row * a.k_row : a.v + row * a.v_row;
    const TI *src = (const TI *)base + (size_t)h0 * HD;
    Quad<TI> r0[B] = {}, r1[B] = {};
    auto load = [&](uint32_t i) __attribute__((always_inline)) {
        if (mine)
#pragma unroll
            for (uint32_t j = 0; j < B; j++)
                if (i + j < n) {
                    r0[j].load_once(src + (i + j) * HD + lo);
                    r1[j].load_once(src + (i + j) * HD + hi);
                }
    };
    load(0);
    V co[4] = {}, sn[4] = {};
    float w0[4] = {1.f, 1.f, 1.f, 1.f}, w1[4] = {1.f, 1.f, 1.f, 1.f};
    const float *w = P == Part::q ? a.qw : a.kw;
    if constexpr (P != Part::v) {
        if (w) {
            ld4(w + lo, w0);
            ld4(w + hi, w1);
        }
        if (rot && mine) {
            float f[4];
            ld4(a.inv_freq + 4 * l, f);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (P == Part::k) sincospi(2.0 * turns(pos, f[e]), &sn[e], &co[e]);
                else sincospif(2.0f * (float)turns(pos, f[e]), &sn[e], &co[e]);
            }
        }
    }
    uint8_t *dst = (P == Part::k ? a.kc : a.vc) + ((size_t)h0 * a.cache_tokens + phys * 16 + slot) * HD;
    float *scale = (P == Part::k ? a.ks : a.vs) + (size_t)phys * a.nkv + h0;
    TQ *out = (TQ *)(a.q_out + row * a.out_row) + (size_t)h0 * HD;
    for (uint32_t i = 0, par = 0; i < n; i += B, par ^= 1) {
        V y0[B][4], y1[B][4];
        uint32_t old[B];
#pragma unroll
        for (int j = 0; j < B; j++) {
            r0[j].get(y0[j]);
            r1[j].get(y1[j]);
            if (P != Part::q) old[j] = __float_as_uint(scale[min(i + j, n - 1)]);
        }
        load(i + B);  // (also where q_out is q: its own dims of other heads)
#pragma unroll
        for (int j = 0; j < B; j++) {
            if (i + j >= n) break;  // uniform
            if constexpr (P != Part::v) turned<V, L>(y0[j], y1[j], w != nullptr, w0, w1, a.eps, rot, co, sn);
            if constexpr (P == Part::q) {
                if (mine) {
                    st4(out + (i + j) * HD + lo, y0[j]);
                    st4(out + (i + j) * HD + hi, y1[j]);
                }
            } else {
                const int t = wave_max(mine ? quads_exp<F>(y0[j], y1[j]) : KV8_LOW);
                if (tid % 64 == 0) top[par][j][tid / 64] = t;
            }
        }
        if constexpr (P != Part::q) {
            lds_bar();  // (the round after the next writes these words, when all threads have passed the next one's)
#pragma unroll
            for (int j = 0; j < B; j++) {
                if (i + j >= n) break;  // uniform
                int t = top[par][j][0];
#pragma unroll
                for (int k = 1; k < NW; k++) t = max(t, top[par][j][k]);
                const float own = __uint_as_float(old[j]), s = block_scale(t, old[j], begun), inv = 1.0f / s;
                uint8_t *to = dst + (size_t)(i + j) * a.cache_tokens * HD;
                if (mine) {
                    *(uint32_t *)(to + lo) = code4<F>(y0[j], s, inv);
                    *(uint32_t *)(to + hi) = code4<F>(y1[j], s, inv);
                } else if (begun) {
                    *(uint32_t *)(to + lo) = 0;
                    *(uint32_t *)(to + hi) = 0;
                } else if (s != own && s == s) {
                    *(uint32_t *)(to + lo) = recode<F>(*(const uint32_t *)(to + lo), own * inv);
                    *(uint32_t *)(to + hi) = recode<F>(*(const uint32_t *)(to + hi), own * inv);
                }
                if (tid == 0) scale[i + j] = s;
            }
        }
    }
}

// The rows' description, checked once a call.
ZH_DEV void check_rows(const Kv8Write &a) {
    if (blockIdx.x || a.unit0) return;
    uint32_t bad = 0;
    for (uint32_t s = threadIdx.x; s < a.n_seq; s += blockDim.x) {
        const Kv8Seq x = kv8_seq(a.row_start, a.seq_lens, s, a.n_rows, bad);
        if (x.n && (x.len - 1) / 16 >= a.stride) bad = 1;
    }
    if (bad) atomicOr(a.err, ZH_DEVERR_KV_ROW);
}

// A page's heads.
template <typename TI, typename TQ, uint32_t F, int HD>
__global__ __launch_bounds__(2 * HD) void k_kv8_write(Kv8Write a) {
    const uint32_t per = a.q_groups + 2 * a.kv_groups, u = a.unit0 + blockIdx.x / per, g = blockIdx.x % per;
    check_rows(a);
    uint32_t s, page, bad;
    auto pages = [&](uint32_t i) {
        const Kv8Seq x = kv8_seq(a.row_start, a.seq_lens, i, a.n_rows, bad);
        return x.n ? (x.len - 1) / 16 - x.pos / 16 + 1 : 0u;
    };
    if (!kv8_find(a.n_seq, u, pages, s, page)) return;
    const Kv8Seq seq = kv8_seq(a.row_start, a.seq_lens, s, a.n_rows, bad);
    page += seq.pos / 16;
    if (g < a.q_groups) {
        page_heads<TI, TQ, F, HD, Part::q>(a, seq, page, 0, g * a.q_heads, min(a.q_heads, a.nq - g * a.q_heads));
        return;
    }
    if (page >= a.stride) return;
    const uint32_t phys = a.tables[(size_t)s * a.stride + page];
    if (phys >= a.cache_tokens / 16) {
        if (threadIdx.x == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
        return;
    }
    const uint32_t h0 = (g - a.q_groups) % a.kv_groups * a.kv_heads, n = min(a.kv_heads, a.nkv - h0);
    if (g - a.q_groups < a.kv_groups) page_heads<TI, TQ, F, HD, Part::k>(a, seq, page, phys, h0, n);
    else page_heads<TI, TQ, F, HD, Part::v>(a, seq, page, phys, h0, n);
}

// 16 head vectors of one row (q's heads, then k's and v's).
template <typename TI, typename TQ, uint32_t F, int HD>
__global__ __launch_bounds__(2 * HD) void k_kv8_rows(Kv8Write a) {
    constexpr uint32_t L = HD / 8;
    __shared__ double2 cs[HD / 2];
    const uint32_t tid = threadIdx.x, l = tid % L, H = a.nq + 2 * a.nkv;
    const uint32_t t = a.unit0 + blockIdx.x / a.q_groups, v = blockIdx.x % a.q_groups * 16 + tid / L, h = min(v, H - 1);
    const bool is_k = h >= a.nq && h < a.nq + a.nkv, is_v = h >= a.nq + a.nkv;
    const uint32_t hh = is_v ? h - a.nq - a.nkv : is_k ? h - a.nq : h;
    check_rows(a);
    uint32_t lo = 8 * l, hi = 8 * l + 4;
    bool rot = false;
    if (!is_v) rot = quads(l, a.rd, lo, hi);
    const TI *src = (const TI *)(is_v ? a.v + t * a.v_row : is_k ? a.k + t * a.k_row : a.q + t * a.q_row) + (size_t)hh * HD;
    Quad<TI> r0, r1;
    r0.load(src + lo);
    r1.load(src + hi);
    const uint32_t len = a.seq_lens[t], pos = len - 1;
    if (len == 0) return;
    // (a vector past the last: nothing stored)
    const bool kv = h >= a.nq && v < H;
    uint32_t phys = 0, old = 0;
    bool ok = kv && pos / 16 < a.stride;
    float *scale = nullptr;
    if (ok) {
        phys = a.tables[(size_t)t * a.stride + pos / 16];
        ok = phys < a.cache_tokens / 16;
        if (!ok && l == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
    }
    if (ok) {
        scale = (is_v ? a.vs : a.ks) + (size_t)phys * a.nkv + hh;
        old = __float_as_uint(*scale);
    }
    if (a.rd) {  // (uniform; a workgroup has a thread for each angle)
        if (tid < a.rd / 2) sincospi(2.0 * turns(pos, a.inv_freq[tid]), &cs[tid].y, &cs[tid].x);
        __syncthreads();
    }
    const float *w = is_k ? a.kw : a.qw;
    float w0[4] = {}, w1[4] = {};
    if (w && !is_v) {
        ld4(w + lo, w0);
        ld4(w + hi, w1);
    }
    int e;
    double x[4], y[4];
    if (h < a.nq) {
        float p[4], q[4], co[4], sn[4];
        r0.get(p);
        r1.get(q);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            co[i] = rot ? (float)cs[4 * l + i].x : 0.f;
            sn[i] = rot ? (float)cs[4 * l + i].y : 0.f;
        }
        turned<float, L>(p, q, w != nullptr, w0, w1, a.eps, rot, co, sn);
        if (v < H) {
            TQ *out = (TQ *)(a.q_out + t * a.out_row) + (size_t)hh * HD;
            st4(out + lo, p);
            st4(out + hi, q);
        }
        return;
    }
    r0.get(x);
    r1.get(y);
    if (is_k) {
        double co[4], sn[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            co[i] = rot ? cs[4 * l + i].x : 0.0;
            sn[i] = rot ? cs[4 * l + i].y : 0.0;
        }
        turned<double, L>(x, y, w != nullptr, w0, w1, a.eps, rot, co, sn);
    }
    e = team_max<L>(quads_exp<F>(x, y));
    if (!ok) return;
    const bool begun = pos % 16 == 0;
    const float own = __uint_as_float(old), s = block_scale(e, old, begun), inv = 1.0f / s;
    uint8_t *to = (is_v ? a.vc : a.kc) + ((size_t)hh * a.cache_tokens + phys * 16) * HD;
    const uint32_t c0 = code4<F>(x, s, inv), c1 = code4<F>(y, s, inv), slot = pos % 16;
    if (begun || (s != own && s == s)) {  // the page's other slots too: 0, or rounded again
        uint32_t o[16][2] = {};
        if (!begun)
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) {
                o[i][0] = *(const uint32_t *)(to + i * HD + lo);
                o[i][1] = *(const uint32_t *)(to + i * HD + hi);
            }
#pragma unroll
        for (uint32_t i = 0; i < 16; i++)
            if (i != slot) {
                *(uint32_t *)(to + i * HD + lo) = begun ? 0u : recode<F>(o[i][0], own * inv);
                *(uint32_t *)(to + i * HD + hi) = begun ? 0u : recode<F>(o[i][1], own * inv);
            }
    }
    *(uint32_t *)(to + slot * HD + lo) = c0;
    *(uint32_t *)(to + slot * HD + hi) = c1;
    if (l == 0) *scale = s;
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
    // the pages (rows) that a launch of fewer than 2^32 threads takes
    const uint64_t per = a.row_start ? 2ull * a.kv_groups + a.q_groups : a.q_groups, most = (1ull << 23) / per;
    for (uint64_t u0 = 0; u0 < units; u0 += most) {  // (per is below 2^18)
        Kv8Write b = a;
        b.unit0 = (uint32_t)u0;
        const dim3 grid((uint32_t)(std::min(units - u0, most) * per));
        if (a.row_start) hipLaunchKernelGGL((k_kv8_write<TI, TQ, F, HD>), grid, dim3(2 * HD), 0, c->stream, b);
        else hipLaunchKernelGGL((k_kv8_rows<TI, TQ, F, HD>), grid, dim3(2 * HD), 0, c->stream, b);
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
    // heads of a workgroup: the more of them, the fewer angles are taken and the more
    // loads are on the way. us at 4 heads of q and 1 of k (of v) / 8 and 2 / 16 and 4,
    // 32 + 16 heads of 128, f16: 100 rows 4.6 / 5.9 / 8.4, 333 6.0 / 6.8 / 8.7, 1000 11.8 /
    // 10.2 / 12.0, 2500 21.8 / 18.8 / 16.6, 8192 71 / 51 / 46; f32 8192 80 / 70 / 75 (for a floor of 58)
    const bool big = units >= 128 && si == 2;
    a.q_heads = units < 48 ? 4 : big ? 16 : 8;
    a.kv_heads = units < 48 ? 1 : big ? 4 : 2;
    a.kv_groups = (a.nkv + a.kv_heads - 1) / a.kv_heads;
    a.q_groups = a.row_start ? (a.nq + a.q_heads - 1) / a.q_heads : (a.nq + 2 * a.nkv + 15) / 16;
    if (si == 4)
        return so == 4 ? kv8_write_type<float, float>(c, a, units, kv->type, kv->head_dim)
                       : kv8_write_type<float, _Float16>(c, a, units, kv->type, kv->head_dim);
    return so == 4 ? kv8_write_type<_Float16, float>(c, a, units, kv->type, kv->head_dim)
                   : kv8_write_type<_Float16, _Float16>(c, a, units, kv->type, kv->head_dim);
}

// ---------------------------------------------------------------------------
// Pages quantised (pack), read back (unpack) and copied. A wave takes one page of
// one cache and head, all of it in registers: the block's largest value is a
// reduction over the wave, no LDS and no barrier. Bound by HBM: 16384 tokens of 16 caches
// read back 157 us, 5.1 TB/s (805 MB, two thirds of them written), 1000 tokens of 32 packed
// 18 us, 5.5 TB/s.
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
    for (int i = 0; i < N; i++) x[i] = __builtin_bit_cast(half8, s[64 * i + lane]);  // (a prompt's pages were just written)
    if (p == a.n_pages - 1) {
#pragma unroll
        for (int i = 0; i < N; i++)
            if ((64 * i + lane) * 8 / HD >= a.last) x[i] = half8{};
    }
    float most = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = fabsf((float)x[i][e]);
            most = fmaxf(most, v);
            sum += v;
        }
    const int t = wave_max(kv8_exp<F>(most, sum));
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
