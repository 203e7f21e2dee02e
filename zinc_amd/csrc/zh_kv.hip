// zh_kv.hip — operators over a paged KV cache for batches: page copies and
// the fused q/k RMSNorm + RoPE + KV write of many tokens.
#include <new>

#include "zh_device.h"
#include "zh_internal.h"
#include "zh_kv.h"

// ---------------------------------------------------------------------------
// Page copies. A page of one cache and head is 16 * head_dim halfs, contiguous
// (4 KB at head_dim 128): nothing is computed, the copy is bound by HBM (or by
// its launch for a few pages). The page numbers travel in the kernel arguments,
// so a call needs no staging memory, is finished with its host arrays when it
// returns and can be captured.
// ---------------------------------------------------------------------------
namespace {

// NC caches and NP pages (numbers of type P) per launch, in 4 KB of arguments.
template <typename P, uint32_t NC, uint32_t NP>
struct KvCopyArgs {
    typedef P Page;
    static constexpr uint32_t caches = NC, n = NP;
    const uint8_t *src[NC];
    uint8_t *dst[NC];
    uint64_t src_head, dst_head;  // bytes of one head of a cache
    uint32_t n_pages, seg;        // seg: bytes of a page of one head
    P pages[NP][2];               // source, destination
};

// One workgroup: KC_U pages of one head and cache, all loads before the stores.
constexpr int KC_U = 2;  // (4 and 8: the same times)
template <bool NT, int U, typename A>
ZH_DEV void kv_copy_pages(const A &a, uint32_t p0, const uint8_t *s, uint8_t *d) {
    for (uint32_t i = threadIdx.x; i < a.seg / 16; i += blockDim.x) {
        u32x4 v[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            const u32x4 *x = (const u32x4 *)(s + (uint64_t)a.pages[p0 + j][0] * a.seg) + i;
            v[j] = NT ? __builtin_nontemporal_load(x) : *x;
        }
#pragma unroll
        for (int j = 0; j < U; j++) {
            u32x4 *x = (u32x4 *)(d + (uint64_t)a.pages[p0 + j][1] * a.seg) + i;
            if (NT) __builtin_nontemporal_store(v[j], x);
            else *x = v[j];
        }
    }
}
template <bool NT, typename A>
__global__ __launch_bounds__(256) void k_kv_copy(A a) {
    const uint32_t p0 = blockIdx.x * KC_U, h = blockIdx.y, c = blockIdx.z;
    const uint8_t *s = a.src[c] + h * a.src_head;
    uint8_t *d = a.dst[c] + h * a.dst_head;
    if (p0 + KC_U <= a.n_pages) kv_copy_pages<NT, KC_U>(a, p0, s, d);
    else
        for (uint32_t p = p0; p < a.n_pages; p++) kv_copy_pages<NT, 1>(a, p, s, d);
}

template <typename A>
int kv_copy_launches(zh_ctx *c, uint32_t n_caches, void *const *dst, const void *const *src, uint32_t dst_tokens,
                     uint32_t src_tokens, uint32_t n_kv_heads, uint32_t head_dim, const uint32_t *dst_pages,
                     const uint32_t *src_pages, uint32_t n_pages) {
    static_assert(sizeof(A) <= 4096, "kernel arguments");
    A a;
    a.seg = 32 * head_dim;
    a.src_head = 2ull * src_tokens * head_dim;
    a.dst_head = 2ull * dst_tokens * head_dim;
    const uint32_t threads = a.seg >= 4096 ? 256u : (a.seg / 16 + 63) / 64 * 64;
    // past what the L2s hold, the pages go by them: 1024 pages of 32 caches of 8
    // heads 382 us (5.6 TB/s read + written) against 408 through them
    const bool nt = (uint64_t)n_caches * n_pages * n_kv_heads * a.seg > (32ull << 20);
    for (uint32_t c0 = 0; c0 < n_caches; c0 += A::caches) {
        const uint32_t nc = n_caches - c0 < A::caches ? n_caches - c0 : A::caches;
        for (uint32_t i = 0; i < nc; i++) {
            a.src[i] = (const uint8_t *)src[c0 + i];
            a.dst[i] = (uint8_t *)dst[c0 + i];
        }
        for (uint32_t p0 = 0; p0 < n_pages; p0 += A::n) {
            a.n_pages = n_pages - p0 < A::n ? n_pages - p0 : A::n;
            for (uint32_t i = 0; i < a.n_pages; i++) {
                a.pages[i][0] = (typename A::Page)src_pages[p0 + i];
                a.pages[i][1] = (typename A::Page)dst_pages[p0 + i];
            }
            const dim3 grid((a.n_pages + KC_U - 1) / KC_U, n_kv_heads, nc);
            if (nt) hipLaunchKernelGGL((k_kv_copy<true, A>), grid, dim3(threads), 0, c->stream, a);
            else hipLaunchKernelGGL((k_kv_copy<false, A>), grid, dim3(threads), 0, c->stream, a);
            ZH_LAUNCH_CHECK(c);
        }
    }
    return ZH_OK;
}

}  // namespace

int zhk_kv_copy(zh_ctx *c, uint32_t n_caches, void *const *dst, const void *const *src, uint32_t dst_tokens,
                uint32_t src_tokens, uint32_t n_kv_heads, uint32_t head_dim, const uint32_t *dst_pages,
                const uint32_t *src_pages, uint32_t n_pages) {
    // the lists that fit the call in the fewest launches: 2400 pages of two caches
    // of one head 16.7 us in three, 50.8 in ten of 256 pages; few pages take short
    // arguments, which the host writes sooner (one page of 64 caches 4.8 us, 6.0)
    auto f = kv_copy_launches<KvCopyArgs<uint32_t, 96, 256>>;
    if (n_pages <= 16) f = kv_copy_launches<KvCopyArgs<uint32_t, 64, 16>>;
    else if (dst_tokens > 16u << 16 || src_tokens > 16u << 16) {}  // (page numbers past 16 bits)
    else if (n_caches <= 4) f = kv_copy_launches<KvCopyArgs<uint16_t, 4, 960>>;
    else if (n_caches <= 64) f = kv_copy_launches<KvCopyArgs<uint16_t, 64, 720>>;
    else f = kv_copy_launches<KvCopyArgs<uint16_t, 96, 592>>;
    return f(c, n_caches, dst, src, dst_tokens, src_tokens, n_kv_heads, head_dim, dst_pages, src_pages, n_pages);
}

constexpr uint32_t KC_MAX = 256;  // caches of a call
static bool caches_ok(const zh_kv_caches *s) {
    if (!s || !s->caches || s->n_caches == 0 || s->n_caches > KC_MAX || s->n_kv_heads == 0 || s->n_kv_heads > 65535 || s->head_dim == 0 ||
        s->head_dim > 1024 || s->cache_tokens == 0 || s->cache_tokens % 16)
        return false;
    for (uint32_t i = 0; i < s->n_caches; i++)
        if (!kv_in_range(s->caches[i], 0, 2ull * s->n_kv_heads * s->cache_tokens * s->head_dim)) return false;
    return true;
}

// The checks of zh_kv_copy_pages, of host data only (exported for the tests; c
// may be null: no message then). `mark` and `call`: see zh_ctx::page_mark.
extern "C" int zh_check_kv_copy_pages(zh_ctx *c, const zh_kv_caches *dst, const zh_kv_caches *src,
                                      const uint32_t *dst_pages, const uint32_t *src_pages, uint32_t n_pages) {
    const bool one = dst && src && dst->caches == src->caches && dst->n_caches == src->n_caches;
    if (!caches_ok(dst) || !(one && dst->cache_tokens == src->cache_tokens && dst->n_kv_heads == src->n_kv_heads &&
                             dst->head_dim == src->head_dim ? true : caches_ok(src)) || dst->n_caches != src->n_caches || dst->n_kv_heads != src->n_kv_heads ||
        dst->head_dim != src->head_dim)
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "kv_copy_pages: cache sets");
    if (n_pages && (!dst_pages || !src_pages))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "kv_copy_pages: no page numbers");
    // one set copied within itself (a cache that it names twice gets the same
    // bytes twice); else the caches' addresses in a small hash table (comparing
    // every pair would take longer than the copy of a few pages)
    bool alias = one;
    if (!one) {
        uint16_t tab[1024] = {};
        auto place = [&](const void *p) {  // p's entry, or the empty one it would take
            uint32_t i = (uint32_t)(((uint64_t)(uintptr_t)p * 0x9E3779B97F4A7C15ull) >> 54);
            while (tab[i] && dst->caches[tab[i] - 1]->ptr != p) i = (i + 1) % 1024;
            return i;
        };
        for (uint32_t i = 0; i < dst->n_caches; i++) {
            uint16_t &e = tab[place(dst->caches[i]->ptr)];
            if (e)
                return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "kv_copy_pages: caches %u and %u of dst are one", e - 1u, i);
            e = (uint16_t)(i + 1);
        }
        for (uint32_t i = 0; i < src->n_caches && !alias; i++) alias = tab[place(src->caches[i]->ptr)] != 0;
    }
    if (alias && dst->cache_tokens != src->cache_tokens)
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "kv_copy_pages: one cache in two sizes");
    const uint32_t np = dst->cache_tokens / 16;
    for (uint32_t i = 0; i < n_pages; i++)
        if (dst_pages[i] >= np || src_pages[i] >= src->cache_tokens / 16)
            return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "kv_copy_pages: copy %u, page %u to %u, outside the cache", i,
                              src_pages[i], dst_pages[i]);
    try {
        std::vector<uint32_t> own;
        std::vector<uint32_t> &mark = c ? c->page_mark : own;
        if (mark.size() < np) mark.resize(np, 0);
        uint32_t one = 0, &call = c ? c->page_call : one;
        if (++call == 0) {  // (wrapped: the old marks go)
            std::fill(mark.begin(), mark.end(), 0u);
            call = 1;
        }
        for (uint32_t i = 0; i < n_pages; i++) {
            if (mark[dst_pages[i]] == call)
                return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "kv_copy_pages: two copies to page %u", dst_pages[i]);
            mark[dst_pages[i]] = call;
        }
        if (alias)
            for (uint32_t i = 0; i < n_pages; i++)
                if (mark[src_pages[i]] == call)
                    return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "kv_copy_pages: page %u is read and written",
                                      src_pages[i]);
    } catch (const std::bad_alloc &) {
        return zh_set_err(c, ZH_ERR_OUT_OF_MEMORY, "kv_copy_pages: host memory");
    }
    return ZH_OK;
}

extern "C" int zh_kv_copy_pages(zh_ctx *c, const zh_kv_caches *dst, const zh_kv_caches *src, const uint32_t *dst_pages,
                                const uint32_t *src_pages, uint32_t n_pages) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    int rc = zh_check_kv_copy_pages(c, dst, src, dst_pages, src_pages, n_pages);
    if (rc) return rc;
    zh_device_scope dev(c);
    void *d[KC_MAX];
    const void *s[KC_MAX];
    for (uint32_t i = 0; i < dst->n_caches; i++) {
        d[i] = dst->caches[i]->ptr;
        s[i] = src->caches[i]->ptr;
    }
    return zhk_kv_copy(c, dst->n_caches, d, s, dst->cache_tokens, src->cache_tokens, dst->n_kv_heads, dst->head_dim,
                       dst_pages, src_pages, n_pages);
}

// ---------------------------------------------------------------------------
// q/k RMSNorm + RoPE + KV write of a batch of rows:
//   h = w (x / sqrt(mean x^2 + eps)) over a head (or x), then dims i and
//   i + r/2 (i < r/2, r = rope_dim): (a cos - b sin, a sin + b cos) with the
//   angle pos * inv_freq[i].
// The angle is a 64-bit product (exact below position 2^29: 29 + 24 bits), taken
// and reduced in 64 bits to a fraction of a turn; at the last positions before 2^32
// it is off by less than 2^-19 radians. In 32 bits a position of 2^17 alone would
// leave an error of 2^-8. Everything else is 32-bit and rounded once, at the store.
// ---------------------------------------------------------------------------
namespace {

struct QkvArgs {
    const uint8_t *q, *k, *v;
    uint8_t *q_out;
    uint64_t q_row, k_row, v_row, out_row;  // bytes between rows
    const float *qw, *kw, *inv_freq;
    uint16_t *kc, *vc;
    const uint32_t *tables, *seq, *pos;
    uint32_t *err;
    uint32_t n_seq, stride, cache_tokens, nq, nkv, hd, rd;
    uint32_t t0;  // rows before this launch's
    float eps;
};

template <typename T>
ZH_DEV void st1(uint8_t *p, uint32_t i, float v) {
    if (sizeof(T) == 4) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = f2h_rn(v);
}
template <typename T>
ZH_DEV float ld1(const uint8_t *p, uint32_t i) {
    return sizeof(T) == 4 ? ((const float *)p)[i] : h2f(((const uint16_t *)p)[i]);
}

// cos and sin of pos * f.
ZH_DEV void turn(uint32_t pos, float f, float &co, float &sn) {
    double a = ((double)pos * (double)f) * 0.15915494309189533576888;  // turns
    a -= __builtin_rint(a);
    sincospif(2.0f * (float)a, &sn, &co);
}

// Any shape and alignment: one wave per head vector, workgroup = (head, row);
// heads [0, nq) are q, then k, then v.
template <typename TI, typename TQ>
__global__ __launch_bounds__(64) void k_qkv_rows(QkvArgs a) {
    const uint32_t t = blockIdx.y, lane = threadIdx.x, head = blockIdx.x;
    const uint32_t pos = a.pos[t];
    if (pos == ZH_POS_NONE) return;
    const bool is_q = head < a.nq, is_v = head >= a.nq + a.nkv;
    const uint32_t h = is_q ? head : (head - a.nq) % a.nkv;
    uint32_t slot = 0;
    if (!is_q) {
        const uint32_t s = a.seq ? a.seq[t] : a.t0 + t;
        if (!kv_slot(a.tables, a.n_seq, a.stride, a.cache_tokens, s, pos, slot)) {
            if (lane == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
            return;
        }
    }
    const uint8_t *x = is_q ? a.q + t * a.q_row : is_v ? a.v + t * a.v_row : a.k + t * a.k_row;
    x += (size_t)h * a.hd * sizeof(TI);
    uint16_t *cache = (is_v ? a.vc : a.kc) + ((size_t)h * a.cache_tokens + slot) * a.hd;
    uint8_t *out = is_q ? a.q_out + t * a.out_row + (size_t)h * a.hd * sizeof(TQ) : (uint8_t *)cache;
    auto put = [&](uint32_t i, float v) __attribute__((always_inline)) {
        if (is_q) st1<TQ>(out, i, v);
        else st1<uint16_t>(out, i, v);
    };
    if (is_v) {
        for (uint32_t i = lane; i < a.hd; i += 64) put(i, ld1<TI>(x, i));
        return;
    }
    const float *w = is_q ? a.qw : a.kw;
    float ri = 1.f;
    if (w) {
        float sq = 0.f;
        for (uint32_t i = lane; i < a.hd; i += 64) {
            const float e = ld1<TI>(x, i);
            sq = fmaf(e, e, sq);
        }
        ri = 1.0f / sqrtf(wave_sum(sq) / (float)a.hd + a.eps);
    }
    auto val = [&](uint32_t i) __attribute__((always_inline)) {
        const float e = ld1<TI>(x, i);
        return w ? w[i] * (e * ri) : e;
    };
    // (a lane reads and writes its own dims only: q_out may be q)
    for (uint32_t i = lane; i < a.rd / 2; i += 64) {
        float co, sn;
        turn(pos, a.inv_freq[i], co, sn);
        const float lo = val(i), hi = val(i + a.rd / 2);
        put(i, lo * co - hi * sn);
        put(i + a.rd / 2, lo * sn + hi * co);
    }
    for (uint32_t i = a.rd + lane; i < a.hd; i += 64) put(i, val(i));
}

// 8 elements of a row as floats / from floats.
ZH_DEV void ld8(const float *p, float (&v)[8]) {
    const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
ZH_DEV void ld8(const _Float16 *p, float (&v)[8]) {
    const half8 a = *(const half8 *)p;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)a[e];
}
ZH_DEV void st8(float *p, const float (&v)[8]) {
    *(f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4 *)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
ZH_DEV void st8(_Float16 *p, const float (&v)[8]) {
    half8 a;
#pragma unroll
    for (int e = 0; e < 8; e++) a[e] = (_Float16)v[e];
    *(half8 *)p = a;
}

// Head dims of 8 L (L = 8, 16, 32 lanes of 8 dims), rope_dim / 16 zero or a
// power of two, 16-byte aligned rows: a workgroup takes R x 256 / L heads of one
// row (blockIdx.x) and works the row's angles out once, in LDS. The rotation's
// partner dims lie rope_dim / 16 lanes away. Bound by HBM: 8192 rows of 32 + 16
// heads in fp16 (201 MB) 42 us, 4.8 TB/s, with R = 4 (3 / 2 / 1: 43.8 / 44.9 /
// 48.4; one wave per head vector, each with its own angles: 190).
template <typename TI, typename TQ, int L, int R>
__global__ __launch_bounds__(256) void k_qkv_rows8(QkvArgs a) {
    constexpr uint32_t HD = 8 * L, NS = 256 / L;
    __shared__ float2 cs[HD / 2];
    const uint32_t t = blockIdx.x, tid = threadIdx.x, l = tid % L, slot8 = tid / L;
    const uint32_t pos = a.pos[t];
    if (pos == ZH_POS_NONE) return;
    const uint32_t h0 = blockIdx.y * (R * NS), H = a.nq + 2 * a.nkv;
    float x[R][8];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const uint32_t h = min(h0 + r * NS + slot8, H - 1);
        const uint8_t *p = h < a.nq ? a.q + t * a.q_row : h < a.nq + a.nkv ? a.k + t * a.k_row : a.v + t * a.v_row;
        const uint32_t hh = h < a.nq ? h : h < a.nq + a.nkv ? h - a.nq : h - a.nq - a.nkv;
        ld8((const TI *)p + hh * HD + 8 * l, x[r]);
    }
    uint32_t slot = 0;
    bool ok = true;
    if (h0 + R * NS > a.nq) {  // (uniform: some k or v head)
        ok = kv_slot(a.tables, a.n_seq, a.stride, a.cache_tokens, a.seq ? a.seq[t] : a.t0 + t, pos, slot);
        if (!ok && tid == 0) atomicOr(a.err, ZH_DEVERR_KV_ROW);
    }
    const uint32_t h2 = a.rd / 2;
    if (h2 && h0 < a.nq + a.nkv) {  // (uniform: some q or k head)
        if (tid < h2) turn(pos, a.inv_freq[tid], cs[tid].x, cs[tid].y);
        __syncthreads();
    }
    const bool rot = 8 * l < a.rd, lower = 8 * l < h2;
    float2 t8[8];
    if (rot) {
        const uint32_t b = lower ? 8 * l : 8 * l - h2;
#pragma unroll
        for (int e = 0; e < 8; e++) t8[e] = cs[b + e];
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const uint32_t h = h0 + r * NS + slot8;
        if (h0 + r * NS >= H) break;  // uniform
        const bool is_q = h < a.nq, is_v = h >= a.nq + a.nkv;
        if (h0 + r * NS < a.nq + a.nkv) {  // (uniform; all lanes take part in the exchanges)
            float y[8], sq = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) sq = fmaf(x[r][e], x[r][e], sq);
            const float *w = is_q ? a.qw : a.kw;
            if (a.qw || a.kw) {
                const float ri = 1.0f / sqrtf(team_sum_dpp<L>(sq) / (float)HD + a.eps);
                if (w && !is_v) {
                    float wv[8];
                    ld8(w + 8 * l, wv);
#pragma unroll
                    for (int e = 0; e < 8; e++) x[r][e] = wv[e] * (x[r][e] * ri);
                }
            }
            if (h2) {
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = __shfl_xor(x[r][e], h2 / 8, 64);
                if (rot && !is_v)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[r][e] = lower ? x[r][e] * t8[e].x - y[e] * t8[e].y : y[e] * t8[e].y + x[r][e] * t8[e].x;
            }
        }
        if (h >= H) continue;
        if (is_q) {
            st8((TQ *)(a.q_out + t * a.out_row) + h * HD + 8 * l, x[r]);
        } else if (ok) {
            const uint32_t hh = is_v ? h - a.nq - a.nkv : h - a.nq;
            st8((_Float16 *)(is_v ? a.vc : a.kc) + ((size_t)hh * a.cache_tokens + slot) * HD + 8 * l, x[r]);
        }
    }
}

}  // namespace

// Bytes from the first to past the last element of `rows` rows of `width` (past 64
// bits: more than any buffer has).
static uint64_t rows_bytes(uint32_t rows, uint32_t stride, uint64_t width, uint32_t size) {
    const uint64_t n = (uint64_t)(rows - 1) * stride + width;
    return n > ~0ull / size ? ~0ull : n * size;
}

bool kv_batch_ok(const zh_kv_batch *kv) {
    return kv && kv->n_seq && kv->table_stride && kv->cache_tokens && kv->cache_tokens % 16 == 0 && kv->n_kv_heads &&
           kv->n_kv_heads <= 65535 && kv->head_dim && kv->head_dim <= 512 &&
           kv_in_range(kv->k_cache, 0, 2ull * kv->n_kv_heads * kv->cache_tokens * kv->head_dim) &&
           kv_in_range(kv->v_cache, 0, 2ull * kv->n_kv_heads * kv->cache_tokens * kv->head_dim) &&
           kv->tables && (uint64_t)kv->n_seq * kv->table_stride <= kv->tables->size / 4 && kv->k_cache->ptr != kv->v_cache->ptr;
}

bool kv_rows_overlap(const zh_buf *a, uint64_t a0, uint64_t an, const zh_buf *b, uint64_t b0, uint64_t bn) {
    const uint64_t pa = (uint64_t)(uintptr_t)a->ptr + a0, pb = (uint64_t)(uintptr_t)b->ptr + b0;
    return pa < pb + bn && pb < pa + an;
}

// The rows with their strides (0: rows without gaps).
static zh_qkv_rows with_strides(const zh_kv_batch *kv, const zh_qkv_rows *r) {
    zh_qkv_rows x = *r;
    if (!x.q_stride) x.q_stride = x.n_q_heads * kv->head_dim;
    if (!x.q_out_stride) x.q_out_stride = x.n_q_heads * kv->head_dim;
    if (!x.k_stride) x.k_stride = kv->n_kv_heads * kv->head_dim;
    if (!x.v_stride) x.v_stride = kv->n_kv_heads * kv->head_dim;
    return x;
}

// The checks of zh_qk_norm_rope_kv_write_batched, of host data only (exported
// for the tests; c may be null: no message then).
extern "C" int zh_check_qkv_rows(zh_ctx *c, const zh_kv_batch *kv, const zh_qkv_rows *rows) {
    if (!kv_batch_ok(kv) || !rows) return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: cache or tables");
    const zh_qkv_rows x = with_strides(kv, rows), *r = &x;
    const uint32_t nkv = kv->n_kv_heads, hd = kv->head_dim, nq = r->n_q_heads, n = r->n_rows;
    if (hd % 2 || nq == 0 || nq > 65535 || nq % nkv || (uint64_t)nq + 2ull * nkv > 65535)
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: heads %u / %u of %u", nq, nkv, hd);
    if (r->rope_dim % 2 || r->rope_dim > hd)
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: rope_dim %u of %u", r->rope_dim, hd);
    if ((r->type != ZH_F32 && r->type != ZH_F16) || (r->q_out_type != ZH_F32 && r->q_out_type != ZH_F16))
        return zh_set_err(c, ZH_ERR_UNSUPPORTED_QUANT_TYPE, "qk_norm_rope_kv batch: types %u, %u", r->type, r->q_out_type);
    if (n == 0) return ZH_OK;
    const uint32_t si = r->type == ZH_F32 ? 4 : 2, so = r->q_out_type == ZH_F32 ? 4 : 2;
    const uint64_t qw = (uint64_t)nq * hd, kw = (uint64_t)nkv * hd;
    if (n > 1 && (r->q_stride < qw || r->k_stride < kw || r->v_stride < kw || r->q_out_stride < qw))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: rows overlap");
    const uint64_t qb = rows_bytes(n, r->q_stride, qw, si), ob = rows_bytes(n, r->q_out_stride, qw, so);
    if (!kv_in_range(r->q, r->q_off, qb) || !kv_in_range(r->k, r->k_off, rows_bytes(n, r->k_stride, kw, si)) ||
        !kv_in_range(r->v, r->v_off, rows_bytes(n, r->v_stride, kw, si)) || !kv_in_range(r->q_out, r->q_out_off, ob) ||
        !kv_in_range(r->pos, 0, 4ull * n) || (r->seq && !kv_in_range(r->seq, 0, 4ull * n)) ||
        (!r->seq && n > kv->n_seq) || (r->q_norm_w && !kv_in_range(r->q_norm_w, 0, 4ull * hd)) ||
        (r->k_norm_w && !kv_in_range(r->k_norm_w, 0, 4ull * hd)) ||
        (r->rope_dim && !kv_in_range(r->inv_freq, 0, 2ull * r->rope_dim)))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: range");
    if (r->q_off % si || r->k_off % si || r->v_off % si || r->q_out_off % so)
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: offset alignment");
    // q_out and the caches: written; q_out q's own rows, or apart from everything
    // that is read
    const zh_buf *const read[] = {kv->tables, r->pos, r->seq, r->q_norm_w, r->k_norm_w, r->rope_dim ? r->inv_freq : nullptr};
    for (const zh_buf *b : read)
        if (b && (b->ptr == r->q_out->ptr || b->ptr == kv->k_cache->ptr || b->ptr == kv->v_cache->ptr))
            return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: an input is written");
    const zh_buf *const rows4[] = {r->q, r->k, r->v, r->q_out};
    for (const zh_buf *b : rows4)
        if (b->ptr == kv->k_cache->ptr || b->ptr == kv->v_cache->ptr)
            return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: rows in a cache");
    const bool same = r->q_out->ptr == r->q->ptr && r->q_out_off == r->q_off && r->q_out_type == r->type &&
                      (r->q_out_stride == r->q_stride || n == 1);
    if ((!same && kv_rows_overlap(r->q_out, r->q_out_off, ob, r->q, r->q_off, qb) &&
         !(r->q_out_type == r->type && r->q_out_stride == r->q_stride && n > 1 &&
           kv_columns_apart(r->q_out, r->q_out_off, r->q, r->q_off, r->q_stride, qw, qw, si))) ||
        (kv_rows_overlap(r->q_out, r->q_out_off, ob, r->k, r->k_off, rows_bytes(n, r->k_stride, kw, si)) &&
         !(r->q_out_type == r->type && r->q_out_stride == r->k_stride &&
           kv_columns_apart(r->q_out, r->q_out_off, r->k, r->k_off, r->k_stride, qw, kw, si))) ||
        (kv_rows_overlap(r->q_out, r->q_out_off, ob, r->v, r->v_off, rows_bytes(n, r->v_stride, kw, si)) &&
         !(r->q_out_type == r->type && r->q_out_stride == r->v_stride &&
           kv_columns_apart(r->q_out, r->q_out_off, r->v, r->v_off, r->v_stride, qw, kw, si))))
        return zh_set_err(c, ZH_ERR_INVALID_ARGUMENT, "qk_norm_rope_kv batch: q_out overlaps rows that are read");
    return ZH_OK;
}

template <typename TI, typename TQ, int L>
static void qkv_launch8(zh_ctx *c, const QkvArgs &a, uint32_t n) {
    constexpr uint32_t NS = 256 / L;
    const uint32_t H = a.nq + 2 * a.nkv;
    // few rows: every workgroup one round of heads, for the most workgroups. us at 1 /
    // 4 rounds, 32 + 16 heads of 128 f32 to f16: 64 rows 3.2 / 4.2, 256 3.9 / 4.5, 512
    // 5.2 / 5.3, 768 6.7 / 6.6, 1024 8.1 / 7.9; f16 of as many heads 512 5.2 / 5.3, 1024
    // 8.0 / 7.4; 32 heads of 64 f32 512 3.5 / 3.7, 2048 6.4 / 7.4 (one round better);
    // 56 of 256 f16 128 5.0 / 5.3, 256 7.0 / 5.6 (four better)
    if (n < 512) hipLaunchKernelGGL((k_qkv_rows8<TI, TQ, L, 1>), dim3(n, (H + NS - 1) / NS), dim3(256), 0, c->stream, a);
    else hipLaunchKernelGGL((k_qkv_rows8<TI, TQ, L, 4>), dim3(n, (H + 4 * NS - 1) / (4 * NS)), dim3(256), 0, c->stream, a);
}

template <typename TI, typename TQ>
static int qkv_launch(zh_ctx *c, const QkvArgs &a, uint32_t n) {
    const uint32_t p2 = a.rd / 16;
    const bool rows16 = (((uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.v |
                          (uint64_t)(uintptr_t)a.q_out | a.q_row | a.k_row | a.v_row | a.out_row) % 16) == 0;
    const bool by8 = rows16 && a.rd % 16 == 0 && (p2 & (p2 - 1)) == 0 && (a.hd == 64 || a.hd == 128 || a.hd == 256);
    // rows of a launch: fewer than 2^32 threads in x, at most 65535 workgroups in y
    const uint32_t most = by8 ? 1u << 23 : 65535u;
    for (uint64_t t0 = 0; t0 < n; t0 += most) {
        const uint32_t m = n - t0 < most ? (uint32_t)(n - t0) : most;
        QkvArgs b = a;
        b.q += t0 * a.q_row;
        b.k += t0 * a.k_row;
        b.v += t0 * a.v_row;
        b.q_out += t0 * a.out_row;
        b.pos += t0;
        if (b.seq) b.seq += t0;
        b.t0 = (uint32_t)t0;
        if (!by8)
            hipLaunchKernelGGL((k_qkv_rows<TI, TQ>), dim3(a.nq + 2 * a.nkv, m), dim3(64), 0, c->stream, b);
        else if (a.hd == 64) qkv_launch8<TI, TQ, 8>(c, b, m);
        else if (a.hd == 128) qkv_launch8<TI, TQ, 16>(c, b, m);
        else qkv_launch8<TI, TQ, 32>(c, b, m);
        ZH_LAUNCH_CHECK(c);
    }
    return ZH_OK;
}

extern "C" int zh_qk_norm_rope_kv_write_batched(zh_ctx *c, const zh_kv_batch *kv, const zh_qkv_rows *rows) {
    if (!c) return ZH_ERR_INVALID_ARGUMENT;
    const int rc = zh_check_qkv_rows(c, kv, rows);
    if (rc || rows->n_rows == 0) return rc;
    const zh_qkv_rows x = with_strides(kv, rows), *r = &x;
    zh_device_scope dev(c);
    const uint32_t si = r->type == ZH_F32 ? 4 : 2, so = r->q_out_type == ZH_F32 ? 4 : 2;
    QkvArgs a = {};
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
    a.kc = (uint16_t *)kv->k_cache->ptr;
    a.vc = (uint16_t *)kv->v_cache->ptr;
    a.tables = (const uint32_t *)kv->tables->ptr;
    a.seq = r->seq ? (const uint32_t *)r->seq->ptr : nullptr;
    a.pos = (const uint32_t *)r->pos->ptr;
    a.err = c->err_dev;
    a.n_seq = kv->n_seq;
    a.stride = kv->table_stride;
    a.cache_tokens = kv->cache_tokens;
    a.nq = r->n_q_heads;
    a.nkv = kv->n_kv_heads;
    a.hd = kv->head_dim;
    a.rd = r->rope_dim;
    a.eps = r->eps;
    if (si == 4) return so == 4 ? qkv_launch<float, float>(c, a, r->n_rows) : qkv_launch<float, _Float16>(c, a, r->n_rows);
    return so == 4 ? qkv_launch<_Float16, float>(c, a, r->n_rows) : qkv_launch<_Float16, _Float16>(c, a, r->n_rows);
}
