"""Operators of a serving batch over a paged KV cache held in 8 bits, as cases
to measure.

  write      a batch's raw q, k and v rows: q and k normalised by head and
             rotated to their positions, k and v quantised into their pages
  pack       whole pages of fp16 caches quantised into 8-bit ones (a prompt
             that was prefilled into fp16 caches)
  unpack     pages of 8-bit caches read back as fp16
  attention  each row's query over its sequence's cached tokens up to its own:
             one row a sequence (decode), a few (drafted tokens to verify) or
             many (chunks of prompts)

A cache holds codes, 8-bit [n_kv_heads][cache_tokens][head_dim], and a scale
for each 16-token page and head, f32 [cache_tokens / 16][n_kv_heads]; a code
stands for its value (a whole number in -127 .. 127, or an e4m3 number) times
the scale, a power of two. Table row s lists sequence s's pages. Codes that an
operator writes come back as e4m3 numbers beside their scales.

`run` computes the operators from elementary torch operations, or, with `own`
set, calls zinc_amd.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
_DEVICE = "cuda"
_LARGEST = 448.0  # of e4m3
_LOWEST = 2.0 ** -64  # of the scales


def listed():
    return [
        # one sequence's decode step: the smallest call, where latency counts
        dict(name="write_1", kind="write", mode="decode", rows=1, seqs=1, heads=32, kv_heads=8, head_dim=128,
             rope_dim=128, type="f32", q_type="f32", norm=True, far=4096),
        # a decode batch at far positions, grouped heads of an odd count, half the head rotated
        dict(name="write_decode_61", kind="write", mode="decode", rows=61, seqs=61, heads=40, kv_heads=8, head_dim=128,
             rope_dim=64, type="f32", q_type="f16", norm=False, far=131072),
        # the largest chunk of prompts of several requests, fp16 throughout
        dict(name="write_prefill_8192", kind="write", mode="prefill", rows=8192, seqs=16, heads=32, kv_heads=8,
             head_dim=128, rope_dim=128, type="f16", q_type="f16", norm=True, far=32768),
        # a prompt of 1000 tokens, prefilled into the fp16 caches of 16 layers
        dict(name="pack_1000", kind="pack", caches=32, kv_heads=8, head_dim=128, tokens=1000, pool=128, cache="e4m3"),
        # long sequences read back for a step that takes fp16 (268 MB read, 537 MB written)
        dict(name="unpack_16384", kind="unpack", caches=16, kv_heads=8, head_dim=128, tokens=16384, pool=2048,
             cache="i8"),
        # two continuations of a short prompt: the smallest attention, where latency counts
        dict(name="attn_2_at_200", kind="attention", mode="decode", rows=2, seqs=2, heads=32, kv_heads=8, head_dim=128,
             past=240, cache="i8", type="f32"),
        # a small batch at middle lengths, 32-bit queries and results
        dict(name="attn_16_at_4096", kind="attention", mode="decode", rows=16, seqs=16, heads=32, kv_heads=8,
             head_dim=128, past=4096, cache="e4m3", type="f32"),
        # unrelated requests, ragged lengths, five query heads to a kv head
        dict(name="attn_48_ragged", kind="attention", mode="ragged", rows=48, seqs=48, heads=40, kv_heads=8,
             head_dim=128, past=4096, cache="i8", type="f32"),
        # many long contexts: the cache is what an 8-bit one is for (2.1 GB)
        dict(name="attn_64_at_16384", kind="attention", mode="decode", rows=64, seqs=64, heads=32, kv_heads=8,
             head_dim=128, past=16384, cache="e4m3", type="f16"),
        # five drafted tokens of each request to verify, heads of 64
        dict(name="verify_24x5_at_3000", kind="attention", mode="verify", rows=120, seqs=24, heads=16, kv_heads=4,
             head_dim=64, past=3000, cache="i8", type="f16"),
        # chunks of several prompts after ragged contexts, 32-bit queries and results
        dict(name="chunk_777", kind="attention", mode="prefill", rows=777, seqs=5, heads=28, kv_heads=4, head_dim=128,
             past=2000, cache="e4m3", type="f32"),
        # the largest chunk: a long document's, after 8192 tokens of it (687 GFLOP)
        dict(name="chunk_4096_at_8192", kind="attention", mode="prefill", rows=4096, seqs=1, heads=32, kv_heads=8,
             head_dim=128, past=8192, cache="e4m3", type="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_SMALLER = {"write": "rows", "pack": "tokens", "unpack": "tokens", "attention": "past"}


def draw(rng):
    case = _draw(rng)
    # no more work than the largest listed call of the operator
    most = [work(c) for c in listed() if c["kind"] == case["kind"]]
    while any(n > max(m.get(k, 0) for m in most) for k, n in work(case).items()):
        k = _SMALLER[case["kind"]]
        if case["kind"] == "attention" and case["past"] <= 64:
            k = "rows"
        if k == "rows" and case["mode"] == "verify":
            each = case["rows"] // case["seqs"]
            case["seqs"] = max(1, case["seqs"] * 3 // 4)
            case["rows"] = case["seqs"] * each
            continue
        case[k] = max(1, case[k] * 3 // 4)
        if "rows" in case and case["mode"] in ("decode", "ragged"):
            case["seqs"] = case["rows"]
        elif "rows" in case and case["mode"] == "prefill":
            case["seqs"] = min(case["seqs"], case["rows"])
    return case


def _draw(rng):
    kind = rng.choice(["write", "write", "pack", "unpack", "attention", "attention", "attention", "attention"])
    kvh, hd = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    if kind in ("pack", "unpack"):
        tokens = _log_int(rng, 1, 32768)
        return dict(kind=kind, caches=2 * _log_int(rng, 1, 16), kv_heads=kvh, head_dim=hd, tokens=tokens,
                    pool=-(-tokens // PAGE) + rng.randint(1, 300),
                    cache="e4m3" if kind == "pack" else rng.choice(["i8", "e4m3"]))
    if kind == "write":
        mode = rng.choice(["decode", "prefill"])
        seqs = _log_int(rng, 1, 256 if mode == "decode" else 32)
        rows = seqs if mode == "decode" else max(seqs, _log_int(rng, 2, 8192))
        types = rng.choice([("f32", "f32"), ("f32", "f16"), ("f16", "f16")])
        return dict(kind=kind, mode=mode, rows=rows, seqs=seqs, heads=rng.choice([1, 2, 4, 5, 7, 8]) * kvh,
                    kv_heads=kvh, head_dim=hd, rope_dim=rng.choice([hd, hd, hd // 2]), type=types[0],
                    q_type=types[1], norm=rng.choice([True, True, False]), far=_log_int(rng, 2048, 262144) + rows)
    mode = rng.choice(["decode", "ragged", "verify", "prefill", "prefill"])
    seqs = _log_int(rng, 1, 16 if mode == "prefill" else 128)
    rows = seqs
    if mode == "verify":
        rows = seqs * rng.randint(2, 8)
    if mode == "prefill":
        rows = max(seqs, _log_int(rng, 16, 4096))
    return dict(kind=kind, mode=mode, rows=rows, seqs=seqs, heads=rng.choice([1, 2, 3, 4, 5, 7, 8, 16]) * kvh,
                kv_heads=kvh, head_dim=hd, past=_log_int(rng, 1, 32768), cache=rng.choice(["i8", "e4m3"]),
                type=rng.choice(["f32", "f16"]))


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------
_TORCH = {"f32": torch.float32, "f16": torch.float16}


class _Gen:
    """Seeded values: large tensors on the device, plans on the host."""

    def __init__(self, seed):
        self.host = np.random.default_rng(seed)
        self.dev = torch.Generator(device=_DEVICE)
        self.dev.manual_seed(seed)

    def normal(self, shape, dtype, scale=1.0):
        t = torch.empty(shape, dtype=dtype, device=_DEVICE).normal_(generator=self.dev)
        return t.mul_(scale) if scale != 1.0 else t

    def codes(self, shape, cache):
        """A cache's codes as bytes: values of about unit size under scales of about 2^-5 (i8), 2^-7 (e4m3)."""
        if cache == "i8":
            return self.normal(shape, torch.float16, 32.0).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        return self.normal(shape, torch.float16, 110.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)

    def scales(self, shape, cache):
        e = torch.randint(-1, 2, shape, generator=self.dev, device=_DEVICE) - (5 if cache == "i8" else 7)
        return torch.exp2(e.float())


def _u32(a):
    """Host integers as a device tensor (int32 holds the same bits)."""
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).to(_DEVICE)


def _page_inputs(case, seed):
    g = _Gen(seed)
    n, pool, nkv, hd = -(-case["tokens"] // PAGE), case["pool"], case["kv_heads"], case["head_dim"]
    shape = (nkv, pool * PAGE, hd)
    x = dict(src=g.host.permutation(pool)[:n].astype(np.uint32), dst=g.host.permutation(pool)[:n].astype(np.uint32))
    if case["kind"] == "pack":  # (heads of different sizes, some channels far larger than the others)
        size = torch.exp2(g.normal((nkv, 1, hd), torch.float32)).half()
        x["half"] = [g.normal(shape, torch.float16).mul_(size) for _ in range(case["caches"])]
    else:
        x["half"] = [g.normal(shape, torch.float16) for _ in range(case["caches"])]
    x["codes"] = [g.codes(shape, case["cache"]) for _ in range(case["caches"])]
    x["scales"] = [g.scales((pool, nkv), case["cache"]) for _ in range(case["caches"])]
    return x


def _cuts(g, rows, seqs):
    """rows split into seqs counts of one or more."""
    cuts = np.sort(g.host.permutation(rows - 1)[:seqs - 1] + 1) if seqs > 1 else np.zeros(0, dtype=np.int64)
    return np.diff(np.concatenate([[0], cuts, [rows]]))


def _write_inputs(case, seed):
    g = _Gen(seed)
    T, S = case["rows"], case["seqs"]
    nh, nkv, hd, rd = case["heads"], case["kv_heads"], case["head_dim"], case["rope_dim"]
    counts = _cuts(g, T, S)
    past = np.array([g.host.integers(0, case["far"] - c + 1) for c in counts])
    stride = -(-case["far"] // PAGE)
    # the tables name pages only where this call writes
    first, last = past // PAGE, (past + counts - 1) // PAGE
    n = T // PAGE + 2 * S  # (at least those)
    perm, at = g.host.permutation(n).astype(np.uint32), 0
    tables = np.zeros((S, stride), dtype=np.uint32)
    for s in range(S):
        k = last[s] - first[s] + 1
        tables[s, first[s]:last[s] + 1] = perm[at:at + k]
        at += k
    x = dict(row_start=_u32(np.concatenate([[0], np.cumsum(counts)])) if case["mode"] == "prefill" else None,
             seq=_u32(np.repeat(np.arange(S), counts)),
             pos=_u32(np.concatenate([p + np.arange(c) for p, c in zip(past, counts)])),
             seq_lens=_u32(past + counts), tables=_u32(tables))
    # q, k and v as one stacked projection leaves them
    x["qkv"] = g.normal((T, (nh + 2 * nkv) * hd), _TORCH[case["type"]], 1.7)
    x["freq"] = (1e6 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)).float().to(_DEVICE)
    x["weights"] = [1 + 0.1 * g.normal((hd,), torch.float32) for _ in range(2)] if case["norm"] else None
    for c in "kv":
        x[c + "_cache"] = g.codes((nkv, n * PAGE, hd), "e4m3")
        x[c + "_scale"] = g.scales((n, nkv), "e4m3")
    return x


def _attn_inputs(case, seed):
    g = _Gen(seed)
    T, S, past = case["rows"], case["seqs"], case["past"]
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    counts = np.full(S, T // S) if case["mode"] != "prefill" else _cuts(g, T, S)
    # tokens before the rows: ragged ones reach from none to `past`, the others lie near it
    low = 0 if case["mode"] == "ragged" or (case["mode"] == "prefill" and S > 1) else past - past // 8
    lens = g.host.integers(low, past + 1, S)
    lens[g.host.integers(S)] = past
    lens = lens + counts
    if S > 8 and case["mode"] == "ragged":
        lens[g.host.integers(S)] = 0  # a free place of a padded batch
    pages = -(-lens // PAGE)
    total = int(max(pages.sum(), 1))
    perm, at = g.host.permutation(total).astype(np.uint32), 0
    tables = np.zeros((S, -(-int(past + counts.max()) // PAGE)), dtype=np.uint32)
    for s, n in enumerate(pages):
        tables[s, :n] = perm[at:at + n]
        at += n
    x = dict(counts=counts, lens=lens, seq_lens=_u32(lens), tables=_u32(tables),
             row_start=_u32(np.concatenate([[0], np.cumsum(counts)])) if T != S else None)
    x["q"] = g.normal((T, nh * hd), _TORCH[case["type"]], 1.5)
    for c in "kv":
        x[c + "_cache"] = g.codes((nkv, total * PAGE, hd), case["cache"])
        x[c + "_scale"] = g.scales((total, nkv), case["cache"])
    return x


def _inputs(case, seed):
    return {"write": _write_inputs, "pack": _page_inputs, "unpack": _page_inputs,
            "attention": _attn_inputs}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------
# The library's buffers
# ---------------------------------------------------------------------------
_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import zinc_amd
        _ctx = zinc_amd.Context(0)
    return _ctx


class _Held:
    """A library buffer, given back with its last reference, and its array."""

    def __init__(self, buf, shape, typestr):
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "version": 2, "strides": None,
                                         "data": (int(buf.device_ptr), False)}

    def __del__(self):
        if getattr(self.buf, "h", None):
            self.buf.free()


_TYPESTR = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4", torch.uint8: "|u1"}


def _place(t):
    """The tensor in a library buffer: (buffer, tensor of it)."""
    buf, view = _empty(t.shape, t.dtype)
    view.copy_(t)
    return buf, view


def _empty(shape, dtype):
    import zinc_amd
    n = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    held = _Held(zinc_amd.Buffer(_context(), max(n, 4)), shape, _TYPESTR[dtype])
    return held.buf, torch.as_tensor(held, device=_DEVICE)


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    if not own:
        return s
    import zinc_amd
    ctx, kind = _context(), case["kind"]
    nkv, hd = case["kv_heads"], case["head_dim"]
    cache = {"i8": zinc_amd.I8, "e4m3": zinc_amd.E4M3}[case.get("cache", "e4m3")]
    if kind in ("pack", "unpack"):
        sets = {}
        for name in ("half", "codes", "scales"):
            placed = [_place(t) for t in s[name]]
            s[name] = [t for _, t in placed]
            sets[name] = [b for b, _ in placed]
        tokens = case["pool"] * PAGE
        s["set16"] = zinc_amd.KvCaches(sets["half"], tokens, nkv, hd)
        s["set8"] = zinc_amd.Kv8Caches(sets["codes"], sets["scales"], tokens, nkv, hd, cache)
        torch.cuda.synchronize()
        return s
    types = {"f32": zinc_amd.F32, "f16": zinc_amd.F16}
    names = ["k_cache", "v_cache", "k_scale", "v_scale", "tables", "seq_lens"]
    names += ["qkv", "freq"] if kind == "write" else ["q"]
    bufs = {"row_start": None}
    for name in names + (["row_start"] if s["row_start"] is not None else []):
        bufs[name], s[name] = _place(s[name])
    s["kv"] = kv = zinc_amd.Kv8Batch(
        bufs["k_cache"], bufs["v_cache"], bufs["k_scale"], bufs["v_scale"], bufs["tables"], bufs["seq_lens"],
        row_start=bufs["row_start"], n_seq=case["seqs"], table_stride=s["tables"].shape[1],
        cache_tokens=s["k_cache"].shape[1], n_kv_heads=nkv, head_dim=hd, type=cache)
    nh, T = case["heads"], case["rows"]
    if kind == "write":
        size = 4 if case["type"] == "f32" else 2
        width = (nh + 2 * nkv) * hd
        w = [_place(t) for t in s["weights"]] if s["weights"] else [(None, None)] * 2
        s["weights"] = [t for _, t in w]
        bufs["q_out"], s["q_out"] = _empty((T, nh * hd), _TORCH[case["q_type"]])
        s["rows"] = zinc_amd.QkvRows(
            q=bufs["qkv"], k=bufs["qkv"], v=bufs["qkv"], k_off=nh * hd * size, v_off=(nh + nkv) * hd * size,
            q_stride=width, k_stride=width, v_stride=width, type=types[case["type"]], q_out=bufs["q_out"],
            q_out_type=types[case["q_type"]], q_norm_w=w[0][0], k_norm_w=w[1][0], inv_freq=bufs["freq"],
            rope_dim=case["rope_dim"], pos=None, n_rows=T, n_q_heads=nh, eps=1e-6)
    else:
        most, longest = int(s["counts"].max()), int(s["lens"].max())
        bufs["out"], s["out"] = _empty((T, nh * hd), _TORCH[case["type"]])
        bufs["ws"], s["ws"] = _empty((ctx.flash_attn_kv8_ws(kv, nh, T, most, longest) // 4 + 1,), torch.int32)
        s["rows"] = zinc_amd.AttnRows(q=bufs["q"], out=bufs["out"], ws=bufs["ws"], n_rows=T, max_rows=most,
                                      max_len=longest, n_heads=nh, type=types[case["type"]])
    torch.cuda.synchronize()
    return s


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"write": _plain_write, "pack": _plain_pack, "unpack": _plain_unpack,
                "attention": _plain_attention}[kind](s)
    if kind == "pack":
        _ctx.kv8_pack_pages(s["set8"], s["set16"], s["dst"], s["src"], s["case"]["tokens"])
        return _packed(s)
    if kind == "unpack":
        _ctx.kv8_unpack_pages(s["set16"], s["set8"], s["dst"], s["src"])
        return s["half"]
    if kind == "write":
        _ctx.qk_norm_rope_kv8_write_batched(s["kv"], s["rows"])
        return _written(s, s["q_out"])
    _ctx.flash_attn_kv8(s["kv"], s["rows"])
    return s["out"]


def _packed(s):
    return {"codes": [c.view(torch.float8_e4m3fn) for c in s["codes"]], "scales": s["scales"]}


def _written(s, q):
    return {"q": q, "k": s["k_cache"].view(torch.float8_e4m3fn), "v": s["v_cache"].view(torch.float8_e4m3fn),
            "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _least_scale(top):
    """The smallest power of two under which no value exceeds e4m3's largest."""
    m, e = torch.frexp(top.double() / _LARGEST)  # m in [1/2, 1)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(top == 0, _LOWEST, torch.ldexp(torch.ones_like(m), e).clamp_min(_LOWEST))


def _values(codes, cache):
    return codes.view(torch.int8 if cache == "i8" else torch.float8_e4m3fn).float()


def _plain_pack(s):
    case = s["case"]
    nkv, hd, n = case["kv_heads"], case["head_dim"], len(s["src"])
    src, dst = (torch.from_numpy(s[k].astype(np.int64)).to(_DEVICE) for k in ("src", "dst"))
    held = torch.arange(n * PAGE, device=_DEVICE).view(n, PAGE) < case["tokens"]
    for half, codes, scales in zip(s["half"], s["codes"], s["scales"]):
        x = half.view(nkv, -1, PAGE, hd)[:, src].float().masked_fill_(~held[..., None], 0)
        scale = _least_scale(x.abs().amax((2, 3)))  # [nkv][n]
        codes.view(nkv, -1, PAGE, hd)[:, dst] = (x / scale.float()[..., None, None]).to(torch.float8_e4m3fn).view(
            torch.uint8)
        scales[dst] = scale.float().t()
    return _packed(s)


def _plain_unpack(s):
    case = s["case"]
    nkv, hd = case["kv_heads"], case["head_dim"]
    src, dst = (torch.from_numpy(s[k].astype(np.int64)).to(_DEVICE) for k in ("src", "dst"))
    for half, codes, scales in zip(s["half"], s["codes"], s["scales"]):
        x = _values(codes.view(nkv, -1, PAGE, hd)[:, src], case["cache"])
        half.view(nkv, -1, PAGE, hd)[:, dst] = (x * scales[src].t()[..., None, None]).half()
    return s["half"]


def _store(codes, scales, x, slot):
    """x [rows][nkv][hd] (64 bits) quantised into its slots: a page takes the
    larger of its scale and the one that its new rows need (its first token
    begins it anew), and what it holds is rounded again to that."""
    nkv, hd = x.shape[1:]
    pages, at = torch.unique(slot // PAGE, return_inverse=True)
    top = torch.zeros(len(pages), nkv, dtype=torch.float64, device=_DEVICE)
    top.index_reduce_(0, at, x.abs().amax(-1), "amax")
    begun = torch.zeros(len(pages), dtype=torch.bool, device=_DEVICE)
    begun[at[slot % PAGE == 0]] = True
    old = scales[pages].double().masked_fill_(begun[:, None], 0)
    scale = torch.maximum(old, _least_scale(top))
    view = codes.view(nkv, -1, PAGE, hd)
    kept = _values(view[:, pages], "e4m3") * (old / scale).float().t()[..., None, None]
    kept = kept.to(torch.float8_e4m3fn).view(torch.uint8)
    kept[:, at, slot % PAGE] = (x / scale[at][..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8).transpose(0, 1)
    view[:, pages] = kept
    scales[pages] = scale.float()


def _plain_write(s):
    case = s["case"]
    nh, nkv, hd, rd = case["heads"], case["kv_heads"], case["head_dim"], case["rope_dim"]
    T = case["rows"]
    x = s["qkv"].view(T, nh + 2 * nkv, hd)
    pos = s["pos"].long()
    angle = (pos.double()[:, None] * s["freq"].double())[:, None]
    w = s["weights"] or [None, None]

    def turned(h, w, cos, sin):
        if w is not None:
            h = w.to(h.dtype) * (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6))
        a, b = h[..., :rd // 2], h[..., rd // 2:rd]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, h[..., rd:]], -1)

    q = turned(x[:, :nh].float(), w[0], angle.cos().float(), angle.sin().float())
    slot = s["tables"][s["seq"].long(), pos // PAGE].long() * PAGE + pos % PAGE
    # (64 bits: a value next to the border of two codes, a largest one next to that of two scales)
    _store(s["k_cache"], s["k_scale"], turned(x[:, nh:nh + nkv].double(), w[1], angle.cos(), angle.sin()), slot)
    _store(s["v_cache"], s["v_scale"], x[:, nh + nkv:].double(), slot)
    return _written(s, q.to(_TORCH[case["q_type"]]).reshape(T, nh * hd))


def _plain_attention(s):
    """Sequences padded to the most rows and the longest, some at a time; one
    softmax over all tokens that a row may see."""
    case = s["case"]
    nh, nkv, hd, S, T = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"], case["rows"]
    G = nh // nkv
    lens, counts = s["seq_lens"].long(), torch.from_numpy(s["counts"]).to(_DEVICE)
    C, M = int(s["counts"].max()), max(int(s["lens"].max()), 1)
    t, i = torch.arange(M, device=_DEVICE), torch.arange(C, device=_DEVICE)
    slots = s["tables"].long()[:, t // PAGE] * PAGE + t % PAGE  # [S][M]
    first = torch.cumsum(counts, 0) - counts
    row = (first[:, None] + i).clamp_max(T - 1)  # [S][C]
    real = i < counts[:, None]
    seen = t < (lens - counts + 1)[:, None, None] + i[:, None]  # [S][C][M]
    q = s["q"].float().view(T, nkv, G, hd) / math.sqrt(hd)
    out = torch.zeros(T, nh * hd, dtype=_TORCH[case["type"]], device=_DEVICE)

    def held(c, a, b):  # [nkv][b - a][M][hd]
        at = slots[a:b]
        v = _values(s[c + "_cache"][:, at], case["cache"])
        return v.mul_(s[c + "_scale"][at // PAGE].permute(2, 0, 1)[..., None])

    step = max(1, 2 ** 29 // (M * nkv * max(hd, C * G)))  # sequences at a time
    for a in range(0, S, step):
        b = min(a + step, S)
        x = q[row[a:b]].permute(2, 0, 1, 3, 4).reshape(nkv, b - a, C * G, hd)
        score = torch.matmul(x, held("k", a, b).transpose(2, 3).contiguous()).view(nkv, b - a, C, G, M)
        score.masked_fill_(~seen[a:b, :, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        p = score.sub_(top.masked_fill_(top == -math.inf, 0)).exp_()
        total = p.sum(-1).clamp_min_(1e-30)[..., None]
        o = torch.matmul(p.view(nkv, b - a, C * G, M), held("v", a, b)).view(nkv, b - a, C, G, hd) / total
        keep = real[a:b]
        out[row[a:b][keep]] = o.permute(1, 2, 0, 3, 4).reshape(b - a, C, nh * hd)[keep].to(out.dtype)
    return out


# ---------------------------------------------------------------------------
# What a call cannot do without
# ---------------------------------------------------------------------------
def work(case):
    nkv, hd = case["kv_heads"], case["head_dim"]
    if case["kind"] in ("pack", "unpack"):
        pages = -(-case["tokens"] // PAGE)
        return {"bytes": case["caches"] * nkv * pages * (3.0 * PAGE * hd + 4) + 8 * pages}
    nh, T, S = case["heads"], case["rows"], case["seqs"]
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "write":
        q_size = 4 if case["q_type"] == "f32" else 2
        values = size * (nh + 2 * nkv) + q_size * nh + 2 * nkv
        return {"bytes": T * values * hd + 8.0 * S + (T / PAGE + S) * (16 * nkv + 4), "flops": T * (nh + nkv) * hd * 7.0}
    past = case["past"] * (0.5 if case["mode"] == "ragged" or (case["mode"] == "prefill" and S > 1) else 15 / 16)
    tokens = S * past + T
    return {"bytes": tokens * nkv * (2 * hd + 8 / PAGE) + 2.0 * T * nh * hd * size + 4 * tokens / PAGE,
            "flops": 4.0 * nh * hd * T * (past + (T / S + 1) / 2)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _held64(codes, cache):
    return codes.view(torch.int8 if cache == "i8" else torch.float8_e4m3fn).double()


def _log2_up(x):
    """The least whole e with x <= 2^e, of positive numbers."""
    e = torch.floor(torch.log2(x)) - 1
    for _ in range(3):  # (whatever the logarithm's rounding)
        e = torch.where(torch.exp2(e) < x, e + 1, e)
    return e


def exact(case, seed):
    """Codes: the unrounded values over the page's scale."""
    x = _inputs(case, seed)
    nkv, hd = case["kv_heads"], case["head_dim"]
    if case["kind"] in ("pack", "unpack"):
        found = {"codes": [], "scales": []}
        halves = []
        for half, codes, scales in zip(x["half"], x["codes"], x["scales"]):
            held, scales, half = _held64(codes, case["cache"]), scales.double(), half.double()
            for i, (a, b) in enumerate(zip(x["src"].tolist(), x["dst"].tolist())) if case["kind"] == "pack" else ():
                n = min(PAGE, case["tokens"] - i * PAGE)
                page = torch.zeros(nkv, PAGE, hd, dtype=torch.float64, device=_DEVICE)
                page[:, :n] = half[:, a * PAGE:a * PAGE + n]
                top = page.abs().flatten(1).max(1).values
                scales[b] = torch.exp2(_log2_up(top.clamp_min(1e-300) / _LARGEST)).clamp_min(_LOWEST)
                held[:, b * PAGE:(b + 1) * PAGE] = page / scales[b][:, None, None]
            if case["kind"] == "unpack":
                at = torch.arange(PAGE, device=_DEVICE)
                a, b = (torch.from_numpy(x[k].astype(np.int64)).to(_DEVICE)[:, None] * PAGE + at for k in ("src", "dst"))
                half[:, b] = held[:, a] * scales[a // PAGE].permute(2, 0, 1)[..., None]
                halves.append(half)
            else:
                found["codes"].append(held)
                found["scales"].append(scales)
        return halves or found
    nh, T, S = case["heads"], case["rows"], case["seqs"]
    tables = x["tables"].cpu().numpy().view(np.uint32).astype(np.int64)
    if case["kind"] == "attention":
        out = torch.zeros(T, nh, hd, dtype=torch.float64, device=_DEVICE)
        first = 0
        for s, (n, c) in enumerate(zip(x["lens"].tolist(), x["counts"].tolist())):
            rows = slice(first, first + c)
            first += c
            if n == 0:
                continue
            t = np.arange(n)
            at = torch.from_numpy(tables[s, t // PAGE] * PAGE + t % PAGE).to(_DEVICE)
            hidden = torch.ones(c, n, dtype=torch.bool, device=_DEVICE).triu_(n - c + 1)
            for h in range(nkv):
                k, v = (_held64(x[m + "_cache"][h, at], case["cache"]) * x[m + "_scale"][at // PAGE, h].double()[:, None]
                        for m in "kv")
                kt = k.t().contiguous()
                for g in range(h * (nh // nkv), (h + 1) * (nh // nkv)):
                    score = (x["q"][rows].double().view(c, nh, hd)[:, g] @ kt) * hd ** -0.5
                    out[rows, g] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
        return out.view(T, nh * hd)
    rd = case["rope_dim"]
    seq, pos = x["seq"].cpu().numpy(), x["pos"].cpu().numpy().astype(np.int64)
    # the rotation as a product of complex numbers
    turn = torch.polar(torch.ones(T, rd // 2, dtype=torch.float64, device=_DEVICE),
                       x["pos"].double()[:, None] * x["freq"].double()[None])
    y = x["qkv"].double().view(T, nh + 2 * nkv, hd).clone()
    for h in range(nh + nkv):
        z = y[:, h]
        if case["norm"]:
            z = z / (z.square().sum(1, keepdim=True) / hd + 1e-6).sqrt() * x["weights"][0 if h < nh else 1].double()
        c = torch.complex(z[:, :rd // 2].contiguous(), z[:, rd // 2:rd].contiguous()) * turn
        y[:, h] = torch.cat([c.real, c.imag, z[:, rd:]], 1)
    found = {"q": y[:, :nh].reshape(T, nh * hd)}
    phys = tables[seq, pos // PAGE]
    runs = np.flatnonzero(np.concatenate([[True], (phys[1:] != phys[:-1])])).tolist() + [T]
    for c, rows in (("k", y[:, nh:nh + nkv]), ("v", y[:, nh + nkv:])):
        held, scales = _held64(x[c + "_cache"], "e4m3"), x[c + "_scale"].double()
        for a, b in zip(runs[:-1], runs[1:]):
            p, first = int(phys[a]), int(pos[a]) % PAGE
            need = rows[a:b].abs().amax((0, 2)).clamp_min(1e-300) / _LARGEST
            need = torch.exp2(_log2_up(need)).clamp_min(_LOWEST)
            old = scales[p].clone() if first else torch.zeros_like(need)
            scales[p] = new = torch.maximum(need, old)
            held[:, p * PAGE:(p + 1) * PAGE] *= (old / new)[:, None, None]
            held[:, p * PAGE + first:p * PAGE + first + b - a] = (rows[a:b] / new[:, None]).transpose(0, 1)
        found[c], found[c + "_scale"] = held, scales
    return found
