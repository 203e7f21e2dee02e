"""Operators of a serving batch over one paged KV cache, as cases to measure.

  copy       pages of a set of caches copied to other pages in one call: the
             last page of a sequence that forks (copy on write), that page for
             many children at once, a pool compacted to its low pages
  rope       a batch's raw q, k and v rows: q and k normalised by head and
             rotated to their positions, k and v written to their pages
  attention  decode attention of a batch (one query a sequence) whose sequences
             share their first prefix_len tokens, which are read once for all

The caches are fp16 [n_kv_heads][cache_tokens][head_dim], addressed through
16-token pages; table row s lists sequence s's pages.

`run` computes the operators from elementary torch operations, or, with `own`
set, calls zinc_amd.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
_DEVICE = "cuda"


def listed():
    return [
        # a request forks: its last, partly filled page, of every layer's K and V
        dict(name="copy_fork_1", kind="copy", op="fork", caches=64, kv_heads=8, head_dim=128, pages=1, pool=64),
        # a prompt sampled 13 times: the partly filled page for each child
        dict(name="copy_fanout_13", kind="copy", op="fanout", caches=48, kv_heads=4, head_dim=64, pages=13, pool=64),
        # a pool after long service, its live pages moved down (1 GB read, 1 GB written)
        dict(name="copy_compact_1024", kind="copy", op="compact", caches=32, kv_heads=8, head_dim=128, pages=1024,
             pool=2048),
        # one sequence's decode step: the smallest call, where latency counts
        dict(name="rope_1", kind="rope", mode="decode", rows=1, seqs=1, heads=32, kv_heads=8, head_dim=128,
             rope_dim=128, type="f32", q_type="f32", norm=True, far=4096),
        # a decode batch at far positions, grouped heads of an odd count, half the head rotated
        dict(name="rope_decode_61", kind="rope", mode="decode", rows=61, seqs=61, heads=40, kv_heads=8, head_dim=128,
             rope_dim=64, type="f32", q_type="f16", norm=False, far=131072),
        # a chunk of prompts of several requests, f32 projections to fp16 queries
        dict(name="rope_prefill_1000", kind="rope", mode="prefill", rows=1000, seqs=7, heads=32, kv_heads=4,
             head_dim=128, rope_dim=128, type="f32", q_type="f16", norm=True, far=16384),
        # the largest chunk, fp16 throughout
        dict(name="rope_prefill_8192", kind="rope", mode="prefill", rows=8192, seqs=16, heads=32, kv_heads=8,
             head_dim=128, rope_dim=128, type="f16", q_type="f16", norm=True, far=32768),
        # two continuations of a short prompt: the smallest call, where latency counts
        dict(name="attn_2_at_200", kind="attention", seqs=2, heads=32, kv_heads=8, head_dim=128, prefix=200, own_max=40,
             type="f32"),
        # sixteen samples of one prompt, 32-bit queries and results
        dict(name="attn_16_at_4096", kind="attention", seqs=16, heads=32, kv_heads=8, head_dim=128, prefix=4096,
             own_max=300, type="f32"),
        # unrelated requests, nothing shared, ragged lengths, five query heads to a kv head
        dict(name="attn_48_ragged", kind="attention", seqs=48, heads=40, kv_heads=8, head_dim=128, prefix=0,
             own_max=4096, type="f32"),
        # many requests under a long common document
        dict(name="attn_64_at_32768", kind="attention", seqs=64, heads=32, kv_heads=8, head_dim=128, prefix=32768,
             own_max=512, type="f16"),
        # a full batch under a long system prompt, eight query heads to a kv head
        dict(name="attn_250_at_8192", kind="attention", seqs=250, heads=32, kv_heads=4, head_dim=128, prefix=8192,
             own_max=256, type="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _draw(rng)
    # no more work than the largest listed call of the operator
    most = [work(c) for c in listed() if c["kind"] == case["kind"]]
    smaller = {"copy": "pages", "rope": "rows", "attention": "seqs"}[case["kind"]]
    while any(n > max(m.get(k, 0) for m in most) for k, n in work(case).items()):
        case[smaller] = max(1, case[smaller] * 3 // 4)
        if case["kind"] == "rope":
            case["seqs"] = min(case["seqs"], case["rows"])
            if case["mode"] == "decode":
                case["seqs"] = case["rows"]
    return case


def _draw(rng):
    kind = rng.choice(["copy", "rope", "rope", "attention", "attention", "attention"])
    kvh, hd = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    if kind == "copy":
        pages = _log_int(rng, 1, 4096)
        return dict(kind=kind, op=rng.choice(["fork", "fanout", "compact"]), caches=2 * _log_int(rng, 1, 32),
                    kv_heads=kvh, head_dim=hd, pages=pages, pool=2 * pages + rng.randint(2, 70))
    if kind == "rope":
        mode = rng.choice(["decode", "prefill"])
        seqs = _log_int(rng, 1, 256 if mode == "decode" else 32)
        rows = seqs if mode == "decode" else max(seqs, _log_int(rng, 2, 8192))
        types = rng.choice([("f32", "f32"), ("f32", "f16"), ("f16", "f16")])
        return dict(kind=kind, mode=mode, rows=rows, seqs=seqs, heads=rng.choice([1, 2, 4, 5, 7, 8]) * kvh,
                    kv_heads=kvh, head_dim=hd, rope_dim=rng.choice([hd, hd, hd // 2]), type=types[0],
                    q_type=types[1], norm=rng.choice([True, True, False]), far=_log_int(rng, 2048, 262144) + rows)
    prefix = rng.choice([0, 1, 1, 1, 1]) * _log_int(rng, 1, 32768)
    return dict(kind=kind, seqs=_log_int(rng, 1, 256), heads=rng.choice([1, 2, 3, 4, 5, 7, 8, 16]) * kvh, kv_heads=kvh,
                head_dim=hd, prefix=prefix, own_max=_log_int(rng, 1, 4096), type=rng.choice(["f32", "f16"]))


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


def _u32(a):
    """Host integers as a device tensor (int32 holds the same bits)."""
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).to(_DEVICE)


def _copy_inputs(case, seed):
    g = _Gen(seed)
    n, pool = case["pages"], case["pool"]
    perm = g.host.permutation(pool)
    if case["op"] == "compact":  # live pages above the boundary, free ones below it
        src, dst = pool // 2 + g.host.permutation(pool - pool // 2)[:n], np.sort(g.host.permutation(pool // 2)[:n])
        src = np.sort(src)
    elif case["op"] == "fanout":
        src, dst = np.repeat(perm[:1], n), perm[1:n + 1]
    else:
        src, dst = perm[:n], perm[n:2 * n]
    shape = (case["kv_heads"], pool * PAGE, case["head_dim"])
    caches = [g.normal(shape, torch.float16) for _ in range(case["caches"])]
    return dict(caches=caches, src=src.astype(np.uint32), dst=dst.astype(np.uint32))


def _tables(g, lens, shared_pages, stride):
    """Page tables of sequences of the given token counts whose first
    shared_pages pages are the same ones; pages in the order a used pool gives
    them out. Returns (tables, tokens of the cache)."""
    pages = [max(0, -(-n // PAGE) - shared_pages) for n in lens]
    total = shared_pages + sum(pages)
    perm = g.host.permutation(max(total, 1)).astype(np.uint32)
    t = np.zeros((len(lens), stride), dtype=np.uint32)
    at = shared_pages
    for s, n in enumerate(pages):
        k = min(shared_pages, stride)
        t[s, :k] = perm[:k]
        t[s, shared_pages:shared_pages + n] = perm[at:at + n]
        at += n
    return t, max(total, 1) * PAGE


def _rope_inputs(case, seed):
    g = _Gen(seed)
    T, S = case["rows"], case["seqs"]
    nh, nkv, hd, rd = case["heads"], case["kv_heads"], case["head_dim"], case["rope_dim"]
    dt = _TORCH[case["type"]]
    # rows of each sequence, consecutive positions after a context of its own
    cuts = np.sort(g.host.permutation(T - 1)[:S - 1] + 1) if S > 1 else np.zeros(0, dtype=np.int64)
    counts = np.diff(np.concatenate([[0], cuts, [T]]))
    seq = np.repeat(np.arange(S), counts)
    start = np.array([g.host.integers(0, case["far"] - c + 1) for c in counts])
    pos = np.concatenate([s + np.arange(c) for s, c in zip(start, counts)])
    stride = -(-case["far"] // PAGE)
    # the tables name pages only where this call writes
    first, last = start // PAGE, (start + counts - 1) // PAGE
    n = T // PAGE + 2 * S  # (at least those)
    perm, at = g.host.permutation(n).astype(np.uint32), 0
    tables = np.zeros((S, stride), dtype=np.uint32)
    for s in range(S):
        k = last[s] - first[s] + 1
        tables[s, first[s]:last[s] + 1] = perm[at:at + k]
        at += k
    tokens = n * PAGE
    # q, k and v as one stacked projection leaves them
    qkv = g.normal((T, (nh + 2 * nkv) * hd), dt, 1.7)
    freq = (1e6 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)).float().to(_DEVICE)
    weights = [1 + 0.1 * g.normal((hd,), torch.float32) for _ in range(2)] if case["norm"] else None
    return dict(qkv=qkv, freq=freq, weights=weights, seq=_u32(seq), pos=_u32(pos), tables=_u32(tables),
                k_cache=g.normal((nkv, tokens, hd), torch.float16), v_cache=g.normal((nkv, tokens, hd), torch.float16))


def _attn_inputs(case, seed):
    g = _Gen(seed)
    S, P, M = case["seqs"], case["prefix"], case["own_max"]
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    lens = P + g.host.integers(1, M + 1, S)
    lens[g.host.integers(S)] = P + M
    if S > 8 and P == 0:
        lens[g.host.integers(S)] = 0  # a free place of a padded batch
    stride = -(-(P + M) // PAGE)
    tables, tokens = _tables(g, lens, P // PAGE, stride)
    kc, vc = (g.normal((nkv, tokens, hd), torch.float16) for _ in range(2))
    if P % PAGE:  # each sequence has its own copy of the page in which the prefix ends
        slots = torch.from_numpy(tables[:, P // PAGE].astype(np.int64) * PAGE).to(_DEVICE)
        for c in (kc, vc):
            for r in range(P % PAGE):
                c[:, slots + r] = c[:, slots[:1] + r].expand(-1, S, -1)
    q = g.normal((S, nh * hd), _TORCH[case["type"]], 1.5)
    return dict(q=q, k_cache=kc, v_cache=vc, tables=_u32(tables), lens=_u32(lens))


def _inputs(case, seed):
    return {"copy": _copy_inputs, "rope": _rope_inputs, "attention": _attn_inputs}[case["kind"]](case, seed)


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


_TYPESTR = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4"}


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
    bufs = s["bufs"] = {}
    nkv, hd = case["kv_heads"], case["head_dim"]
    if kind == "copy":
        placed = []
        for i in range(len(s["caches"])):
            placed.append(_place(s["caches"][i]))
            s["caches"][i] = placed[-1][1]
        s["set"] = zinc_amd.KvCaches([p[0] for p in placed], case["pool"] * PAGE, nkv, hd)
        torch.cuda.synchronize()
        return s
    types = {"f32": zinc_amd.F32, "f16": zinc_amd.F16}
    names = ["k_cache", "v_cache", "tables"]
    names += ["qkv", "freq", "seq", "pos"] if kind == "rope" else ["q", "lens"]
    for name in names:
        bufs[name], s[name] = _place(s[name])
    s["kv"] = kv = zinc_amd.KvBatch(bufs["k_cache"], bufs["v_cache"], bufs["tables"], n_seq=case["seqs"],
                                    table_stride=s["tables"].shape[1], cache_tokens=s["k_cache"].shape[1],
                                    n_kv_heads=nkv, head_dim=hd)
    nh = case["heads"]
    if kind == "rope":
        size = 4 if case["type"] == "f32" else 2
        width = (nh + 2 * nkv) * hd
        w = [_place(t) for t in s["weights"]] if s["weights"] else [(None, None)] * 2
        s["weights"] = [t for _, t in w]
        bufs["q_out"], s["q_out"] = _empty((case["rows"], nh * hd), _TORCH[case["q_type"]])
        s["rows"] = zinc_amd.QkvRows(
            q=bufs["qkv"], k=bufs["qkv"], v=bufs["qkv"], k_off=nh * hd * size, v_off=(nh + nkv) * hd * size,
            q_stride=width, k_stride=width, v_stride=width, type=types[case["type"]], q_out=bufs["q_out"],
            q_out_type=types[case["q_type"]], q_norm_w=w[0][0], k_norm_w=w[1][0], inv_freq=bufs["freq"],
            rope_dim=case["rope_dim"], seq=bufs["seq"], pos=bufs["pos"], n_rows=case["rows"], n_q_heads=nh, eps=1e-6)
    else:
        longest = case["prefix"] + case["own_max"]
        bufs["out"], s["out"] = _empty((case["seqs"], nh * hd), _TORCH[case["type"]])
        bufs["ws"], s["ws"] = _empty((ctx.flash_decode_shared_ws(kv, nh, case["prefix"], longest) // 4 + 1,),
                                     torch.int32)
        s["rows"] = zinc_amd.DecodeRows(q=bufs["q"], out=bufs["out"], seq_lens=bufs["lens"], ws=bufs["ws"], n_heads=nh,
                                        prefix_len=case["prefix"], max_len=longest, type=types[case["type"]])
    torch.cuda.synchronize()
    return s


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"copy": _plain_copy, "rope": _plain_rope, "attention": _plain_attention}[kind](s)
    if kind == "copy":
        _ctx.kv_copy_pages(s["set"], s["set"], s["dst"], s["src"])
        return s["caches"]
    if kind == "rope":
        _ctx.qk_norm_rope_kv_write_batched(s["kv"], s["rows"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    _ctx.flash_decode_shared(s["kv"], s["rows"])
    return s["out"]


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_copy(s):
    src, dst = (torch.from_numpy(s[k].astype(np.int64)).to(_DEVICE) for k in ("src", "dst"))
    for c in s["caches"]:
        pages = c.view(c.shape[0], -1, PAGE, c.shape[2])
        pages[:, dst] = pages[:, src]
    return s["caches"]


def _plain_rope(s):
    case = s["case"]
    nh, nkv, hd, rd = case["heads"], case["kv_heads"], case["head_dim"], case["rope_dim"]
    T = case["rows"]
    x = s["qkv"].float().view(T, nh + 2 * nkv, hd)
    pos = s["pos"].long()
    angle = pos.double()[:, None] * s["freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(h, w):
        if w is not None:
            h = w * (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6))
        a, b = h[..., :rd // 2], h[..., rd // 2:rd]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, h[..., rd:]], -1)

    w = s["weights"] or [None, None]
    q = turned(x[:, :nh], w[0]).to(_TORCH[case["q_type"]]).reshape(T, nh * hd)
    slot = s["tables"][s["seq"].long(), pos // PAGE].long() * PAGE + pos % PAGE
    s["k_cache"][:, slot] = turned(x[:, nh:nh + nkv], w[1]).half().transpose(0, 1)
    s["v_cache"][:, slot] = x[:, nh + nkv:].half().transpose(0, 1)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    """The prefix as one product for all sequences, the own tokens padded to
    the longest, one softmax over both."""
    case = s["case"]
    S, P, M = case["seqs"], case["prefix"], case["own_max"]
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    G = nh // nkv
    lens, tables = s["lens"].long(), s["tables"].long()
    t = torch.arange(P + M, device=_DEVICE)
    slots = tables[:, t // PAGE] * PAGE + t % PAGE  # [S][P + M]
    q = s["q"].float().view(S, nkv, G, hd).transpose(0, 1).reshape(nkv, S * G, hd) / math.sqrt(hd)
    seen = t[None] < lens[:, None]
    out = torch.zeros(nkv, S * G, hd, device=_DEVICE)
    top = torch.full((nkv, S * G, 1), -math.inf, device=_DEVICE)
    total = torch.zeros(nkv, S * G, 1, device=_DEVICE)
    parts = []
    if P:
        k = s["k_cache"][:, slots[0, :P]].float().transpose(1, 2).contiguous()
        rows = seen[:, None, :P].expand(S, G, P).reshape(S * G, P)
        parts.append(torch.matmul(q, k).masked_fill_(~rows, -math.inf))
    step = max(1, 2 ** 28 // (M * nkv * hd))  # sequences at a time
    scores = []
    for a in range(0, S, step):
        k = s["k_cache"][:, slots[a:a + step, P:]].float()  # [nkv][n][M][hd]
        n = k.shape[1]
        sc = torch.matmul(q.view(nkv, S, G, hd)[:, a:a + n], k.transpose(2, 3).contiguous())
        scores.append(sc.masked_fill_(~seen[a:a + n, None, P:], -math.inf).view(nkv, n * G, M))
    parts.append(torch.cat(scores, 1))
    for p in parts:
        top = torch.maximum(top, p.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0)
    parts = [(p - top).exp_() for p in parts]
    for p in parts:
        total = total + p.sum(-1, keepdim=True)
    if P:
        out += torch.matmul(parts[0], s["v_cache"][:, slots[0, :P]].float())
    for a in range(0, S, step):
        v = s["v_cache"][:, slots[a:a + step, P:]].float()
        n = v.shape[1]
        v = v.masked_fill_(~seen[a:a + n, P:, None], 0)
        o = torch.matmul(parts[-1].view(nkv, S, G, M)[:, a:a + n].contiguous(), v)
        out.view(nkv, S, G, hd)[:, a:a + n] += o
    out = out / total.masked_fill(total == 0, 1)
    return out.view(nkv, S, G, hd).transpose(0, 1).reshape(S, nh * hd).to(_TORCH[case["type"]])


# ---------------------------------------------------------------------------
# What a call cannot do without
# ---------------------------------------------------------------------------
def work(case):
    nkv, hd = case["kv_heads"], case["head_dim"]
    if case["kind"] == "copy":
        page = case["caches"] * nkv * PAGE * hd * 2
        return {"bytes": page * (case["pages"] + (1 if case["op"] == "fanout" else case["pages"]))}
    nh = case["heads"]
    if case["kind"] == "rope":
        T = case["rows"]
        size, q_size = (4 if case[k] == "f32" else 2 for k in ("type", "q_type"))
        values = size * (nh + 2 * nkv) + q_size * nh + 2 * 2 * nkv
        return {"bytes": T * (values * hd + 12), "flops": T * (nh + nkv) * hd * 7.0}
    S, P, M = case["seqs"], case["prefix"], case["own_max"]
    tokens = S * (M + 1) / 2  # own tokens: 1 to M
    size = 4 if case["type"] == "f32" else 2
    return {"bytes": (P + tokens) * (4 * nkv * hd + 4 / PAGE) + 2 * S * nh * hd * size + 4 * S,
            "flops": 4.0 * nh * hd * (S * P + tokens)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence or row at a time
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "copy":
        return None  # nothing is computed
    x = _inputs(case, seed)
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    tables = x["tables"].cpu().numpy().view(np.uint32).astype(np.int64)
    if case["kind"] == "attention":
        lens = x["lens"].cpu().numpy()
        out = torch.zeros(case["seqs"], nh, hd, dtype=torch.float64, device=_DEVICE)
        for s, n in enumerate(lens):
            if n == 0:
                continue
            t = np.arange(n)
            at = torch.from_numpy(tables[s, t // PAGE] * PAGE + t % PAGE).to(_DEVICE)
            k, v = x["k_cache"][:, at].double(), x["v_cache"][:, at].double()
            for h in range(nkv):
                group = slice(h * (nh // nkv), (h + 1) * (nh // nkv))
                score = (x["q"][s].double().view(nh, hd)[group] @ k[h].t().contiguous()) * hd ** -0.5
                out[s, group] = torch.softmax(score, -1) @ v[h]
        return out.view(case["seqs"], nh * hd)
    rd, T = case["rope_dim"], case["rows"]
    q = torch.empty(T, nh, hd, dtype=torch.float64, device=_DEVICE)
    kc, vc = x["k_cache"].double(), x["v_cache"].double()
    seq, pos = x["seq"].cpu().numpy(), x["pos"].cpu().numpy()
    at = torch.from_numpy(tables[seq, pos // PAGE] * PAGE + pos % PAGE).to(_DEVICE)
    # the rotation as a product of complex numbers
    turn = torch.polar(torch.ones(T, rd // 2, dtype=torch.float64, device=_DEVICE),
                       x["pos"].double()[:, None] * x["freq"].double()[None])
    for h in range(nh + nkv):
        y = x["qkv"][:, h * hd:(h + 1) * hd].double()
        if case["norm"]:
            w = x["weights"][0 if h < nh else 1].double()
            y = y / (y.square().sum(1, keepdim=True) / hd + 1e-6).sqrt() * w
        z = torch.complex(y[:, :rd // 2].contiguous(), y[:, rd // 2:rd].contiguous()) * turn
        y = torch.cat([z.real, z.imag, y[:, rd:]], 1)
        if h < nh:
            q[:, h] = y
        else:
            kc[h - nh, at] = y
    for h in range(nkv):
        vc[h, at] = x["qkv"][:, (nh + nkv + h) * hd:(nh + nkv + h + 1) * hd].double()
    return {"q": q.view(T, nh * hd), "k_cache": kc, "v_cache": vc}
