"""The values of a decode step on the device: embedding rows, normalised and rotated queries and keys with the key-value cache that
they fill, and attention over that cache with an optional sliding window. What the witness generators read is made of them.

`listed()` names twelve cases, `draw()` gives more from the same ranges, `prepare()` builds what a program holds before the call,
`run()` is one call of one operator: in plain torch, or, where `own` is true, through the library. `work()` gives the bytes and
operations a call cannot do without, `exact()` the outputs from the definitions in 64 bits."""
import math

import numpy as np
import torch

own = False

THETA, EPS = 10000.0, 1e-6


def listed():
    return [
        # One decoded token's row of an int8 embedding table: latency alone.
        dict(name="embed 1 x 4096", kind="embed", tokens=1, width=4096, vocab=32000, table="int8", out="bf16", segment=0),
        # Prompts of a batch.
        dict(name="embed 16384 x 4096", kind="embed", tokens=16384, width=4096, vocab=32000, table="int8", out="bf16", segment=0),
        # One decoded token of each of eight streams, into a cache of the model's own type.
        dict(name="rope 8 streams", kind="rope", seqs=8, rows=1, length=2048, ragged=True, q_heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, norm=True, cache="bf16", source="bf16"),
        # Prompts of unequal lengths into an int8 cache.
        dict(name="rope 4 x 2048 int8", kind="rope", seqs=4, rows=2048, length=2048, ragged=True, q_heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, norm=True, cache="int8", source="bf16"),
        # The token block of a dequantize component, read where that component leaves it: rotation alone, of half of each head.
        dict(name="rope 512 words", kind="rope", seqs=1, rows=512, length=2048, ragged=False, q_heads=32, kv_heads=8, dim=128, rotary=64,
             interleaved=True, norm=False, cache="bf16", source="words"),
        # The smallest segment: 32 tokens against a context of 128, two heads of 32 on one.
        dict(name="attend 32 of 128", kind="attend", seqs=1, rows=32, length=128, ragged=False, q_heads=2, kv_heads=1, dim=32, window=0, sinks=0,
             cache="bf16", out="words"),
        # One token of one stream at the model's context length.
        dict(name="attend 1 of 2048", kind="attend", seqs=1, rows=1, length=2048, ragged=False, q_heads=32, kv_heads=8, dim=128, window=0, sinks=0,
             cache="int8", out="bf16"),
        # The token block of a segment against that context.
        dict(name="attend 32 of 2048", kind="attend", seqs=1, rows=32, length=2048, ragged=False, q_heads=32, kv_heads=8, dim=128, window=0, sinks=0,
             cache="int8", out="words"),
        # One token of each of 64 streams of unequal lengths.
        dict(name="attend 64 x 1 of 8192", kind="attend", seqs=64, rows=1, length=8192, ragged=True, q_heads=32, kv_heads=8, dim=128, window=0,
             sinks=0, cache="int8", out="bf16"),
        # Long streams behind a window, the first tokens staying visible.
        dict(name="attend 16 x 1 window", kind="attend", seqs=16, rows=1, length=32768, ragged=True, q_heads=32, kv_heads=8, dim=128, window=1024,
             sinks=4, cache="bf16", out="bf16"),
        # Whole prompts.
        dict(name="attend 4 x 2048", kind="attend", seqs=4, rows=2048, length=2048, ragged=True, q_heads=32, kv_heads=8, dim=128, window=0, sinks=0,
             cache="bf16", out="bf16"),
        # A long prompt behind a window.
        dict(name="attend 8192 window", kind="attend", seqs=1, rows=8192, length=8192, ragged=False, q_heads=32, kv_heads=8, dim=128, window=1024,
             sinks=4, cache="int8", out="bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "rope", "rope", "attend", "attend", "attend", "attend"])
    if kind == "embed":
        width = rng.choice([_between(rng, 64, 8192), 8 * _between(rng, 8, 1024)])
        segment = rng.choice([0, 0, max(1, width // 8)])
        return dict(kind=kind, tokens=_between(rng, 1, 16384 * 4096 // max(width, 4096)), width=width, vocab=_between(rng, 100, 50000),
                    table=rng.choice(["int8", "bf16"]), out=rng.choice(["bf16", "words"]), segment=segment)
    kv_heads, group, dim = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 4, 4, 5, 8]), rng.choice([32, 64, 128, 128])
    seqs, cache = _between(rng, 1, 64), rng.choice(["bf16", "int8"])
    if kind == "rope":
        rows = rng.choice([1, 1, _between(rng, 1, max(1, 8192 // seqs))])
        return dict(kind=kind, seqs=seqs, rows=rows, length=rows + _between(rng, 1, 4096), ragged=rng.random() < 0.5, q_heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, 16, dim // 2]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.7, cache=cache, source=rng.choice(["bf16", "bf16", "words"]))
    window = rng.choice([0, 0, 0, _between(rng, 1, 4096)])
    sinks = rng.choice([0, _between(rng, 1, 64)]) if window else 0
    if rng.random() < 0.5:  # one token or a few of each stream
        rows = rng.choice([1, 1, 1, _between(rng, 2, 8)])
        length = rows + _between(rng, 1, min(32768, 64 * 8192 // seqs))
    else:  # prompts and token blocks
        seqs = min(seqs, 8)
        rows = _between(rng, 8, max(8, 8192 // seqs))
        length = rows + rng.choice([0, 0, _between(rng, 1, 2048)])
        while seqs * kv_heads * group * rows * length > 32 * 8192 * 8192:
            seqs, rows, length = max(1, seqs // 2), max(8, rows // 2), max(8, length // 2)
    return dict(kind=kind, seqs=seqs, rows=rows, length=length, ragged=rng.random() < 0.5, q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                window=window, sinks=sinks, cache=cache, out=rng.choice(["bf16", "bf16", "words"]))


# ---- shapes ------------------------------------------------------------------------------------------------------------------------
def _shape(case):
    """(rows of this step, tokens in all) of each sequence: unequal ones are down to half of the longest."""
    out = []
    for b in range(case["seqs"]):
        cut = (b * 37 % 100) / 200 if case["ragged"] else 0.0
        rows = max(1, int(case["rows"] * (1 - cut)))
        out.append((rows, max(rows, int(case["length"] * (1 - cut)))))
    return out


def _visible(case, rows, length):
    """(pairs of a row and a key it sees, keys that some row sees) of one sequence."""
    w, s = case["window"] or length, case["sinks"] if case["window"] else 0
    p = np.arange(length - rows, length, dtype=np.int64)
    near = np.minimum(p + 1, w)
    pairs = int((near + np.minimum(s, p + 1 - near)).sum())
    first = max(0, int(p[0]) - w + 1)
    return pairs, length - first + min(s, first)


def work(case):
    if case["kind"] == "embed":
        n = case["tokens"] * case["width"]
        per = (1 if case["table"] == "int8" else 2) + (2 if case["out"] == "bf16" else 4)
        return {"bytes": n * per + case["tokens"] * (8 if case["table"] == "int8" else 4), "flops": n}
    shape, d = _shape(case), case["dim"]
    rows = sum(r for r, _ in shape)
    value, scale = (1, 4) if case["cache"] == "int8" else (2, 0)
    if case["kind"] == "rope":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        read = rows * heads * d * (2 if case["source"] == "bf16" else 4)
        return {"bytes": read + rows * (case["q_heads"] * d * 2 + 2 * case["kv_heads"] * (d * value + scale)), "flops": 10 * rows * heads * d}
    seen = [_visible(case, r, n) for r, n in shape]
    keys = sum(k for _, k in seen) * case["kv_heads"] * 2 * (d * value + scale)
    return {"bytes": keys + rows * case["q_heads"] * d * (2 + (2 if case["out"] == "bf16" else 4)), "flops": 4 * d * case["q_heads"] * sum(p for p, _ in seen)}


# ---- what a program holds ----------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _codes(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def _words(x):
    """bf16 values as patterns in the low halves of 32-bit words."""
    return x.view(torch.int16).to(torch.int32) & 0xFFFF


def _of_words(x):
    return (x << 16).view(torch.float32)


def _values(x):
    """The bf16 values of words, where they lie: the low halves come first."""
    return x.view(torch.bfloat16)[..., ::2]


def _batch(case):
    """The device arrays that say which rows and how many tokens each sequence has."""
    shape = _shape(case)
    first = np.concatenate([[0], np.cumsum([r for r, _ in shape])]).astype(np.int32)
    return dict(first=torch.from_numpy(first).cuda(), lens=torch.tensor([n for _, n in shape], dtype=torch.int32, device="cuda"), n_rows=int(first[-1]),
                max_rows=max(r for r, _ in shape), max_len=max(n for _, n in shape))


def prepare(case, seed):
    g, s = _gen(seed), dict(case=case)
    if case["kind"] == "embed":
        v, w, t = case["vocab"], case["width"], case["tokens"]
        s["table"] = _codes(g, v, w) if case["table"] == "int8" else _normal(g, v, w).bfloat16()
        s["row_scale"] = (0.5 + torch.rand(v, generator=g, device="cuda")) / 4096 if case["table"] == "int8" else None
        s["scale"] = 1.0 if case["table"] == "int8" else math.sqrt(w)
        s["ids"] = torch.randint(0, v, (t,), generator=g, device="cuda", dtype=torch.int32)
        if t >= 64:
            s["ids"][t // 3::97] = -1  # padding
        seg = case["segment"] or w
        s["out"] = torch.zeros(t, -(-w // seg), 2 if case["segment"] else 1, seg, device="cuda", dtype=torch.bfloat16 if case["out"] == "bf16" else torch.int32)
        return s
    s.update(_batch(case))
    n, hq, hk, d, cap, seqs = s["n_rows"], case["q_heads"], case["kv_heads"], case["dim"], case["length"], case["seqs"]
    if case["kind"] == "rope":
        heads = hq + 2 * hk
        rows = (_normal(g, n, heads, d) * torch.exp2(_normal(g, n, heads, 1))).bfloat16()
        # words: as a dequantize component leaves them, the last token and the last head first
        s["rows"] = rows if case["source"] == "bf16" else _words(rows).flip(0, 1).contiguous()
        s["q_weight"], s["k_weight"] = ((1 + 0.2 * _normal(g, d)).bfloat16() for _ in range(2)) if case["norm"] else (None, None)
        half = case["rotary"] // 2
        s["freq"] = THETA ** (-np.arange(half, dtype=np.float64) / half)
        s["q"] = torch.zeros(n, hq, d, device="cuda", dtype=torch.bfloat16)
        kind = torch.int8 if case["cache"] == "int8" else torch.bfloat16
        s["k"], s["v"] = (torch.zeros(seqs, hk, cap, d, device="cuda", dtype=kind) for _ in range(2))
        if case["cache"] == "int8":
            s["k_scale"], s["v_scale"] = (torch.zeros(seqs, hk, cap, device="cuda") for _ in range(2))
            s["k_values"], s["v_values"] = (torch.zeros(seqs, hk, cap, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        return s
    s["q"] = _normal(g, n, hq, d).bfloat16()
    if case["cache"] == "int8":
        s["k"], s["v"] = (_codes(g, seqs, hk, cap, d) for _ in range(2))
        s["k_scale"], s["v_scale"] = ((0.5 + torch.rand(seqs, hk, cap, generator=g, device="cuda")) / 73 for _ in range(2))
    else:
        s["k"], s["v"] = (torch.empty(seqs, hk, cap, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g) for _ in range(2))
    # words: one row of leaves a head, its second half the attention's
    s["out"] = torch.zeros(n, hq, d, device="cuda", dtype=torch.bfloat16) if case["out"] == "bf16" else torch.zeros(n, hq, 2, d, device="cuda", dtype=torch.int32)
    return s


def run(s):
    return {"embed": _embed, "rope": _rope, "attend": _attend}[s["case"]["kind"]](s)


# ---- embedding rows ------------------------------------------------------------------------------------------------------------------
def _embed(s):
    if own:
        _context().step_embed(_kept(s, _embed_args))
        return (s["out"] if s["case"]["out"] == "bf16" else _values(s["out"]))[:, :, -1]
    case, ids = s["case"], s["ids"].long()
    inside = (ids >= 0) & (ids < case["vocab"])
    at = torch.where(inside, ids, 0)
    by = (s["row_scale"][at] * s["scale"])[:, None] if s["row_scale"] is not None else s["scale"]
    x = torch.where(inside[:, None], s["table"][at].float() * by, 0.0).bfloat16()
    seg = case["segment"] or case["width"]
    pad = -case["width"] % seg
    x = torch.cat([x, x.new_zeros(x.shape[0], pad)], 1) if pad else x
    return x.view(case["tokens"], -1, seg)


# ---- norms, rotation, the cache ------------------------------------------------------------------------------------------------------
def _positions(s):
    """(sequence, position) of every row."""
    rows = torch.arange(s["n_rows"], device="cuda")
    seq = torch.searchsorted(s["first"][1:].long(), rows, right=True)
    return seq, s["lens"][seq].long() - s["first"][seq + 1].long() + rows


def _split(s, rows):
    hq, hk = s["case"]["q_heads"], s["case"]["kv_heads"]
    return rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]


def _rotated(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1 if interleaved else -2).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _rope(s):
    case = s["case"]
    if own:
        ctx = _context()
        ctx.step_norm_rope(_kept(s, _rope_args))
        if case["cache"] == "bf16":
            return dict(q=s["q"], k=s["k"], v=s["v"])
        with torch.cuda.stream(_stream()):  # the cache's values: codes times scales
            return dict(q=s["q"], k=torch.mul(s["k"], s["k_scale"].unsqueeze(-1), out=s["k_values"]), v=torch.mul(s["v"], s["v_scale"].unsqueeze(-1), out=s["v_values"]))
    rows = s["rows"].float() if case["source"] == "bf16" else _of_words(s["rows"].flip(0, 1))
    q, k, v = _split(s, rows)
    seq, pos = _positions(s)
    angle = pos.double()[:, None, None] * torch.from_numpy(s["freq"]).cuda()
    cos, sin = angle.cos().float(), angle.sin().float()
    if case["norm"]:
        q, k = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float() for x, w in ((q, s["q_weight"]), (k, s["k_weight"])))
    q, k = (_rotated(x, cos, sin, case["interleaved"]) for x in (q, k))
    s["q"].copy_(q)
    if case["cache"] == "bf16":
        s["k"][seq, :, pos], s["v"][seq, :, pos] = k.bfloat16(), v.bfloat16()
        return dict(q=s["q"], k=s["k"], v=s["v"])
    for name, x in (("k", k), ("v", v)):
        by = x.abs().amax(-1, keepdim=True) / 127
        code = torch.round(x / torch.where(by > 0, by, 1.0)).clamp(-127, 127)
        s[name + "_values"][seq, :, pos] = (code * by).bfloat16()
    return dict(q=s["q"], k=s["k_values"], v=s["v_values"])


# ---- attention -----------------------------------------------------------------------------------------------------------------------
def _attend(s):
    case = s["case"]
    if own:
        _context().step_attention(_kept(s, _attend_args))
        return s["out"] if case["out"] == "bf16" else _values(s["out"])[:, :, 1]
    hq, hk, d, seqs, most, length = case["q_heads"], case["kv_heads"], case["dim"], case["seqs"], s["max_rows"], s["max_len"]
    group = hq // hk
    first, lens = s["first"].long(), s["lens"].long()
    counts = first[1:] - first[:-1]
    r, j = torch.arange(most, device="cuda"), torch.arange(length, device="cuda")
    at = torch.where(r < counts[:, None], first[:-1, None] + r, 0)
    pos = (lens - counts)[:, None] + r  # [sequence, row]
    gap = pos[:, :, None] - j
    seen = (gap >= 0) & (j < lens[:, None, None])
    if case["window"]:
        seen &= (gap < case["window"]) | (j < case["sinks"])
    q = s["q"].float()[at].view(seqs, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * most, d)
    k, v = s["k"][:, :, :length].float(), s["v"][:, :, :length].float()
    if case["cache"] == "int8":
        k, v = k * s["k_scale"][:, :, :length, None], v * s["v_scale"][:, :, :length, None]
    score = torch.matmul(q, k.transpose(-1, -2)).view(seqs, hk, group, most, length)
    score.mul_(1 / math.sqrt(d)).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, hk, group * most, length), v).view(seqs, hk, group, most, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, most, hq, d)[r < counts[:, None]].bfloat16()
    return o


# ---- the library's calls -------------------------------------------------------------------------------------------------------------
_one = {}


def _context():
    if "context" not in _one:
        import zk_inference_prover_b200 as zkb

        _one["context"] = zkb.Context(device=0, max_log_size=10)
    return _one["context"]


def _stream():
    if "stream" not in _one:
        _one["stream"] = torch.cuda.ExternalStream(_context().stream())
    return _one["stream"]


def _kept(s, make):
    """The call's description, built once for the buffers that it names."""
    if "call" not in s:
        import zk_inference_prover_b200 as zkb

        s["call"] = make(s, zkb)
    return s["call"]


def _embed_args(s, zkb):
    case, out = s["case"], s["out"]
    seg = out.shape[3]
    return zkb.StepEmbed(ids=s["ids"].data_ptr(), n_tokens=case["tokens"], table=s["table"].data_ptr(), table_type=zkb.VALUE_INT8 if case["table"] == "int8" else zkb.VALUE_BF16,
                         vocab=case["vocab"], width=case["width"], table_stride=case["width"], row_scale=s["row_scale"].data_ptr() if s["row_scale"] is not None else 0,
                         scale=s["scale"], out=out.data_ptr() + (seg * out.element_size() if case["segment"] else 0), out_type=zkb.VALUE_BF16 if case["out"] == "bf16" else zkb.VALUE_WORD,
                         out_stride=out.stride(0), segment=seg, segment_stride=out.stride(1))


def _cache_of(s, zkb):
    k = s["k"]
    c = zkb.KvCache(k=k.data_ptr(), v=s["v"].data_ptr(), type=zkb.VALUE_INT8 if s["case"]["cache"] == "int8" else zkb.VALUE_BF16, n_seqs=k.shape[0], n_heads=k.shape[1],
                    head_dim=k.shape[3], capacity=k.shape[2], seq_stride=k.stride(0), head_stride=k.stride(1), token_stride=k.stride(2))
    if s["case"]["cache"] == "int8":
        c.k_scale, c.v_scale, c.scale_seq_stride, c.scale_head_stride = s["k_scale"].data_ptr(), s["v_scale"].data_ptr(), s["k_scale"].stride(0), s["k_scale"].stride(1)
    return c


def _rows_of(s, zkb):
    return zkb.StepRows(first=s["first"].data_ptr(), kv_len=s["lens"].data_ptr(), n_rows=s["n_rows"], max_rows=s["max_rows"], max_len=s["max_len"])


def _rope_args(s, zkb):
    case, rows = s["case"], s["rows"]
    heads, d = rows.shape[1], rows.shape[2]
    down = case["source"] == "words"
    sign, size = (-1, 4) if down else (1, 2)
    head = lambda h: rows.data_ptr() + size * ((rows.numel() - d - h * d) if down else h * d)  # noqa: E731
    stride = sign * heads * d
    return zkb.StepNormRope(cache=_cache_of(s, zkb), rows=_rows_of(s, zkb), q=head(0), k=head(case["q_heads"]), v=head(case["q_heads"] + case["kv_heads"]),
                            type=zkb.VALUE_WORD if down else zkb.VALUE_BF16, q_heads=case["q_heads"], q_stride=stride, k_stride=stride, v_stride=stride,
                            head_stride=sign * d, q_weight=s["q_weight"].data_ptr() if case["norm"] else 0, k_weight=s["k_weight"].data_ptr() if case["norm"] else 0,
                            eps=EPS, rotary_dim=case["rotary"], interleaved=case["interleaved"], h_inv_freq=s["freq"].ctypes.data,
                            q_out=s["q"].data_ptr(), q_out_stride=s["q"].stride(0), q_out_head_stride=s["q"].stride(1))


def _attend_args(s, zkb):
    case, q, out = s["case"], s["q"], s["out"]
    words = case["out"] == "words"
    return zkb.StepAttention(cache=_cache_of(s, zkb), rows=_rows_of(s, zkb), q=q.data_ptr(), q_heads=case["q_heads"], q_stride=q.stride(0), q_head_stride=q.stride(1),
                             out=out.data_ptr() + (4 * case["dim"] if words else 0), out_type=zkb.VALUE_WORD if words else zkb.VALUE_BF16, out_stride=out.stride(0),
                             out_head_stride=out.stride(1), scale=1 / math.sqrt(case["dim"]), window=case["window"], sinks=case["sinks"])


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        out = torch.zeros(case["tokens"], case["width"], device="cuda", dtype=torch.float64)
        ok = s["ids"] >= 0
        picked = torch.index_select(s["table"], 0, s["ids"][ok]).double() * s["scale"]
        out[ok] = picked * s["row_scale"].double()[s["ids"][ok].long()].unsqueeze(1) if s["row_scale"] is not None else picked
        seg = case["segment"] or case["width"]
        full = torch.zeros(case["tokens"], -(-case["width"] // seg) * seg, device="cuda", dtype=torch.float64)
        full[:, :case["width"]] = out
        return full.view(case["tokens"], -1, seg)
    return _exact_rope(s) if case["kind"] == "rope" else _exact_attend(s)


def _exact_rope(s):
    case, hq, hk, d = s["case"], s["case"]["q_heads"], s["case"]["kv_heads"], s["case"]["dim"]
    x = s["rows"].double() if case["source"] == "bf16" else torch.flip(_of_words(s["rows"]).double(), (0, 1))
    out_q = torch.empty(s["n_rows"], hq, d, device="cuda", dtype=torch.float64)
    cache = [torch.zeros(case["seqs"], hk, case["length"], d, device="cuda", dtype=torch.float64) for _ in range(2)]
    half, at = case["rotary"] // 2, 0
    i = np.arange(half)
    one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    for b, (rows, n) in enumerate(_shape(case)):
        y = x[at:at + rows].clone()
        if case["norm"]:
            w = torch.ones(hq + 2 * hk, d, device="cuda", dtype=torch.float64)
            w[:hq], w[hq:hq + hk] = s["q_weight"].double(), s["k_weight"].double()
            root = (y.square().sum(-1, keepdim=True) / d + EPS).sqrt()
            root[:, hq + hk:] = 1
            y = y / root * w
        turn = torch.arange(n - rows, n, device="cuda", dtype=torch.float64)[:, None] * torch.tensor(s["freq"], device="cuda")
        z = torch.complex(y[:, :hq + hk, one], y[:, :hq + hk, two]) * torch.polar(torch.ones_like(turn), turn)[:, None]
        y[:, :hq + hk, one], y[:, :hq + hk, two] = z.real, z.imag
        out_q[at:at + rows] = y[:, :hq]
        for c, part in zip(cache, (y[:, hq:hq + hk], y[:, hq + hk:])):
            if case["cache"] == "int8":
                step = part.abs().amax(-1, keepdim=True) / 127
                part = torch.where(step > 0, torch.round(part / step.clamp_min(1e-300)), 0.0) * step
            c[b, :, n - rows:n] = part.transpose(0, 1)
        at += rows
    return dict(q=out_q, k=cache[0], v=cache[1])


def _exact_attend(s):
    case, hq, hk, d = s["case"], s["case"]["q_heads"], s["case"]["kv_heads"], s["case"]["dim"]
    if work(case)["flops"] > 4e12:
        return None
    out, at = torch.zeros(s["n_rows"], hq, d, device="cuda", dtype=torch.float64), 0
    for b, (rows, n) in enumerate(_shape(case)):
        for lo in range(0, rows, 512):
            hi = min(rows, lo + 512)
            p = torch.arange(n - rows + lo, n - rows + hi, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = j > p
            if case["window"]:
                hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
            for h in range(hk):
                k, v = s["k"][b, h, :n].double(), s["v"][b, h, :n].double()
                if case["cache"] == "int8":
                    k, v = k * s["k_scale"][b, h, :n].double()[:, None], v * s["v_scale"][b, h, :n].double()[:, None]
                heads = slice(h * hq // hk, (h + 1) * hq // hk)
                t = torch.einsum("rgd,jd->grj", s["q"][at + lo:at + hi, heads].double(), k) / math.sqrt(d)
                t = torch.softmax(t.masked_fill(hidden, -math.inf), -1)
                out[at + lo:at + hi, heads] = torch.einsum("grj,jd->rgd", t, v)
        at += rows
    return out
