"""What a decode step computes between its attention and its answer: the norm of the residual stream with 8-bit codes, products of codes with
4-bit and 8-bit weights, the gate between the feed-forward products, and log probabilities of the output head.

`listed()` names twelve cases, `draw()` gives more from the same ranges, `prepare()` builds what a program holds before the call,
`run()` is one call of one operator: in plain torch, or, where `own` is true, through the library. `work()` gives the bytes and
operations a call cannot do without, `exact()` the outputs from the definitions in 64 bits."""
import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # One decoded token's residual stream: latency alone.
        dict(name="norm 1 x 4096", kind="norm", rows=1, width=4096, source="bf16", residual=True, out="codes"),
        # Prompts of a batch.
        dict(name="norm 8191 x 4096", kind="norm", rows=8191, width=4096, source="bf16", residual=True, out="codes"),
        # The token block of a layer segment, between its feed-forward products.
        dict(name="gate 32 x 14336", kind="gate", rows=32, width=14336, source="words", gated=True, out="codes"),
        # The same for prompts.
        dict(name="gate 4096 x 14336", kind="gate", rows=4096, width=14336, source="bf16", gated=True, out="codes"),
        # One decoded token through an attention output's 4-bit weights.
        dict(name="product 1 x 4096 x 4096 int4", kind="product", rows=1, n_in=4096, n_out=4096, weights="int4", group=128, out="bf16"),
        # Sixteen streams' tokens through the way back from the feed-forward width.
        dict(name="product 16 x 14336 x 4096 int4", kind="product", rows=16, n_in=14336, n_out=4096, weights="int4", group=64, out="bf16"),
        # A prompt through 4-bit weights.
        dict(name="product 2001 x 4096 x 6144 int4", kind="product", rows=2001, n_in=4096, n_out=6144, weights="int4", group=128, out="bf16"),
        # One decoded token's logits.
        dict(name="product 1 x 4096 x 32000 int8", kind="product", rows=1, n_in=4096, n_out=32000, weights="int8", group=0, out="f32"),
        # The token block of a layer segment: the accumulators that its dequantize component proves.
        dict(name="product 32 x 4096 x 28672 int8", kind="product", rows=32, n_in=4096, n_out=28672, weights="int8", group=0, out="int32"),
        # Prompts through one feed-forward product.
        dict(name="product 4096 x 4096 x 14336 int8", kind="product", rows=4096, n_in=4096, n_out=14336, weights="int8", group=0, out="bf16"),
        # The answer to one token.
        dict(name="logprobs 1 x 32000", kind="logprobs", rows=1, vocab=32000, type="f32", top=8, given=1, masked=False, scale=1.0),
        # The score of given prompts; a vocabulary of an odd size, some of it masked.
        dict(name="logprobs 4096 x 32003", kind="logprobs", rows=4096, vocab=32003, type="bf16", top=5, given=1, masked=True, scale=1.0),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """The same, odd or a multiple of some power of two."""
    n = _between(rng, lo, hi)
    to = rng.choice([1, 1, 8, 16, 128, 128])
    return n if n < to else n // to * to


def draw(rng):
    kind = rng.choice(["norm", "gate", "product", "product", "product", "logprobs", "logprobs"])
    if kind in ("norm", "gate"):
        width = _size(rng, 64, 16384)
        case = dict(kind=kind, rows=_between(rng, 1, min(8191, 8191 * 4096 // width)), width=width, source=rng.choice(["bf16", "bf16", "words"]))
        case.update(dict(residual=rng.random() < 0.8) if kind == "norm" else dict(gated=rng.random() < 0.8))
        return dict(case, out=rng.choice(["codes", "codes", "bf16", "words"]))
    if kind == "product":
        n_in, n_out, weights = _size(rng, 64, 16384), _size(rng, 64, 32000), rng.choice(["int4", "int8"])
        while n_in * n_out > 4096 * 32000:
            n_out //= 2
        most = 4096 * 4096 * 14336 // (n_in * n_out)
        rows = rng.choice([1, _between(rng, 2, 64), _between(rng, 64, 4096)])
        return dict(kind=kind, rows=max(1, min(rows, most // 2)), n_in=n_in, n_out=n_out, weights=weights, group=rng.choice([32, 64, 128]) if weights == "int4" else 0,
                    out=rng.choice(["bf16", "words", "f32"] + ["int32"] * 2 * (weights == "int8")))
    vocab = _size(rng, 100, 50000)
    return dict(kind=kind, rows=_between(rng, 1, min(4096, 4096 * 32003 // vocab // 2)), vocab=vocab, type=rng.choice(["bf16", "words", "f32"]), top=rng.choice([0, 1, 5, 20]),
                given=rng.choice([1, 1, 4]), masked=rng.random() < 0.4, scale=rng.choice([1.0, 1.0, 1.25]))


def work(case):
    rows = case["rows"]
    if case["kind"] in ("norm", "gate"):
        n, size = rows * case["width"], {"bf16": 2, "words": 4}
        two = case["residual"] if case["kind"] == "norm" else case["gated"]
        read = n * size[case["source"]] * (2 if two and case["kind"] == "gate" else 1) + (2 * n if two and case["kind"] == "norm" else 0)
        wrote = (n + 4 * rows if case["out"] == "codes" else n * size[case["out"]]) + (2 * n if two and case["kind"] == "norm" else 0)
        return {"bytes": read + wrote, "flops": 8 * n}
    if case["kind"] == "product":
        k, n = case["n_in"], case["n_out"]
        held = n * k + 4 * n if case["weights"] == "int8" else n * ((k + 1) // 2) + 2 * n * -(-k // case["group"])
        return {"bytes": held + rows * (k + 4) + rows * n * (2 if case["out"] == "bf16" else 4), "flops": 2 * rows * k * n}
    n = rows * case["vocab"]
    return {"bytes": n * (2 if case["type"] == "bf16" else 4) + rows * (8 * case["given"] + 8 * case["top"] + 4), "flops": 6 * n}


# ---- what a program holds ----------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _words(x):
    """bf16 values as patterns in the low halves of 32-bit words."""
    return x.view(torch.int16).to(torch.int32) & 0xFFFF


def _of_words(x):
    return (x << 16).view(torch.float32)


def _as(kind, x):
    return _words(x) if kind == "words" else x


def _floats(x):
    return _of_words(x) if x.dtype == torch.int32 else x.float()


def _room(kind, *shape):
    return torch.zeros(*shape, device="cuda", dtype={"bf16": torch.bfloat16, "words": torch.int32, "f32": torch.float32, "int32": torch.int32, "codes": torch.int8}[kind])


def prepare(case, seed):
    g, s, rows = _gen(seed), dict(case=case), case["rows"]
    if case["kind"] in ("norm", "gate"):
        w = case["width"]
        s["x"] = _as(case["source"], _normal(g, rows, w).bfloat16())
        # a residual stream: channels of unlike sizes
        s["residual"] = (_normal(g, rows, w) * torch.exp2(_normal(g, 1, w))).bfloat16() if case.get("residual") else None
        s["weight"] = (1 + 0.2 * _normal(g, w)).bfloat16()
        s["gate"] = _as(case["source"], (2 * _normal(g, rows, w)).bfloat16()) if case.get("gated") else None
        s["sum"] = _room("bf16", rows, w) if case.get("residual") else None
        s["out"] = _room(case["out"], rows, w)
        if case["out"] == "codes":
            s["scale"], s["values"] = torch.zeros(rows, device="cuda"), _room("bf16", rows, w)
        return s
    if case["kind"] == "product":
        k, n = case["n_in"], case["n_out"]
        # rows of activations: a row's largest is 127
        s["x"] = (_normal(g, rows, k) * 32).round().clamp(-127, 127).to(torch.int8)
        s["x_scale"] = (0.5 + torch.rand(rows, generator=g, device="cuda")) / 32
        if case["weights"] == "int8":
            s["w"] = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
            s["w_scale"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / (73 * math.sqrt(k))
        else:  # two codes of -8 .. 7 a byte, the first in the low half
            s["w"] = torch.randint(-128, 128, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.int8)
            s["w_scale"] = ((0.5 + torch.rand(n, -(-k // case["group"]), generator=g, device="cuda")) / (4.6 * math.sqrt(k))).bfloat16()
        s["out"] = _room(case["out"], rows, n)
        return s
    v = case["vocab"]
    x = _normal(g, rows, v) * 2.5
    x[:, v // 3] += 12 * torch.rand(rows, generator=g, device="cuda")  # a favourite, certain in some rows
    if case["masked"]:
        x.masked_fill_(torch.rand(v, generator=g, device="cuda") < 0.3, -math.inf)
        x[:, -3:] = torch.finfo(torch.bfloat16).min  # padding of the table
    s["logits"] = x if case["type"] == "f32" else _as(case["type"], x.bfloat16())
    del x
    s["ids"] = torch.randint(0, v - 3, (rows, case["given"]), generator=g, device="cuda", dtype=torch.int32)
    s["ids"][3::11] = -1  # nothing is asked of these rows
    s["logprobs"], s["entropy"] = _room("f32", rows, case["given"]), _room("f32", rows)
    s["top_ids"], s["top_logprobs"] = _room("int32", rows, case["top"]), _room("f32", rows, case["top"])
    return s


def run(s):
    return {"norm": _norm, "gate": _gate, "product": _product, "logprobs": _logprobs}[s["case"]["kind"]](s)


# ---- rows to codes -------------------------------------------------------------------------------------------------------------------
def _coded(s, y):
    """y as the case holds its output: bf16, words, or the values that 8-bit codes and a row's scale stand for."""
    if s["case"]["out"] == "codes":
        by = y.abs().amax(-1, keepdim=True) / 127
        return (torch.round(y / torch.where(by > 0, by, 1.0)).clamp(-127, 127) * by).bfloat16()
    return y.bfloat16()


def _given(s):
    """The library's output of a call that writes codes or values, laid out as _coded does."""
    out = s["out"]
    if s["case"]["out"] == "codes":
        with torch.cuda.stream(_stream()):
            return torch.mul(out, s["scale"].unsqueeze(-1), out=s["values"])
    return out.view(torch.bfloat16)[..., ::2] if out.dtype == torch.int32 else out


def _norm(s):
    if own:
        _context().step_residual_norm(_kept(s, _norm_args))
        return dict(sum=s["sum"], y=_given(s)) if s["residual"] is not None else dict(y=_given(s))
    h = _floats(s["x"])
    out = {}
    if s["residual"] is not None:
        out["sum"] = (h + s["residual"].float()).bfloat16()
        h = out["sum"].float()
    out["y"] = _coded(s, h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float())
    return out


def _gate(s):
    if own:
        _context().step_gate(_kept(s, _gate_args))
        return _given(s)
    y = _floats(s["x"])
    if s["gate"] is not None:
        a = _floats(s["gate"])
        y = y * a / (1 + torch.exp(-a))
    return _coded(s, y)


# ---- products ------------------------------------------------------------------------------------------------------------------------
def _unpacked(w, k):
    """The codes of bytes that hold two each."""
    low = (w << 4) >> 4  # (in 8 bits: the sign comes along)
    return torch.stack([low, w >> 4], -1).flatten(-2)[:, :k]


def _product(s):
    case = s["case"]
    if own:
        _context().step_product(_kept(s, _product_args))
        out = s["out"]
        return out.view(torch.bfloat16)[..., ::2] if case["out"] == "words" else out
    if case["out"] == "int32":  # whole numbers past 2^24
        return torch.matmul(s["x"].double(), s["w"].double().T).to(torch.int32)
    if case["weights"] == "int8":
        w = s["w"].float() * s["w_scale"][:, None]
    else:
        w = _unpacked(s["w"], case["n_in"]).float() * s["w_scale"].float().repeat_interleave(case["group"], -1)[:, :case["n_in"]]
    y = torch.matmul(s["x"].float(), w.T) * s["x_scale"][:, None]
    return y if case["out"] == "f32" else y.bfloat16()


# ---- log probabilities -----------------------------------------------------------------------------------------------------------------
def _logprobs(s):
    case, ids = s["case"], s["ids"]
    if own:
        _context().step_logprobs(_kept(s, _logprobs_args))
        return dict(logprobs=s["logprobs"], entropy=s["entropy"], top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
    x = _floats(s["logits"])
    d = (x - x.amax(-1, keepdim=True)) * case["scale"]
    p = torch.exp(d)
    total = p.sum(-1, keepdim=True)
    log = torch.log(total)
    entropy = (log - (p * torch.where(p > 0, d, 0.0)).sum(-1, keepdim=True) / total).squeeze(-1)
    known = ids >= 0
    given = torch.where(known, d.gather(-1, torch.where(known, ids, 0).long()) - log, 0.0)
    # ties to the lowest index: the order of floats as whole numbers (of -0 and 0 as one), the index behind it
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * 2 ** 20 + (2 ** 20 - 1 - torch.arange(case["vocab"], device="cuda"))
    top = torch.topk(key, case["top"], -1).indices if case["top"] else torch.zeros(case["rows"], 0, device="cuda", dtype=torch.int64)
    return dict(logprobs=given, entropy=entropy, top_ids=top.int(), top_logprobs=d.gather(-1, top) - log)


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


def _at(x):
    return x.data_ptr() if x is not None else 0


def _held(zkb, kind):
    return {"bf16": zkb.VALUE_BF16, "words": zkb.VALUE_WORD, "f32": zkb.VALUE_F32, "int32": zkb.VALUE_INT32, "codes": zkb.VALUE_INT8}[kind]


def _norm_args(s, zkb):
    case, w = s["case"], s["case"]["width"]
    return zkb.StepResidualNorm(x=_at(s["x"]), x_type=_held(zkb, case["source"]), x_stride=w, residual=_at(s["residual"]), residual_type=zkb.VALUE_BF16, residual_stride=w, weight=_at(s["weight"]),
                                sum_out=_at(s["sum"]), sum_type=zkb.VALUE_BF16, sum_stride=w, out=_at(s["out"]), out_type=_held(zkb, case["out"]), out_scale=_at(s.get("scale")), out_stride=w,
                                n_rows=case["rows"], width=w, eps=EPS)


def _gate_args(s, zkb):
    case, w = s["case"], s["case"]["width"]
    return zkb.StepGate(gate=_at(s["gate"]), gate_stride=w, x=_at(s["x"]), x_stride=w, x_type=_held(zkb, case["source"]), out=_at(s["out"]), out_type=_held(zkb, case["out"]), out_scale=_at(s.get("scale")),
                        out_stride=w, n_rows=case["rows"], width=w)


def _product_args(s, zkb):
    case = s["case"]
    int4 = case["weights"] == "int4"
    return zkb.StepProduct(x=_at(s["x"]), x_stride=case["n_in"], x_scale=0 if case["out"] == "int32" else _at(s["x_scale"]), w=_at(s["w"]), w_type=zkb.VALUE_INT4 if int4 else zkb.VALUE_INT8,
                           w_stride=s["w"].stride(0) * (2 if int4 else 1), w_scale=0 if case["out"] == "int32" else _at(s["w_scale"]), group=case["group"],
                           w_scale_stride=s["w_scale"].stride(0) if int4 else 0, out=_at(s["out"]), out_type=_held(zkb, case["out"]), out_stride=case["n_out"], n_rows=case["rows"], n_in=case["n_in"],
                           n_out=case["n_out"])


def _logprobs_args(s, zkb):
    case = s["case"]
    return zkb.StepLogprobs(logits=_at(s["logits"]), type=_held(zkb, case["type"]), logits_stride=case["vocab"], scale=case["scale"], n_rows=case["rows"], vocab=case["vocab"], ids=_at(s["ids"]),
                            n_given=case["given"], logprobs=_at(s["logprobs"]), entropy=_at(s["entropy"]), n_top=case["top"], top_ids=_at(s["top_ids"]) if case["top"] else 0,
                            top_logprobs=_at(s["top_logprobs"]) if case["top"] else 0)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "gate"):
        return _exact_rows(s)
    return _exact_product(s) if case["kind"] == "product" else _exact_logprobs(s)


def _wide(x):
    """Values in 64 bits, of words by their patterns."""
    return x.to(torch.int16).view(torch.bfloat16).double() if x.dtype == torch.int32 else x.double()


def _exact_rows(s):
    case, y, total = s["case"], _wide(s["x"]), None
    if case["kind"] == "norm":
        if case["residual"]:
            total = y + s["residual"].double()
            y = total.to(torch.bfloat16).double()  # what is normed is the stream as it is held
        y = y / torch.sqrt(torch.linalg.vector_norm(y, dim=-1, keepdim=True) ** 2 / case["width"] + EPS) * s["weight"].double()
    elif case["gated"]:
        y = y * torch.nn.functional.silu(_wide(s["gate"]))
    if case["out"] == "codes":
        step = torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True) / 127
        y = torch.where(step > 0, torch.round(y / step.clamp_min(1e-300)), 0.0) * step
    if case["kind"] == "gate":
        return y
    return dict(sum=total, y=y) if case["residual"] else dict(y=y)


def _exact_product(s):
    case, x, w, k = s["case"], s["x"].double(), s["w"], s["case"]["n_in"]
    if case["weights"] == "int8":
        y = torch.einsum("tk,ck->tc", x, w.double())
        if case["out"] == "int32":
            return y.to(torch.int32)
        y = y * s["w_scale"].double()
    else:
        byte = w.to(torch.int16) & 255
        code = torch.empty(w.shape[0], 2 * w.shape[1], device="cuda", dtype=torch.float64)
        code[:, 0::2], code[:, 1::2] = byte % 16, byte // 16
        code = torch.where(code >= 8, code - 16, code)[:, :k]
        y = torch.zeros(case["rows"], case["n_out"], device="cuda", dtype=torch.float64)
        for i, at in enumerate(range(0, k, case["group"])):
            y.addcmul_(x[:, at:at + case["group"]] @ code[:, at:at + case["group"]].T, s["w_scale"][:, i].double())
    return y * s["x_scale"].double().unsqueeze(1)


def _exact_logprobs(s):
    case, parts = s["case"], []
    for at in range(0, case["rows"], 512):
        x = s["logits"][at:at + 512]
        z = _wide(x) * case["scale"]
        lp = torch.log_softmax(z, -1)
        ids = s["ids"][at:at + 512].long()
        given = torch.take_along_dim(lp, ids.clamp_min(0), 1).masked_fill(ids < 0, 0.0)
        entropy = torch.special.entr(lp.exp()).sum(-1)
        top = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        parts.append((given, entropy, top.int(), torch.take_along_dim(lp, top, 1)))
    return dict(zip(("logprobs", "entropy", "top_ids", "top_logprobs"), (torch.cat(p) for p in zip(*parts))))
