"""What lies between the values of a decode step and behind them (zkb_step_residual_norm, zkb_step_gate, zkb_step_product, zkb_step_logprobs).

CPU: what the calls refuse. GPU: each against its definition in 64 bits at the sizes, layouts and masks where it can go wrong, with bounds counted
from the roundings, and a layer's calls one after another."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from step_cases import Batch, Cache, attention_reference, rope_reference, values_of, words
from test_step_values import done, gen, refuse  # noqa: F401

gpu = pytest.mark.gpu
BF16, WORD, INT8, F32, INT32, INT4 = range(6)
HALF = 2.0 ** -8  # a rounding to bf16


# ---- what is refused -----------------------------------------------------------------------------------------------------------------------
def _norm_args(zkb, **other):
    return zkb.StepResidualNorm(**{**dict(x=64, residual=64, weight=64, sum_out=128, out=256, out_scale=64, x_stride=64, residual_stride=64, sum_stride=64, out_stride=64, n_rows=2, width=64, x_type=0,
                                          residual_type=0, sum_type=0, out_type=2, eps=1e-5), **other})


@pytest.mark.parametrize("other,want", [(dict(x_type=2), "x_type"), (dict(residual_type=3), "residual_type"), (dict(sum_type=2), "sum_type"), (dict(out_type=3), "out_type"), (dict(width=0), "width"),
                                        (dict(width=32769), "width"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(n_rows=1 << 31), "n_rows"), (dict(x=0), "a.x"), (dict(out=0), "a.out"),
                                        (dict(out_scale=0), "out_scale"), (dict(out_type=0), "out_scale"), (dict(x=65), "aligned"), (dict(weight=65), "weight"), (dict(out_scale=66), "out_scale"),
                                        (dict(sum_type=1, sum_out=130), "sum_out"), (dict(out_stride=63), "out_stride"), (dict(sum_stride=63), "sum_stride"),
                                        (dict(sum_out=64, sum_stride=128), "sum_stride"), (dict(sum_out=64, sum_type=1), "sum_type")])
def test_residual_norm_refuses(zkb, refuse, other, want):  # noqa: F811
    refuse("zkb_step_residual_norm", _norm_args(zkb, **other), want)


def _gate_args(zkb, **other):
    return zkb.StepGate(**{**dict(gate=64, x=64, out=256, out_scale=64, gate_stride=64, x_stride=64, out_stride=64, n_rows=2, width=64, x_type=0, out_type=2), **other})


@pytest.mark.parametrize("other,want", [(dict(x_type=3), "x_type"), (dict(out_type=5), "out_type"), (dict(width=0), "width"), (dict(width=1 << 16), "width"), (dict(n_rows=1 << 31), "n_rows"), (dict(x=0), "a.x"),
                                        (dict(out=0), "a.out"), (dict(out_scale=0), "out_scale"), (dict(out_type=1), "out_scale"), (dict(gate=65), "gate"), (dict(x_type=1, x=66), "aligned"),
                                        (dict(out_stride=10), "out_stride")])
def test_gate_refuses(zkb, refuse, other, want):  # noqa: F811
    refuse("zkb_step_gate", _gate_args(zkb, **other), want)


def _product_args(zkb, **other):
    return zkb.StepProduct(**{**dict(x=64, x_scale=64, w=64, w_scale=64, out=64, x_stride=256, w_stride=256, w_scale_stride=2, out_stride=8, n_rows=2, n_in=256, n_out=8, w_type=5, group=128, out_type=0), **other})


@pytest.mark.parametrize("other,want", [(dict(w_type=0), "w_type"), (dict(out_type=2), "out_type"), (dict(out_type=4), "out_type"), (dict(group=0), "group"), (dict(group=16), "group"), (dict(w_type=2), "group"),
                                        (dict(n_in=0), "n_in"), (dict(n_in=131072), "n_in"), (dict(n_out=0), "n_out"), (dict(n_out=(1 << 24) + 1), "n_out"), (dict(n_rows=(1 << 18) + 1), "n_rows"), (dict(x=0), "a.x"),
                                        (dict(x_scale=0), "x_scale"), (dict(w_scale=0), "w_scale"), (dict(w_type=2, group=0, out_type=4), "x_scale"), (dict(out=65), "aligned"), (dict(out_type=3, out=66), "aligned"),
                                        (dict(w_scale=65), "w_scale"), (dict(w_type=2, group=0, w_scale=66), "w_scale"), (dict(w_stride=254), "w_stride"), (dict(w_stride=257), "w_stride"),
                                        (dict(w_scale_stride=1), "w_scale_stride"), (dict(x_stride=255), "x_stride"), (dict(out_stride=7), "out_stride"), (dict(x_stride=-256), "x_stride")])
def test_product_refuses(zkb, refuse, other, want):  # noqa: F811
    refuse("zkb_step_product", _product_args(zkb, **other), want)


def _logprobs_args(zkb, **other):
    return zkb.StepLogprobs(**{**dict(logits=64, ids=64, logprobs=64, entropy=64, top_ids=64, top_logprobs=64, logits_stride=100, n_rows=2, vocab=100, n_given=1, n_top=3, type=0, scale=1.0), **other})


@pytest.mark.parametrize("other,want", [(dict(type=2), "type"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 19) + 1), "vocab"), (dict(n_rows=(1 << 26) + 1), "n_rows"), (dict(n_top=33), "n_top"),
                                        (dict(n_given=(1 << 19) + 1), "n_given"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=2.0 ** -101), "scale"), (dict(scale=math.nan), "scale"), (dict(logits=0), "logits"),
                                        (dict(logits=65), "logits"), (dict(type=3, logits=66), "logits"), (dict(ids=0), "ids"), (dict(logprobs=0), "logprobs"), (dict(top_ids=0), "top_ids"),
                                        (dict(top_logprobs=66), "top_logprobs"), (dict(entropy=66), "entropy"), (dict(off_table=68), "off_table")])
def test_logprobs_refuses(zkb, refuse, other, want):  # noqa: F811
    refuse("zkb_step_logprobs", _logprobs_args(zkb, **other), want)


def test_a_layer_call_without_arguments_or_context_or_rows(zkb):
    lib, blank = zkb.load_library(), C.create_string_buffer(1 << 16)
    at = C.cast(blank, C.c_void_p)
    for name, make in (("residual_norm", _norm_args), ("gate", _gate_args), ("product", _product_args), ("logprobs", _logprobs_args)):
        call = getattr(lib, "zkb_step_" + name)
        assert call(None, None) == -1 and call(at, None) == -1
        assert call(at, C.byref(make(zkb, n_rows=0, out=0) if name != "logprobs" else make(zkb, n_rows=0, logits=0))) == 0


# ---- rows ------------------------------------------------------------------------------------------------------------------------------------
class Rows:
    """Rows of values [row][width] with `pad` values behind each, from a multiple of 16 bytes + `off` values on; `words`: patterns; `down`: the last row, and the last segment, first."""

    def __init__(self, x, kind="bf16", pad=0, off=0, segment=0, down=False):
        n, w = x.shape
        self.x, self.segment = x, segment
        held = words(x) | 0x31F20000 if kind == "words" else x
        seg = segment or w
        n_seg = -(-w // seg)
        full = torch.zeros(n, n_seg * seg, device="cuda", dtype=held.dtype)
        full[:, :w] = held
        full = full.view(n, n_seg, seg)
        room = torch.full((n * n_seg * (seg + pad) + off,), 77, device="cuda", dtype=held.dtype)
        laid = room[off:].view(n, n_seg, seg + pad)
        laid[..., :seg] = full.flip(0, 1) if down else full
        self.keep, step = room, seg + pad
        self.stride, self.segment_stride = (-n_seg * step, -step) if down else (n_seg * step, step)
        self.ptr = laid.data_ptr() + held.element_size() * ((n * n_seg - 1) * step if down else 0)
        self.type = WORD if kind == "words" else BF16


def room(kind, n, w, pad=0, off=0):
    dtype = {"bf16": torch.bfloat16, "words": torch.int32, "codes": torch.int8, "f32": torch.float32, "int32": torch.int32}[kind]
    full = torch.full((n * (w + pad) + off,), 55, device="cuda", dtype=dtype)
    return full, full[off:].view(n, w + pad)[:, :w]


TYPES = dict(bf16=BF16, words=WORD, codes=INT8, f32=F32, int32=INT32)


def untouched(full, view, off):
    """What lies behind the rows and before the first one is as it was."""
    rest = full[off:].view(view.shape[0], view.stride(0))[:, view.shape[1]:]
    assert bool((rest == 55).all()) and bool((full[:off] == 55).all())


def check_out(out, scale, kind, y, rel):
    """An output against y in 64 bits, itself off by `rel` of its size (a number or a tensor). A code is half a step off at most, and the step itself and the
    quotient by it 127 times a few roundings."""
    if kind != "codes":
        assert bool(((values_of(out) - y).abs() <= (HALF * (1 + rel) + rel) * y.abs() + 2.0 ** -133).all())
        return
    most = y.abs().amax(-1, keepdim=True)
    s = scale.double()[:, None]
    worst = rel.amax(-1, keepdim=True) if torch.is_tensor(rel) else rel
    assert bool(((s - most / 127).abs() <= (worst + 2.0 ** -23) * most / 127 + 2.0 ** -149).all())
    assert bool(((out.double() * s - y).abs() <= s * (0.5 + 127 * (worst + 2.0 ** -21)) + rel * y.abs() + 2.0 ** -140).all())
    assert bool((out.double().abs().amax(-1)[most.squeeze(-1) > 1e-30] == 127).all())


ROW_CASES = [  # rows, width, source, residual, sum, out, pad, off, segment, down
    (1, 1, "bf16", None, None, "codes", 0, 0, 0, False), (1, 4096, "bf16", "bf16", "bf16", "codes", 0, 0, 0, False), (3, 4096, "words", "bf16", "words", "codes", 0, 0, 128, True),
    (700, 64, "bf16", "bf16", "bf16", "codes", 0, 0, 0, False), (5, 63, "words", "words", None, "words", 3, 1, 0, False), (33, 1000, "bf16", "bf16", "bf16", "bf16", 8, 0, 0, False),
    (1200, 2056, "bf16", "words", "bf16", "codes", 0, 8, 0, False), (9, 777, "words", "bf16", "bf16", "codes", 1, 1, 37, True), (2, 32768, "bf16", "bf16", "bf16", "codes", 0, 0, 0, False),
    (700, 14336, "bf16", None, "bf16", "words", 0, 0, 0, False), (2, 32767, "bf16", "bf16", "bf16", "codes", 0, 0, 0, False), (600, 16384, "bf16", "bf16", None, "codes", 16, 0, 4096, False),
    (650, 8200, "bf16", "bf16", "bf16", "codes", 0, 0, 0, False), (4000, 8, "bf16", "bf16", "bf16", "codes", 0, 0, 0, False), (601, 300, "words", "bf16", "words", "bf16", 0, 0, 12, True),
]


def norm_reference(s, weight, eps):
    y = s.double()
    y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if weight is None else y * weight.double()


@gpu
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("rows,width,source,residual,summed,out,pad,off,segment,down", ROW_CASES)
def test_residual_norm(ctx, zkb, weighted, rows, width, source, residual, summed, out, pad, off, segment, down):
    """The sum is bit for bit a 32-bit one rounded once. A sum of squares in 32 bits goes through 64 additions in a thread and 10 across, 74 roundings, half of which the root
    keeps; the root, two products: below 2^-18 of y in all."""
    g = gen(rows + width)
    x = (torch.randn(rows, width, generator=g, device="cuda") * torch.exp2(2 * torch.randn(rows, 1, generator=g, device="cuda"))).bfloat16()
    h = (3 * torch.randn(rows, width, generator=g, device="cuda")).bfloat16()
    weight = (1 + 0.3 * torch.randn(width + 1, generator=g, device="cuda")).bfloat16()[off % 2:off % 2 + width] if weighted else None
    xs, hs = Rows(x, source, pad, off, segment, down), Rows(h, residual, pad, off) if residual else None
    sum_full, sum_out = room(summed, rows, width, pad, off) if summed else (None, None)
    out_full, got = room(out, rows, width, pad, off)
    scale = torch.full((rows,), -1.0, device="cuda") if out == "codes" else None
    torch.cuda.synchronize()
    ctx.step_residual_norm(zkb.StepResidualNorm(
        x=xs.ptr, x_type=xs.type, x_stride=xs.stride, x_segment=segment, x_segment_stride=xs.segment_stride, residual=hs.ptr if hs else 0, residual_type=hs.type if hs else 0,
        residual_stride=hs.stride if hs else 0, weight=weight.data_ptr() if weighted else 0, sum_out=sum_out.data_ptr() if summed else 0, sum_type=TYPES[summed] if summed else 0,
        sum_stride=sum_out.stride(0) if summed else 0, out=got.data_ptr(), out_type=TYPES[out], out_scale=scale.data_ptr() if scale is not None else 0, out_stride=got.stride(0), n_rows=rows, width=width, eps=1e-5))
    done(ctx)
    s = (h.float() + x.float()).bfloat16() if residual else x
    if summed:
        assert torch.equal(sum_out, words(s) if summed == "words" else s)
        untouched(sum_full, sum_out, off)
    check_out(got, scale, out, norm_reference(s, weight, 1e-5), 2.0 ** -18)
    untouched(out_full, got, off)


@gpu
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("rows,width,source,residual,summed,out,pad,off,segment,down", ROW_CASES)
def test_gate(ctx, zkb, gated, rows, width, source, residual, summed, out, pad, off, segment, down):
    """The exponential of |g| is off by 2 + 1.173 |g| units of 2^-23 (the documented bound), the quotient by 2, three products by half of one each."""
    g = gen(rows + width)
    x = (torch.randn(rows, width, generator=g, device="cuda") * torch.exp2(2 * torch.randn(rows, 1, generator=g, device="cuda"))).bfloat16()
    a = (4 * torch.randn(rows, width, generator=g, device="cuda")).bfloat16()
    xs, gs = Rows(x, source, pad, off, segment, down), Rows(a, source, pad, off, segment, down)
    out_full, got = room(out, rows, width, pad, off)
    scale = torch.full((rows,), -1.0, device="cuda") if out == "codes" else None
    torch.cuda.synchronize()
    ctx.step_gate(zkb.StepGate(gate=gs.ptr if gated else 0, gate_stride=gs.stride, x=xs.ptr, x_stride=xs.stride, x_type=xs.type, segment=segment, segment_stride=xs.segment_stride, out=got.data_ptr(),
                               out_type=TYPES[out], out_scale=scale.data_ptr() if scale is not None else 0, out_stride=got.stride(0), n_rows=rows, width=width))
    done(ctx)
    y, rel = x.double(), 0.0
    if gated:
        y, rel = y * a.double() / (1 + torch.exp(-a.double())), (6 + 1.2 * a.double().abs()) * 2.0 ** -23
    check_out(got, scale, out, y, rel)
    untouched(out_full, got, off)


@gpu
@pytest.mark.parametrize("width", [64, 777, 4096])
@pytest.mark.parametrize("kind", ["codes", "bf16"])
def test_rows_of_nothing_and_of_no_numbers_and_far_from_one(ctx, zkb, width, kind):
    """Rows of zeros, of the smallest and the largest values, with a NaN and an infinity. Squares outside of what 32 bits hold are summed in 64."""
    g = gen(width)
    base = torch.randn(8, width, generator=g, device="cuda")
    size = torch.tensor([0.0, 1e-30, 1e-38, 1e37, 1.0, 1.0, 2.0 ** 62, 1e18], device="cuda")[:, None]
    x = (base * size).bfloat16()
    x[4, width // 2], x[5, 3] = math.nan, math.inf
    for eps in (1e-5, 0.0):
        full, got = room(kind, 8, width)
        scale = torch.full((8,), -1.0, device="cuda") if kind == "codes" else None
        torch.cuda.synchronize()
        ctx.step_residual_norm(zkb.StepResidualNorm(x=x.data_ptr(), x_stride=width, out=got.data_ptr(), out_type=TYPES[kind], out_scale=scale.data_ptr() if kind == "codes" else 0, out_stride=width, n_rows=8,
                                                    width=width, eps=eps))
        done(ctx)
        y = norm_reference(x, None, eps)
        ok = torch.tensor([eps > 0, True, True, True, False, False, True, True], device="cuda")
        check_out(got[ok], scale[ok] if kind == "codes" else None, kind, y[ok], 2.0 ** -18)
        for row in (~ok).nonzero().flatten().tolist():
            assert bool(torch.isnan(scale[row]) and (got[row] == 0).all()) if kind == "codes" else bool(torch.equal(torch.isnan(got[row].float()), torch.isnan(y[row])))


@gpu
def test_codes_of_the_smallest_and_of_infinite_rows(ctx, zkb):
    """Scales down to the smallest float; an infinite largest value leaves its scale and no codes."""
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    x[0, 5], x[0, 6] = 2.0 ** -126, -(2.0 ** -127)
    x[1, 7] = 2.0 ** -133
    x[2, 9], x[2, 1] = math.inf, 1.0
    x[3, 2], x[3, 3] = 3e38, -1.5e38
    out, scale = torch.full((4, 64), 9, device="cuda", dtype=torch.int8), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    ctx.step_gate(zkb.StepGate(x=x.data_ptr(), x_stride=64, out=out.data_ptr(), out_type=INT8, out_scale=scale.data_ptr(), out_stride=64, n_rows=4, width=64))
    done(ctx)
    assert out[0, 5] == 127 and out[0, 6] in (-64, -63) and int((out[0] != 0).sum()) == 2
    assert abs(float(scale[0]) * 127 / 2.0 ** -126 - 1) < 127 * 2.0 ** -22  # a denormal scale: steps of 2^-149
    # bf16's smallest value, 2^-133, over 127 is 2^-140, no zero: its code is the largest
    assert out[1, 7] == 127 and int((out[1] != 0).sum()) == 1 and abs(float(scale[1]) * 127 / 2.0 ** -133 - 1) < 127 * 2.0 ** -16
    assert scale[2] == math.inf and not bool(out[2].any())
    assert out[3, 2] == 127 and out[3, 3] in (-64, -63)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "words"])
def test_the_stream_may_be_added_to_where_it_is(ctx, zkb, kind):
    g = gen(3)
    x, h = (torch.randn(37, 512, generator=g, device="cuda").bfloat16() for _ in range(2))
    held = words(h) if kind == "words" else h.clone()
    out = torch.zeros(37, 512, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    ctx.step_residual_norm(zkb.StepResidualNorm(x=x.data_ptr(), x_stride=512, residual=held.data_ptr(), residual_type=TYPES[kind], residual_stride=512, sum_out=held.data_ptr(), sum_type=TYPES[kind], sum_stride=512,
                                                out=out.data_ptr(), out_stride=512, n_rows=37, width=512, eps=1e-6))
    done(ctx)
    s = (x.float() + h.float()).bfloat16()
    assert torch.equal(held, words(s) if kind == "words" else s)
    check_out(out, None, "bf16", norm_reference(s, None, 1e-6), 2.0 ** -18)


# ---- products ----------------------------------------------------------------------------------------------------------------------------------
class Weights:
    def __init__(self, g, kind, n_out, n_in, group=0, pad=0, off=0):
        self.kind, self.group, self.n_in, self.n_out = kind, group, n_in, n_out
        bytes_ = n_in if kind == "int8" else (n_in + 1) // 2
        self.keep = torch.randint(-128, 128, (n_out * (bytes_ + pad) + off,), generator=g, device="cuda", dtype=torch.int8)
        self.w = self.keep[off:].view(n_out, bytes_ + pad)
        if kind == "int8":
            self.scale = (0.5 + torch.rand(n_out, generator=g, device="cuda")) / 100
            self.codes = self.w[:, :n_in].double()
        else:
            b = self.w[:, :bytes_].to(torch.int16) & 255
            c = torch.stack([b % 16, b // 16], -1).flatten(1)[:, :n_in].double()
            self.codes = torch.where(c > 7, c - 16, c)
            self.scale = ((torch.rand(n_out, -(-n_in // group) + 3, generator=g, device="cuda") - 0.3) / 10).bfloat16()  # (some below zero)

    def values(self, rows):
        """sum over groups of scale * sum, and the sizes of its parts of 32 codes, in 64 bits."""
        x = rows.double()
        if self.kind == "int8":
            return x @ self.codes.T
        y, size = (torch.zeros(x.shape[0], self.n_out, device="cuda", dtype=torch.float64) for _ in range(2))
        for at in range(0, self.n_in, 32):
            part = (x[:, at:at + 32] @ self.codes[:, at:at + 32].T) * self.scale[:, at // self.group].double()
            y += part
            size += part.abs()
        return y, size


def run_product(ctx, zkb, x, x_scale, w, out):
    """x [row][n_in] with any row stride, out a view."""
    types = {torch.bfloat16: BF16, torch.float32: F32}
    kind = out[0]
    int32 = kind == "int32"
    y = out[1]
    int4 = w.kind == "int4"
    assert kind in ("int32", "words") or types[y.dtype] == TYPES[kind]
    ctx.step_product(zkb.StepProduct(x=x.data_ptr(), x_stride=x.stride(0), x_scale=0 if int32 else x_scale.data_ptr(), w=w.w.data_ptr(), w_stride=w.w.stride(0) * (2 if int4 else 1), w_type=INT4 if int4 else INT8,
                                     w_scale=0 if int32 else w.scale.data_ptr(), w_scale_stride=w.scale.stride(0) if int4 else 0, group=w.group, out=y.data_ptr(), out_type=TYPES[kind], out_stride=y.stride(0),
                                     n_rows=x.shape[0], n_in=w.n_in, n_out=w.n_out))


def check_product(kind, y, x, x_scale, w):
    """INT32 is exact. Of 8-bit weights: the sum as a float, the product of the scales and the last product are a rounding each. Of 4-bit ones: the sums of 32 codes are
    exact; a sum of n / 32 of them in any order, each a float by itself, is at no point larger than the sum of their sizes, and is off by a rounding of that for each addition."""
    if w.kind == "int8":
        acc = w.values(x)
        if kind == "int32":
            assert torch.equal(y.double(), acc)
            return
        want = acc * x_scale.double()[:, None] * w.scale.double()
        bound = 4 * 2.0 ** -24 * want.abs()
    else:
        want, size = w.values(x)
        want, size = want * x_scale.double()[:, None], size * x_scale.double().abs()[:, None]
        bound = (w.n_in / 32 + 40) * 2.0 ** -24 * size
    if kind != "f32":
        bound = bound + HALF * (want.abs() + bound)
    got = values_of(y) if kind != "f32" else y.double()
    assert bool(((got - want).abs() <= bound + 2.0 ** -133).all()), float(((got - want).abs() - bound).max())


def codes_of(g, rows, n_in, pad=0, off=0):
    keep = torch.randint(-128, 128, (rows * (n_in + pad) + off,), generator=g, device="cuda", dtype=torch.int8)
    return keep[off:].view(rows, n_in + pad)[:, :n_in]


PRODUCT_SIZES = [  # rows, n_in, n_out, pad, off
    (1, 1, 1, 0, 0), (1, 4096, 512, 0, 0), (2, 31, 5, 0, 0), (3, 33, 130, 0, 0), (1, 2000, 333, 0, 1), (5, 130, 129, 14, 0), (8, 512, 256, 0, 0), (9, 1024, 128, 0, 0), (15, 1000, 700, 0, 0), (16, 4096, 384, 0, 0),
    (17, 999, 257, 0, 3), (31, 2048, 136, 0, 0), (33, 160, 1000, 16, 0), (64, 14336, 130, 0, 0), (65, 352, 300, 0, 0), (100, 4095, 200, 0, 0), (128, 640, 640, 0, 16), (130, 97, 129, 0, 0), (200, 1056, 513, 0, 0),
    (257, 512, 384, 0, 0), (300, 8192, 100, 0, 0), (513, 333, 1025, 5, 7), (1000, 768, 900, 0, 0), (2050, 256, 2100, 0, 0), (1, 131071, 40, 0, 0), (70, 20000, 9, 0, 0), (40, 4096, 6144, 0, 0), (600, 64, 4, 0, 0),
]


@gpu
@pytest.mark.parametrize("rows,n_in,n_out,pad,off", PRODUCT_SIZES)
@pytest.mark.parametrize("kind", ["int32", "bf16", "words", "f32"])
def test_product_of_8_bit_weights(ctx, zkb, rows, n_in, n_out, pad, off, kind):
    g = gen(rows + n_in + n_out)
    x, w = codes_of(g, rows, n_in, pad, off), Weights(g, "int8", n_out, n_in, 0, pad, off)
    x_scale = torch.rand(rows, generator=g, device="cuda") + 0.1
    full, y = room(kind, rows, n_out, pad, off)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, (kind, y))
    done(ctx)
    check_product(kind, y, x, x_scale, w)
    untouched(full, y, off)


@gpu
@pytest.mark.parametrize("rows,n_in,n_out,pad,off", PRODUCT_SIZES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", ["bf16", "words", "f32"])
def test_product_of_4_bit_weights(ctx, zkb, rows, n_in, n_out, pad, off, group, kind):
    g = gen(rows + n_in + n_out)
    x, w = codes_of(g, rows, n_in, pad, off), Weights(g, "int4", n_out, n_in, group, pad, off)
    x_scale = torch.rand(rows, generator=g, device="cuda") + 0.1
    full, y = room(kind, rows, n_out, pad, off)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, (kind, y))
    done(ctx)
    check_product(kind, y, x, x_scale, w)
    untouched(full, y, off)


@gpu
@pytest.mark.parametrize("rows", [1, 7, 40, 300])
def test_the_largest_sums_do_not_leave_32_bits(ctx, zkb, rows):
    """Every code -128: 131071 products of 2^14 each."""
    g, n_in, n_out = gen(1), 131071, 130
    x, w = torch.full((rows, n_in + 1), -128, device="cuda", dtype=torch.int8)[:, :n_in], Weights(g, "int8", n_out, n_in, 0, 1)
    w.w.fill_(-128)
    y = torch.zeros(rows, n_out, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, None, w, ("int32", y))
    done(ctx)
    assert bool((y == 131071 * 2 ** 14).all())


@gpu
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 64)])
@pytest.mark.parametrize("rows,n_in,n_out", [(1, 4096, 1000), (16, 14336, 256), (300, 2048, 700)])
def test_products_give_the_same_bits_each_time(ctx, zkb, kind, group, rows, n_in, n_out):
    g = gen(rows)
    x, w, x_scale = codes_of(g, rows, n_in), Weights(g, kind, n_out, n_in, group), torch.rand(rows, generator=g, device="cuda")
    ys = [torch.zeros(rows, n_out, device="cuda") for _ in range(5)]
    torch.cuda.synchronize()
    for y in ys:
        run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    assert all(torch.equal(ys[0], y) for y in ys[1:])


@gpu
@pytest.mark.parametrize("rows", [1, 200])
def test_products_past_32_bits(ctx, zkb, rows):
    """Weights, rows and outputs whose last ones lie more than 2^32 bytes behind the first."""
    g, n_in, n_out = gen(5), 512, 300
    stride = (1 << 32) // (n_out - 1) // 16 * 16 + 512
    room_w = torch.empty(stride * n_out, device="cuda", dtype=torch.int8)
    w = Weights(g, "int8", n_out, n_in)
    at = room_w.view(n_out, stride)
    at[:, :n_in] = w.w
    w.w = at
    x, y = codes_of(g, rows, n_in), torch.zeros(rows, n_out, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, None, w, ("int32", y))
    done(ctx)
    check_product("int32", y, x, None, w)


# ---- log probabilities ---------------------------------------------------------------------------------------------------------------------------
def answer(ctx, zkb, logits, kind, ids, n_top, scale=1.0, off_table=None, entropy=True):
    """logits [row][vocab] as held, with any row stride."""
    rows, vocab = logits.shape
    lp = torch.full((rows, ids.shape[1]), 9.0, device="cuda")
    ent = torch.full((rows,), 9.0, device="cuda")
    top, top_lp = torch.full((rows, n_top), 9, device="cuda", dtype=torch.int32), torch.full((rows, n_top), 9.0, device="cuda")
    torch.cuda.synchronize()
    ctx.step_logprobs(zkb.StepLogprobs(logits=logits.data_ptr(), type=TYPES[kind], logits_stride=logits.stride(0), scale=scale, n_rows=rows, vocab=vocab, ids=ids.data_ptr() if ids.numel() else 0,
                                       n_given=ids.shape[1], logprobs=lp.data_ptr() if ids.numel() else 0, entropy=ent.data_ptr() if entropy else 0, n_top=n_top, top_ids=top.data_ptr() if n_top else 0,
                                       top_logprobs=top_lp.data_ptr() if n_top else 0, off_table=off_table.data_ptr() if off_table is not None else 0))
    done(ctx)
    return lp, ent, top, top_lp


def check_answer(got, x, ids, n_top, scale=1.0):
    """x in 64 bits. z - max and its product with the scale are off by 2^-23 of themselves; a weight by 2^-22 and by 3 * 2^-24 of its exponent, which for weights that count is below
    40; sums by a rounding for each of 64 additions in a thread and a hundred across: all terms of a log probability, and of the entropy, have one sign, so 2^-15 of the result
    covers them. Weights below 2^-126 count for nothing: 2^-100."""
    lp, ent, top, top_lp = got
    scale = float(np.float32(scale))
    for t in range(x.shape[0]):
        z = x[t] * scale
        odd, none = bool((torch.isnan(z) | (z == math.inf)).any()), bool((z == -math.inf).all())
        if odd:
            assert bool(torch.isnan(ent[t])) and bool((top[t] == -1).all()) and bool(torch.isnan(top_lp[t]).all())
            inside = (ids[t] >= 0) & (ids[t] < x.shape[1])
            assert bool(torch.isnan(lp[t][inside]).all()) and bool((lp[t][~inside] == 0).all())
            continue
        d = z - z.max() if not none else z
        w = torch.exp(d)
        at = int(torch.argmax(d))
        others = w.sum() - w[at] if not none else w.sum()
        rest = torch.cat([w[:at], w[at + 1:]]).sum() if not none else others
        log = torch.log1p(rest) if not none else torch.zeros_like(rest)
        want = d - log
        want_ent = 0.0 if none else float(log - (w * torch.where(w > 0, d, 0.0)).sum() / w.sum())
        assert abs(float(ent[t]) - want_ent) <= 2.0 ** -15 * want_ent + 2.0 ** -100, (t, float(ent[t]), want_ent)
        for i, id in enumerate(ids[t].tolist()):
            ref = float(want[id]) if 0 <= id < x.shape[1] else 0.0
            assert float(lp[t, i]) == ref or abs(float(lp[t, i]) - ref) <= 2.0 ** -15 * abs(ref) + 2.0 ** -100, (t, id, float(lp[t, i]), ref)
        order = torch.sort(x[t] + 0.0, descending=True, stable=True).indices
        order = order[x[t][order] > -math.inf][:n_top]
        assert top[t, :len(order)].tolist() == order.tolist(), (t, top[t].tolist(), order.tolist())
        assert bool(((top_lp[t, :len(order)].double() - want[order]).abs() <= 2.0 ** -15 * want[order].abs() + 2.0 ** -100).all())
        assert bool((top[t, len(order):] == -1).all()) and bool((top_lp[t, len(order):] == -math.inf).all())


def held_logits(x, kind, pad=0, off=0):
    """x as it is held, and what that stands for in 64 bits."""
    held = x if kind == "f32" else words(x.bfloat16()) | 0x12340000 if kind == "words" else x.bfloat16()
    r = torch.full((x.shape[0] * (x.shape[1] + pad) + off,), 33, device="cuda", dtype=held.dtype)
    view = r[off:].view(x.shape[0], x.shape[1] + pad)[:, :x.shape[1]]
    view.copy_(held)
    return view, (x if kind == "f32" else x.bfloat16()).double()


LOGIT_CASES = [(1, 1, 1), (2, 2, 3), (3, 7, 5), (40, 100, 5), (1, 32000, 8), (2, 32003, 20), (5, 50001, 1), (17, 4096, 32), (33, 33000, 5), (300, 1001, 5), (9, 131072, 6), (150, 20000, 0), (1, 1 << 19, 32), (80, (1 << 17) + 5, 9),
               (1, 4097, 32), (20, 40000, 32), (700, 129, 32), (1, 65, 32)]


@gpu
@pytest.mark.parametrize("rows,vocab,n_top", LOGIT_CASES)
@pytest.mark.parametrize("kind", ["bf16", "words", "f32"])
@pytest.mark.parametrize("pad,off", [(0, 0), (1, 3), (5, 0)])
def test_logprobs(ctx, zkb, rows, vocab, n_top, kind, pad, off):
    g = gen(rows + vocab)
    x = 3 * torch.randn(rows, vocab, generator=g, device="cuda")
    x[:, vocab // 2] += 30 * torch.rand(rows, generator=g, device="cuda")
    ids = torch.randint(-1, vocab + 1, (rows, 3), generator=g, device="cuda", dtype=torch.int32)
    ids[0, 0], ids[0, 1], ids[0, 2] = vocab // 2, -(2 ** 31), 2 ** 31 - 1
    held, values = held_logits(x, kind, pad, off)
    count = torch.zeros(1, device="cuda", dtype=torch.int64)
    got = answer(ctx, zkb, held, kind, ids, n_top, 1.25, count)
    few = slice(0, rows) if rows < 60 else slice(0, rows, rows // 40)
    check_answer(tuple(y[few] for y in got), values[few], ids[few], n_top, 1.25)
    assert int(count) == int(((ids < 0) | (ids >= vocab)).sum())


@gpu
@pytest.mark.parametrize("kind", ["bf16", "words", "f32"])
@pytest.mark.parametrize("vocab", [50, 3000, 32000, 100003])
@pytest.mark.parametrize("rows", [12, 320])
def test_logprobs_of_rows_that_are_masked_equal_and_no_numbers(ctx, zkb, kind, vocab, rows):
    """Rows: nothing left; one token left; all equal; zeros of both signs; a few distinct values; the type's lowest value beside others and alone; ascending; descending; a NaN; +infinity;
    one token all but certain."""
    g = gen(vocab)
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    lowest = torch.finfo(torch.bfloat16).min
    i = torch.arange(vocab, device="cuda").float()
    for t, row in enumerate((torch.full((vocab,), -math.inf), torch.where(i == vocab - 1, 2.0, -math.inf), torch.full((vocab,), 1.5), torch.where(i % 3 == 1, -0.0, 0.0), (i * 7 % 5 == 2).float(),
                             torch.where(i % 2 == 0, lowest, x[5]), torch.full((vocab,), lowest), i, -i)):
        x[t] = row.cuda()
    x[9, vocab // 3], x[10, vocab - 2], x[11] = math.nan, math.inf, x[11].clamp(max=3) + torch.where(i == 5, 40.0, 0.0)
    if rows > 12:
        x[12:] = x[:12].repeat(-(-rows // 12), 1)[12:rows]
    ids = torch.tensor([[0, vocab - 1, vocab // 3, 5, -1]], device="cuda", dtype=torch.int32).expand(rows, -1).contiguous()
    held, values = held_logits(x, kind, 3, 1)
    for n_top, scale in ((5, 1.0), (32, 0.7), (0, 1e-30)):
        got = answer(ctx, zkb, held, kind, ids, n_top, scale)
        some = list(range(12)) + [rows - 1]
        check_answer(tuple(y[some] for y in got), values[some], ids[some], n_top, scale)


@gpu
def test_logprobs_where_nothing_is_asked(ctx, zkb):
    x = torch.randn(3, 100, generator=gen(0), device="cuda")
    lp, ent, top, top_lp = answer(ctx, zkb, x, "f32", torch.zeros(3, 0, device="cuda", dtype=torch.int32), 0, entropy=False)
    assert bool((ent == 9).all())


@gpu
def test_logits_past_32_bits(ctx, zkb):
    stride = (1 << 30) + 12
    r = torch.empty(2 * stride, device="cuda", dtype=torch.float32)
    x = r.view(2, stride)[:, :3001]
    x.copy_(torch.randn(2, 3001, generator=gen(2), device="cuda"))
    ids = torch.tensor([[5], [3000]], device="cuda", dtype=torch.int32)
    check_answer(answer(ctx, zkb, x, "f32", ids, 4), x.double(), ids, 4)


# ---- a layer -----------------------------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("weights,group", [("int8", 0), ("int4", 64)])
@pytest.mark.parametrize("rows,before", [(1, 90), (32, 40), (150, 0)])
def test_a_layer_and_an_answer(ctx, zkb, weights, group, rows, before):
    """A decoder layer and the output head on one stream, nothing waits in between; each call against its definition on what it was given."""
    g, d, hq, hk, inner, vocab = gen(rows), 32, 4, 2, 320, 1003
    width, heads = hq * d, hq + 2 * hk
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    blank = lambda dtype, *s: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    bf, i8, f32 = torch.bfloat16, torch.int8, torch.float32
    batch, cache = Batch([(rows, before + rows)]), Cache(g, "int8", 1, hk, before + rows + 3, d)
    table, table_scale = torch.randint(-127, 128, (vocab, width), generator=g, device="cuda", dtype=i8), (0.5 + torch.rand(vocab, generator=g, device="cuda")) / 100
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    w_qkv, w_o, w_up, w_down, w_head = (Weights(g, weights, n, k, group) for n, k in ((heads * d, width), (width, width), (2 * inner, width), (width, inner), (vocab, width)))
    norms = [(1 + 0.2 * rand(width)).bfloat16() for _ in range(3)]
    qk_norm = [(1 + 0.2 * rand(d)).bfloat16() for _ in range(2)]
    freq = 1e4 ** (-np.arange(d // 2) / (d // 2))
    h, qkv, q, att, o, up, down, h1, h2, h3 = (blank(bf, rows, n) for n in (width, heads * d, width, width, width, 2 * inner, width, width, width, width))
    code, scale = [blank(i8, rows, n) for n in (width, width, width, inner, width)], [blank(f32, rows) for _ in range(5)]
    logits, lp, ent = blank(f32, rows, vocab), blank(f32, rows, 1), blank(f32, rows)
    top, top_lp = blank(torch.int32, rows, 4), blank(f32, rows, 4)
    next_ids = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()

    def norm(x, residual, summed, weight, i):
        ctx.step_residual_norm(zkb.StepResidualNorm(x=x.data_ptr(), x_stride=width, residual=residual.data_ptr() if residual is not None else 0, residual_stride=width, sum_out=summed.data_ptr(), sum_stride=width,
                                                    weight=weight.data_ptr(), out=code[i].data_ptr(), out_type=INT8, out_scale=scale[i].data_ptr(), out_stride=width, n_rows=rows, width=width, eps=1e-5))

    ctx.step_embed(zkb.StepEmbed(ids=ids.data_ptr(), table=table.data_ptr(), row_scale=table_scale.data_ptr(), out=h.data_ptr(), table_stride=width, out_stride=width, n_tokens=rows, vocab=vocab, width=width,
                                 table_type=INT8, out_type=BF16, scale=1.0))
    norm(h, None, h1, norms[0], 0)
    run_product(ctx, zkb, code[0], scale[0], w_qkv, ("bf16", qkv))
    at = lambda n: qkv.data_ptr() + 2 * n * d  # noqa: E731
    ctx.step_norm_rope(zkb.StepNormRope(cache=cache.args(zkb), rows=batch.args(zkb), q=at(0), k=at(hq), v=at(hq + hk), q_weight=qk_norm[0].data_ptr(), k_weight=qk_norm[1].data_ptr(), h_inv_freq=freq.ctypes.data,
                                        q_out=q.data_ptr(), q_stride=heads * d, k_stride=heads * d, v_stride=heads * d, head_stride=d, q_out_stride=width, q_out_head_stride=d, type=BF16, q_heads=hq, rotary_dim=d,
                                        eps=1e-6))
    ctx.step_attention(zkb.StepAttention(cache=cache.args(zkb), rows=batch.args(zkb), q=q.data_ptr(), out=att.data_ptr(), q_stride=width, q_head_stride=d, out_stride=width, out_head_stride=d, q_heads=hq,
                                         out_type=BF16, scale=d ** -0.5))
    ctx.step_gate(zkb.StepGate(x=att.data_ptr(), x_stride=width, out=code[1].data_ptr(), out_type=INT8, out_scale=scale[1].data_ptr(), out_stride=width, n_rows=rows, width=width))
    run_product(ctx, zkb, code[1], scale[1], w_o, ("bf16", o))
    norm(o, h1, h2, norms[1], 2)
    run_product(ctx, zkb, code[2], scale[2], w_up, ("bf16", up))
    ctx.step_gate(zkb.StepGate(gate=up.data_ptr(), gate_stride=2 * inner, x=up.data_ptr() + 2 * inner, x_stride=2 * inner, out=code[3].data_ptr(), out_type=INT8, out_scale=scale[3].data_ptr(), out_stride=inner,
                               n_rows=rows, width=inner))
    run_product(ctx, zkb, code[3], scale[3], w_down, ("bf16", down))
    norm(down, h2, h3, norms[2], 4)
    run_product(ctx, zkb, code[4], scale[4], w_head, ("f32", logits))
    ctx.step_logprobs(zkb.StepLogprobs(logits=logits.data_ptr(), type=F32, logits_stride=vocab, scale=1.0, n_rows=rows, vocab=vocab, ids=next_ids.data_ptr(), n_given=1, logprobs=lp.data_ptr(),
                                       entropy=ent.data_ptr(), n_top=4, top_ids=top.data_ptr(), top_logprobs=top_lp.data_ptr()))
    done(ctx)
    assert torch.equal(h, (table[ids.long()].float() * table_scale[ids.long()][:, None]).bfloat16()) and torch.equal(h1, h)
    check_out(code[0], scale[0], "codes", norm_reference(h, norms[0], 1e-5), 2.0 ** -18)
    check_product("bf16", qkv, code[0], scale[0], w_qkv)
    y, size = rope_reference(batch, qkv.view(rows, heads, d)[:, :hq + hk], [qk_norm[0]] * hq + [qk_norm[1]] * hk, 1e-6, freq, 0)
    assert bool(((q.view(rows, hq, d).double() - y[:, :hq]).abs() <= HALF * y[:, :hq].abs() + 2.0 ** -18 * size[:, :hq]).all())
    ref, bound = attention_reference(batch, cache, q.view(rows, hq, d), d ** -0.5, 0, 0)
    assert bool(((att.view(rows, hq, d).double() - ref).abs() <= bound).all())
    check_out(code[1], scale[1], "codes", att.double(), 0.0)
    check_product("bf16", o, code[1], scale[1], w_o)
    assert torch.equal(h2, (h1.float() + o.float()).bfloat16())
    check_out(code[2], scale[2], "codes", norm_reference(h2, norms[1], 1e-5), 2.0 ** -18)
    check_product("bf16", up, code[2], scale[2], w_up)
    a, b = up[:, :inner].double(), up[:, inner:].double()
    check_out(code[3], scale[3], "codes", b * a / (1 + torch.exp(-a)), (6 + 1.2 * a.abs()) * 2.0 ** -23)
    check_product("bf16", down, code[3], scale[3], w_down)
    assert torch.equal(h3, (h2.float() + down.float()).bfloat16())
    check_out(code[4], scale[4], "codes", norm_reference(h3, norms[2], 1e-5), 2.0 ** -18)
    check_product("f32", logits, code[4], scale[4], w_head)
    check_answer((lp, ent, top, top_lp), logits.double(), next_ids, 4)


@gpu
def test_accumulators_between_norm_and_dequantize(ctx, zkb, oracle):
    """As a proof makes its values: codes of a norm, their exact products as the accumulators of zkb_witness_dequant, and what that leaves (words, tokens and channel blocks descending)
    read as the next rows of the residual stream."""
    from zk_inference_prover_b200 import witness_cases as wc

    g, tokens, chunks, per_row, width = gen(8), 32, 8, 32, 512
    n_out = chunks * per_row
    dq = wc.dequant_case(3, 1, tokens, chunks, per_row, 13, 1, 1)
    cfg, rows = dq["cfg"], dq["rows"]
    x, weight, w = torch.randn(tokens, width, generator=g, device="cuda").bfloat16(), (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).bfloat16(), Weights(g, "int8", n_out, width)
    code, scale, acc = torch.zeros(tokens, width, device="cuda", dtype=torch.int8), torch.zeros(tokens, device="cuda"), torch.zeros(tokens, n_out, device="cuda", dtype=torch.int32)
    h, h_next, y = torch.randn(tokens, n_out, generator=g, device="cuda").bfloat16(), torch.zeros(tokens, n_out, device="cuda", dtype=torch.bfloat16), torch.zeros(tokens, n_out, device="cuda", dtype=torch.bfloat16)
    sx, sw = (ctx.upload_bytes(np.ascontiguousarray(dq[k])) for k in ("sx", "sw"))
    norm3, mul2 = ctx.upload(dq["norm3"].reshape(-1)), ctx.upload(dq["mul2"].reshape(-1))
    base, pre = [ctx.alloc(rows).zero() for _ in range(dq["n_base"])], [ctx.alloc(rows).zero() for _ in range(dq["n_pre"])]
    ms = [ctx.alloc(cfg[k]).zero() for k in ("n_norm", "n_frac", "n_mul", "n_r8")]
    counts, want = ctx.alloc(4).zero(), ctx.alloc(rows * per_row).zero()
    torch.cuda.synchronize()
    ctx.step_residual_norm(zkb.StepResidualNorm(x=x.data_ptr(), x_stride=width, weight=weight.data_ptr(), out=code.data_ptr(), out_type=INT8, out_scale=scale.data_ptr(), out_stride=width, n_rows=tokens, width=width,
                                                eps=1e-5))
    run_product(ctx, zkb, code, None, w, ("int32", acc))
    ctx.witness_dequant(cfg, acc.data_ptr(), 0, 0, sx.ptr, sw.ptr, norm3.ptr, mul2.ptr, [b.ptr for b in base], [p.ptr for p in pre], *[m.ptr for m in ms], counts.ptr, want.ptr)
    ctx.step_residual_norm(zkb.StepResidualNorm(x=want.ptr + 4 * per_row * (tokens * chunks - 1), x_type=WORD, x_stride=-n_out, x_segment=per_row, x_segment_stride=-per_row, residual=h.data_ptr(),
                                                residual_stride=n_out, sum_out=h_next.data_ptr(), sum_stride=n_out, out=y.data_ptr(), out_type=BF16, out_stride=n_out, n_rows=tokens, width=n_out, eps=1e-5))
    done(ctx)
    check_out(code, scale, "codes", norm_reference(x, weight, 1e-5), 2.0 ** -18)
    check_product("int32", acc, code, None, w)
    o = oracle.witness_dequant(acc.cpu().numpy(), dq["jx"], dq["jw"], dq["sx"], dq["sw"], dq["norm3"], dq["mul2"], dq["n_base"], dq["n_pre"], cfg)
    given = want.download()[:rows * per_row]
    assert np.array_equal(given, np.asarray(o["want"]).reshape(-1))
    came = (torch.from_numpy(given.astype(np.int32)).cuda().view(tokens, chunks, per_row).flip(0, 1).reshape(tokens, n_out) << 16).view(torch.float32)
    finite = torch.isfinite(came).all(-1)
    s = (h.float() + came).bfloat16()
    assert torch.equal(h_next[finite], s[finite]) and int(finite.sum()) > 0
    check_out(y[finite], None, "bf16", norm_reference(s[finite], None, 1e-5), 2.0 ** -18)


class Answer:
    """A norm, a product and the log probabilities of what they leave, described once."""

    def __init__(self, zkb, seed, rows, width=256, vocab=999):
        g = gen(seed)
        self.x, self.h = (torch.randn(rows, width, generator=g, device="cuda").bfloat16() for _ in range(2))
        self.s, self.code, self.scale = torch.zeros_like(self.x), torch.zeros(rows, width, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")
        self.w, self.logits = Weights(g, "int4" if seed % 2 else "int8", vocab, width, 64 if seed % 2 else 0), torch.zeros(rows, vocab, device="cuda")
        self.ids = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda", dtype=torch.int32)
        self.out = torch.zeros(rows, 1, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(rows, 5, device="cuda", dtype=torch.int32), torch.zeros(rows, 5, device="cuda")
        lp, ent, top, top_lp = self.out
        self.norm = zkb.StepResidualNorm(x=self.x.data_ptr(), x_stride=width, residual=self.h.data_ptr(), residual_stride=width, sum_out=self.s.data_ptr(), sum_stride=width, out=self.code.data_ptr(), out_type=INT8,
                                         out_scale=self.scale.data_ptr(), out_stride=width, n_rows=rows, width=width, eps=1e-5)
        self.answer = zkb.StepLogprobs(logits=self.logits.data_ptr(), type=F32, logits_stride=vocab, scale=1.0, n_rows=rows, vocab=vocab, ids=self.ids.data_ptr(), n_given=1, logprobs=lp.data_ptr(),
                                       entropy=ent.data_ptr(), n_top=5, top_ids=top.data_ptr(), top_logprobs=top_lp.data_ptr())
        self.zkb = zkb
        torch.cuda.synchronize()

    def run(self, ctx):
        ctx.step_residual_norm(self.norm)
        run_product(ctx, self.zkb, self.code, self.scale, self.w, ("f32", self.logits))
        ctx.step_logprobs(self.answer)

    def check(self):
        s = (self.x.float() + self.h.float()).bfloat16()
        assert torch.equal(self.s, s)
        check_out(self.code, self.scale, "codes", norm_reference(s, None, 1e-5), 2.0 ** -18)
        check_product("f32", self.logits, self.code, self.scale, self.w)
        check_answer(self.out, self.logits.double(), self.ids, 5)


@gpu
@pytest.mark.parametrize("rows", [1, 40, 140])
def test_captured_answers_side_by_side(ctx, zkb, rows):
    """Two graphs of one context's calls, replayed side by side on other streams with other inputs: no workspace is shared."""
    a, b = Answer(zkb, 1, rows), Answer(zkb, 2, rows)
    stream = torch.cuda.ExternalStream(ctx.stream())
    graphs = []
    for one in (a, b):
        one.run(ctx)  # (kernels' attributes are set before a capture)
        ctx.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            one.run(ctx)
        graphs.append(graph)
    others = [torch.cuda.Stream() for _ in graphs]
    for turn in range(3):
        for one in (a, b):
            one.x.copy_(torch.randn(one.x.shape, generator=gen(50 + turn), device="cuda"))
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, s in zip(graphs, others):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        a.check(), b.check()


@gpu
def test_layer_calls_of_contexts_on_threads(zkb):
    import threading

    contexts, steps, wrong = [zkb.Context(device=0, max_log_size=10) for _ in range(3)], [Answer(zkb, 10 + i, (1, 33, 140)[i]) for i in range(3)], []

    def work(c, s):
        try:
            for _ in range(20):
                s.run(c)
            c.sync()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(contexts, steps)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for s in steps:
        s.check()
    for c in contexts:
        c.close()
