"""Norms and gates (zkb_step_residual_norm, zkb_step_gate) of values at the ends of the 32-bit floats."""
import math

import pytest
import torch

from test_step_layer import HALF, INT8, TYPES, check_out, norm_reference, room
from test_step_layer import values_of
from test_step_values import done, gen

gpu = pytest.mark.gpu


def norms(ctx, zkb, x, w, kind, eps):
    rows, width = x.shape
    full, got = room(kind, rows, width)
    scale = torch.zeros(rows, device="cuda") if kind == "codes" else None
    torch.cuda.synchronize()
    ctx.step_residual_norm(zkb.StepResidualNorm(x=x.data_ptr(), x_stride=width, weight=w.data_ptr(), out=got.data_ptr(), out_type=TYPES[kind], out_scale=scale.data_ptr() if scale is not None else 0,
                                                out_stride=width, n_rows=rows, width=width, eps=eps))
    done(ctx)
    return got, scale


@gpu
@pytest.mark.parametrize("kind", ["codes", "bf16", "words"])
@pytest.mark.parametrize("width", [64, 777, 4096, 20000])
@pytest.mark.parametrize("small", [-7, -9, -12, -20, -44, -60])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -60])
def test_weights_of_unlike_sizes(ctx, zkb, kind, width, small, eps):
    """Small rows with weights of which one is near 1 and others are so small that values times them have few bits in 32, or none, though the norm has all. A norm in 32 bits is off by
    2^-18 (test_residual_norm); where products were taken at up to 2^10 times less than the norm they are off by 2^-150 each, of the least bf16 steps, 2^-133, by 2^-7."""
    g = gen(width)
    x = (torch.randn(7, width, generator=g, device="cuda") * 2.0 ** small).bfloat16()
    x[0] = 2.0 ** small
    w = ((1 + torch.rand(width, generator=g, device="cuda")) * torch.exp2(-140.0 * torch.rand(width, generator=g, device="cuda").double())).bfloat16()
    w[0], w[1], w[2] = 1.0, 1.297 * 2.0 ** -101, 1.3 * 2.0 ** -126
    got, scale = norms(ctx, zkb, x, w, kind, eps)
    y = norm_reference(x, w, eps)
    if kind == "codes":
        check_out(got, scale, kind, y, 2.0 ** -18)
    else:
        assert bool(((values_of(got) - y).abs() <= (HALF + 2.0 ** -17) * y.abs() + (0.5 + 2.0 ** -7) * 2.0 ** -133).all())


@gpu
@pytest.mark.parametrize("source,width", [("bf16", 64), ("bf16", 333), ("words", 4096), ("words", 77)])
@pytest.mark.parametrize("kind", ["codes", "bf16", "words"])
def test_gates_of_minus_infinity_are_closed(ctx, zkb, source, width, kind):
    """0 below -87, down to -infinity; x that are no numbers and gates that are NaN stay what they are."""
    from step_cases import words

    g = gen(width)
    x, a = (torch.randn(4, width, generator=g, device="cuda").bfloat16() for _ in range(2))
    a[0, ::3], a[1], a[2, 5], a[3, 7] = -math.inf, -math.inf, math.nan, -math.inf
    x[3, 7] = math.inf
    out, scale = room(kind, 4, width)[1], torch.full((4,), -1.0, device="cuda")
    xs, gs = (words(v) if source == "words" else v for v in (x, a))
    torch.cuda.synchronize()
    ctx.step_gate(zkb.StepGate(gate=gs.data_ptr(), gate_stride=width, x=xs.data_ptr(), x_stride=width, x_type=TYPES[source], out=out.data_ptr(), out_type=TYPES[kind],
                               out_scale=scale.data_ptr() if kind == "codes" else 0, out_stride=width, n_rows=4, width=width))
    done(ctx)
    d = a.double()
    y = x.double() * torch.where(d == -math.inf, 0.0, d / (1 + torch.exp(-d)))
    rel = (6 + 1.2 * d.abs().clamp(max=87)) * 2.0 ** -23
    rows = slice(0, 2)
    check_out(out[rows], scale[rows] if kind == "codes" else None, kind, y[rows], rel[rows])
    if kind == "codes":
        assert bool(torch.isnan(scale[2:]).all()) and not bool(out[2:].any()) and scale[1] == 0
    else:
        assert bool(torch.equal(torch.isnan(values_of(out)), torch.isnan(y)))


def codes_to_even(y):
    """y * 127 / max|y| of rows in 64 bits that hold 127 y exactly, rounded to nearest even without a rounding on the way, and how far from halfway between two codes (a quotient of
    exact numbers) each one is."""
    size, most = 127 * y.abs(), y.abs().amax(-1, keepdim=True)
    k = torch.floor(size / most)
    k = k - (k * most > size).double()
    k = k + ((k + 1) * most <= size).double()
    twice = 2 * (size - k * most) - most  # exact: of 24 bits each
    up = (twice > 0) | ((twice == 0) & (k % 2 == 1))
    return torch.sign(y) * (k + up.double()), (twice / most).abs()


@gpu
@pytest.mark.parametrize("rows,width,source", [(700, 64, "bf16"), (33, 4096, "bf16"), (9, 777, "words"), (650, 1000, "words"), (64, 14336, "bf16")])
def test_values_halfway_between_two_codes_go_to_the_even_one(ctx, zkb, rows, width, source):
    """Rows of bf16 values whose largest has few bits hold many. A value of c codes that is not halfway is 2^-17 c and more from it (eight bits over eight), and the kernel's error is 2^-23 c at most: all
    codes are those of the definition."""
    from step_cases import words

    g = gen(width)
    x = torch.randn(rows, width, generator=g, device="cuda").bfloat16()
    top = torch.tensor([1, 3, 5, 7, 96, 127, 255, 129], device="cuda").float()[torch.arange(rows, device="cuda") % 8] * torch.exp2(torch.arange(rows, device="cuda") % 40 - 20.0)
    x = (x.float() / x.float().abs().amax(-1, keepdim=True) * top[:, None]).bfloat16()
    x[:, 5] = -top.bfloat16()
    held = words(x) if source == "words" else x
    out, scale = room("codes", rows, width)[1], torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ctx.step_gate(zkb.StepGate(x=held.data_ptr(), x_stride=width, x_type=TYPES[source], out=out.data_ptr(), out_type=INT8, out_scale=scale.data_ptr(), out_stride=width, n_rows=rows, width=width))
    done(ctx)
    want, far = codes_to_even(x.double())
    assert int((far == 0).sum()) > 10
    assert torch.equal(out.double(), want)


@gpu
@pytest.mark.parametrize("rows,width", [(700, 64), (33, 4096), (9, 777), (64, 14336), (2000, 4096)])
def test_norms_halfway_between_two_codes_go_to_the_even_one(ctx, zkb, rows, width):
    """Products of bf16 values and weights, sixteen bits over sixteen: what is not halfway may be as near to it as the kernel's error, 2^-23 of 127 codes."""
    g = gen(width)
    x, w = torch.randn(rows, width, generator=g, device="cuda").clamp(-3, 3), 1 + 0.2 * torch.randn(width, generator=g, device="cuda")
    w[::2] = 3.0
    x[:, 0], x[:, 2], x[:, 4], x[:, 6] = 8.0, 4.0, -4.0, -2.0  # the largest is 24; 12 is half of it
    x[1::2] = torch.randint(-200, 200, (rows // 2, width), generator=g, device="cuda").float()  # the largest is 762, six times 127: odd ones times 3 are halfway
    x[1::2, 0] = 254.0
    x[1::2, 1::2] *= 0.125
    x, w = x.bfloat16(), w.bfloat16()
    got, scale = norms(ctx, zkb, x, w, "codes", 1e-5)
    want, far = codes_to_even(x.double() * w.double())
    assert int((far == 0).sum()) >= 2 * rows
    off = got.double() != want
    assert not bool((off & ((far == 0) | (far > 2.0 ** -15))).any()), (int(off.sum()), int((off & (far == 0)).sum()))
