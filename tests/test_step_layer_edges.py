"""Calls between a step's attention and its answer that other tests do not make: refused clusters, scales and values that are no numbers, rows after rows of one thread block, more
questions than threads, the borders of the rules that choose a kernel."""
import math

import pytest
import torch

from test_step_layer import (INT8, TYPES, Rows, Weights, answer, check_answer, check_out, check_product, codes_of, held_logits, norm_reference, room, run_product, untouched, values_of)
from test_step_values import done, gen

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("most", [1, 2, 8])
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 128), ("int4", 32)])
@pytest.mark.parametrize("rows,n_in,n_out", [(20, 4096, 300), (40, 8192, 130), (64, 3000, 256), (17, 700, 100)])
def test_products_whose_clusters_are_refused(ctx, zkb, monkeypatch, most, kind, group, rows, n_in, n_out):
    monkeypatch.setenv("ZKB_STEP_CLUSTERS", str(most))
    g = gen(rows)
    x, w, x_scale = codes_of(g, rows, n_in), Weights(g, kind, n_out, n_in, group), torch.rand(rows, generator=g, device="cuda") + 0.1
    y = torch.zeros(rows, n_out, device="cuda")
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    check_product("f32", y, x, x_scale, w)


@gpu
@pytest.mark.parametrize("most", [1, 2, 8])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_logprobs_whose_clusters_are_refused(ctx, zkb, monkeypatch, most, kind):
    monkeypatch.setenv("ZKB_STEP_CLUSTERS", str(most))
    g = gen(most)
    held, values = held_logits(3 * torch.randn(2, 200001, generator=g, device="cuda"), kind)
    ids = torch.randint(0, 200001, (2, 2), generator=g, device="cuda", dtype=torch.int32)
    check_answer(answer(ctx, zkb, held, kind, ids, 32), values, ids, 32)


@gpu
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 32), ("int4", 64), ("int4", 128)])
@pytest.mark.parametrize("rows", [1, 2, 5, 13, 30, 60, 140, 300])
@pytest.mark.parametrize("pad", [0, 1])
def test_scales_that_are_no_numbers_stay_with_their_outputs(ctx, zkb, kind, group, rows, pad):
    """Of one output's weights, of one of its groups, of one row: what they do not scale has the same bits as without them."""
    g, n_in, n_out = gen(rows), 1024, 300
    x, w, x_scale = codes_of(g, rows, n_in, pad), Weights(g, kind, n_out, n_in, group, pad), torch.rand(rows, generator=g, device="cuda") + 0.1
    clean, y = torch.zeros(rows, n_out, device="cuda"), torch.zeros(rows, n_out, device="cuda")
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, ("f32", clean))
    done(ctx)
    check_product("f32", clean, x, x_scale, w)
    if kind == "int8":
        w.scale[7], w.scale[131] = math.nan, math.inf
    else:
        w.scale[7, n_in // group - 1], w.scale[131, 1], w.scale[200, n_in // group:] = math.nan, math.inf, math.nan
    x_scale[rows - 1] = math.nan if rows > 1 else x_scale[0]
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    odd = torch.zeros(rows, n_out, device="cuda", dtype=torch.bool)
    odd[:, 7] = odd[:, 131] = True
    if rows > 1:
        odd[rows - 1] = True
    assert torch.equal(y[~odd], clean[~odd]) and not bool(torch.isfinite(y[odd]).any())


@gpu
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 32), ("int4", 64), ("int4", 128)])
@pytest.mark.parametrize("rows", [2, 3, 4, 8, 9, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_products_at_the_borders_between_kernels(ctx, zkb, kind, group, rows):
    g = gen(rows)
    for n_in, n_out, pad in ((512, 260, 0), (513, 130, 0), (96, 4200, 3)):
        x, w, x_scale = codes_of(g, rows, n_in, pad), Weights(g, kind, n_out, n_in, group, pad), torch.rand(rows, generator=g, device="cuda") + 0.1
        full, y = room("f32", rows, n_out, 2)
        torch.cuda.synchronize()
        run_product(ctx, zkb, x, x_scale, w, ("f32", y))
        done(ctx)
        check_product("f32", y, x, x_scale, w)
        untouched(full, y, 0)


@gpu
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 64)])
def test_products_of_more_tiles_than_the_gpu_holds(ctx, zkb, kind, group):
    """Thread blocks that have one tile after the other, with and without the tensor memory unit's copies."""
    g = gen(9)
    for rows, n_in, n_out in ((3000, 384, 4000), (2999, 385, 3001), (20, 256, 40000), (50, 300, 20000)):
        x, w, x_scale = codes_of(g, rows, n_in), Weights(g, kind, n_out, n_in, group), torch.rand(rows, generator=g, device="cuda") + 0.1
        y = torch.zeros(rows, n_out, device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        run_product(ctx, zkb, x, x_scale, w, ("bf16", y))
        done(ctx)
        check_product("bf16", y, x, x_scale, w)


@gpu
def test_two_rows_and_weights_that_share_their_memory(ctx, zkb):
    """Rows that overlap one another are read alone: each begins 16 codes behind the one before; outputs' weights all the same."""
    g, n_in = gen(4), 256
    line, w = torch.randint(-128, 128, (n_in + 16 * 40,), generator=g, device="cuda", dtype=torch.int8), Weights(g, "int8", 130, n_in)
    x = torch.stack([line[16 * t:16 * t + n_in] for t in range(40)])
    y = torch.zeros(40, 130, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    with pytest.raises(zkb.ZkbError, match="x_stride"):  # a stride shorter than a row is refused
        ctx.step_product(zkb.StepProduct(x=line.data_ptr(), x_stride=16, w=w.w.data_ptr(), w_stride=n_in, w_type=INT8, out=y.data_ptr(), out_type=TYPES["int32"], out_stride=130, n_rows=40, n_in=n_in, n_out=130))
    run_product(ctx, zkb, x, None, w, ("int32", y))
    done(ctx)
    check_product("int32", y, x, None, w)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "words", "f32"])
@pytest.mark.parametrize("rows,vocab,n_top", [(1300, 4000, 32), (1500, 3001, 0), (700, 8001, 7), (400, 16001, 1), (330, 32768 - 9, 20)])
def test_logprobs_of_row_after_row(ctx, zkb, kind, rows, vocab, n_top):
    """More rows than the GPU holds at once: every border between a thread block's rows. Some rows are masked, some all equal (too many ties for a list), some hold a NaN."""
    g = gen(rows)
    x = 2 * torch.randn(rows, vocab, generator=g, device="cuda")
    x[::7] = 0.5
    x[1::7, vocab // 3:] = -math.inf
    x[2::7, 11] = math.nan
    x[3::7] = -math.inf
    x[4::7, vocab - 1] = 60.0
    held, values = held_logits(x, kind, 1, 1)
    ids = torch.randint(-1, vocab, (rows, 2), generator=g, device="cuda", dtype=torch.int32)
    count = torch.zeros(1, device="cuda", dtype=torch.int64)
    got = answer(ctx, zkb, held, kind, ids, n_top, 1.0, count)
    again = answer(ctx, zkb, held, kind, ids, n_top)
    assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(got, again))
    some = list(range(0, 14)) + list(range(rows - 14, rows)) + list(range(290, 304))
    check_answer(tuple(y[some] for y in got), values[some], ids[some], n_top)
    assert int(count) == int((ids < 0).sum())


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 50), (3, 40000), (1300, 4000)])
def test_more_tokens_are_asked_for_than_there_are_threads(ctx, zkb, rows, vocab):
    g = gen(vocab)
    held, values = held_logits(3 * torch.randn(rows, vocab, generator=g, device="cuda"), "bf16")
    ids = torch.randint(0, vocab, (rows, 1700), generator=g, device="cuda", dtype=torch.int32)
    ids[:, 1] = ids[:, 0]  # the same one twice
    lp = answer(ctx, zkb, held, "bf16", ids, 2)[0]
    want = torch.log_softmax(values, -1).gather(1, ids.long())
    assert bool(((lp.double() - want).abs() <= 2.0 ** -15 * want.abs() + 2.0 ** -100).all()) and torch.equal(lp[:, 0], lp[:, 1])


@gpu
def test_gates_that_are_no_numbers_and_far_from_zero(ctx, zkb):
    """The limits of g / (1 + exp(-g)): g itself, and 0 below -87, where the factor is less than 10^-35 in size."""
    gates = torch.tensor([0.0, -0.0, 100.0, 3e38, math.inf, -100.0, -87.5, -3e38, math.nan, 1e-30, -1e-30, -80.0], device="cuda").bfloat16().repeat(4)[None]
    x = torch.full_like(gates, 2.0)
    out = torch.zeros_like(gates)
    torch.cuda.synchronize()
    ctx.step_gate(zkb.StepGate(gate=gates.data_ptr(), gate_stride=48, x=x.data_ptr(), x_stride=48, out=out.data_ptr(), out_stride=48, n_rows=1, width=48))
    done(ctx)
    a, y = gates.double(), out.double()
    want = 2 * a / (1 + torch.exp(-a))
    assert bool(torch.isnan(y[torch.isnan(a)]).all()) and bool((y[a == math.inf] == math.inf).all()) and bool((y[a < -88].abs() < 1e-35).all())
    # twice 3e38 is more than the largest float, 3.403e38: rounded, it is infinite
    large = want > 3.41e38
    assert bool((y[large] == math.inf).all())
    ok = torch.isfinite(a) & (a > -87) & ~large
    assert bool(((y - want)[ok].abs() <= (2.0 ** -8 + (8 + 1.2 * a.abs()[ok]) * 2.0 ** -23) * want[ok].abs() + 2.0 ** -133).all())


@gpu
@pytest.mark.parametrize("rows", [1, 5, 591, 593, 1200])
@pytest.mark.parametrize("width", [256, 264, 512, 520, 4096, 8192, 8200, 16384, 16392, 32768])
def test_rows_at_the_borders_of_their_layouts(ctx, zkb, rows, width):
    if rows * width > 1 << 23:
        rows = (1 << 23) // width
    g = gen(width + rows)
    x, h = (torch.randn(rows, width, generator=g, device="cuda").bfloat16() for _ in range(2))
    s, code, scale = torch.zeros_like(x), torch.zeros(rows, width, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ctx.step_residual_norm(zkb.StepResidualNorm(x=x.data_ptr(), x_stride=width, residual=h.data_ptr(), residual_stride=width, sum_out=s.data_ptr(), sum_stride=width, out=code.data_ptr(), out_type=INT8,
                                                out_scale=scale.data_ptr(), out_stride=width, n_rows=rows, width=width, eps=1e-5))
    done(ctx)
    want = (x.float() + h.float()).bfloat16()
    assert torch.equal(s, want)
    check_out(code, scale, "codes", norm_reference(want, None, 1e-5), 2.0 ** -18)


@gpu
def test_rows_of_outputs_that_descend(ctx, zkb):
    """Negative strides of what is written: the last row first."""
    g = gen(2)
    x = torch.randn(50, 128, generator=g, device="cuda").bfloat16()
    out, scale = torch.zeros(50, 128, device="cuda", dtype=torch.int8), torch.zeros(50, device="cuda")
    xs = Rows(x, "bf16", down=True)
    torch.cuda.synchronize()
    ctx.step_gate(zkb.StepGate(x=xs.ptr, x_stride=xs.stride, out=out.data_ptr() + 49 * 128, out_type=INT8, out_scale=scale.data_ptr(), out_stride=-128, n_rows=50, width=128))
    done(ctx)
    check_out(out.flip(0), scale, "codes", x.double(), 0.0)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "words", "f32"])
@pytest.mark.parametrize("rows,vocab", [(3, 4097), (1, 100003), (400, 20011), (2, 50)])
def test_logprobs_of_temperatures_near_zero(ctx, zkb, kind, rows, vocab):
    """Scales so large that a step of the largest logit decides, up to the largest that is taken: the likeliest token, or those that tie, have everything."""
    g = gen(rows + vocab)
    x = 10 + 30 * torch.randn(rows, vocab, generator=g, device="cuda")
    x[0, vocab // 3] = x[0, vocab // 2] = 200.0
    x[:, vocab - 7] = -math.inf
    ids = torch.tensor([[vocab // 3, vocab // 2, 0, vocab - 7]], device="cuda", dtype=torch.int32).expand(rows, -1).contiguous()
    held, values = held_logits(x, kind, 1, 0)
    few = slice(0, rows, -(-rows // 20))
    for scale in (3e5, 3e7, 1e9, 2.0 ** 100):
        got = answer(ctx, zkb, held, kind, ids, 4, scale)
        check_answer(tuple(y[few] for y in got), values[few], ids[few], 4, scale)
    # products that no float holds: what is below the largest logit has nothing
    held, values = held_logits(torch.where(x > 0, x * 1e35, x), kind, 1, 0)
    for scale in (1e6, 2.0 ** 100):
        lp, entropy, top, top_lp = answer(ctx, zkb, held, kind, ids, 4, scale)
        ties = (values == values.amax(-1, keepdim=True)).sum(-1).double()
        assert bool(((entropy - ties.log()).abs() <= 2.0 ** -15 * ties.log()).all()) and bool(((top_lp[:, 0] + ties.log()).abs() <= 2.0 ** -15 * ties.log()).all())
        assert bool((values.gather(1, top[:, :1].long()) == values.amax(-1, keepdim=True)).all())
        assert not bool(torch.isnan(lp).any()) and bool((lp[1:] == -math.inf).sum() >= rows - 1)


@gpu
@pytest.mark.parametrize("kind", ["codes", "bf16", "words"])
@pytest.mark.parametrize("width", [64, 777, 4096])
def test_norms_whose_products_with_the_weights_are_tiny(ctx, zkb, kind, width):
    """Small rows and small weights, with a norm that is a number all the same. (x^2 has a mean of 2^-80 about, and weights of 2^-100: products of 2^-140, norms of 2^-100.)"""
    g = gen(width)
    x = (torch.randn(5, width, generator=g, device="cuda") * 2.0 ** -40).bfloat16()
    w = ((1 + torch.rand(width, generator=g, device="cuda")) * 2.0 ** -100).bfloat16()
    full, got = room(kind, 5, width)
    scale = torch.zeros(5, device="cuda")
    torch.cuda.synchronize()
    ctx.step_residual_norm(zkb.StepResidualNorm(x=x.data_ptr(), x_stride=width, weight=w.data_ptr(), out=got.data_ptr(), out_type=TYPES[kind], out_scale=scale.data_ptr() if kind == "codes" else 0,
                                                out_stride=width, n_rows=5, width=width, eps=0.0))
    done(ctx)
    y = norm_reference(x, w, 0.0)
    if kind == "codes":  # (in units of 2^-100: what is compared has absolute terms)
        scale, y = scale.double() * 2.0 ** 100, y * 2.0 ** 100
        check_out(got, scale, kind, y, 2.0 ** -18)
    else:
        assert bool(((values_of(got) - y).abs() <= (2.0 ** -8 + 2.0 ** -17) * y.abs()).all())


@gpu
@pytest.mark.parametrize("kind,group,rows,n_out", [
    # as many tiles as the GPU holds at once, and one more: of 32, 64 and 128 rows
    ("int8", 0, 33, 18944), ("int8", 0, 64, 18945), ("int8", 0, 63, 19100), ("int8", 0, 65, 12673), ("int8", 0, 128, 12640), ("int8", 0, 256, 18944), ("int8", 0, 250, 18945), ("int8", 0, 513, 7681),
    ("int4", 128, 33, 18945), ("int4", 32, 64, 9472), ("int4", 64, 65, 9473), ("int4", 128, 128, 9472), ("int4", 32, 129, 6273), ("int4", 64, 192, 6272)])
@pytest.mark.parametrize("n_in,pad", [(256, 0), (208, 0), (163, 1)])
def test_products_at_the_borders_between_tiles(ctx, zkb, kind, group, rows, n_out, n_in, pad):
    g = gen(rows + n_out)
    x, w, x_scale = codes_of(g, rows, n_in, pad), Weights(g, kind, n_out, n_in, group, pad), torch.rand(rows, generator=g, device="cuda") + 0.1
    full, y = room("f32", rows, n_out, 1)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    check_product("f32", y, x, x_scale, w)
    untouched(full, y, 0)


@gpu
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 32), ("int4", 128)])
@pytest.mark.parametrize("n_in", [1024, 2816, 3000, 4096, 4224, 9000])
def test_products_of_few_tiles_and_more_steps(ctx, zkb, kind, group, n_in):
    """One row tile and a few outputs' tiles, with as many codes as are, and are not, spread over several thread blocks."""
    g = gen(n_in)
    for rows, n_out in ((17, 200), (40, 1000), (33, 4300), (128, 600)):
        x, w, x_scale = codes_of(g, rows, n_in), Weights(g, kind, n_out, n_in, group), torch.rand(rows, generator=g, device="cuda") + 0.1
        y = torch.zeros(rows, n_out, device="cuda")
        torch.cuda.synchronize()
        run_product(ctx, zkb, x, x_scale, w, ("f32", y))
        done(ctx)
        check_product("f32", y, x, x_scale, w)
