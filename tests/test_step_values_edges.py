"""zkb_step_* where their definitions and their layouts have corners: hints that do not fit the batch, values that are no numbers, scales and windows at the ends of their
ranges, launches that are refused. The references and bounds are those of tests/step_cases.py."""
import math

import numpy as np
import pytest
import torch

from step_cases import Batch, Cache, attention_reference, rope_reference, values_of, words
from test_step_values import _attention_args, check_attention, done, gen, refuse  # noqa: F401

gpu = pytest.mark.gpu


@pytest.mark.parametrize("n_rows,group,heads", [((1 << 30) - 1, 2, 1), ((1 << 30) - 127, 2, 1), (((1 << 31) - 254) // 3 + 1, 3, 1), ((1 << 30) - 1, 2, 3), (1 << 29, 2, 2)])
def test_attention_refuses_more_rows_of_a_head_than_it_can_number(zkb, refuse, n_rows, group, heads):  # noqa: F811
    """Up to 2^31 - 256 rows of a kv head: tiles are numbered by the row behind their last one."""
    refuse("zkb_step_attention", _attention_args(zkb, dict(n_heads=heads), dict(n_rows=n_rows), q_heads=group * heads), "n_rows")


def hinted(batch, max_rows, max_len):
    """The batch with these hints instead of its own."""
    args = batch.args

    def other(zkb, hints=True):
        r = args(zkb, hints)
        r.max_rows, r.max_len = max_rows, max_len
        return r

    batch.args = other
    return batch


# Hints that call for the large products, and cover fewer pairs of tiles than the batch has: a unit goes on with the same sequence's other pairs.
@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
@pytest.mark.parametrize("shape,hk", [([(1300, 1400)], 2), ([(900, 900)], 1), ([(900, 1000), (0, 4), (1300, 1300), (17, 600), (600, 700)], 2), ([(700, 800)] * 12, 3)])
def test_attention_of_more_rows_than_the_hint_says(ctx, zkb, kind, window, sinks, shape, hk):
    g = gen(hk + window)
    batch = hinted(Batch(shape, behind=2), 400, 1400)
    cache = Cache(g, kind, len(shape), hk, max(n for _, n in shape), 64)
    q = torch.randn(batch.n_rows, 4 * hk, 64, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "bf16" if window else "words", window, sinks)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_a_captured_call_serves_a_batch_of_longer_sequences(ctx, zkb, kind):
    """Captured for sequences of up to 500 rows, replayed for one of 600 and for one that has all 1,500."""
    g, hq, hk, d, cap = gen(3), 8, 2, 64, 1600
    cache = Cache(g, kind, 3, hk, cap, d)
    batch = hinted(Batch([(500, 500)] * 3), 500, 500)
    q = torch.randn(batch.n_rows, hq, d, generator=g, device="cuda").bfloat16()
    out = torch.zeros(batch.n_rows, hq, d, device="cuda", dtype=torch.bfloat16)
    call = zkb.StepAttention(cache=cache.args(zkb), rows=batch.args(zkb), q=q.data_ptr(), out=out.data_ptr(), q_stride=hq * d, q_head_stride=d, out_stride=hq * d, out_head_stride=d, q_heads=hq,
                             scale=d ** -0.5)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctx.stream())):
        ctx.step_attention(call)
    for shape in ([(500, 500)] * 3, [(600, 700), (300, 1600), (600, 600)], [(0, 0), (1500, 1600), (0, 9)]):
        other = Batch(shape)
        batch.first.copy_(other.first)
        batch.lens.copy_(other.lens)
        out.fill_(-3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        other.args = lambda zkb, hints=True: zkb.StepRows(first=other.first.data_ptr(), kv_len=other.lens.data_ptr(), n_rows=other.n_rows, max_rows=500, max_len=500)
        got = check_attention(ctx, zkb, other, cache, q, "bf16", 0, 0)
        assert torch.equal(got, replayed)
    del graph


def attend(ctx, zkb, batch, cache, q, out, window=0, sinks=0, scale=None):
    """The call, into `out` [row][head][dim] as it lies."""
    torch.cuda.synchronize()
    ctx.step_attention(zkb.StepAttention(cache=cache.args(zkb), rows=batch.args(zkb), q=q.data_ptr(), out=out.data_ptr(), q_stride=q.stride(0), q_head_stride=q.stride(1), out_stride=out.stride(0),
                                         out_head_stride=out.stride(1), q_heads=q.shape[1], out_type=zkb.VALUE_WORD if out.dtype == torch.int32 else zkb.VALUE_BF16, window=window, sinks=sinks,
                                         scale=q.shape[2] ** -0.5 if scale is None else scale))
    done(ctx)
    return out


def same(got, want, bound):
    """Infinities and NaN where the definition has them, the rest within the bound."""
    x, fine = values_of(got), torch.isfinite(want)
    assert torch.equal(torch.isnan(x), torch.isnan(want)) and torch.equal(x[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    over = ((x - want).abs() - bound)[fine]
    assert not over.numel() or float(over.max()) <= 0, (float(over.max()), int((over > 0).sum()), over.numel())


# Rows of one warp that go different ways: of unlike alignment, with and without values that are no numbers, behind the last one.
@gpu
@pytest.mark.parametrize("kind,out", [("bf16", "bf16"), ("bf16", "words"), ("int8", "bf16")])
@pytest.mark.parametrize("shape,hk,d,window", [([(201, 500)], 1, 64, 0), ([(201, 500)], 40, 128, 0), ([(77, 300), (130, 131), (50, 90)], 60, 32, 40)])
def test_attention_rows_of_a_warp_go_different_ways(ctx, zkb, kind, out, shape, hk, d, window):
    g, group = gen(d + hk), 3
    batch, hq = Batch(shape, behind=1), group * hk
    cache = Cache(g, kind, len(shape), hk, max(n for _, n in shape), d)
    q = torch.randn(batch.n_rows, hq, d, generator=g, device="cuda").bfloat16()
    if kind == "bf16":
        for b, at, rows, pos in batch.each():
            cache.v[b, :, pos + rows // 2, 3] = math.inf
            cache.v[b, :, pos + rows - 3, ::7] = math.nan
    room = torch.full((batch.n_rows * hq * (d + 1) + 1,), -3, device="cuda", dtype=torch.int32 if out == "words" else torch.bfloat16)
    got = attend(ctx, zkb, batch, cache, q, room[1:].view(batch.n_rows, hq, d + 1)[..., :d], window, 2)
    want, bound = attention_reference(batch, cache, q, d ** -0.5, window, 2)
    last = sum(r for r, _ in shape)
    same(got[:last], want[:last], bound[:last])
    assert bool((got[last:] == -3).all()) and bool((room[1:].view(-1, d + 1)[:, d] == -3).all())


@gpu
@pytest.mark.parametrize("source", ["bf16", "words"])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("d,rotary,interleaved", [(64, 0, 0), (64, 0, 1), (64, 16, 0), (128, 64, 1), (32, 16, 0), (128, 128, 0)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_of_values_that_are_no_numbers(ctx, zkb, source, kind, d, rotary, interleaved, norm):
    """What does not turn stays as it is, bit for bit, whatever lies beside it; what turns has infinities and NaN where the definition has them."""
    g, hq, hk, rows = gen(d + rotary), 6, 3, 21
    batch, cache = Batch([(rows, rows + 50)], behind=1), Cache(gen(0), kind, 1, hk, rows + 55, d, blank=True)
    x = torch.randn(batch.n_rows, hq + 2 * hk, d, generator=g, device="cuda").bfloat16()
    x[::2, :, rotary // 2::5] = -0.0
    for i, (h, at) in enumerate([(0, d - 1), (1, rotary % d), (2, max(0, rotary - 1)), (hq, d - 3), (hq + 1, rotary // 2), (hq + hk, d // 2), (hq + hk + 1, 1)]):
        x[3 + i, h, at] = [math.inf, -math.inf, math.nan][i % 3]
        x[11 + i, h, at] = math.inf
    weight = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).bfloat16()
    freq = 10000.0 ** (-np.arange(rotary // 2) / max(1, rotary // 2))
    laid, out = words(x) if source == "words" else x, torch.zeros(batch.n_rows, hq, d, device="cuda", dtype=torch.bfloat16)
    at = lambda h: laid.data_ptr() + laid.element_size() * h * d  # noqa: E731
    s, w = laid.stride(0), weight.data_ptr() if norm else 0
    torch.cuda.synchronize()
    ctx.step_norm_rope(zkb.StepNormRope(cache=cache.args(zkb), rows=batch.args(zkb), q=at(0), k=at(hq), v=at(hq + hk), q_weight=w, k_weight=w, h_inv_freq=freq.ctypes.data, q_out=out.data_ptr(),
                                        q_stride=s, k_stride=s, v_stride=s, head_stride=d, q_out_stride=out.stride(0), q_out_head_stride=d, type=1 if source == "words" else 0, q_heads=hq,
                                        rotary_dim=rotary, interleaved=interleaved, eps=1e-6))
    done(ctx)
    y, size = rope_reference(batch, x[:, :hq + hk], [weight if norm else None] * (hq + hk), 1e-6, freq, interleaved)
    y, size, v = y[:rows], size[:rows], x[:rows, hq + hk:]
    same(out[:rows], y[:, :hq], 2.0 ** -8 * y[:, :hq].abs() + 2.0 ** -18 * size[:, :hq])
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    alike = lambda a, b: bool(((bits(a) == bits(b)) | (a.isnan() & b.isnan())).all())  # noqa: E731
    if not norm:
        assert alike(out[:rows, :, rotary:], x[:rows, :hq, rotary:])
    for part, scale, want, room in ((cache.k, cache.k_scale, y[:, hq:], size[:, hq:]), (cache.v, cache.v_scale, v.double(), 0 * v.double())):
        got = part[0, :, 50:50 + rows].transpose(0, 1)
        if kind == "bf16":
            same(got, want, 2.0 ** -8 * want.abs() + 2.0 ** -18 * room)
            if not norm:
                old = x[:rows, hq:hq + hk] if part is cache.k else v
                begin = rotary if part is cache.k else 0
                assert alike(got[..., begin:], old[..., begin:])
        else:  # one scale a head: an infinity's is infinite, a NaN's NaN
            step, most = scale[0, :, 50:50 + rows].T.double(), want.abs().amax(-1)
            same(step, most / 127, 2.0 ** -18 * (room.amax(-1) + most))
            fine = torch.isfinite(most)
            over = (got.double() * step[..., None] - want).abs() - step[..., None] * (0.5 + 127 * 2.0 ** -22) - 2.0 ** -18 * room.amax(-1, keepdim=True)
            assert bool((over[fine] <= 0).all())


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,hk", [(1, 2), (3, 2), (300, 2), (300, 40)])
def test_attention_rows_whose_scores_are_all_minus_infinity_get_zeros(ctx, zkb, kind, rows, hk):
    """Whatever the values are that they see, some of them no numbers."""
    g, d, n = gen(rows), 64, rows + 150
    batch, cache = Batch([(rows, n)]), Cache(g, kind, 1, hk, n, d)
    q = torch.randn(rows, 4 * hk, d, generator=g, device="cuda").bfloat16()
    q[..., 0] = q[..., 0].abs() + 0.25
    if kind == "int8":
        cache.k.zero_()
        cache.k[..., 0] = -1
        cache.k_scale.fill_(math.inf)
        cache.v_scale[:, :, ::11] = math.nan
    else:
        cache.k[..., 0] = -math.inf
        cache.v[:, :, ::11, ::3] = math.inf
    q[rows // 2, 1, 0] = 0 if kind == "int8" else q[rows // 2, 1, 0]  # 0 times an infinity: NaN
    got = attend(ctx, zkb, batch, cache, q, torch.full_like(q, 7))
    if kind == "int8":
        assert bool(got[rows // 2, 1].isnan().all())
        got[rows // 2, 1] = 0
    assert bool((got == 0).all())


def far_apart(g, shape, hq, d):
    """Queries whose scores (by a scale of 3) lie so far apart that most weights are below the smallest float."""
    return (6 * torch.randn(shape, hq, d, generator=g, device="cuda")).bfloat16()


# A token's value that is no number reaches every row that sees the token, however small its weight: in blocks that all rows see and in others, with keys spread and not.
@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("shape,hk,d,window", [([(1, 1500)], 2, 128, 0), ([(3, 700), (2, 90)], 3, 64, 0), ([(300, 2000)], 1, 128, 0), ([(300, 1500)], 40, 64, 0), ([(200, 1200), (90, 90)], 30, 32, 400),
                                               ([(100, 900)], 1, 64, 0)])
def test_attention_values_that_are_no_numbers_under_weights_of_nothing(ctx, zkb, kind, shape, hk, d, window):
    g, hq = gen(d + hk), 4 * hk
    batch = Batch(shape)
    cache = Cache(g, kind, len(shape), hk, max(n for _, n in shape), d)
    for b, _, rows, pos in batch.each():
        for i, j in enumerate([0, 5, 130, pos - 200, pos - 1]):
            if 0 <= j < pos:
                x = [math.inf, -math.inf, math.nan][(i + b) % 3]
                if kind == "int8":
                    cache.v[b, :, j][cache.v[b, :, j] == 0] = 1  # of a code of zero and an infinity the product is NaN: kept out of the comparison
                    cache.v_scale[b, i % hk, j] = x
                else:
                    cache.v[b, i % hk, j, i::9] = x
    q = far_apart(g, batch.n_rows, hq, d)
    check_attention(ctx, zkb, batch, cache, q, "words" if window else "bf16", window, 4, scale=3.0)
    check_attention(ctx, zkb, batch, cache, q, "bf16", window, 4, scale=-0.05)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,hk", [(1, 2), (3, 2), (300, 2), (300, 40)])
def test_attention_values_that_are_no_numbers_of_a_token_whose_score_is_minus_infinity(ctx, zkb, kind, rows, hk):
    """They reach the rows that see it like any other's; the other tokens' weights are as without it."""
    g, d, n = gen(rows), 64, rows + 300
    batch, cache = Batch([(rows, n)]), Cache(g, kind, 1, hk, n, d)
    q = torch.randn(rows, 4 * hk, d, generator=g, device="cuda").bfloat16()
    q[..., 0] = q[..., 0].abs() + 0.25
    for j in (7, 200, n - 3):
        if kind == "int8":
            cache.k[0, :, j] = 0
            cache.k[0, :, j, 0] = -1
            cache.k_scale[0, :, j] = math.inf
        else:
            cache.k[0, :, j] = 0.5
            cache.k[0, :, j, 0] = -math.inf
        if j == 200 and kind == "bf16":
            cache.v[0, 0, j, 1::5] = math.inf
        elif j == 200:
            cache.v[0, 0, j] = 3
            cache.v_scale[0, 0, j] = -math.inf
    got = attend(ctx, zkb, batch, cache, q, torch.full_like(q, 7))
    cache.k[0, :, [7, 200, n - 3]] = 0  # a definition without products of zero and infinity: those tokens' scores by hand
    if kind == "int8":
        cache.k_scale[0, :, [7, 200, n - 3]] = 1
    k, v = cache.values()
    p, j = torch.arange(n - rows, n, device="cuda")[:, None], torch.arange(n, device="cuda")
    for h in range(4 * hk):
        s = (q[:, h].double() @ k[0, h // 4].T * d ** -0.5).masked_fill(j > p, -math.inf)
        s[:, [7, 200, n - 3]] = -math.inf
        w, bad = torch.softmax(s, -1), ~torch.isfinite(v[0, h // 4])
        want = w @ v[0, h // 4].masked_fill(bad, 0) + torch.where(bad[200], v[0, h // 4, 200], 0.0)
        # as attention_reference counts: weights by 2^-8 and scores by 68 roundings of 2^-24 of magnitudes below 2^8, the result by 2^-8
        bound = (2.0 ** -8 + 2.0 ** -9) * (w @ v[0, h // 4].masked_fill(bad, 0).abs() + want.abs())
        same(got[:, h], want, bound)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows", [1, 3, 300])
@pytest.mark.parametrize("window,sinks", [((1 << 31) - 10, 0), ((1 << 31) - 250, 3), ((1 << 31) + 5, 0), ((1 << 32) - 1, 7), ((1 << 30) + 3, 2)])
def test_attention_windows_of_more_than_2_to_the_30(ctx, zkb, kind, rows, window, sinks):
    """The rows of the last positions that there are, over the first tokens: what a window of about as many leaves of them."""
    g, cap = gen(rows), 70
    batch, cache = Batch([(rows, (1 << 31) - 1), (rows, 60)]), Cache(g, kind, 2, 4, cap, 64)
    q = torch.randn(batch.n_rows, 16, 64, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "bf16", window, sinks)


@gpu
@pytest.mark.parametrize("source", ["bf16", "words"])
@pytest.mark.parametrize("d", [32, 128])
def test_int8_codes_of_the_smallest_heads(ctx, zkb, source, d):
    """Heads down to the smallest bf16 number, 2^-133, whose scales are among the smallest floats (steps of 2^-149: a scale is off by up to 2^-150, a value of 127 of them by 2^-143)."""
    g, hk, rows = gen(d), 2, 140
    batch, cache = Batch([(rows, rows)]), Cache(gen(0), "int8", 1, hk, rows, d, blank=True)
    x = torch.rand(rows, 3 * hk, d, generator=g, device="cuda", dtype=torch.float64) * 2 - 1
    x = (x * torch.exp2(-torch.arange(rows, device="cuda", dtype=torch.float64))[:, None, None]).bfloat16()
    x[7:] *= torch.randint(0, 2, (rows - 7, 3 * hk, 1), generator=g, device="cuda")  # heads of zeros among them
    laid, out = words(x) if source == "words" else x, torch.zeros(rows, hk, d, device="cuda", dtype=torch.bfloat16)
    at = lambda h: laid.data_ptr() + laid.element_size() * h * d  # noqa: E731
    s = laid.stride(0)
    torch.cuda.synchronize()
    ctx.step_norm_rope(zkb.StepNormRope(cache=cache.args(zkb), rows=batch.args(zkb), q=at(0), k=at(hk), v=at(2 * hk), q_out=out.data_ptr(), q_stride=s, k_stride=s, v_stride=s, head_stride=d,
                                        q_out_stride=out.stride(0), q_out_head_stride=d, type=1 if source == "words" else 0, q_heads=hk, rotary_dim=0, eps=1e-6))
    done(ctx)
    for part, scale, h in ((cache.k, cache.k_scale, hk), (cache.v, cache.v_scale, 2 * hk)):
        y, codes, step = x[:, h:h + hk].double(), part[0].transpose(0, 1).double(), scale[0].T.double()
        most = y.abs().amax(-1)
        assert bool(((step - most / 127).abs() <= 2.0 ** -24 * most / 127 + 2.0 ** -150).all())
        ideal = y * 127 / torch.where(most > 0, most, 1.0)[..., None]
        assert bool(((codes - ideal).abs() <= 0.5 + 127 * 2.0 ** -22).all())
        assert bool(((codes * step[..., None] - y).abs() <= step[..., None] * (0.5 + 127 * 2.0 ** -22) + 2.0 ** -142).all())


@gpu
def test_attention_weights_are_rounded_once(ctx, zkb):
    """Weights of the first half of a block whose second half has a score more than 2^8 times above: 63 alike, so that their roundings add up, for 512 weights a row apiece and 64 later
    scores. The bound has one rounding of a weight and the result's."""
    rows, hq, d = 512, 64, 64
    n = rows + 128
    batch, cache = Batch([(rows, n)]), Cache(gen(0), "bf16", 1, 1, n, d, blank=True)
    q = torch.zeros(rows, hq, d, device="cuda")
    q[..., 0], q[..., 1] = torch.linspace(0.01, 3.9, rows, device="cuda")[:, None], torch.linspace(8.6, 14, hq, device="cuda")
    cache.k[0, 0, :63, 0] = -1
    cache.k[0, 0, 64, 1] = 1
    cache.k[0, 0, 65:, 1] = -16
    cache.v[0, 0, :63] = 1
    check_attention(ctx, zkb, batch, cache, q.bfloat16(), "bf16", 0, 0, scale=math.log(2.0))


# What the few rows' kernel says of its weights: two bf16 numbers, off by 2^-16. Means of a few hundred values of either sign are so far below them that one number's 2^-8
# would show (worked out with one: 57 of 1,024 values of 300 tokens and 128 dimensions are out of the bound).
@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("shape,hq,hk,d,window,long", [([(1, 300)], 32, 8, 128, 0, False), ([(1, 200), (1, 64), (1, 333)], 8, 2, 128, 0, False), ([(3, 333), (2, 64)], 6, 3, 32, 0, False),
                                                       ([(4, 250)], 16, 2, 64, 0, False), ([(1, 3000)] * 6, 16, 4, 64, 200, False), ([(8, 300)], 16, 4, 128, 0, True), ([(5, 250), (8, 200)], 16, 4, 64, 0, True)])
def test_attention_weights_of_few_rows(ctx, zkb, kind, shape, hq, hk, d, window, long):
    """`long`: caches that have room for 1,600 tokens and hints that say so, for which int8 caches have sixteen rows a product."""
    g = gen(d + hq)
    batch, cache = Batch(shape), Cache(g, kind, len(shape), hk, 1600 if long else max(n for _, n in shape), d)
    if long:
        hinted(batch, max(r for r, _ in shape), 1600)
    q = torch.randn(batch.n_rows, hq, d, generator=g, device="cuda").bfloat16()
    got = attend(ctx, zkb, batch, cache, q, torch.zeros_like(q), window, 4)
    same(got, *attention_reference(batch, cache, q, d ** -0.5, window, 4, weight=2.0 ** -16))


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("most", [1, 2, 4, 8])
def test_attention_whose_clusters_are_refused(ctx, zkb, monkeypatch, kind, most):
    """Keys spread over fewer thread blocks than planned: a token of one sequence and several, few rows of a long cache, many rows."""
    monkeypatch.setenv("ZKB_STEP_CLUSTERS", str(most))
    for shape, hk, d, window in (([(1, 3000)], 2, 128, 0), ([(1, 900), (2, 2100)], 3, 64, 0), ([(8, 2500)], 1, 32, 0), ([(300, 2000)], 1, 128, 0), ([(90, 1700), (100, 1500)], 2, 64, 900)):
        g = gen(d + hk)
        batch, cache = Batch(shape), Cache(g, kind, len(shape), hk, max(n for _, n in shape), d)
        q = torch.randn(batch.n_rows, 4 * hk, d, generator=g, device="cuda").bfloat16()
        check_attention(ctx, zkb, batch, cache, q, "bf16", window, 5)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("shape,d", [([(8, 300)], 128), ([(5, 250), (8, 200)], 64), ([(3, 290), (4, 150)], 32)])
def test_attention_weights_of_few_rows_of_many_heads(ctx, zkb, kind, shape, d):
    """As above where eight rows a product would have thread blocks share SMs."""
    test_attention_weights_of_few_rows(ctx, zkb, kind, shape, 64, 16, d, 0, True)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows", [1, 3, 300])
@pytest.mark.parametrize("scale", [0.0, 1e-39, -1e-38, 2e-38])
def test_attention_scales_of_nothing_and_nearly(ctx, zkb, kind, rows, scale):
    """Products of 10^38 and a scale that makes less than one, or nothing, of them: by nothing all keys that a row sees weigh alike."""
    g, d, n = gen(rows), 64, rows + 200
    batch, cache = Batch([(rows, n)]), Cache(g, kind, 1, 4, n, d)
    q = torch.randn(rows, 16, d, generator=g, device="cuda").bfloat16()
    q[..., 0] = 1e19
    cache.k[..., 0] = 0
    if kind == "int8":
        cache.k[:, :, ::3, 0] = 100
        cache.k_scale.fill_(1e17)
    else:
        cache.k[:, :, ::3, 0] = 1e19
    check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0, scale=scale)


class Backwards(Cache):
    """The same cache, laid out with its tokens, heads or sequences descending: the address is that of the first one, behind the others."""

    def args(self, zkb):
        c = super().args(zkb)
        size, (s, h, t, _), k = self.k.element_size(), self.dims, self.k
        self.room = [x.flip([dict(s=0, h=1, t=2)[y] for y in self.down]).contiguous() for x in (self.k, self.v)]
        seq, head, token = h * t * k.shape[3], t * k.shape[3], k.shape[3]
        off = (s - 1) * seq * ("s" in self.down) + (h - 1) * head * ("h" in self.down) + (t - 1) * token * ("t" in self.down)
        c.k, c.v = (x.data_ptr() + size * off for x in self.room)
        c.seq_stride, c.head_stride, c.token_stride = (-x if y in self.down else x for x, y in ((seq, "s"), (head, "h"), (token, "t")))
        torch.cuda.synchronize()
        return c


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("down", ["t", "h", "s", "sht"])
@pytest.mark.parametrize("shape,window", [([(1, 300), (2, 77)], 0), ([(200, 400), (90, 200)], 60)])
def test_caches_laid_out_backwards(ctx, zkb, kind, down, shape, window):
    g = gen(len(down))
    batch, cache = Batch(shape), Backwards(g, kind, 2, 8, 400, 64)
    cache.down = down
    q = torch.randn(batch.n_rows, 32, 64, generator=g, device="cuda").bfloat16()
    if kind == "bf16":
        cache.v[0, 1, 9, 5] = math.inf
    check_attention(ctx, zkb, batch, cache, q, "words", window, 3)
    x = torch.randn(batch.n_rows, 32 + 16, 64, generator=g, device="cuda").bfloat16()
    args, freq = cache.args(zkb), 1e4 ** (-np.arange(32) / 32)
    torch.cuda.synchronize()
    out = torch.zeros(batch.n_rows, 32, 64, device="cuda", dtype=torch.bfloat16)
    ctx.step_norm_rope(zkb.StepNormRope(cache=args, rows=batch.args(zkb), q=x.data_ptr(), k=x[:, 32:].data_ptr(), v=x[:, 40:].data_ptr(), h_inv_freq=freq.ctypes.data, q_out=out.data_ptr(),
                                        q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0), head_stride=64, q_out_stride=out.stride(0), q_out_head_stride=64, q_heads=32,
                                        rotary_dim=64, eps=1e-6))
    done(ctx)
    cache.v = cache.room[1].flip([dict(s=0, h=1, t=2)[y] for y in down])
    for b, at, rows, pos in batch.each():
        got, want = cache.values()[1][b, :, pos:pos + rows].transpose(0, 1), x[at:at + rows, 40:].double()
        step = cache.v_scale[b, :, pos:pos + rows].T.double()[..., None] if kind == "int8" else 0
        assert bool(((got - want).abs() <= step * (0.5 + 127 * 2.0 ** -22)).all())


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,length", [(1, 500), (70, 400)])
def test_sequences_that_share_a_cache(ctx, zkb, kind, rows, length):
    """A sequence stride of zero: each sees its own first tokens of the same ones."""
    g = gen(rows)
    batch, cache = Batch([(rows, length), (rows, length - 100), (rows, length)]), Cache(g, kind, 3, 8, length, 64)
    for x in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if x is not None:
            x[1:] = x[:1]
    own = cache.args

    def shared(zkb):
        c = own(zkb)
        c.seq_stride = c.scale_seq_stride = 0
        return c

    cache.args = shared
    q = torch.randn(batch.n_rows, 32, 64, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("shape,hk,window", [([(1, 3000)], 8, 0), ([(32, 2048)], 8, 0), ([(500, 900), (3, 70), (300, 300)], 8, 0), ([(700, 1500)], 1, 200)])
def test_attention_gives_the_same_bits_each_time(ctx, zkb, kind, shape, hk, window):
    """Sums have one order, whichever thread blocks come first."""
    g = gen(hk)
    batch, cache = Batch(shape), Cache(g, kind, len(shape), hk, max(n for _, n in shape), 128)
    q = torch.randn(batch.n_rows, 4 * hk, 128, generator=g, device="cuda").bfloat16()
    first = attend(ctx, zkb, batch, cache, q, torch.zeros_like(q), window, 3)
    for _ in range(10):
        assert torch.equal(attend(ctx, zkb, batch, cache, q, torch.full_like(q, 5), window, 3), first)
