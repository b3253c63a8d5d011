"""The values of a decode step (zkb_step_embed, zkb_step_norm_rope, zkb_step_attention).

CPU: what the calls refuse. GPU: each against its definition in 64 bits at the sizes, layouts and masks where it can go wrong, with
bounds counted from the roundings (tests/step_cases.py), and the calls one after another with the witness generators around them."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from step_cases import Batch, Cache, attention_reference, rope_reference, values_of, words

gpu = pytest.mark.gpu


# ---- what is refused: arguments are looked at before anything is asked of a device, so a blank context will do -----------------------------
@pytest.fixture()
def refuse(zkb):
    lib, blank = zkb.load_library(), C.create_string_buffer(1 << 16)

    def call(name, args, want):
        assert getattr(lib, name)(C.cast(blank, C.c_void_p), C.byref(args)) == -1, want
        assert want in lib.zkb_last_error(C.cast(blank, C.c_void_p)).decode()

    return call


def _embed_args(zkb, **other):
    return zkb.StepEmbed(**{**dict(ids=64, table=64, row_scale=64, out=64, table_stride=64, out_stride=64, n_tokens=2, vocab=10, width=64, table_type=2, out_type=0, scale=1.0), **other})


@pytest.mark.parametrize("other,want", [(dict(table_type=1), "table_type"), (dict(out_type=2), "out_type"), (dict(width=0), "width"), (dict(width=1 << 24), "width"),
                                        (dict(scale=math.nan), "scale"), (dict(ids=0), "ids"), (dict(row_scale=0), "row_scale"), (dict(table_type=0), "row_scale"),
                                        (dict(out=65), "aligned"), (dict(out_type=1, out=66), "aligned"), (dict(out_stride=63), "out_stride"), (dict(table=0), "table"),
                                        (dict(segment=16, segment_stride=15), "segment_stride")])
def test_embed_refuses(zkb, refuse, other, want):
    refuse("zkb_step_embed", _embed_args(zkb, **other), want)


CACHE = dict(k=64, v=64, k_scale=64, v_scale=64, type=2, n_seqs=2, n_heads=2, head_dim=64, capacity=10, seq_stride=1280, head_stride=640, token_stride=64)
ROWS = dict(first=64, kv_len=64, n_rows=3)
CACHE_REFUSALS = [(dict(type=1), {}, "cache.type"), (dict(head_dim=96), {}, "head_dim"), (dict(k=0), {}, "cache.k"), (dict(k_scale=0), {}, "k_scale"),
                  (dict(type=0, v=65), {}, "boundary"), (dict(n_seqs=0), {}, "n_seqs"), (dict(n_heads=0), {}, "n_heads"), (dict(capacity=0), {}, "capacity"),
                  (dict(token_stride=63), {}, "token_stride"), ({}, dict(first=0), "rows.first"), ({}, dict(n_rows=1 << 31), "n_rows")]


def _rope_args(zkb, cache={}, rows={}, **other):
    freq = np.ones(32)
    a = zkb.StepNormRope(**{**dict(cache=zkb.KvCache(**{**CACHE, **cache}), rows=zkb.StepRows(**{**ROWS, **rows}), q=64, k=64, v=64, h_inv_freq=freq.ctypes.data, q_out=64, q_stride=512,
                                   k_stride=512, v_stride=512, head_stride=64, q_out_stride=256, q_out_head_stride=64, type=0, q_heads=4, rotary_dim=64, eps=1e-6), **other})
    a.keep = freq
    return a


@pytest.mark.parametrize("other,want", [(dict(ids=66), "ids"), (dict(row_scale=70), "row_scale"), (dict(off_table=68), "off_table")])
def test_embed_refuses_arrays_off_their_boundaries(zkb, refuse, other, want):
    refuse("zkb_step_embed", _embed_args(zkb, **other), want)


@pytest.mark.parametrize("cache,rows,want", [(dict(k_scale=66), {}, "k_scale"), (dict(v_scale=65), {}, "v_scale"), (dict(token_stride=(1 << 29) + 1), {}, "2^29"), (dict(token_stride=-(1 << 30)), {}, "2^29"),
                                             (dict(capacity=(1 << 30) + 1), {}, "capacity"), (dict(n_heads=1025), {}, "n_heads"), (dict(n_seqs=65536), {}, "n_seqs"), ({}, dict(kv_len=0), "kv_len"),
                                             ({}, dict(first=66), "boundary"), ({}, dict(kv_len=65), "boundary")])
def test_caches_and_rows_past_their_limits_are_refused(zkb, refuse, cache, rows, want):
    refuse("zkb_step_norm_rope", _rope_args(zkb, cache, rows), want)
    refuse("zkb_step_attention", _attention_args(zkb, cache, rows), want)


def test_attention_refuses_more_rows_of_heads_than_it_can_number(zkb, refuse):
    refuse("zkb_step_attention", _attention_args(zkb, {}, dict(n_rows=1 << 29), q_heads=4), "q_heads")


@pytest.mark.parametrize("cache,rows,want", CACHE_REFUSALS)
def test_norm_rope_refuses_caches_and_rows(zkb, refuse, cache, rows, want):
    refuse("zkb_step_norm_rope", _rope_args(zkb, cache, rows), want)


@pytest.mark.parametrize("other,want", [(dict(type=2), "type"), (dict(rotary_dim=24), "rotary_dim"), (dict(rotary_dim=80), "rotary_dim"), (dict(interleaved=2), "interleaved"),
                                        (dict(h_inv_freq=0), "h_inv_freq"), (dict(eps=-1.0), "eps"), (dict(eps=math.inf), "eps"), (dict(q=0), "a.q"), (dict(q_out=0), "q_out"), (dict(v=65), "aligned"),
                                        (dict(type=1, k=66), "aligned"), (dict(q_heads=3), "q_heads"), (dict(q_out_head_stride=32), "q_out_head_stride"), (dict(q_out_stride=8), "q_out_stride")])
def test_norm_rope_refuses(zkb, refuse, other, want):
    refuse("zkb_step_norm_rope", _rope_args(zkb, **other), want)


def test_norm_rope_refuses_frequencies_without_a_value(zkb, refuse):
    a = _rope_args(zkb)
    a.keep[5] = math.nan
    refuse("zkb_step_norm_rope", a, "h_inv_freq")


def _attention_args(zkb, cache={}, rows={}, **other):
    return zkb.StepAttention(**{**dict(cache=zkb.KvCache(**{**CACHE, **cache}), rows=zkb.StepRows(**{**ROWS, **rows}), q=64, out=64, q_stride=256, q_head_stride=64, out_stride=256,
                                       out_head_stride=64, q_heads=4, scale=0.1), **other})


@pytest.mark.parametrize("cache,rows,want", CACHE_REFUSALS)
def test_attention_refuses_caches_and_rows(zkb, refuse, cache, rows, want):
    refuse("zkb_step_attention", _attention_args(zkb, cache, rows), want)


@pytest.mark.parametrize("other,want", [(dict(out_type=2), "out_type"), (dict(scale=math.inf), "scale"), (dict(q=0), "a.q"), (dict(out=65), "aligned"), (dict(out_type=1, out=66), "aligned"),
                                        (dict(q_heads=5), "q_heads"), (dict(q_heads=0), "q_heads"), (dict(q_heads=130), "q_heads"), (dict(out_head_stride=63), "out_head_stride"),
                                        (dict(out_stride=63), "out_stride")])
def test_attention_refuses(zkb, refuse, other, want):
    refuse("zkb_step_attention", _attention_args(zkb, **other), want)


def test_a_call_without_arguments_or_context_is_refused(zkb, refuse):
    lib, blank = zkb.load_library(), C.create_string_buffer(1 << 16)
    for name in ("zkb_step_embed", "zkb_step_norm_rope", "zkb_step_attention"):
        assert getattr(lib, name)(None, None) == -1
        assert getattr(lib, name)(C.cast(blank, C.c_void_p), None) == -1


def test_a_step_without_rows_is_nothing_to_do(zkb):
    lib, blank = zkb.load_library(), C.create_string_buffer(1 << 16)
    for name, args in (("zkb_step_embed", _embed_args(zkb, n_tokens=0)), ("zkb_step_norm_rope", _rope_args(zkb, {}, dict(n_rows=0))), ("zkb_step_attention", _attention_args(zkb, {}, dict(n_rows=0)))):
        assert getattr(lib, name)(C.cast(blank, C.c_void_p), C.byref(args)) == 0


# ---- GPU ---------------------------------------------------------------------------------------------------------------------------------------
def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def done(ctx):
    """Inputs are made on torch's stream, calls run on the context's."""
    torch.cuda.synchronize()
    ctx.sync()


@gpu
@pytest.mark.parametrize("tokens,width,table,out,segment,pad,offset", [(1, 4096, "int8", "bf16", 0, 0, 0), (1, 1, "int8", "words", 0, 0, 0), (7, 4096, "int8", "words", 128, 0, 0), (300, 1001, "int8", "bf16", 0, 0, 0),
                                                                     (33, 2056, "bf16", "bf16", 0, 8, 0), (40, 264, "bf16", "words", 88, 3, 0), (5000, 512, "int8", "bf16", 0, 0, 0),
                                                                     (3, 96, "int8", "bf16", 0, 0, 1), (70, 30, "bf16", "bf16", 7, 0, 0), (2, 8, "int8", "words", 8, 0, 0), (9000, 33, "int8", "words", 0, 1, 0)])
def test_embed(ctx, zkb, tokens, width, table, out, segment, pad, offset):
    """Bit for bit: the code times the scale in 32 bits and one rounding are what the definition says."""
    g, vocab = gen(tokens + width), 131
    room = torch.randint(-128, 128, (vocab, width + pad + offset), generator=g, device="cuda", dtype=torch.int8) if table == "int8" else torch.randn(vocab, width + pad + offset, generator=g, device="cuda").bfloat16()
    tab = room[:, offset:offset + width]
    scales = torch.rand(vocab, generator=g, device="cuda") if table == "int8" else None
    ids = torch.randint(0, vocab, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    ids[::5] = torch.tensor([-1, vocab, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32, device="cuda")[torch.arange(len(ids[::5]), device="cuda") % 4]
    if tokens == 1:
        ids[0] = vocab - 1
    seg = segment or width
    n_seg, mark = -(-width // seg), -7
    dst = torch.full((tokens, n_seg, 2, seg), mark, device="cuda", dtype=torch.int32 if out == "words" else torch.bfloat16)
    off = torch.zeros(1, device="cuda", dtype=torch.int64)
    torch.cuda.synchronize()
    ctx.step_embed(zkb.StepEmbed(ids=ids.data_ptr(), table=tab.data_ptr(), row_scale=scales.data_ptr() if table == "int8" else 0, out=dst.data_ptr(), off_table=off.data_ptr(), table_stride=tab.stride(0),
                                 out_stride=dst.stride(0), segment_stride=dst.stride(1), n_tokens=tokens, vocab=vocab, width=width, segment=segment, table_type=2 if table == "int8" else 0,
                                 out_type=1 if out == "words" else 0, scale=1.7))
    done(ctx)
    inside = (ids >= 0) & (ids < vocab)
    x = tab[torch.where(inside, ids, 0).long()].float() * (scales[torch.where(inside, ids, 0).long()] * np.float32(1.7))[:, None] if table == "int8" else tab[torch.where(inside, ids, 0).long()].float() * np.float32(1.7)
    want = torch.where(inside[:, None], x, 0.0).bfloat16()
    got = dst[:, :, 0].reshape(tokens, -1)
    assert torch.equal(got[:, :width] if out == "bf16" else got[:, :width], want if out == "bf16" else words(want))
    assert int(off) == int((~inside).sum())
    assert bool((dst[:, :, 1] == mark).all()) and bool((got[:, width:] == mark).all())  # what lies between the segments and behind a row stays


ROPE_CASES = [  # shape, q heads, kv heads, dim, rotary, interleaved, norm, cache, source, order, pad, down
    ([(1, 1)], 1, 1, 32, 32, 0, True, "bf16", "bf16", "shtd", 0, False),
    ([(1, 2000), (1, 1), (0, 7), (1, 500)], 32, 8, 128, 128, 0, True, "int8", "bf16", "shtd", 0, False),
    ([(40, 40), (3, 90)], 6, 2, 64, 32, 0, True, "int8", "words", "sthd", 0, True),
    ([(17, 30), (0, 0), (64, 64)], 5, 5, 128, 64, 1, False, "bf16", "words", "tshd", 8, True),
    ([(9, 100)], 8, 1, 32, 16, 0, True, "int8", "bf16", "shtd", 3, False),
    ([(100, 150)], 4, 4, 64, 0, 0, True, "bf16", "bf16", "hstd", 0, False),
    ([(33, 64), (1, 64)], 12, 3, 128, 16, 1, True, "int8", "bf16", "shtd", 0, False),
    ([(700, 1000)], 8, 8, 32, 32, 1, False, "bf16", "bf16", "shtd", 5, False),
    ([(1, 20 + b) for b in range(70)], 4, 2, 64, 64, 0, True, "int8", "bf16", "shtd", 0, False),
]


@gpu
@pytest.mark.parametrize("shape,hq,hk,d,rotary,interleaved,norm,kind,source,order,pad,down", ROPE_CASES)
def test_norm_rope(ctx, zkb, shape, hq, hk, d, rotary, interleaved, norm, kind, source, order, pad, down):
    """Norms are sums of D squares, a reciprocal root and two products: below 2^-20 of a value; angles are off by 2 pi 2^-25 and their sines by
    2^-23 beside it, three roundings of a turned pair: below 2^-19 of |a| + |b| in all. bf16 adds 2^-8 of the value."""
    g = gen(hq + d + rotary)
    batch, cap = Batch(shape, behind=3, gap=2), max(n for _, n in shape) + 4
    cache = Cache(g, kind, len(shape), hk, cap, d, order, pad, blank=True)
    heads = hq + 2 * hk
    x = (torch.randn(batch.n_rows, heads, d + pad, generator=g, device="cuda") * torch.exp2(torch.randn(batch.n_rows, heads, 1, generator=g, device="cuda"))).bfloat16()
    x[batch.gap, 0] = 0  # a head without length
    rows = words(x) if source == "words" else x
    if source == "words":
        rows = rows | 0x5A5A0000  # the high halves do not count
    laid = rows.flip(0, 1).contiguous() if down else rows
    at = lambda h: laid.data_ptr() + laid.element_size() * ((batch.n_rows - 1) * laid.stride(0) + (heads - 1 - h) * laid.stride(1) if down else h * laid.stride(1))  # noqa: E731
    sign = -1 if down else 1
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).bfloat16() for _ in range(2))
    freq = 10000.0 ** (-np.arange(rotary // 2) / max(1, rotary // 2))
    out = torch.full((batch.n_rows, hq, d), 77.0, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    ctx.step_norm_rope(zkb.StepNormRope(cache=cache.args(zkb), rows=batch.args(zkb), q=at(0), k=at(hq), v=at(hq + hk), q_weight=wq.data_ptr() if norm else 0, k_weight=wk.data_ptr() if norm else 0,
                                        h_inv_freq=freq.ctypes.data, q_out=out.data_ptr(), q_stride=sign * laid.stride(0), k_stride=sign * laid.stride(0), v_stride=sign * laid.stride(0),
                                        head_stride=sign * laid.stride(1), q_out_stride=out.stride(0), q_out_head_stride=out.stride(1), type=1 if source == "words" else 0, q_heads=hq, rotary_dim=rotary,
                                        interleaved=interleaved, eps=1e-6))
    done(ctx)
    x = x[..., :d]
    weights = [wq if norm else None] * hq + [wk if norm else None] * hk
    y, size = rope_reference(batch, x[:, :hq + hk], weights, 1e-6, freq, interleaved)
    v = x[:, hq + hk:].double()
    inside = torch.zeros(batch.n_rows, dtype=torch.bool, device="cuda")
    k_got, v_got = cache.values()
    touched = torch.zeros(cache.dims[:3], dtype=torch.bool, device="cuda")
    for b, r0, r, p0 in batch.each():
        inside[r0:r0 + r] = True
        touched[b, :, p0:p0 + r] = True
        for got, want, s, scale in ((k_got, y[r0:r0 + r, hq:], size[r0:r0 + r, hq:], cache.k_scale), (v_got, v[r0:r0 + r], 0 * v[r0:r0 + r], cache.v_scale)):
            d_ = (got[b, :, p0:p0 + r].transpose(0, 1) - want).abs()
            if kind == "bf16":
                assert bool((d_ <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * s).all())
            else:  # half a step, a rounding of each of scale and quotient, and what the value itself is off
                step = scale[b, :, p0:p0 + r].T.double()[..., None]
                assert bool((d_ <= step * (0.5 + 127 * 2.0 ** -22) + 2.0 ** -18 * s.amax(-1, keepdim=True)).all())
                assert bool(((step[..., 0] * 127 - want.abs().amax(-1)).abs() <= 2.0 ** -18 * (s.amax(-1) + want.abs().amax(-1))).all())
    got = out.double()
    assert bool(((got - y[:, :hq]).abs() <= 2.0 ** -8 * y[:, :hq].abs() + 2.0 ** -18 * size[:, :hq])[inside].all())
    assert bool((out[~inside] == 77).all())
    for part in (cache.k, cache.v):
        assert bool((part[~touched] == 0).all())


def run_attention(ctx, zkb, batch, cache, q, out_kind, window, sinks, scale, hints=True, down=False):
    n, hq, d = q.shape
    room = torch.full((n, hq, 2, d), -3, device="cuda", dtype=torch.int32 if out_kind == "words" else torch.bfloat16)
    at = room.data_ptr() + room.element_size() * ((n - 1) * room.stride(0) + (hq - 1) * room.stride(1) if down else 0)
    sign = -1 if down else 1
    torch.cuda.synchronize()
    ctx.step_attention(zkb.StepAttention(cache=cache.args(zkb), rows=batch.args(zkb, hints), q=q.data_ptr(), out=at, q_stride=q.stride(0), q_head_stride=q.stride(1), out_stride=sign * room.stride(0),
                                         out_head_stride=sign * room.stride(1), q_heads=hq, out_type=1 if out_kind == "words" else 0, window=window, sinks=sinks, scale=scale))
    done(ctx)
    assert bool((room[:, :, 1] == -3).all())
    got = room[:, :, 0]
    return got.flip(0, 1) if down else got


def check_attention(ctx, zkb, batch, cache, q, out_kind, window, sinks, scale=None, hints=True, down=False):
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    got = run_attention(ctx, zkb, batch, cache, q, out_kind, window, sinks, scale, hints, down)
    want, bound = attention_reference(batch, cache, q, scale, window, sinks)
    inside = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for _, at, rows, _ in batch.each():
        inside[at:at + rows] = True
    assert bool((got[~inside] == -3).all())  # rows of no sequence are left as they were
    x, y, b = values_of(got[inside]), want[inside], bound[inside]
    fine = torch.isfinite(y)
    assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x[~fine & ~torch.isnan(y)], y[~fine & ~torch.isnan(y)])
    over = ((x - y).abs() - b)[fine]
    assert not over.numel() or float(over.max()) <= 0, (float(over.max()), int((over > 0).sum()), over.numel())
    return got


ATTENTION_CASES = [  # shape, q heads, kv heads, dim, cache, out, window, sinks, order, pad
    ([(1, 1)], 1, 1, 32, "bf16", "bf16", 0, 0, "shtd", 0),
    ([(1, 1), (1, 2), (0, 5), (1, 17)], 4, 1, 128, "int8", "words", 0, 0, "shtd", 0),
    ([(1, 2048)], 32, 8, 128, "int8", "bf16", 0, 0, "shtd", 0),
    ([(1, 5000), (1, 129), (1, 128), (1, 127)], 8, 2, 128, "bf16", "bf16", 0, 0, "sthd", 0),
    ([(1, 700), (1, 30)], 5, 1, 64, "int8", "bf16", 100, 4, "shtd", 0),
    ([(1, 4000)], 16, 2, 64, "bf16", "words", 1, 0, "shtd", 8),
    ([(3, 333), (2, 64)], 6, 3, 32, "int8", "words", 7, 20, "tshd", 0),
    ([(4, 1500), (4, 4)], 8, 2, 128, "bf16", "bf16", 0, 0, "shtd", 0),
    ([(5, 600)], 64, 1, 64, "int8", "bf16", 0, 0, "shtd", 0),
    ([(32, 128)], 2, 1, 32, "bf16", "words", 0, 0, "shtd", 0),
    ([(32, 2048)], 8, 2, 128, "int8", "words", 0, 0, "shtd", 0),
    ([(33, 700), (0, 0), (1, 90), (64, 64)], 12, 4, 64, "bf16", "bf16", 0, 0, "sthd", 0),
    ([(300, 300), (129, 500)], 4, 1, 128, "bf16", "bf16", 0, 0, "shtd", 0),
    ([(257, 300), (128, 128)], 3, 3, 128, "int8", "bf16", 0, 0, "shtd", 0),
    ([(400, 1000)], 4, 2, 64, "bf16", "bf16", 130, 3, "shtd", 0),
    ([(500, 600), (63, 64)], 2, 1, 128, "int8", "words", 50, 200, "shtd", 0),
    ([(200, 200)], 5, 1, 32, "int8", "bf16", 1, 1, "shtd", 3),
    ([(150, 160)], 9, 3, 64, "bf16", "bf16", 0, 0, "shtd", 1),
    ([(1, 300), (90, 300)], 3, 1, 128, "bf16", "bf16", 0, 0, "shtd", 4),
    ([(1, 10 + 13 * b) for b in range(80)], 4, 2, 64, "int8", "bf16", 64, 2, "shtd", 0),
]


@gpu
@pytest.mark.parametrize("shape,hq,hk,d,kind,out,window,sinks,order,pad", ATTENTION_CASES)
def test_attention(ctx, zkb, shape, hq, hk, d, kind, out, window, sinks, order, pad):
    g = gen(hq * d + window)
    batch = Batch(shape, behind=2)
    cache = Cache(g, kind, len(shape), hk, max(n for _, n in shape) + 3, d, order, pad)
    q = torch.randn(batch.n_rows, hq, d + pad, generator=g, device="cuda").bfloat16()[..., :d]
    check_attention(ctx, zkb, batch, cache, q, out, window, sinks, hints=len(shape) % 2 == 0, down=out == "words")


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("order,pad", [("shtd", 0), ("tshd", 0), ("hstd", 3)])
@pytest.mark.parametrize("shape,hq,hk,window,sinks", [([(129, 400), (40, 390), (0, 3), (1, 60), (86, 86)], 24, 8, 0, 0), ([(129, 400), (40, 390), (0, 3), (1, 60), (86, 86)], 24, 8, 33, 5),
                                                      ([(100, 700), (90, 600)], 32, 4, 0, 0), ([(100, 700), (90, 600)], 32, 4, 300, 2)])
def test_attention_of_many_rows(ctx, zkb, kind, d, order, pad, shape, hq, hk, window, sinks):
    """Batches whose rows fill the large products, with and without their keys spread over thread blocks, in caches that can be copied by tiles and in one that cannot."""
    g = gen(d + window)
    batch = Batch(shape, behind=1, gap=1)
    cache = Cache(g, kind, len(shape), hk, max(n for _, n in shape) + 1, d, order, pad)
    q = torch.randn(batch.n_rows, hq, d, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "bf16" if window else "words", window, sinks)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_attention_rows_before_the_cache_and_behind_it(ctx, zkb, kind, rows):
    """More rows than tokens: the first rows see nothing and get zeros; lengths past the capacity: what is there is seen."""
    g = gen(rows)
    batch = Batch([(rows, rows // 2), (rows, 0), (rows, 100), (rows, 64 + rows // 2)])
    cache = Cache(g, kind, 4, 2, 64, 64)
    q = torch.randn(batch.n_rows, 4, 64, generator=g, device="cuda").bfloat16()
    got = check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0)
    assert bool((got[rows:2 * rows] == 0).all())
    check_attention(ctx, zkb, batch, cache, q, "bf16", 20, 3)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,length,d,window,sinks", [(1, 300, 128, 50, 2), (3, 200, 64, 0, 0), (3, 200, 32, 9, 1), (60, 200, 128, 0, 0), (150, 400, 128, 70, 5), (150, 400, 64, 0, 0), (20, 40, 32, 5, 3)])
def test_attention_what_is_hidden_does_not_reach_a_row(ctx, zkb, kind, rows, length, d, window, sinks):
    """NaN and infinities behind the last token, outside the window and among the step's own later tokens."""
    g = gen(rows + d)
    batch = Batch([(rows, length)])
    cache = Cache(g, kind, 1, 2, length + 70, d)
    q = torch.randn(rows, 4, d, generator=g, device="cuda").bfloat16()
    places = list(range(length, length + 70)) + ([sinks + 1, length - rows - window] if window else []) + ([length - 1, length - rows + rows // 2] if rows > 1 else [])
    for i, p in enumerate(p for p in places if 0 <= p < length + 70):
        x = math.nan if kind == "int8" and length - rows <= p < length else [math.nan, math.inf, -math.inf][i % 3]
        for part, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            if part is cache.k and p < length and i % 2:
                continue
            if kind == "int8":
                scale[0, :, p] = x
                part[0, :, p][part[0, :, p] == 0] = 1  # a code of zero times infinity would be NaN: kept out of the comparison
            else:
                part[0, :, p, ::3] = x
    check_attention(ctx, zkb, batch, cache, q, "bf16", window, sinks)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,length", [(1, 500), (2, 700), (130, 260)])
def test_attention_scores_far_apart(ctx, zkb, kind, rows, length):
    """One key's score far above the others (the softmax is that key's value), and scores of a size that the exponential cannot take as they are."""
    g = gen(rows)
    batch, d = Batch([(rows, length)]), 64
    cache = Cache(g, kind, 1, 1, length, d)
    q = (torch.randn(rows, 2, d, generator=g, device="cuda") * 6).bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0, scale=3.0)
    check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0, scale=-3.0)
    check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0, scale=0.0)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,length,d,window,sinks", [(5000, 5000, 64, 0, 0), (4000, 4200, 128, 300, 40), (100, 3000, 128, 0, 0)])
def test_attention_of_many_units(ctx, zkb, kind, rows, length, d, window, sinks):
    """More pairs of tiles than thread blocks, and keys spread over many thread blocks; infinities in one token's values that the last rows see."""
    g = gen(rows)
    batch, cache = Batch([(rows, length)]), Cache(g, kind, 1, 4, length, d)
    q = torch.randn(rows, 16, d, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "bf16", window, sinks)
    if kind == "bf16":
        cache.v[0, 1, length - 20, 5:9] = math.inf
        cache.v[0, 2, length - 30, 7] = -math.inf
        check_attention(ctx, zkb, batch, cache, q, "bf16", window, sinks)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("order,pad", [("shtd", 0), ("hstd", 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1600, 7)])
def test_attention_of_several_rows_over_long_caches(ctx, zkb, kind, d, order, pad, window, sinks):
    """Rows that fill one small product and part of the next, and a sequence of fewer."""
    g = gen(d + window)
    batch = Batch([(3, 2500), (0, 0), (5, 1801), (1, 2500), (4, 2)])
    cache = Cache(g, kind, 5, 2, 2501, d, order, pad)
    q = torch.randn(batch.n_rows, 14, d, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "words", window, sinks)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("most,length", [(30, 120), (30, 250), (120, 250), (1, 2)])
def test_attention_of_many_short_sequences(ctx, zkb, kind, most, length):
    """Several sequences a thread block, of one tile or two and of one block of keys or two; some without rows, some without tokens."""
    g, rng = gen(most + length), np.random.default_rng(most)
    shape = [(int(r), int(n)) for r, n in zip(rng.integers(0, most + 1, 300), rng.integers(0, length + 1, 300))] + [(most, length)]
    batch, cache = Batch(shape, behind=1), Cache(g, kind, len(shape), 4, length, 64)
    q = torch.randn(batch.n_rows, 16, 64, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "words", 0, 0)


@gpu
def test_attention_values_that_are_no_numbers_in_a_long_cache(ctx, zkb):
    """Every row sees an infinity among 30,000 tokens, so that all outputs go the slow way, for longer than a wait within the kernel may take without a reason."""
    g, rows, length, heads, d = gen(8), 300, 30000, 40, 128
    batch, cache = Batch([(rows, length)]), Cache(g, "bf16", 1, heads, length, d)
    cache.v[0, :, 11, 3::7] = math.inf
    cache.v[0, :, length - rows, 4::7] = -math.inf
    q = torch.randn(rows, heads, d, generator=g, device="cuda").bfloat16()
    check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0)


@gpu
def test_as_many_sequences_as_there_may_be(ctx, zkb):
    """65,535 sequences of a token: written, and seen, each by its own row."""
    g, seqs, d, cap = gen(6), 65535, 32, 3
    pos = torch.arange(seqs, device="cuda") % cap
    first, lens = torch.arange(seqs + 1, device="cuda", dtype=torch.int32), (pos + 1).int()
    k, v = (torch.randn(seqs, 1, cap, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    x = torch.randn(seqs, 3, d, generator=g, device="cuda").bfloat16()
    q, out = x[:, :1].clone(), torch.zeros(seqs, 1, d, device="cuda", dtype=torch.bfloat16)
    cache = zkb.KvCache(k=k.data_ptr(), v=v.data_ptr(), type=zkb.VALUE_BF16, n_seqs=seqs, n_heads=1, head_dim=d, capacity=cap, seq_stride=cap * d, head_stride=cap * d, token_stride=d)
    rows = zkb.StepRows(first=first.data_ptr(), kv_len=lens.data_ptr(), n_rows=seqs, max_rows=1, max_len=cap)
    torch.cuda.synchronize()
    ctx.step_norm_rope(zkb.StepNormRope(cache=cache, rows=rows, q=x.data_ptr(), k=x[:, 1:].data_ptr(), v=x[:, 2:].data_ptr(), q_out=q.data_ptr(), q_stride=3 * d, k_stride=3 * d, v_stride=3 * d,
                                        head_stride=d, q_out_stride=d, q_out_head_stride=d, q_heads=1, rotary_dim=0, eps=1e-6))
    ctx.step_attention(zkb.StepAttention(cache=cache, rows=rows, q=q.data_ptr(), out=out.data_ptr(), q_stride=d, q_head_stride=d, out_stride=d, out_head_stride=d, q_heads=1, scale=0.2))
    done(ctx)
    each = torch.arange(seqs, device="cuda")
    assert torch.equal(q, x[:, :1]) and torch.equal(k[each, 0, pos], x[:, 1]) and torch.equal(v[each, 0, pos], x[:, 2])
    s = torch.einsum("sd,std->st", q[:, 0].double(), k[:, 0].double()) * 0.2
    w = torch.softmax(s.masked_fill(torch.arange(cap, device="cuda") > pos[:, None], -math.inf), -1)
    want, size = (torch.einsum("st,std->sd", w, y) for y in (v[:, 0].double(), v[:, 0].double().abs()))
    # as attention_reference counts: weights off by 2^-8 and scores by 36 roundings of 2^-24 of magnitudes below 64, the result's own 2^-8
    assert bool(((out[:, 0].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -11) * (size + want.abs())).all())


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("max_rows,max_len", [(1, 1), (0, 1), (1, 0), (1 << 31, 1 << 31), (7, 900)])
def test_attention_hints_that_are_wrong_change_no_result(ctx, zkb, kind, max_rows, max_len):
    """Fewer rows and tokens than there are, and more; both ways of laying out the work meet them."""
    g = gen(max_rows % 100)
    for shape in ([(300, 700), (2, 5)], [(1, 1500), (3, 40)]):
        batch, d = Batch(shape, behind=1), 64
        cache = Cache(g, kind, 2, 2, 1500, d)
        q = torch.randn(batch.n_rows, 8, d, generator=g, device="cuda").bfloat16()
        args = batch.args

        def hinted(zkb, hints=True):
            r = args(zkb, hints)
            r.max_rows, r.max_len = max_rows, max_len
            return r

        batch.args = hinted
        check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0)
        check_attention(ctx, zkb, batch, cache, q, "words", 100, 4)


@gpu
@pytest.mark.parametrize("first,lens", [([0, 9, 4, 30], [20, 20, 20]), ([-5, 3, 60, 10], [50, -3, 7]), ([40, 30, 20, 10], [5, 5, 5]), ([0, 2 ** 31 - 1, -(2 ** 31), 24], [2 ** 31 - 1, -(2 ** 31), 40])])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,heads", [(24, 4), (24, 64)])
def test_arrays_that_describe_no_batch_stay_inside_the_buffers(ctx, zkb, first, lens, kind, rows, heads):
    """Borders that descend, or lie outside the rows; lengths below zero and past the capacity: what the rows get is undefined, what lies around them is not touched."""
    g, d, cap = gen(rows), 64, 50 if heads == 4 else 600  # few rows a product, and many
    cache = Cache(g, kind, 5, 2, cap, d)
    before = [x.clone() for x in (cache.k, cache.v)]
    f, n = torch.tensor(first, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    c = cache.args(zkb)
    size = cache.k.element_size()
    c.n_seqs, c.k, c.v = 3, c.k + size * cache.k.stride(0), c.v + size * cache.k.stride(0)  # sequences 0 and 4 lie around it
    if kind == "int8":
        c.k_scale, c.v_scale = c.k_scale + 4 * cache.k_scale.stride(0), c.v_scale + 4 * cache.k_scale.stride(0)
    batch = zkb.StepRows(first=f.data_ptr(), kv_len=n.data_ptr(), n_rows=rows)
    x = torch.randn(rows, heads + 4, d, generator=g, device="cuda").bfloat16()
    out = torch.full((rows + 2, heads, d), -3.0, device="cuda", dtype=torch.bfloat16)
    freq = np.ones(16)
    torch.cuda.synchronize()
    ctx.step_norm_rope(zkb.StepNormRope(cache=c, rows=batch, q=x.data_ptr(), k=x[:, heads:].data_ptr(), v=x[:, heads + 2:].data_ptr(), h_inv_freq=freq.ctypes.data, q_out=out[1].data_ptr(),
                                        q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0), head_stride=d, q_out_stride=out.stride(0), q_out_head_stride=d, q_heads=heads, rotary_dim=32, eps=1e-6))
    ctx.step_attention(zkb.StepAttention(cache=c, rows=batch, q=x.data_ptr(), out=out[1].data_ptr(), q_stride=x.stride(0), q_head_stride=d, out_stride=out.stride(0), out_head_stride=d, q_heads=heads, scale=0.1))
    done(ctx)
    assert bool((out[0] == -3).all()) and bool((out[-1] == -3).all())
    for x, y in zip((cache.k, cache.v), before):
        assert torch.equal(x[0], y[0]) and torch.equal(x[4], y[4])


@gpu
@pytest.mark.parametrize("d,order,heads", [(128, "thsd", 8), (64, "hstd", 2), (64, "shtd", 2)])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_offsets_past_32_bits(ctx, zkb, kind, d, order, heads):
    """Tokens, heads or sequences so far apart that the last ones lie more than 2^32 bytes into the cache: written by norm_rope, read by the attention, by one row and by many."""
    size, cap = 1 if kind == "int8" else 2, 33
    far = dict(t=(1 << 32) // 30 // size, s=(1 << 32) // size, h=(1 << 32) // size)[order[0]] // 64 * 64
    stride = {"thsd": dict(t=far, h=2 * d, s=d), "hstd": dict(h=far, s=cap * d, t=d), "shtd": dict(s=far, h=cap * d, t=d)}[order]
    seqs = 2
    need = (seqs - 1) * stride["s"] + (heads - 1) * stride["h"] + (cap - 1) * stride["t"] + d
    assert need * size > 1 << 32
    g = gen(d)
    cache = Cache(g, kind, seqs, heads, cap, d, blank=True)
    rooms = [torch.zeros(need, device="cuda", dtype=cache.k.dtype) for _ in range(2)]
    cache.k, cache.v = (r.as_strided((seqs, heads, cap, d), (stride["s"], stride["h"], stride["t"], 1)) for r in rooms)
    for rows in (cap - 2, 1):
        batch = Batch([(rows, cap), (rows, cap - 1)])
        x = torch.randn(batch.n_rows, 4 * heads, d, generator=g, device="cuda").bfloat16()
        q = x[:, :2 * heads]
        freq = 1e4 ** (-np.arange(d // 2) / (d // 2))
        out = torch.zeros(batch.n_rows, 2 * heads, d, device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        ctx.step_norm_rope(zkb.StepNormRope(cache=cache.args(zkb), rows=batch.args(zkb), q=x.data_ptr(), k=x[:, 2 * heads:].data_ptr(), v=x[:, 3 * heads:].data_ptr(), h_inv_freq=freq.ctypes.data,
                                            q_out=out.data_ptr(), q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0), head_stride=d, q_out_stride=out.stride(0), q_out_head_stride=d,
                                            q_heads=2 * heads, rotary_dim=d, eps=1e-6))
        done(ctx)
        k, v = cache.values()
        for b, r0, r, p0 in batch.each():
            want = x[r0:r0 + r, 3 * heads:].double().transpose(0, 1)
            step = cache.v_scale[b, :, p0:p0 + r].double()[..., None] if kind == "int8" else 0
            assert bool(((v[b, :, p0:p0 + r] - want).abs() <= step * (0.5 + 127 * 2.0 ** -22)).all())
            assert bool((k[b, :, p0:p0 + r] != 0).any(-1).all())
        check_attention(ctx, zkb, batch, cache, q, "bf16", 0, 0)
    del rooms, cache
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("table", ["bf16", "int8"])
def test_embedding_rows_past_32_bits(ctx, zkb, table):
    g, vocab, width, stride = gen(3), 1100, 40, 1 << 22
    dtype = torch.int8 if table == "int8" else torch.bfloat16
    room = torch.zeros((vocab - 1) * stride + width, device="cuda", dtype=dtype)
    tab = room.as_strided((vocab, width), (stride, 1))
    tab.copy_(torch.randint(-100, 100, (vocab, width), generator=g, device="cuda"))
    scales = torch.rand(vocab, generator=g, device="cuda")
    ids = torch.tensor([vocab - 1, 0, 3, vocab - 1, 1024, vocab - 1], dtype=torch.int32, device="cuda")
    out = torch.zeros(len(ids), width, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    ctx.step_embed(zkb.StepEmbed(ids=ids.data_ptr(), table=tab.data_ptr(), row_scale=scales.data_ptr() if table == "int8" else 0, out=out.data_ptr(), table_stride=stride, out_stride=width,
                                 n_tokens=len(ids), vocab=vocab, width=width, table_type=2 if table == "int8" else 0, out_type=0, scale=1.0))
    done(ctx)
    want = tab[ids.long()].float() * (scales[ids.long()][:, None] if table == "int8" else 1.0)
    assert torch.equal(out, want.bfloat16())
    del room, tab
    torch.cuda.empty_cache()


@gpu
def test_queries_may_be_turned_where_they_are(ctx, zkb):
    g, d, heads = gen(9), 64, 6
    batch, cache = Batch([(50, 60), (1, 9)], behind=2), Cache(gen(1), "bf16", 2, 2, 64, 64, blank=True)
    x = torch.randn(batch.n_rows, heads + 4, d, generator=g, device="cuda").bfloat16()
    freq, results = 1e4 ** (-np.arange(16) / 16), []
    for inside in (False, True):
        rows = x.clone()
        out = rows if inside else x.clone()
        torch.cuda.synchronize()
        ctx.step_norm_rope(zkb.StepNormRope(cache=cache.args(zkb), rows=batch.args(zkb), q=rows.data_ptr(), k=rows[:, heads:].data_ptr(), v=rows[:, heads + 2:].data_ptr(), h_inv_freq=freq.ctypes.data,
                                            q_out=out.data_ptr(), q_stride=rows.stride(0), k_stride=rows.stride(0), v_stride=rows.stride(0), head_stride=d, q_out_stride=out.stride(0), q_out_head_stride=d,
                                            q_heads=heads, rotary_dim=32, eps=1e-6))
        done(ctx)
        results.append(out)
    assert torch.equal(*results) and not torch.equal(results[0], x)


class Step:
    """A whole step on buffers of its own: embedding rows, norms and rotation, attention."""

    def __init__(self, zkb, seed, kind, rows, cap=300, seqs=3, d=64, hq=8, hk=2):
        self.zkb, self.g, self.dims = zkb, gen(seed), (seqs, rows, cap, d, hq, hk)
        self.cache = Cache(self.g, kind, seqs, hk, cap, d, blank=True)
        self.table = torch.randn(50, (hq + 2 * hk) * d, generator=self.g, device="cuda").bfloat16()
        n = seqs * rows
        self.ids, self.first, self.lens = (torch.zeros(x, dtype=torch.int32, device="cuda") for x in (n, seqs + 1, seqs))
        self.x = torch.zeros(n, hq + 2 * hk, d, device="cuda", dtype=torch.bfloat16)
        self.q, self.out = (torch.zeros(n, hq, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        self.freq = 1e4 ** (-np.arange(d // 2) / (d // 2))
        self.weight = torch.randn(d, generator=self.g, device="cuda").bfloat16()
        rows_ = zkb.StepRows(first=self.first.data_ptr(), kv_len=self.lens.data_ptr(), n_rows=n)
        c, w, s = self.cache.args(zkb), self.x.stride(0), self.q.stride(0)
        self.calls = (zkb.StepEmbed(ids=self.ids.data_ptr(), table=self.table.data_ptr(), out=self.x.data_ptr(), table_stride=w, out_stride=w, n_tokens=n, vocab=50, width=w, scale=1.0),
                      zkb.StepNormRope(cache=c, rows=rows_, q=self.x.data_ptr(), k=self.x[:, hq:].data_ptr(), v=self.x[:, hq + hk:].data_ptr(), q_weight=self.weight.data_ptr(),
                                       k_weight=self.weight.data_ptr(), h_inv_freq=self.freq.ctypes.data, q_out=self.q.data_ptr(), q_stride=w, k_stride=w, v_stride=w, head_stride=d, q_out_stride=s,
                                       q_out_head_stride=d, q_heads=hq, rotary_dim=d, eps=1e-6),
                      zkb.StepAttention(cache=c, rows=rows_, q=self.q.data_ptr(), out=self.out.data_ptr(), q_stride=s, q_head_stride=d, out_stride=s, out_head_stride=d, q_heads=hq, scale=d ** -0.5))

    def batch(self, shape, seed):
        """Other tokens of another batch into the arrays that the calls read."""
        self.shape = shape
        self.ids.copy_(torch.randint(0, 50, self.ids.shape, generator=gen(seed), device="cuda", dtype=torch.int32))
        self.first.copy_(torch.tensor(np.concatenate([[0], np.cumsum([r for r, _ in shape])]), dtype=torch.int32))
        self.lens.copy_(torch.tensor([n for _, n in shape], dtype=torch.int32))
        self.out.fill_(-3)
        torch.cuda.synchronize()

    def run(self, ctx):
        ctx.step_embed(self.calls[0])
        ctx.step_norm_rope(self.calls[1])
        ctx.step_attention(self.calls[2])

    def check(self):
        """The attention over what the cache holds now; the cache's new tokens against the table's."""
        batch = Batch(self.shape)
        seqs, rows, cap, d, hq, hk = self.dims
        n = batch.n_rows
        want, bound = attention_reference(batch, self.cache, self.q[:n], d ** -0.5, 0, 0)
        assert bool(((self.out[:n].double() - want).abs() <= bound).all()) and bool((self.out[n:] == -3).all())
        x = self.table[self.ids.long()].view(-1, hq + 2 * hk, d)
        assert torch.equal(self.x, x)
        _, v = self.cache.values()
        for b, at, r, pos in batch.each():
            step = self.cache.v_scale[b, :, pos:pos + r].double()[..., None] if self.cache.kind == "int8" else 0
            assert bool(((v[b, :, pos:pos + r].transpose(0, 1) - x[at:at + r, hq + hk:].double()).abs() <= (step.transpose(0, 1) if self.cache.kind == "int8" else 0) * (0.5 + 127 * 2.0 ** -22)).all())


SHAPES = {1: [[(1, 5), (1, 300), (1, 77)], [(1, 6), (0, 300), (1, 1)]], 90: [[(90, 90), (1, 250), (90, 300)], [(3, 3), (80, 200), (0, 0)]]}


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows", [1, 90])
def test_captured_steps_serve_other_batches_side_by_side(ctx, zkb, kind, rows):
    """Two steps of two contexts captured into graphs, replayed on streams of their own at the same time, for batches that were not there when they were captured;
    what a replay computes is what the same call computes."""
    other = zkb.Context(device=0, max_log_size=10)
    try:
        steps = [Step(zkb, 1 + i, kind, rows) for i in range(2)]
        graphs = []
        for step, c in zip(steps, (ctx, other)):
            step.batch([(0, 0)] * 3, 0)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(c.stream())):
                step.run(c)
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in steps]
        for shape in SHAPES[rows]:
            for i, step in enumerate(steps):
                step.batch(shape, 5 + i)
            for _ in range(3):
                for graph, stream in zip(graphs, streams):
                    with torch.cuda.stream(stream):
                        graph.replay()
            torch.cuda.synchronize()
            for step, c in zip(steps, (ctx, other)):
                step.check()
                replayed = step.out.clone(), step.cache.k.clone()
                step.batch(shape, 5 + steps.index(step))
                step.run(c)
                done(c)
                assert torch.equal(step.out, replayed[0]) and torch.equal(step.cache.k, replayed[1])
        del graphs
    finally:
        other.close()


@gpu
def test_contexts_on_threads_of_their_own(zkb):
    """Steps of four contexts at once, each from a thread of its own: one token a sequence and many."""
    import threading

    contexts = [zkb.Context(device=0, max_log_size=10) for _ in range(4)]
    steps, wrong = [Step(zkb, 20 + i, ("bf16", "int8")[i % 2], (1, 90)[i // 2]) for i in range(4)], []
    for i, s in enumerate(steps):
        s.batch(SHAPES[s.dims[1]][0], i)

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
    torch.cuda.synchronize()
    for s in steps:
        s.check()
    for c in contexts:
        c.close()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_a_step_between_the_witness_generators(ctx, zkb, oracle, kind):
    """The run of all calls as a proof makes its values: zkb_witness_dequant leaves a block of tokens' queries, keys and values as words, descending; they are normed, turned
    and cached; the attention over the cache and the embedding's rows go straight into the leaves of zkb_witness_residual_stream, which adds them. Nothing waits in between."""
    from zk_inference_prover_b200 import witness_cases as wc

    g, tokens, d, hq, hk, before = gen(4), 32, 32, 4, 2, 40
    heads, n = hq + 2 * hk, hq * d
    dq = wc.dequant_case(3, 1, tokens, heads, d, 13, 1, 1)
    cfg, rows = dq["cfg"], dq["rows"]
    rs = wc.residual_stream_case(5, "pairs", n, 5, tokens, kind=0, spread=6)
    up, ml = ctx.upload, rs["m_len"]
    acc, sx, sw = (ctx.upload_bytes(np.ascontiguousarray(dq[k])) for k in ("acc", "sx", "sw"))
    norm3, mul2 = up(dq["norm3"].reshape(-1)), up(dq["mul2"].reshape(-1))
    base, pre = [ctx.alloc(rows).zero() for _ in range(dq["n_base"])], [ctx.alloc(rows).zero() for _ in range(dq["n_pre"])]
    ms = [ctx.alloc(cfg[k]).zero() for k in ("n_norm", "n_frac", "n_mul", "n_r8")]
    counts, want = ctx.alloc(4).zero(), ctx.alloc(rows * d).zero()
    table = torch.randint(-127, 128, (60, n), generator=g, device="cuda", dtype=torch.int8)
    scales = (0.5 + torch.rand(60, generator=g, device="cuda")) / 50
    ids = torch.randint(0, 60, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    batch, cache = Batch([(tokens, before + tokens)]), Cache(g, kind, 1, hk, before + tokens + 5, d)
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).bfloat16() for _ in range(2))
    freq = 1e4 ** (-np.arange(d // 2) / (d // 2))
    q = torch.zeros(tokens, hq, d, device="cuda", dtype=torch.bfloat16)
    wit = torch.full((tokens, 2 * n), -1, device="cuda", dtype=torch.int32)
    r_norm, r_smul = up(rs["norm3"]), ctx.upload_bytes(np.ascontiguousarray(rs["smul3"], np.int32))
    cols = [ctx.alloc(32).zero() for _ in range(rs["n_cols"])]
    out_pat, out_nat, in_nat = ctx.alloc(32 * n).zero(), ctx.alloc(64 * n).zero(), ctx.alloc(128 * n).zero()
    r_ms, r_counts = {k: ctx.alloc(ml[k]).zero() for k in ("pow", "norm", "val", "frac", "smul")}, ctx.alloc(4).zero()
    torch.cuda.synchronize()
    ctx.witness_dequant(cfg, acc.ptr, 0, 0, sx.ptr, sw.ptr, norm3.ptr, mul2.ptr, [b.ptr for b in base], [p.ptr for p in pre], *[m.ptr for m in ms], counts.ptr, want.ptr)
    at = lambda h: want.ptr + 4 * d * ((tokens - 1) * heads + heads - 1 - h)  # noqa: E731  head h of token 0
    ctx.step_norm_rope(zkb.StepNormRope(cache=cache.args(zkb), rows=batch.args(zkb), q=at(0), k=at(hq), v=at(hq + hk), q_weight=wq.data_ptr(), k_weight=wk.data_ptr(), h_inv_freq=freq.ctypes.data,
                                        q_out=q.data_ptr(), q_stride=-heads * d, k_stride=-heads * d, v_stride=-heads * d, head_stride=-d, q_out_stride=n, q_out_head_stride=d, type=zkb.VALUE_WORD,
                                        q_heads=hq, rotary_dim=d, eps=1e-6))
    ctx.step_embed(zkb.StepEmbed(ids=ids.data_ptr(), table=table.data_ptr(), row_scale=scales.data_ptr(), out=wit.data_ptr(), table_stride=n, out_stride=2 * n, n_tokens=tokens, vocab=60, width=n,
                                 table_type=zkb.VALUE_INT8, out_type=zkb.VALUE_WORD, scale=1.0))
    ctx.step_attention(zkb.StepAttention(cache=cache.args(zkb), rows=batch.args(zkb), q=q.data_ptr(), out=wit.data_ptr() + 4 * n, q_stride=n, q_head_stride=d, out_stride=2 * n, out_head_stride=d,
                                         q_heads=hq, out_type=zkb.VALUE_WORD, scale=d ** -0.5))
    ctx.witness_residual_stream(rs["lowered_groups"], rs["lowered_slots"], rs["out_slot"], rs["kind"], rs["sticky"], rs["kmax"], r_norm.ptr, len(rs["norm3"]) // 3, r_smul.ptr, len(rs["smul3"]) // 3, [],
                                rs["n_val"], wit.data_ptr(), tokens, 5, [c.ptr for c in cols], out_pat.ptr, out_nat.ptr, in_nat.ptr, {k: (v.ptr, ml[k]) for k, v in r_ms.items()}, [], r_counts.ptr)
    done(ctx)
    o = oracle.witness_dequant(dq["acc"], dq["jx"], dq["jw"], dq["sx"], dq["sw"], dq["norm3"], dq["mul2"], dq["n_base"], dq["n_pre"], cfg)
    given = want.download()[:rows * d]
    assert np.array_equal(given, np.asarray(o["want"]).reshape(-1))
    x = torch.from_numpy(given.astype(np.int32)).cuda().view(tokens, heads, d).flip(0, 1)
    x = (x << 16).view(torch.float32)
    y, size = rope_reference(batch, x[:, :hq + hk], [wq] * hq + [wk] * hk, 1e-6, freq, 0)
    assert bool(((q.double() - y[:, :hq]).abs() <= 2.0 ** -8 * y[:, :hq].abs() + 2.0 ** -18 * size[:, :hq]).all())
    k, v = cache.values()
    for got, ref, s, scale in ((k, y[:, hq:], size[:, hq:], cache.k_scale), (v, x[:, hq + hk:].double(), 0 * x[:, hq + hk:].double(), cache.v_scale)):
        diff = (got[0, :, before:before + tokens].transpose(0, 1) - ref).abs()
        if kind == "bf16":
            assert bool((diff <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * s).all())
        else:
            assert bool((diff <= scale[0, :, before:before + tokens].T.double()[..., None] * (0.5 + 127 * 2.0 ** -22) + 2.0 ** -18 * s.amax(-1, keepdim=True)).all())
    assert torch.equal(wit[:, :n], words((table[ids.long()].float() * scales[ids.long()][:, None]).bfloat16()))
    ref, bound = attention_reference(batch, cache, q, d ** -0.5, 0, 0)
    assert bool(((values_of(wit[:, n:].reshape(tokens, hq, d)) - ref).abs() <= bound).all())
    summed = oracle.witness_residual_stream({**rs, "wit": wit.cpu().numpy().astype(np.uint32).reshape(-1)})
    assert np.array_equal(out_pat.download()[:32 * n], summed["out_pat"])
