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
