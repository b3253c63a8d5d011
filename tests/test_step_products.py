"""Products of codes (zkb_step_product): the ways that their sizes and layouts lead to, beside those of test_step_layer.py and test_step_layer_edges.py."""
import math

import pytest
import torch

from test_step_layer import INT8, TYPES, Weights, check_product, codes_of, room, run_product, untouched
from test_step_values import done, gen

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n_in,n_out", [(20, 14336, 4096), (40, 14336, 14336), (64, 4096, 9472), (100, 4096, 1500), (128, 8192, 4096)])
def test_weights_that_arrive_in_any_order(ctx, zkb, group, rows, n_in, n_out):
    """Tiles of 4-bit weights while copies on another stream keep the memory busy: the sums are right, and have the same bits each time."""
    g = gen(rows + group)
    x, w, x_scale = codes_of(g, rows, n_in), Weights(g, "int4", n_out, n_in, group), torch.rand(rows, generator=g, device="cuda") + 0.1
    ys, other = [torch.zeros(rows, n_out, device="cuda") for _ in range(12)], torch.cuda.Stream()
    a, b = (torch.empty(1 << 28, device="cuda", dtype=torch.int8) for _ in range(2))
    torch.cuda.synchronize()
    for y in ys:
        with torch.cuda.stream(other):
            b.copy_(a)
        run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    other.synchronize()
    check_product("f32", ys[0], x, x_scale, w)
    assert all(torch.equal(ys[0], y) for y in ys[1:])


@gpu
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 32), ("int4", 128)])
@pytest.mark.parametrize("rows", [1, 2, 5, 13, 40, 300])
@pytest.mark.parametrize("short", [1, 15, 16, 17, 31])
def test_arrays_that_end_inside_a_block_of_memory(ctx, zkb, kind, group, rows, short):
    """Rows and weights on odd boundaries whose last bytes lie `short` before a multiple of 32 bytes; what is behind them is no part of the sums."""
    g, n_out = gen(rows + short), 37
    n_in = 1024 + 33 if kind == "int8" else 1024 + 2 * 33
    bytes_ = n_in if kind == "int8" else n_in // 2
    x, w = codes_of(g, rows, n_in, 0, -(rows * n_in + short) % 32), Weights(g, kind, n_out, n_in, group, 0, -(n_out * bytes_ + short) % 32)
    assert (x.data_ptr() + rows * n_in) % 32 == 32 - short and (w.w.data_ptr() + n_out * bytes_) % 32 == 32 - short
    x_scale, y = torch.rand(rows, generator=g, device="cuda") + 0.1, torch.zeros(rows, n_out, device="cuda")
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    check_product("f32", y, x, x_scale, w)


def with_scales(w, pad, off):
    """w's scales laid out with `pad` more behind each output's, from `off` scales behind a multiple of 16 bytes on, NaN in between and behind."""
    groups = -(-w.n_in // w.group)
    keep = torch.full((w.scale.shape[0] * (groups + pad) + off,), math.nan, device="cuda", dtype=torch.bfloat16)
    scale = keep[off:].view(-1, groups + pad)
    scale[:, :groups] = w.scale[:, :groups]
    assert keep.data_ptr() % 16 == 0
    w.scale = scale
    return w


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("pad,off", [(0, 0), (8, 0), (0, 1), (0, 2), (0, 4), (1, 0), (3, 2), (8, 4), (4, 8)])
@pytest.mark.parametrize("rows,n_out", [(1, 200), (2, 130), (5, 300), (16, 260), (20, 256), (40, 300), (64, 1), (150, 257), (300, 700)])
def test_scales_wherever_they_lie(ctx, zkb, group, pad, off, rows, n_out):
    """Groups by eights and not, in rows that follow one another and that do not, on every boundary that is taken; codes spread over clusters where they are many."""
    g = gen(rows + group)
    for n_in in (group * 8, 4096, 4096 + group, 14336):
        x, w, x_scale = codes_of(g, rows, n_in), with_scales(Weights(g, "int4", n_out, n_in, group), pad, off), torch.rand(rows, generator=g, device="cuda") + 0.1
        y = torch.zeros(rows, n_out, device="cuda")
        torch.cuda.synchronize()
        run_product(ctx, zkb, x, x_scale, w, ("f32", y))
        done(ctx)
        check_product("f32", y, x, x_scale, w)


@gpu
@pytest.mark.parametrize("rows", [3, 8, 9, 16])
@pytest.mark.parametrize("n_in,n_out", [(4096, 9000), (14336, 2400), (131071, 300), (1024, 40001), (4100, 8200), (2049, 17000)])
@pytest.mark.parametrize("pad,off", [(0, 0), (16, 0), (1, 3)])
@pytest.mark.parametrize("kind", ["int32", "bf16"])
def test_few_rows_and_many_8_bit_weights(ctx, zkb, rows, n_in, n_out, pad, off, kind):
    """More than 2^25 weights: tiles of sixteen rows, spread over clusters or one after the other in a thread block, on 16-byte boundaries and others."""
    assert n_in * n_out > 1 << 25
    g = gen(rows + n_in)
    pad += -n_in % 16 if pad == 16 else 0
    x, w, x_scale = codes_of(g, rows, n_in, pad, off), Weights(g, "int8", n_out, n_in, 0, pad, off), torch.rand(rows, generator=g, device="cuda") + 0.1
    full, y = room(kind, rows, n_out, pad, off)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, (kind, y))
    done(ctx)
    check_product(kind, y, x, x_scale, w)
    untouched(full, y, off)


@gpu
@pytest.mark.parametrize("most", [1, 2, 4])
@pytest.mark.parametrize("n_in,n_out", [(4096, 9000), (14336, 2400), (131071, 300)])
def test_few_rows_and_many_8_bit_weights_whose_clusters_are_refused(ctx, zkb, monkeypatch, most, n_in, n_out):
    monkeypatch.setenv("ZKB_STEP_CLUSTERS", str(most))
    g = gen(most)
    x, w = codes_of(g, 11, n_in, -n_in % 16), Weights(g, "int8", n_out, n_in, 0, -n_in % 16)
    y = torch.zeros(11, n_out, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, None, w, ("int32", y))
    done(ctx)
    check_product("int32", y, x, None, w)


@gpu
@pytest.mark.parametrize("rows", [33, 50, 64])
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 32), ("int4", 128)])
@pytest.mark.parametrize("n_in,n_out,pad", [(256, 128256, 0), (1024, 40000, 0), (272, 37889, 0), (300, 40000, 1)])
def test_tiles_of_64_rows_one_after_the_other(ctx, zkb, rows, kind, group, n_in, n_out, pad):
    """More outputs' tiles of 33 to 64 rows than the GPU holds at once: an output head."""
    g = gen(rows + n_out)
    x, w, x_scale = codes_of(g, rows, n_in, pad), Weights(g, kind, n_out, n_in, group, pad), torch.rand(rows, generator=g, device="cuda") + 0.1
    full, y = room("f32", rows, n_out, 3)
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    check_product("f32", y, x, x_scale, w)
    untouched(full, y, 0)


@gpu
@pytest.mark.parametrize("rows", [1, 2, 7, 40, 200])
@pytest.mark.parametrize("kind,group", [("int8", 0), ("int4", 64)])
def test_rows_and_weights_of_one_buffer(ctx, zkb, rows, kind, group):
    """Rows of x that lie behind each output's weights, and that are the weights themselves."""
    g, n_in, n_out = gen(rows), 256, 130
    w = Weights(g, kind, n_out, n_in, group, n_in)
    lines = w.w  # [output][weights, and 256 codes behind them]
    x = lines[:, -n_in:][:rows] if rows <= n_out else torch.cat([lines, lines])[:rows, -n_in:]
    x_scale = torch.rand(rows, generator=g, device="cuda") + 0.1
    y = torch.zeros(rows, n_out, device="cuda")
    torch.cuda.synchronize()
    run_product(ctx, zkb, x, x_scale, w, ("f32", y))
    done(ctx)
    check_product("f32", y, x, x_scale, w)
    if kind == "int8":  # rows as the weights, too
        rows = min(rows, n_out)
        y = torch.zeros(rows, rows, device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
        ctx.step_product(zkb.StepProduct(x=x.data_ptr(), x_stride=x.stride(0), w=x.data_ptr(), w_stride=x.stride(0), w_type=INT8, out=y.data_ptr(), out_type=TYPES["int32"], out_stride=rows, n_rows=rows,
                                         n_in=n_in, n_out=rows))
        done(ctx)
        assert torch.equal(y.double(), x[:rows].double() @ x[:rows].double().T)
