"""Products of codes (zkb_step_product): the ways that their sizes and layouts lead to, beside those of test_step_layer.py and test_step_layer_edges.py."""
import math

import pytest
import torch

from test_step_layer import Weights, check_product, codes_of, run_product
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
