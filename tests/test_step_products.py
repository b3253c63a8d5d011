"""Products of codes (zkb_step_product): the ways that their sizes and layouts lead to, beside those of test_step_layer.py and test_step_layer_edges.py."""
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
