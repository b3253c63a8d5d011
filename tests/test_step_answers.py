"""Log probabilities (zkb_step_logprobs) at the ends of the 32-bit floats."""
import pytest
import torch

from test_step_layer import answer, check_answer, held_logits
from test_step_values import gen

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("kind", ["bf16", "words", "f32"])
@pytest.mark.parametrize("rows,vocab", [(2, 50), (1, 100003), (400, 5000), (1300, 8192 * 2)])
@pytest.mark.parametrize("scale", [2.0 ** -100, 1e-20, 0.25, 0.6])
def test_logits_that_lie_further_apart_than_a_float(ctx, zkb, kind, rows, vocab, scale):
    """The largest logit and others of the other sign: their difference leaves the 32-bit floats, scaled it is in them. A token that can be has no log probability of -infinity.
    Products with the scale are rounded once each and so is their difference: within the bound of check_answer."""
    g = gen(rows + vocab)
    x = 1e38 * torch.randn(rows, vocab, generator=g, device="cuda").clamp(-3, 3)
    x[:, vocab // 3], x[:, vocab // 2], x[:, 1] = 3.3e38, -3.3e38, -3e38
    x[0, 2] = -float("inf")
    held, values = held_logits(x, kind, 1, 1)
    ids = torch.tensor([[vocab // 3, vocab // 2, 1, 0, 2]], device="cuda", dtype=torch.int32).expand(rows, -1).contiguous()
    got = answer(ctx, zkb, held, kind, ids, 32, scale)
    few = slice(0, rows, -(-rows // 20))
    exact = (values - values.amax(-1, keepdim=True)) * scale
    assert bool((exact[:, vocab // 2] > -3.402e38).all()) == (scale < 0.5)
    if scale < 0.5:
        check_answer(tuple(y[few] for y in got), values[few], ids[few], 32, scale)
        assert bool(torch.isfinite(got[0][1:]).all()) and got[0][0, 4] == -float("inf")
    else:  # what no float holds is -infinity, as a rounding of it is
        assert bool((got[0][:, 1] == -float("inf")).all()) and bool((got[0][:, 0] == 0).all())
