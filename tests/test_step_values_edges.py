"""zkb_step_* where their definitions and their layouts have corners: hints that do not fit the batch, values that are no numbers, scales and windows at the ends of their
ranges, launches that are refused. The references and bounds are those of tests/step_cases.py."""
import pytest
import torch

from step_cases import Batch, Cache
from test_step_values import check_attention, gen

gpu = pytest.mark.gpu


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
