"""The values of a decode step, from their definitions in 64 bits: batches, caches and references for the tests of zkb_step_*."""
import math

import numpy as np
import torch

INF = math.inf


class Batch:
    """Sequences of (rows, tokens in all); `behind` rows follow the last sequence, `gap` rows precede the first."""

    def __init__(self, shape, behind=0, gap=0):
        self.shape, self.gap = list(shape), gap
        first = gap + np.concatenate([[0], np.cumsum([r for r, _ in self.shape])])
        self.n_rows = int(first[-1]) + behind
        self.first = torch.tensor(first, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor([n for _, n in self.shape], dtype=torch.int32, device="cuda")

    def args(self, zkb, hints=True):
        return zkb.StepRows(first=self.first.data_ptr(), kv_len=self.lens.data_ptr(), n_rows=self.n_rows, max_rows=max(r for r, _ in self.shape) if hints else 0,
                            max_len=max(0, max(n for _, n in self.shape)) if hints else 0)

    def each(self):
        """(sequence, its first row, rows, position of the first row)."""
        at = self.gap
        for b, (r, n) in enumerate(self.shape):
            yield b, at, r, n - r
            at += r


class Cache:
    """A cache [sequence][head][token][dim] laid out as `order` says ("shtd" outermost first), with `pad` values behind each token's row."""

    def __init__(self, g, kind, seqs, heads, capacity, dim, order="shtd", pad=0, blank=False):
        self.kind, self.dims = kind, (seqs, heads, capacity, dim)
        size = dict(s=seqs, h=heads, t=capacity, d=dim + pad)
        back = [order.index(x) for x in "shtd"]

        def room(dtype):
            full = torch.zeros([size[x] for x in order], device="cuda", dtype=dtype)
            return full.permute(back)[..., :dim]

        self.k, self.v = (room(torch.int8 if kind == "int8" else torch.bfloat16) for _ in range(2))
        self.k_scale = self.v_scale = None
        if kind == "int8":
            self.k_scale, self.v_scale = (torch.zeros(heads, seqs, capacity, device="cuda").permute(1, 0, 2) for _ in range(2))
        if not blank:
            for x, s in ((self.k, self.k_scale), (self.v, self.v_scale)):
                if kind == "int8":
                    x.copy_(torch.randint(-128, 128, x.shape, generator=g, device="cuda", dtype=torch.int8))
                    s.copy_((0.5 + torch.rand(s.shape, generator=g, device="cuda")) / 73)
                else:
                    x.copy_(torch.randn(x.shape, generator=g, device="cuda"))

    def args(self, zkb):
        k, s = self.k, self.k_scale
        assert self.v.stride() == k.stride() and k.stride(3) == 1
        c = zkb.KvCache(k=k.data_ptr(), v=self.v.data_ptr(), type=zkb.VALUE_INT8 if self.kind == "int8" else zkb.VALUE_BF16, n_seqs=self.dims[0], n_heads=self.dims[1],
                        head_dim=self.dims[3], capacity=self.dims[2], seq_stride=k.stride(0), head_stride=k.stride(1), token_stride=k.stride(2))
        if s is not None:
            c.k_scale, c.v_scale, c.scale_seq_stride, c.scale_head_stride = s.data_ptr(), self.v_scale.data_ptr(), s.stride(0), s.stride(1)
        return c

    def values(self):
        """k and v in 64 bits."""
        if self.kind == "int8":
            return self.k.double() * self.k_scale.double()[..., None], self.v.double() * self.v_scale.double()[..., None]
        return self.k.double(), self.v.double()


def attention_reference(batch, cache, q, scale, window, sinks, weight=2.0 ** -8):
    """(out, bound): the definition in 64 bits, nan in rows of no sequence, and how far an output may be from it.

    Scores are sums of D products in 32 bits: off by D + 4 roundings of 2^-24 of the sum of their magnitudes B, and so the weights by that
    much relatively, by 2^-20 for the exponential and the scores' own size in it, and by a bf16 rounding 2^-8 (`weight`; two bf16 numbers: 2^-16); the sum of n weights in 32 bits adds n 2^-24.
    The result takes another 2^-8. None of this is relative below 2^-126, where 32-bit floats and bf16 have a fixed step of at most 2^-133, or nothing:
    a weight is then off by up to 2^-126, n of them by n 2^-126 of the largest value, the result by another 2^-126."""
    n, hq, d = q.shape
    seqs, hk, cap, _ = cache.dims
    k, v = cache.values()
    out, bound = torch.full((n, hq, d), math.nan, device="cuda", dtype=torch.float64), torch.zeros(n, hq, d, device="cuda", dtype=torch.float64)
    for b, at, rows, pos0 in batch.each():
        if not rows:
            continue
        p = torch.arange(pos0, pos0 + rows, device="cuda")[:, None]
        j = torch.arange(cap, device="cuda")[None]
        seen = j <= p
        if window:
            seen &= (p - j < window) | (j < sinks)
        for h in range(hq):
            kk, vv, qq = k[b, h * hk // hq], v[b, h * hk // hq], q[at:at + rows, h].double()
            s = (qq @ kk.T * scale).masked_fill(~seen, -INF)
            size = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~seen, 0)
            top = s.amax(-1, keepdim=True)
            w = torch.exp(s - torch.where(top == -INF, 0.0, top)).masked_fill(~seen, 0)
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total == 0, 1.0, total)
            bad = ~torch.isfinite(vv)
            clean = vv.masked_fill(bad, 0)
            o, a = w @ clean, w @ clean.abs()
            for key in bad.any(-1).nonzero().flatten().tolist():
                o = o + torch.where(seen[:, key, None] & bad[key], vv[key], torch.zeros_like(vv[key]))
            out[at:at + rows, h] = o
            rel = weight + 2 * (d + 4) * 2.0 ** -24 * size.amax(-1, keepdim=True) + 2.0 ** -19 + seen.sum(-1, keepdim=True) * 2.0 ** -24
            least = 2.0 ** -126 * (1 + seen.sum(-1, keepdim=True) * clean.abs().amax(0))
            bound[at:at + rows, h] = (rel * a) * (1 + 2.0 ** -8) + 2.0 ** -8 * o.abs() + least
    return out, bound


def rope_reference(batch, x, weights, eps, freq, interleaved):
    """(y, size): norm and rotation of heads x [row][head][dim] in 64 bits, weights [head][dim] or None for a head that is left as it is
    (rows of no sequence: nan), and |a| + |b| of each value's pair before its rotation."""
    y, half = x.double().clone(), len(freq)
    n, heads, d = y.shape
    for h in range(heads):
        if weights[h] is not None:
            y[:, h] = y[:, h] / (y[:, h].square().mean(-1, keepdim=True) + eps).sqrt() * weights[h].double()
    out, size = torch.full_like(y, math.nan), y.abs().clone()
    i = np.arange(half)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    for b, at, rows, pos0 in batch.each():
        part = y[at:at + rows].clone()
        if half:
            angle = (torch.arange(pos0, pos0 + rows, device="cuda", dtype=torch.float64)[:, None] * torch.tensor(freq, device="cuda"))[:, None]
            u, w = y[at:at + rows][..., one], y[at:at + rows][..., two]
            part[..., one], part[..., two] = u * angle.cos() - w * angle.sin(), w * angle.cos() + u * angle.sin()
            size[at:at + rows][..., one] = size[at:at + rows][..., two] = u.abs() + w.abs()
        out[at:at + rows] = part
    return out, size


def values_of(x):
    """bf16 tensors and tensors of words, in 64 bits; a word's high half is zero."""
    if x.dtype == torch.int32:
        assert int((x >> 16 != 0).sum()) == 0
        return (x << 16).view(torch.float32).double()
    return x.double()


def words(x):
    return x.view(torch.int16).to(torch.int32) & 0xFFFF
