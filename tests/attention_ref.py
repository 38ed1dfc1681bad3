"""The attention half of a decoder layer in 64 bits, from its definitions, and
batches for its tests: pages in a random order, unwritten slots NaN."""
from __future__ import annotations

import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


class Case:
    """Sequences with `rows` new tokens and `lengths` cached ones (both lists),
    with their pools, page table and query rows on the CPU (`to_device` moves
    them)."""

    def __init__(self, rows, lengths, q_heads, kv_heads, dim, page=16, kv="f16", window=0,
                 sinks=0, seed=0, spare=0, layout="heads", extra_pages=2, q_scale=1.5,
                 scale=None):
        self.rows, self.lengths = list(rows), list(lengths)
        self.q_heads, self.kv_heads, self.dim, self.page = q_heads, kv_heads, dim, page
        self.kv, self.window, self.sinks = kv, window, sinks
        self.scale = dim ** -0.5 if scale is None else scale
        self.k_scale, self.v_scale = (1 / 64, 1 / 32) if kv == "e4m3" else (1.0, 1.0)
        g = torch.Generator().manual_seed(seed)
        self.g = g
        n = len(self.rows)
        per = max(1, -(-max(self.lengths) // page))
        pages = n * per + extra_pages
        self.table = torch.randperm(pages, generator=g)[:n * per].view(n, per).to(torch.int32)
        self.starts = torch.tensor([0, *np.cumsum(self.rows)], dtype=torch.int32)
        self.total = int(self.starts[-1]) + spare
        shape = (pages, kv_heads, page, dim)

        def pool(s):
            x = torch.randn(shape, generator=g)
            x = x.to(torch.float16) if kv == "f16" else (x / s).to(E4M3)
            if layout == "tokens":  # heads inside the tokens
                x = x.transpose(1, 2).contiguous().transpose(1, 2)
            return x

        self.k, self.v = pool(self.k_scale), pool(self.v_scale)
        written = torch.zeros(pages, page, dtype=torch.bool)
        for s, length in enumerate(self.lengths):
            for t in range(length):
                written[int(self.table[s, t // page]), t % page] = True
        where = ~written[:, None, :, None].expand(shape)
        for x in (self.k, self.v):
            if kv == "f16":
                x.masked_fill_(where, math.nan)
            else:
                x.view(torch.uint8).masked_fill_(where, 0x7F)
        self.q = (torch.randn(max(1, self.total), q_heads, dim, generator=g) * q_scale).half()

    def slot(self, s, t):
        return int(self.table[s, t // self.page]), t % self.page

    def put(self, which, s, t, head, value):
        """Writes `value` to all elements of one cached token of one head."""
        i, j = self.slot(s, t)
        x = getattr(self, which)
        x[i, head, j] = torch.full((self.dim,), value).to(x.dtype)

    def tokens(self, which, s):
        """Sequence s's cached tokens of one pool in 64 bits, [length, heads, dim]."""
        x = getattr(self, which)
        n = self.lengths[s]
        ids = self.table[s].long()[: max(1, -(-n // self.page))]
        scale = self.k_scale if which == "k" else self.v_scale
        return x[ids].double().transpose(1, 2).reshape(-1, self.kv_heads, self.dim)[:n] * scale

    def visible(self, pos, length):
        j = torch.arange(length)
        see = j <= pos
        if self.window:
            see &= (pos - j < self.window) | (j < self.sinks)
        return see

    def attention(self):
        """Outputs in 64 bits and, per element, how far an fp16 result may be off."""
        group = self.q_heads // self.kv_heads
        out = torch.zeros(self.total, self.q_heads, self.dim, dtype=torch.float64)
        tol = torch.zeros_like(out)
        for s, (n, length) in enumerate(zip(self.rows, self.lengths)):
            k, v = self.tokens("k", s), self.tokens("v", s)
            for i in range(n):
                r, pos = int(self.starts[s]) + i, length - n + i
                see = self.visible(pos, length)
                if pos < 0 or not bool(see.any()):
                    continue
                ks, vs = k[see], v[see]
                for h in range(self.q_heads):
                    q = self.q[r, h].double()
                    kh, vh = ks[:, h // group], vs[:, h // group]
                    p = torch.softmax(kh @ q * self.scale, 0)
                    out[r, h] = p @ vh
                    # Each weight is off by its rounding to fp16 (half a step, 2^-11), by
                    # its logit's fp32 sum (dim + 8 roundings of at most the sum of the
                    # products' sizes) twice, in the weight and in the total, and by
                    # the exponential and the sums over the keys in fp32; the result
                    # by its own rounding, half a step, and fp16's smallest step.
                    logit = (kh.abs() @ q.abs()).max() * abs(self.scale) * (self.dim + 8) * 2.0 ** -24
                    rel = 2.0 ** -11 + 2 * logit + (len(vh) + 64) * 2.0 ** -23
                    tol[r, h] = 2.0 ** -11 * out[r, h].abs() + (p @ vh.abs()) * rel + 2.0 ** -24
        return out, tol

    def to_device(self):
        d = {}
        for name in ("k", "v"):
            x = getattr(self, name)
            d[name] = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
            d[name].view(torch.uint8 if self.kv == "e4m3" else torch.int16).copy_(
                x.view(torch.uint8 if self.kv == "e4m3" else torch.int16))
        for name in ("table", "lengths", "starts", "q"):
            x = getattr(self, name)
            x = torch.tensor(x, dtype=torch.int32) if isinstance(x, list) else x
            d[name] = x.cuda()
        return d


def assert_near(got, want, tol, what=""):
    """Every element within its tolerance; NaN and infinities in the same places."""
    got = got.double().cpu()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got) & ~nan, inf), f"{what}: infinities in other places"
    fine = ~(nan | inf)
    assert torch.equal(got[inf], want[inf])
    over = ((got - want).abs() - tol)[fine]
    if over.numel():
        worst = int(over.argmax())
        assert float(over[worst]) <= 0, (
            f"{what}: {float(got[fine][worst])} for {float(want[fine][worst])}, allowed "
            f"{float(tol[fine][worst])}")


def append_reference(q, k, v, pos, q_weight, k_weight, inv_freq, rot, interleaved, eps,
                     normalize_v):
    """Rows [n, heads, dim] normed and turned in 64 bits, with what fp32 may be off."""
    def norm(x, w):
        x = x.double()
        y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        return y if w is None else y * w.double()

    def turn(y):
        size = y.abs().clone()
        if rot:
            a = pos.double()[:, None] * inv_freq.double()
            cos, sin = a.cos()[:, None], a.sin()[:, None]
            first = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
            second = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
            u, w = y[..., first].clone(), y[..., second].clone()
            y = y.clone()
            y[..., first], y[..., second] = u * cos - w * sin, w * cos + u * sin
            size[..., first] = size[..., second] = u.abs() + w.abs()
        # the sum of squares in fp32 (halved by the root), the square root, division and
        # products, and v_sin_f32 / v_cos_f32, for which 2^-18 of a unit is allowed
        return y, size * ((y.shape[-1] / 2 + 16) * 2.0 ** -24 + 2.0 ** -18)

    qn = norm(q, q_weight) if q_weight is not None else q.double()
    kn = norm(k, k_weight) if k_weight is not None else k.double()
    vn = norm(v, None) if normalize_v else v.double()
    return turn(qn), turn(kn), (vn, vn.abs() * (v.shape[-1] / 2 + 16) * 2.0 ** -24)
