"""Logits of every kind where sequences share a prefix: minus infinity in the prefix, behind it and
throughout, scales of either sign and none."""
from __future__ import annotations

import math

import pytest
import torch

from tests.attention_ref import Case, assert_near
from tests.test_gpu_attention import ctx, launch, tsg  # noqa: F401 (fixtures)
from tests.test_gpu_attention_shared import call, check, share

pytestmark = pytest.mark.gpu

PREFIX = 192


def batch(dim=64, heads=(8, 2), scale=None, prefix=PREFIX, seqs=8):
    c = Case([2] * seqs, [prefix + 20 + 31 * s for s in range(seqs)], *heads, dim, seed=20, scale=scale)
    return share(c, [0, seqs], [prefix])


@pytest.mark.parametrize("dim,heads", [(64, (8, 2)), (128, (4, 2)), (256, (16, 2)), (512, (8, 1))])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales(tsg, ctx, dim, heads, scale):  # noqa: F811
    check(tsg, ctx, batch(dim, heads, scale * dim ** -0.5, prefix=512))


@pytest.mark.parametrize("dim,heads", [(64, (8, 2)), (128, (4, 2)), (256, (16, 2)), (512, (8, 1))])
@pytest.mark.parametrize("where", ["one", "a tile", "prefix", "own", "all"])
def test_logits_of_minus_infinity(tsg, ctx, dim, heads, where):  # noqa: F811
    """Keys whose logits are minus infinity count for nothing; rows without others are NaN."""
    c = batch(dim, heads)
    c.q[:, :, 0] = c.q[:, :, 0].abs() + 0.5
    longest = max(c.lengths)
    hidden = {"one": range(70, 71), "a tile": range(64, 128), "prefix": range(PREFIX),
              "own": range(PREFIX, longest), "all": range(longest)}[where]
    for s, n in enumerate(c.lengths):
        for t in hidden:
            if t < n:
                i, j = c.slot(s, t)
                c.k[i, :, j, 0] = -math.inf
    got = call(tsg, ctx, c)
    ctx.synchronize()
    want = torch.full(got.shape, math.nan, dtype=torch.float64)
    if where != "all":
        seen = [torch.tensor([t for t in range(n) if t not in hidden]) for n in c.lengths]
        want, tol = without(c, seen)
        assert_near(got, want, tol)
    else:
        assert bool(torch.isnan(got).all())
    assert_near(launch(tsg, ctx, c, "decode"), want, 0.0 * want if where == "all" else tol)


def without(c, seen):
    """Case.attention over some of each sequence's keys."""
    want = torch.zeros(c.total, c.q_heads, c.dim, dtype=torch.float64)
    tol, group = torch.zeros_like(want), c.q_heads // c.kv_heads
    for s, n in enumerate(c.rows):
        k, v = c.tokens("k", s), c.tokens("v", s)
        for i in range(n):
            r = int(c.starts[s]) + i
            see = seen[s][seen[s] <= c.lengths[s] - n + i]
            for h in range(c.q_heads):
                kh, vh, q = k[see, h // group], v[see, h // group], c.q[r, h].double()
                p = torch.softmax(kh @ q * c.scale, 0)
                want[r, h] = p @ vh
                # as Case.attention derives it
                logit = (kh.abs() @ q.abs()).max() * abs(c.scale) * (c.dim + 8) * 2.0 ** -24
                rel = 2.0 ** -11 + 2 * logit + (len(vh) + 64) * 2.0 ** -23
                tol[r, h] = 2.0 ** -11 * want[r, h].abs() + (p @ vh.abs()) * rel + 2.0 ** -24
    return want, tol


@pytest.mark.parametrize("dim", [8, 128])
def test_a_prefix_of_a_thousand_million_tokens(tsg, ctx, dim):  # noqa: F811
    """All on one page of keys of 0 and values of 1: sums that fp32 holds exactly (multiples of
    2^12 up to 2^30)."""
    seqs, page, tokens = 64, 4096, 1 << 30
    attn = tsg.Attention(ctx, 1, 1, dim, page)
    k = torch.zeros(1, 1, page, dim, dtype=torch.float16, device="cuda")
    table = torch.zeros(seqs, tokens // page, dtype=torch.int32, device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.ones(seqs, 1, dim, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, -77.0)
    attn.encode_decode_shared(attn.cache(k, torch.ones_like(k)),
                              attn.batch(table, ints(*[tokens] * seqs), seqs),
                              attn.prefixes(ints(0, seqs), ints(tokens - page)), q, out)
    ctx.synchronize()
    assert bool((out == 1).all())
