"""Attention at the edges of its values' ranges: logits far from zero, rows whose
result is one value, infinities that some rows see, in every kernel's width."""
from __future__ import annotations

import pytest
import torch

from tests.attention_ref import Case, assert_near
from tests.test_gpu_attention import ctx, launch, tsg  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def set_products(c, base, steps):
    """Queries and keys of small whole numbers with q . k = base + steps[j] for key j of
    every sequence and head, exact in fp32 in any order (every partial sum is below 2^24)."""
    half = c.dim // 2
    c.q[:] = 0
    c.q[..., :half] = 1024.0
    c.q[..., half] = 1.0
    for s, length in enumerate(c.lengths):
        for t in range(length):
            i, j = c.slot(s, t)
            row = torch.zeros(c.dim)
            row[:half] = base / (1024.0 * half) / c.k_scale
            row[half] = float(steps[t % len(steps)]) / c.k_scale
            assert torch.equal(row.to(c.k.dtype).float(), row)
            c.k[i, :, j] = row.to(c.k.dtype)


def products_tolerance(c, out):
    """Products are exact here, so a weight is off by its rounding to fp16 (half a step, 2^-11),
    by its exponent (at most 40 powers of two matter; scale log2(e) in fp32 and two roundings of
    the multiply-add: 3 x 40 x 2^-24, under 2^-16), and by the sums in fp32; the result by its
    own rounding."""
    size = torch.zeros_like(out)
    for s, n in enumerate(c.rows):
        first = int(c.starts[s])
        size[first:first + n] = c.tokens("v", s).abs().amax((0, 2))[
            torch.arange(c.q_heads) // (c.q_heads // c.kv_heads)][:, None]
    return (2.0 ** -11 * out.abs()
            + size * (2.0 ** -11 + 2.0 ** -16 + (max(c.lengths) + 64) * 2.0 ** -23) + 2.0 ** -24)


@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("base", [1 << 21, -(1 << 21)])
@pytest.mark.parametrize("scale", [0.5, 37.0, 1e4])
def test_logits_far_from_zero(tsg, ctx, op, dim, base, scale):  # noqa: F811
    """Logits of 10^6 to 2 10^10 whose differences are exact: the weights are those of the
    differences, and a row that sees one key returns its value. The maximum comes step by
    step, and (3001 keys, split) lies in one split only."""
    steps = [-9.0, -8.0, -7.0, -7.0, -8.0, -6.0, -9.0]
    c = Case([2, 2, 2], [2, 150, 3001], 4, 2, dim, page=64, scale=scale, seed=dim)
    set_products(c, base, steps)
    for length, t in ((150, 77), (3001, 40), (3001, 2000)):
        i, j = c.slot(c.lengths.index(length), t)
        c.k[i, :, j, dim // 2] = -4.0 if t != 2000 else 0.0
    got = launch(tsg, ctx, c, op, uniform=True)
    ctx.synchronize()
    want, _ = c.attention()
    assert bool(torch.isfinite(want).all())
    assert_near(got, want, products_tolerance(c, want), op)
    assert_near(got[:1], want[:1], 2.0 ** -11 * want[:1].abs(), "a single key")


@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("scale", [40.0, 3e5])
def test_logits_far_from_zero_e4m3(tsg, ctx, op, scale):  # noqa: F811
    c = Case([1, 1], [1, 700], 4, 2, 128, kv="e4m3", scale=scale, seed=1)
    set_products(c, 4.0 * 1024 * 64, [-0.125, -0.25, 0.0, -0.125])
    got = launch(tsg, ctx, c, op, uniform=True)
    ctx.synchronize()
    want, _ = c.attention()
    assert_near(got, want, products_tolerance(c, want), op)


@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_equal_values_come_back(tsg, ctx, op, dim):  # noqa: F811
    """Where all keys have one value the result is that value, whatever the weights: their
    rounding to fp16 is in the sum as well. Two keys count, the later one 3.4 .. 4 powers of two
    above the earlier, so that the reference lags behind it."""
    n = 300  # so many that the keys are not split
    c = Case([1] * n, [80] * n, 2, 1, dim, page=64, scale=1.0, seed=dim)
    c.q[:] = 0
    c.q[..., 0] = 1.0
    c.k[:] = 0
    c.k[..., 0] = -100.0
    c.v[:] = 1.9990234375  # half a step is 2^-12 of it
    for s in range(n):
        i, j = c.slot(s, 4)
        c.k[i, :, j, 0] = 0.0
        i, j = c.slot(s, 68)  # another tile of the same wave, in decode too
        c.k[i, :, j, 0] = (3.4 + 0.6 * s / n) * 0.6931
    got = launch(tsg, ctx, c, op, uniform=True)
    ctx.synchronize()
    assert bool((got == 1.9990234375).all())


@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("length", [40, 3000])
def test_logits_of_minus_infinity(tsg, ctx, op, length):  # noqa: F811
    """Weight 0 beside finite logits; a row that sees no others is 0 / 0; rows
    without a token stay zeros."""
    c = Case([4, 4, 4], [length, length, 2], 4, 2, 64, window=30, seed=60)
    c.q[..., 0] = c.q[..., 0].abs() + 0.5
    for t in range(length - 33, length):
        for s in (0, 1):
            i, j = c.slot(s, t)
            if s == 0 or t % 3 == 0:
                c.k[i, 0, j, 0] = -float("inf")
    got = launch(tsg, ctx, c, op, uniform=True)
    ctx.synchronize()
    want, tol = c.attention()
    assert bool(torch.isnan(want[:4, :2]).all()) and int(torch.isnan(want).sum()) == 4 * 2 * 64
    # the tolerance of attention_ref, its logits' sizes those of the finite keys
    k, v = c.tokens("k", 1), c.tokens("v", 1)
    k[torch.isinf(k)] = 0.0
    size = torch.einsum("jhd,rhgd->rhg", k.abs().amax(0, keepdim=True),
                        c.q[4:8].view(4, 2, 2, 64).abs().double()).reshape(4, 4, 1) * c.scale
    rel = 2.0 ** -11 + 2 * size * 72 * 2.0 ** -24 + (length + 64) * 2.0 ** -23
    tol[:4, :2] = 0.0
    tol[4:8] = 2.0 ** -11 * want[4:8].abs() + v.abs().max() * rel + 2.0 ** -24
    assert_near(got, want, tol, op)
    assert bool((got[8:10] == 0).all())


def test_decode_more_key_tiles_than_32_bits_count(tsg, ctx):  # noqa: F811
    """64 sequences of 2^30 tokens, all on one shared page: 2^32 tiles of 16 keys. Keys of 0
    and values of 1 give sums that fp32 holds exactly (multiples of a power of two)."""
    seqs, page = 64, 4096
    attn = tsg.Attention(ctx, 1, 1, 8, page)
    k = torch.zeros(1, 1, page, 8, dtype=torch.float16, device="cuda")
    table = torch.zeros(seqs, (1 << 30) // page, dtype=torch.int32, device="cuda")
    lengths = torch.full((seqs,), 1 << 30, dtype=torch.int32, device="cuda")
    q = torch.ones(seqs, 1, 8, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, -77.0)
    attn.encode_decode(attn.cache(k, torch.ones_like(k)), attn.batch(table, lengths, seqs), q, out)
    ctx.synchronize()
    assert bool((out == 1).all())


@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("dim", [64, 80, 128, 256, 512])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("window", [0, 45])
def test_single_elements_that_a_row_does_not_see(tsg, ctx, op, dim, kv, window):  # noqa: F811
    """+inf, -inf and NaN in one element each of tokens that some of the rows see (e4m3 has NaN
    only), in a short sequence and in one that is split: they reach their element of the rows
    that see them and nothing else. 140 rows of two heads take the prefill kernel at any width."""
    rows = 4 if op == "decode" else 140
    c = Case([rows] * 2, [rows + 90, 1500], 2, 1, dim, kv=kv, page=64, window=window, seed=dim)
    bad = [float("inf"), -float("inf"), float("nan")]
    places = [(2, dim - 1), (rows // 2, dim // 2 + 5), (rows // 2 + 44, 3)]  # before the last row
    for s, length in enumerate(c.lengths):
        for value, (back, element) in zip(bad, places):
            i, j = c.slot(s, length - back)
            if kv == "e4m3":
                c.v.view(torch.uint8)[i, 0, j, element] = 0x7F
            else:
                c.v[i, 0, j, element] = value
    got = launch(tsg, ctx, c, op, uniform=True)
    ctx.synchronize()
    want, tol = c.attention()
    seen = ~torch.isfinite(want)
    assert bool(seen.any()) and int(seen.sum(-1).max()) <= 3 and int(seen.sum(-1).min()) < 3
    assert_near(got, want, tol, op)


@pytest.mark.parametrize("scale", [0.0, -0.2])
@pytest.mark.parametrize("dim", [64, 512])
def test_prefill_scales(tsg, ctx, scale, dim):  # noqa: F811
    c = Case([270], [300], 2, 1, dim, page=64, seed=61, scale=scale)
    got = launch(tsg, ctx, c, "prefill", uniform=True)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(got, want, tol)
