"""Attention over the paged cache against its definition in 64 bits: decode and
prefill at the sizes and masks where they can go wrong, the append, bad device
data, graphs, streams, and the three together behind int4 projections."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.attention_ref import E4M3, Case, append_reference, assert_near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tsg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import tsugumi_amd
    return tsugumi_amd


@pytest.fixture(scope="module")
def ctx(tsg):
    return tsg.Context(0)


def plan(tsg, ctx, c):
    return tsg.Attention(ctx, c.q_heads, c.kv_heads, c.dim, c.page, kv_type=c.kv, window=c.window,
                         sinks=c.sinks, scale=c.scale, k_scale=c.k_scale, v_scale=c.v_scale)


def launch(tsg, ctx, c, op, d=None, out=None, uniform=None):
    """One call of `op` on the case; rows that belong to no sequence keep a mark."""
    d = d or c.to_device()
    attn = plan(tsg, ctx, c)
    if uniform is None:
        uniform = op == "decode"
    batch = attn.batch(d["table"], d["lengths"], c.total, None if uniform else d["starts"])
    cache = attn.cache(d["k"], d["v"])
    if out is None:
        out = torch.full((c.total, c.q_heads, c.dim), -77.0, dtype=torch.float16, device="cuda")
    call = attn.encode_decode if op == "decode" else attn.encode_prefill
    call(cache, batch, d["q"], out)
    return out


def check_attention(tsg, ctx, c, op, **more):
    got = launch(tsg, ctx, c, op, **more)
    ctx.synchronize()
    want, tol = c.attention()
    used = int(c.starts[-1])
    assert_near(got[:used], want[:used], tol[:used], op)
    assert bool((got[used:] == -77.0).all()), "rows behind the last sequence were written"
    return got


# -------------------------------------------------------------------- decode

DIMS = [(4, 2, 16), (8, 1, 64), (6, 2, 80), (2, 2, 96), (8, 2, 128), (5, 1, 192), (16, 8, 256),
        (3, 1, 264), (8, 1, 512)]


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("q_heads,kv_heads,dim", DIMS)
def test_decode_head_layouts(tsg, ctx, q_heads, kv_heads, dim, kv):
    if kv == "e4m3" and dim % 16:
        dim += 8
    c = Case([1, 1], [45, 211], q_heads, kv_heads, dim, kv=kv, seed=dim)
    check_attention(tsg, ctx, c, "decode")


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255,
                                    257, 511, 513, 1000])
def test_decode_lengths(tsg, ctx, length):
    check_attention(tsg, ctx, Case([1], [length], 4, 2, 64, seed=length), "decode")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_decode_page_sizes(tsg, ctx, page):
    check_attention(tsg, ctx, Case([1, 1, 1], [1, 300, 129], 8, 2, 64, page=page, seed=page),
                    "decode")


@pytest.mark.parametrize("rows", [2, 3, 5, 8])
@pytest.mark.parametrize("heads", [(2, 2), (12, 2), (24, 3)])
def test_decode_blocks_of_rows(tsg, ctx, rows, heads):
    c = Case([rows] * 3, [rows, 40, 301], *heads, 64, seed=rows)
    check_attention(tsg, ctx, c, "decode")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 0), (31, 1), (64, 4), (100, 33),
                                          (100, 90), (500, 5), (4000, 9)])
@pytest.mark.parametrize("rows", [1, 4])
def test_decode_windows_and_sinks(tsg, ctx, window, sinks, rows):
    c = Case([rows] * 4, [rows, 77, 190, 300], 4, 2, 64, window=window, sinks=sinks, seed=window)
    check_attention(tsg, ctx, c, "decode")


def test_decode_empty_sequences_and_padded_rows(tsg, ctx):
    """Length 0, and fewer tokens than rows: the rows without a token are zeros."""
    c = Case([3, 3, 3, 3], [0, 1, 2, 50], 4, 2, 64, seed=5)
    got = check_attention(tsg, ctx, c, "decode")
    assert bool((got[:3] == 0).all()) and bool((got[3:5] == 0).all())
    assert not bool((got[5] == 0).all())


def test_decode_long_split(tsg, ctx):
    """One sequence whose keys are split over many workgroups and joined."""
    c = Case([1], [20011], 8, 2, 128, page=64, seed=3)
    check_attention(tsg, ctx, c, "decode")


@pytest.mark.parametrize("op,rows", [("decode", 4), ("prefill", 4), ("prefill", 70)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("window", [0, 24])
def test_values_that_a_row_does_not_see(tsg, ctx, op, rows, value, window):
    """NaN and infinities in the cache reach the rows that see their token only:
    a token inside the new rows, and one that the window has left behind."""
    c = Case([rows], [rows + 90], 4, 2, 64, window=window, seed=11)
    inside, behind = rows + 90 - 2, rows + 90 - rows // 2 - 30
    c.put("v", 0, inside, 0, value)
    if window:
        c.put("v", 0, behind, 1, value)
    got = launch(tsg, ctx, c, op)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(got, want, tol, f"{op} {value}")
    assert bool(torch.isfinite(want).any()) and not bool(torch.isfinite(want).all())


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_key_values_that_a_row_does_not_see(tsg, ctx, op):
    c = Case([4], [70], 4, 2, 64, window=20, seed=12)
    c.put("k", 0, 68, 0, math.nan)
    c.put("k", 0, 10, 1, math.inf)
    got = launch(tsg, ctx, c, op)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(got, want, tol, op)


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_far_apart_logits(tsg, ctx, op):
    """Logits from -900 to 900: one key takes all, with no overflow, wherever it lies."""
    c = Case([2], [200], 4, 2, 64, seed=13, q_scale=60.0, scale=1.0)
    check_attention(tsg, ctx, c, op)


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_one_large_weight_and_many_small(tsg, ctx, op):
    """A key of weight e^11 among 4000 of weight 1 (each 2^-16 of it): the small
    weights' sum counts."""
    c = Case([1], [4001], 1, 1, 64, page=64, seed=14, scale=1.0)
    c.q[:] = 0
    c.q[0, 0, 0] = 11.0
    k, v = c.k.float(), c.v.float()
    k[:] = 0
    c.k.copy_(torch.where(torch.isnan(c.k), c.k, k.half()))
    i, j = c.slot(0, 17)
    c.k[i, 0, j, 0] = 1.0
    c.v.copy_(torch.where(torch.isnan(v), v, v.abs() + 1).half())
    check_attention(tsg, ctx, c, op)


@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales(tsg, ctx, scale):
    check_attention(tsg, ctx, Case([2], [90], 4, 2, 64, seed=15, scale=scale), "decode")


# ------------------------------------------------------------------- prefill

@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("q_heads,kv_heads,dim", DIMS)
def test_prefill_head_layouts(tsg, ctx, q_heads, kv_heads, dim, kv):
    if kv == "e4m3" and dim % 16:
        dim += 8
    c = Case([19, 70], [45, 70], q_heads, kv_heads, dim, kv=kv, seed=dim)
    check_attention(tsg, ctx, c, "prefill")


@pytest.mark.parametrize("rows,before", [(1, 0), (2, 0), (9, 0), (31, 1), (32, 0), (33, 500),
                                         (64, 64), (65, 0), (127, 3), (128, 0), (129, 31),
                                         (200, 333)])
def test_prefill_lengths(tsg, ctx, rows, before):
    c = Case([rows], [rows + before], 2, 1, 64, seed=rows)
    check_attention(tsg, ctx, c, "prefill")


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (7, 1), (16, 2), (40, 1)])
def test_prefill_groups(tsg, ctx, heads):
    check_attention(tsg, ctx, Case([37, 5], [50, 5], *heads, 64, seed=heads[0]), "prefill")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_prefill_page_sizes(tsg, ctx, page):
    check_attention(tsg, ctx, Case([90, 1, 33], [200, 129, 40], 4, 2, 64, page=page, seed=page),
                    "prefill")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 0), (31, 1), (64, 4), (70, 33),
                                          (100, 90), (200, 5), (4000, 9)])
def test_prefill_windows_and_sinks(tsg, ctx, window, sinks):
    c = Case([150, 40], [150, 290], 4, 2, 64, window=window, sinks=sinks, seed=window)
    check_attention(tsg, ctx, c, "prefill")


@pytest.mark.parametrize("dim", [128, 256, 512])
def test_prefill_window_wide_heads(tsg, ctx, dim):
    c = Case([140], [260], 2, 1, dim, window=75, sinks=2, seed=dim)
    check_attention(tsg, ctx, c, "prefill")


def test_prefill_ragged_with_empty_padded_and_spare(tsg, ctx):
    """Sequences without rows, without tokens, with fewer tokens than rows, and
    rows behind the last sequence."""
    c = Case([5, 0, 40, 12, 0, 9], [30, 7, 0, 4, 0, 9], 4, 2, 64, seed=6, spare=13)
    got = check_attention(tsg, ctx, c, "prefill")
    assert bool((got[5:45] == 0).all()) and bool((got[45:53] == 0).all())


def test_prefill_many_sequences(tsg, ctx):
    """More sequences than a wave has lanes."""
    rng = np.random.default_rng(1)
    rows = rng.integers(0, 7, 150).tolist()
    lengths = [r + int(rng.integers(0, 20)) for r in rows]
    check_attention(tsg, ctx, Case(rows, lengths, 4, 2, 32, seed=7, spare=3), "prefill")


def test_prefill_uniform_equals_ragged(tsg, ctx):
    c = Case([20] * 3, [40, 20, 77], 4, 2, 64, seed=8)
    d = c.to_device()
    a = launch(tsg, ctx, c, "prefill", d=d, uniform=True)
    b = launch(tsg, ctx, c, "prefill", d=d, uniform=False)
    ctx.synchronize()
    assert torch.equal(a, b)


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("dim,heads,rows", [(256, (4, 2), 1), (256, (4, 2), 32), (256, (4, 2), 33),
                                            (512, (8, 1), 31), (512, (8, 1), 33), (272, (2, 1), 128),
                                            (272, (2, 1), 130)])
def test_prefill_uniform_few_rows_of_wide_heads(tsg, ctx, dim, heads, rows, kv):
    """On both sides of the sizes at which the kernels change."""
    c = Case([rows] * 2, [rows + 300, rows], *heads, dim, kv=kv, window=170, sinks=3, seed=rows)
    check_attention(tsg, ctx, c, "prefill", uniform=True)


def test_prefill_few_rows_over_a_long_cache(tsg, ctx):
    c = Case([12], [9001], 8, 2, 64, page=64, seed=9)
    check_attention(tsg, ctx, c, "prefill")


# ------------------------------------------------------- layouts and buffers

@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
def test_tokens_outside_heads(tsg, ctx, op, kv):
    c = Case([3, 3], [50, 131], 6, 3, 64, kv=kv, layout="tokens", seed=16)
    check_attention(tsg, ctx, c, op)


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_strided_rows(tsg, ctx, op):
    """q as a part of a fused buffer, out in wider rows: what lies between stays."""
    c = Case([2, 2], [50, 131], 4, 2, 64, seed=17)
    d = c.to_device()
    wide = torch.randn(4, 4 * 64 + 128, device="cuda").half()
    wide[:, 64:320] = d["q"].view(4, 256)
    d["q"] = wide[:, 64:320]
    out = torch.full((4, 512), -77.0, dtype=torch.float16, device="cuda")
    launch(tsg, ctx, c, op, d=d, out=out[:, 128:384])
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(out[:, 128:384].reshape(4, 4, 64), want, tol, op)
    assert bool((out[:, :128] == -77).all()) and bool((out[:, 384:] == -77).all())


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_pages_past_4_gib(tsg, ctx, op):
    """Pages at the end of pools of 4.5 GiB."""
    c = Case([2], [60], 4, 2, 128, page=64, seed=18, extra_pages=0)
    d = c.to_device()
    pages = (9 << 29) // (2 * 64 * 128 * 2)
    for name in ("k", "v"):
        big = torch.empty(pages, 2, 64, 128, dtype=torch.float16, device="cuda")
        big[-1] = d[name][0]
        d[name] = big
    d["table"] = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    got = launch(tsg, ctx, c, op, d=d)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(got, want, tol, op)


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_same_bits_each_time(tsg, ctx, op):
    c = Case([4], [5003], 8, 2, 128, seed=19)
    d = c.to_device()
    first = launch(tsg, ctx, c, op, d=d)
    for _ in range(5):
        assert torch.equal(launch(tsg, ctx, c, op, d=d), first)


# ----------------------------------------------------------- bad device data

@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_bad_page_is_reported(tsg, ctx, op):
    """A page past the pool: its rows are NaN, the other sequence's are right."""
    c = Case([2, 2], [100, 90], 4, 2, 64, seed=20)
    d = c.to_device()
    d["table"][0, 3] = d["k"].shape[0]
    got = launch(tsg, ctx, c, op, d=d)
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert e.value.status == 1 and "page table" in str(e.value)
    ctx.synchronize()  # reported once
    want, tol = c.attention()
    assert bool(torch.isnan(got[:2]).all())
    assert_near(got[2:], want[2:], tol[2:], op)


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_bad_page_that_no_row_sees(tsg, ctx, op):
    c = Case([1], [100], 4, 2, 64, window=20, seed=21)
    d = c.to_device()
    d["table"][0, 1] = -1
    got = launch(tsg, ctx, c, op, d=d)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(got, want, tol, op)


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_too_long_is_reported(tsg, ctx, op):
    c = Case([1, 1], [100, 90], 4, 2, 64, seed=22)
    d = c.to_device()
    d["lengths"][0] = d["table"].shape[1] * 16 + 1
    got = launch(tsg, ctx, c, op, d=d)
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert e.value.status == 1 and "longer" in str(e.value)
    want, tol = c.attention()
    assert bool(torch.isnan(got[0]).all())
    assert_near(got[1:], want[1:], tol[1:], op)


@pytest.mark.parametrize("starts", [[0, 9, 5], [0, 5, 99], [0, -1, 9]])
def test_bad_row_starts_are_reported(tsg, ctx, starts):
    c = Case([5, 4], [30, 20], 4, 2, 64, seed=23)
    d = c.to_device()
    d["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    launch(tsg, ctx, c, "prefill", d=d)
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert e.value.status == 1 and "row starts" in str(e.value)


# ------------------------------------------------- larger batches, refusals

@pytest.mark.parametrize("seqs,rows", [(70, 1), (130, 3), (256, 1), (300, 1)])
def test_decode_many_sequences(tsg, ctx, seqs, rows):
    """Runs found over several scans of the lengths, and (past 256) one run a sequence."""
    rng = np.random.default_rng(seqs)
    lengths = np.where(rng.random(seqs) < 0.1, rng.integers(rows, 900, seqs),
                       rng.integers(0, 60, seqs))
    lengths = np.maximum(lengths, np.where(rng.random(seqs) < 0.05, 0, rows)).tolist()
    check_attention(tsg, ctx, Case([rows] * seqs, lengths, 6, 2, 32, seed=seqs), "decode")


def test_decode_rows_past_one_tile_over_splits(tsg, ctx):
    """Eight rows of groups of five: three row tiles of each head, split and joined."""
    c = Case([8] * 3, [3000, 40, 1500], 10, 2, 256, seed=50, window=2500, sinks=3)
    check_attention(tsg, ctx, c, "decode")


def test_prefill_ragged_splits_with_window(tsg, ctx):
    c = Case([12, 3, 40, 0, 1], [5000, 900, 2100, 9, 1], 6, 2, 64, page=32, window=1800, sinks=5,
             seed=51, spare=4)
    check_attention(tsg, ctx, c, "prefill")


@pytest.mark.parametrize("dim", [256, 512])
def test_prefill_wide_heads_over_splits(tsg, ctx, dim):
    check_attention(tsg, ctx, Case([33], [1500], 4, 1, dim, seed=dim), "prefill")


@pytest.mark.parametrize("op,lengths", [("decode", [50, 3000]), ("prefill", [50, 3000])])
def test_in_place(tsg, ctx, op, lengths):
    c = Case([3, 3], lengths, 8, 2, 128, seed=52)
    d = c.to_device()
    launch(tsg, ctx, c, op, d=d, out=d["q"])
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(d["q"], want, tol, op)


def test_call_refusals(tsg, ctx):
    """Nothing is launched: the outputs keep their marks."""
    c = Case([9, 9], [30, 40], 4, 2, 64, seed=53)
    d = c.to_device()
    attn = plan(tsg, ctx, c)
    cache = attn.cache(d["k"], d["v"])
    uniform = attn.batch(d["table"], d["lengths"], 18)
    ragged = attn.batch(d["table"], d["lengths"], 18, d["starts"])
    out = torch.full_like(d["q"], -77.0)

    def refused(status, call, *args):
        with pytest.raises(tsg.TsgError) as e:
            call(*args)
        assert e.value.status == status

    refused(4, attn.encode_decode, cache, uniform, d["q"], out)  # nine rows: declined
    refused(1, attn.encode_decode, cache, ragged, d["q"], out)
    refused(1, attn.encode_prefill, cache, ragged, d["q"][:5], out)
    refused(1, attn.encode_prefill, cache, ragged, d["q"].float(), out)
    refused(1, attn.encode_prefill, cache, ragged, d["q"].cpu(), out)
    refused(1, attn.encode_prefill, cache, ragged, d["q"].transpose(1, 2), out)
    off = torch.zeros(18 * 256 + 8, dtype=torch.float16, device="cuda")[2:18 * 256 + 2].view(18, 256)
    refused(2, attn.encode_prefill, cache, ragged, off, out)
    refused(2, attn.encode_prefill, cache, ragged, d["q"], off)
    rope = tsg.HeadNormRope(inv_freq=torch.ones(20, device="cuda"))
    kv = torch.zeros(18, 2, 64, dtype=torch.float16, device="cuda")
    refused(3, attn.encode_append, cache, ragged, d["q"], kv, kv, rope, out)  # 40 of 64
    wide = tsg.HeadNormRope(torch.ones(32, device="cuda").bfloat16())
    refused(1, attn.encode_append, cache, ragged, d["q"], kv, kv, wide, out)
    refused(1, tsg.HeadNormRope, torch.ones(64, device="cuda"))
    refused(1, attn.cache, d["k"], d["v"].float())
    refused(1, attn.cache, d["k"][:, :1], d["v"][:, :1])
    refused(1, attn.batch, d["table"], d["lengths"].long(), 18)
    refused(1, attn.batch, d["table"], d["lengths"], 17)
    refused(1, tsg.Attention, ctx, 4, 2, 64, 16, "f32")
    refused(3, tsg.Attention, ctx, 4, 2, 60, 16)
    ctx.synchronize()
    assert bool((out == -77).all())


# -------------------------------------------------------------------- append

def append_case(tsg, ctx, c, rot, interleaved=False, normalize_v=False, weights=True, seed=0,
                in_place=False, k_is_v=False, uniform=False):
    g = torch.Generator().manual_seed(seed)
    n, width = c.total, (c.q_heads + 2 * c.kv_heads) * c.dim
    qkv = (torch.randn(n, width, generator=g) * 2).half()
    qw = (1 + 0.3 * torch.randn(c.dim, generator=g)).to(torch.bfloat16) if weights else None
    kw = (1 + 0.3 * torch.randn(c.dim, generator=g)).to(torch.bfloat16) if weights else None
    inv = (10000.0 ** (-torch.arange(0, rot, 2).double() / max(1, rot))).float() if rot else None
    d, eps = c.to_device(), 1e-5
    rope = tsg.HeadNormRope(None if qw is None else qw.cuda(), None if kw is None else kw.cuda(),
                            None if inv is None else inv.cuda(), interleaved, normalize_v, eps)
    attn = plan(tsg, ctx, c)
    dq, dk, dv = qkv.cuda().split((c.q_heads * c.dim, c.kv_heads * c.dim, c.kv_heads * c.dim), 1)
    if k_is_v:
        dv = dk
    out = dq if in_place else torch.full((n, c.q_heads, c.dim), -77.0, dtype=torch.float16,
                                         device="cuda")
    batch = attn.batch(d["table"], d["lengths"], n, None if uniform else d["starts"])
    attn.encode_append(attn.cache(d["k"], d["v"]), batch, dq, dk, dv, rope, out)
    ctx.synchronize()
    q, k, v = (x.view(n, -1, c.dim) for x in qkv.split(
        (c.q_heads * c.dim, c.kv_heads * c.dim, c.kv_heads * c.dim), 1))
    if k_is_v:
        v = k
    pos = torch.cat([torch.arange(length - r, length) for r, length in zip(c.rows, c.lengths)])
    used = len(pos)
    (qr, qt), (kr, kt), (vr, vt) = append_reference(
        q[:used], k[:used], v[:used], pos, qw, kw, inv, rot, interleaved, eps, normalize_v)
    zero = pos < 0
    qr[zero], qt[zero] = 0, 0
    got = out.reshape(n, c.q_heads, c.dim)
    assert_near(got[:used], qr, qt + qr.abs() * 2.0 ** -11 + 2.0 ** -25, "q")
    if not in_place:
        assert bool((got[used:] == -77).all())
    for name, ref, tol, scale in (("k", kr, kt, c.k_scale), ("v", vr, vt, c.v_scale)):
        pool = getattr(c, name).double()
        slack = torch.zeros_like(pool)
        for r in range(used):
            if pos[r] < 0:
                continue
            s = int(torch.searchsorted(c.starts, torch.tensor(r), right=True)) - 1
            i, j = c.slot(s, int(pos[r]))
            if c.kv == "f16":
                pool[i, :, j] = ref[r]
                slack[i, :, j] = tol[r] + ref[r].abs() * 2.0 ** -11 + 2.0 ** -25
            else:  # codes of value / scale, half a step or half the smallest
                code = (ref[r] / scale).clamp(-448, 448)
                pool[i, :, j] = code
                slack[i, :, j] = tol[r] / scale + torch.clamp(code.abs() * 2.0 ** -4, min=2.0 ** -10)
        assert_near(d[name].double().cpu(), pool, slack, name)


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,rot", [
    (4, 2, 16, 16), (8, 2, 64, 64), (6, 2, 80, 48), (3, 1, 96, 0), (32, 8, 128, 128),
    (5, 5, 192, 96), (16, 8, 256, 256), (16, 8, 256, 64), (8, 1, 512, 512), (8, 1, 512, 128)])
def test_append_head_layouts(tsg, ctx, q_heads, kv_heads, dim, rot, kv):
    c = Case([1, 3, 20], [1, 40, 20], q_heads, kv_heads, dim, kv=kv, seed=dim + rot)
    append_case(tsg, ctx, c, rot, seed=rot)


def test_append_odd_width(tsg, ctx):
    append_case(tsg, ctx, Case([2, 7], [9, 30], 3, 1, 72, seed=31), 32, seed=31)
    append_case(tsg, ctx, Case([2, 7], [9, 30], 3, 1, 8, seed=32), 0, seed=32)


@pytest.mark.parametrize("interleaved,normalize_v,weights", [(True, False, True),
                                                             (False, True, True),
                                                             (True, True, False)])
@pytest.mark.parametrize("kv", ["f16", "e4m3"])
def test_append_forms(tsg, ctx, interleaved, normalize_v, weights, kv):
    c = Case([4, 1, 9], [20, 30, 9], 8, 2, 128, kv=kv, seed=33)
    append_case(tsg, ctx, c, 64, interleaved, normalize_v, weights, seed=33)


def test_append_in_place_and_shared_rows(tsg, ctx):
    append_case(tsg, ctx, Case([4, 5], [20, 30], 8, 2, 128, seed=34), 128, seed=34, in_place=True)
    append_case(tsg, ctx, Case([4, 5], [20, 30], 8, 2, 128, seed=35), 32, seed=35, k_is_v=True,
                normalize_v=True)


def test_append_padded_empty_and_spare(tsg, ctx):
    c = Case([5, 0, 4, 3], [30, 7, 0, 1], 4, 2, 64, seed=36, spare=6)
    append_case(tsg, ctx, c, 64, seed=36)


def test_append_uniform_and_tokens_layout(tsg, ctx):
    c = Case([3, 3], [100, 3], 4, 2, 64, seed=37, layout="tokens", page=64)
    append_case(tsg, ctx, c, 64, seed=37, uniform=True)


def test_append_far_position(tsg, ctx):
    """Position 1,000,002: an angle formed in fp32 would be off by hundredths of a radian."""
    c = Case([3], [48], 2, 1, 64, seed=38)
    d = c.to_device()
    far = 1000003
    pages = -(-far // 4096)
    attn = tsg.Attention(ctx, 2, 1, 64, 4096)
    k = torch.zeros(2, 1, 4096, 64, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.ones(1, pages, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([far], dtype=torch.int32, device="cuda")
    inv = (1e6 ** (-torch.arange(0, 64, 2).double() / 64)).float()
    out = torch.empty_like(d["q"])
    kv_rows = torch.randn(3, 64, generator=c.g).half()
    attn.encode_append(attn.cache(k, v), attn.batch(table, lengths, 3), d["q"], kv_rows.cuda(),
                       kv_rows.cuda(), tsg.HeadNormRope(inv_freq=inv.cuda()), out)
    ctx.synchronize()
    (qr, qt), (kr, kt), _ = append_reference(c.q, kv_rows[:, None], kv_rows[:, None],
                                             torch.arange(far - 3, far), None, None, inv, 64,
                                             False, 1e-6, False)
    assert_near(out, qr, qt + qr.abs() * 2.0 ** -11 + 2.0 ** -25, "q")
    at = (far - 3) % 4096
    assert_near(k[1, 0, at:at + 3], kr[:, 0], kt[:, 0] + kr[:, 0].abs() * 2.0 ** -11 + 2.0 ** -25, "k")
    assert torch.equal(v[1, 0, at:at + 3].cpu(), kv_rows)


def test_append_saturates_and_keeps_nan(tsg, ctx):
    """e4m3: past the largest code the largest, NaN stays NaN."""
    c = Case([1], [1], 1, 1, 16, kv="e4m3", seed=39)
    d = c.to_device()
    attn = tsg.Attention(ctx, 1, 1, 16, 16, kv_type="e4m3", k_scale=1.0, v_scale=0.5)
    row = torch.tensor([[450.0, -460, 465, 1e4, -6e4, math.inf, -math.inf, math.nan, 0, -0.0,
                         2.0 ** -10, 2.0 ** -9, 448, 440, 17, -17]]).half()
    attn.encode_append(attn.cache(d["k"], d["v"]), attn.batch(d["table"], d["lengths"], 1),
                       d["q"], row.cuda(), row.cuda(), tsg.HeadNormRope(), d["q"])
    ctx.synchronize()
    i, j = c.slot(0, 0)
    for name, scale in (("k", 1.0), ("v", 0.5)):
        want = (row[0].float() / scale).clamp(-448, 448).to(E4M3).float()
        got = d[name][i, 0, j].float().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(), want.nan_to_num())


def test_append_bad_page_and_length(tsg, ctx):
    """Nothing goes to the cache, the query rows are NaN, the others are right."""
    c = Case([2, 2], [40, 30], 4, 2, 64, seed=40)
    for break_length in (False, True):
        d = c.to_device()
        if break_length:
            d["lengths"][0] = 10 ** 6
        else:
            d["table"][0, 2] = 10 ** 6
        attn = plan(tsg, ctx, c)
        k0, v0 = d["k"].clone(), d["v"].clone()
        rows = torch.randn(4, 2, 64, device="cuda").half()
        out = torch.empty_like(d["q"])
        attn.encode_append(attn.cache(d["k"], d["v"]), attn.batch(d["table"], d["lengths"], 4),
                           d["q"], rows, rows, tsg.HeadNormRope(), out)
        with pytest.raises(tsg.TsgError):
            ctx.synchronize()
        assert bool(torch.isnan(out[:2]).all()) and torch.equal(out[2:], d["q"][2:])
        same = torch.ones(k0.shape[0], 16, dtype=torch.bool)
        for t in (28, 29):
            i, j = c.slot(1, t)
            same[i, j] = False
            assert torch.equal(d["k"][i, :, j], rows[2 + t - 28])
        for new, old in ((d["k"], k0), (d["v"], v0)):
            where = same.cuda()[:, None, :, None].expand_as(old)
            assert torch.equal(new.view(torch.int16)[where], old.view(torch.int16)[where])


# -------------------------------------------------- graphs, streams, together

def test_graph_replays_with_new_lengths(tsg, ctx):
    """append + decode captured once; each replay appends the next token."""
    c = Case([1, 1], [60, 300], 8, 2, 64, seed=41)
    attn = plan(tsg, ctx, c)
    d, e = c.to_device(), c.to_device()
    rope = tsg.HeadNormRope(inv_freq=torch.linspace(1, 0.01, 32).cuda())
    rows = torch.empty(2, 12 * 64, dtype=torch.float16, device="cuda")
    start = torch.tensor([40, 120], dtype=torch.int32, device="cuda")

    def step(x, out):
        q, k, v = rows.split((512, 128, 128), 1)
        cache, batch = attn.cache(x["k"], x["v"]), attn.batch(x["table"], x["lengths"], 2)
        attn.encode_append(cache, batch, q, k, v, rope, x["q"])
        attn.encode_decode(cache, batch, x["q"], out)

    outs = [torch.empty(2, 8, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        d["lengths"].copy_(start)
        rows.normal_()
        step(d, outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(d, outs[0])
    d["k"].copy_(e["k"])
    d["v"].copy_(e["v"])
    for i in range(4):
        for x in (d, e):
            x["lengths"].copy_(start + 7 * i)
        rows.normal_()
        graph.replay()
        torch.cuda.synchronize()
        step(e, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]), i
        assert torch.equal(d["k"].view(torch.int16), e["k"].view(torch.int16))
    ctx.synchronize()


def test_two_plans_on_two_streams(tsg, ctx):
    """Calls of two plans beside each other, each on a stream of its own."""
    cases = [Case([1] * 2, [4000, 777], 8, 2, 128, seed=42),
             Case([2], [6001], 4, 1, 64, seed=43, window=3000)]
    devices = [c.to_device() for c in cases]
    want = [launch(tsg, ctx, c, "decode", d=d) for c, d in zip(cases, devices)]
    plans = [plan(tsg, ctx, c) for c in cases]
    outs = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for c, d, p, o, s in zip(cases, devices, plans, outs, streams):
            p.encode_decode(p.cache(d["k"], d["v"]), p.batch(d["table"], d["lengths"], c.total),
                            d["q"], o, stream=s)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_layer_front_together(tsg):
    """A prompt, then a token, through int4 projections, append, attention and
    the O projection; the token's row also as the last row of a longer prompt."""
    import oracle
    from tests.gpu_util import dev
    ctx = tsg.Context(0, group_size=32, scheme="sym")
    hidden, hq, hk, dim, n = 256, 8, 2, 64, 70
    rng = np.random.default_rng(4)

    def projection(m, k):
        w = dev(rng.integers(0, 256, m * k // 2, dtype=np.uint8))
        s = dev(oracle.bf16_bits(np.abs(rng.normal(0, 0.02, m * k // 32)).astype(np.float32) / 7))
        return w, s

    wq, wk, wv, wo = (projection(m, k) for m, k in (
        (hq * dim, hidden), (hk * dim, hidden), (hk * dim, hidden), (hidden, hq * dim)))
    gemm, gemv = tsg.PrefillInt4QMM(ctx), tsg.DequantInt4GEMV(ctx)
    attn = tsg.Attention(ctx, hq, hk, dim, 16, window=40, sinks=2)
    x = torch.randn(n + 1, hidden, generator=torch.Generator().manual_seed(1)).half().cuda()
    weight = torch.ones(dim, dtype=torch.bfloat16, device="cuda")
    inv = (10000.0 ** (-torch.arange(0, dim, 2).double() / dim)).float().cuda()
    rope = tsg.HeadNormRope(weight, weight, inv)
    table = torch.arange(5, dtype=torch.int32, device="cuda").flip(0).view(1, 5).contiguous()

    def pools():
        return [torch.full((5, hk, 16, dim), math.nan, dtype=torch.float16, device="cuda")
                for _ in range(2)]

    def rows(m, k):
        return torch.empty(m, k, dtype=torch.float16, device="cuda")

    def prompt(count, k_pool, v_pool):
        q, k, v, o, y = (rows(count, w) for w in (hq * dim, hk * dim, hk * dim, hq * dim, hidden))
        for (w, s), out in ((wq, q), (wk, k), (wv, v)):
            gemm.encode(w, s, s, x[:count], out, count, out.shape[1], hidden)
        lengths = torch.tensor([count], dtype=torch.int32, device="cuda")
        batch, cache = attn.batch(table, lengths, count), attn.cache(k_pool, v_pool)
        attn.encode_append(cache, batch, q, k, v, rope, q)
        attn.encode_prefill(cache, batch, q, o)
        gemm.encode(*wo, wo[1], o, y, count, hidden, hq * dim)
        return q, o, y

    k1, v1 = pools()
    prompt(n, k1, v1)
    q, k, v, o, y = (rows(1, w) for w in (hq * dim, hk * dim, hk * dim, hq * dim, hidden))
    for (w, s), out in ((wq, q), (wk, k), (wv, v)):
        gemv.encode(w, s, s, x[n], out, out.shape[1], hidden)
    lengths = torch.tensor([n + 1], dtype=torch.int32, device="cuda")
    batch, cache = attn.batch(table, lengths, 1), attn.cache(k1, v1)
    attn.encode_append(cache, batch, q, k, v, rope, q)
    attn.encode_decode(cache, batch, q, o)
    gemv.encode(*wo, wo[1], o, y, hidden, hq * dim)
    k2, v2 = pools()
    q2, o2, y2 = prompt(n + 1, k2, v2)
    ctx.synchronize()

    # the prompt's attention against 64 bits over the cache that was written
    c = Case([n + 1], [n + 1], hq, hk, dim, window=40, sinks=2)
    c.table, c.k, c.v, c.q = table.cpu(), k2.cpu(), v2.cpu(), q2.view(-1, hq, dim).cpu()
    want, tol = c.attention()
    assert_near(o2.view(-1, hq, dim), want, tol, "prompt")
    c = Case([1], [n + 1], hq, hk, dim, window=40, sinks=2)
    c.table, c.k, c.v, c.q = table.cpu(), k1.cpu(), v1.cpu(), q.view(1, hq, dim).cpu()
    want, tol = c.attention()
    assert_near(o.view(1, hq, dim), want, tol, "token")
    # the two paths of the same token: fp16 rounding of each projection and weight
    assert float((o - o2[n:]).norm() / o2[n:].norm()) < 5e-3
    assert float((y - y2[n:]).norm() / y2[n:].norm()) < 5e-3
