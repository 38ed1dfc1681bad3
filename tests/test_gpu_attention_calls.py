"""Attention calls as programs make them: errors of several calls, plans and their
caches, streams."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.attention_ref import Case, assert_near
from tests.gpu_util import dev, empty
from tests.test_gpu_attention import ctx, launch, plan, tsg  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def test_every_error_is_reported(tsg, ctx):  # noqa: F811
    """A page past the pool, a sequence past its table, row starts that pass the rows and a
    grouping's expert past the layer, in four calls: all are in the one report, the
    attention's first, since its NaN rows can cause others."""
    c = Case([2, 2], [40, 30], 4, 2, 64, seed=70)
    for wrong in ("page", "length", "starts"):
        d = c.to_device()
        if wrong == "page":
            d["table"][0, 0] = 10 ** 6
        elif wrong == "length":
            d["lengths"][1] = 10 ** 6
        else:
            d["starts"][2] = 9
        launch(tsg, ctx, c, "prefill", d=d)
    tokens, k, experts, tile = 16, 2, 8, 32
    idx = np.tile(np.arange(k, dtype=np.uint32), (tokens, 1))
    idx[5, 1] = experts + 3
    g = tsg.PrefillGroupedRoutedMoE(tsg.MoE(ctx))
    blocks = tokens * k // tile + experts + 1
    g.group_pairs_device(
        dev(idx), dev(np.full((tokens, k), 0x3800, np.uint16)), tokens, k, experts,
        empty(tokens * k * 4, np.uint32), empty(experts, np.uint32), empty(experts, np.uint32),
        empty(blocks * 4, np.uint32), blocks, empty(1, np.uint32),
        empty(g.scratch_bytes(tokens, k, experts) // 4 + 1, np.uint32), tile_rows=tile)
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert e.value.status == 1
    text = str(e.value)
    places = [text.find(part) for part in ("page table entry", "longer than its page table",
                                           "row starts", "expertOutOfRange")]
    assert -1 not in places and places == sorted(places)
    ctx.synchronize()  # reported once


def refused(tsg, call, *args, text=""):  # noqa: F811
    with pytest.raises(tsg.TsgError) as e:
        call(*args)
    assert e.value.status == 1 and text in str(e.value)


def test_closed_context_and_plan(tsg):  # noqa: F811
    """A plan points into its context: after the context's end its calls are refused."""
    c = Case([1], [20], 2, 1, 64, seed=71)
    d = c.to_device()
    own = tsg.Context(0)
    attn, other = plan(tsg, own, c), plan(tsg, own, c)
    cache, batch = attn.cache(d["k"], d["v"]), attn.batch(d["table"], d["lengths"], 1)
    out = torch.full_like(d["q"], -77.0)
    rows = torch.zeros(1, 64, dtype=torch.float16, device="cuda")
    calls = [(attn.encode_decode, cache, batch, d["q"], out),
             (attn.encode_prefill, cache, batch, d["q"], out),
             (attn.encode_append, cache, batch, d["q"], rows, rows, tsg.HeadNormRope(), out)]
    other.close()
    refused(tsg, other.encode_decode, cache, batch, d["q"], out)
    own.close()
    for call in calls:
        refused(tsg, *call, text="closed")
    torch.cuda.synchronize()
    assert bool((out == -77).all())
    attn.close()  # needs no context


def test_caches_and_batches_of_another_kind(tsg, ctx):  # noqa: F811
    """A cache of another type, head or page size is refused (its bytes would be read as the
    plan's own), as is a batch whose table counts other pages; those of a plan that differs in
    window or query heads only are taken."""
    c = Case([2], [40], 4, 2, 64, kv="e4m3", seed=72)
    d = c.to_device()
    codes = plan(tsg, ctx, c)
    cache, batch = codes.cache(d["k"], d["v"]), codes.batch(d["table"], d["lengths"], 2)
    out = torch.full_like(d["q"], -77.0)
    rows = torch.zeros(2, 128, dtype=torch.float16, device="cuda")
    pool = torch.zeros(4, 2, 32, 64, dtype=torch.float16, device="cuda")
    half, wide_pages = tsg.Attention(ctx, 4, 2, 64, 16), tsg.Attention(ctx, 4, 2, 64, 32)
    one_head = tsg.Attention(ctx, 4, 1, 64, 16, "e4m3")
    for attn in (half, one_head):
        refused(tsg, attn.encode_decode, cache, batch, d["q"], out, text="a cache of")
        refused(tsg, attn.encode_prefill, cache, batch, d["q"], out, text="a cache of")
    refused(tsg, half.encode_append, cache, batch, d["q"], rows, rows, tsg.HeadNormRope(), out,
            text="a cache of")
    refused(tsg, wide_pages.encode_decode, wide_pages.cache(pool, pool), batch, d["q"], out,
            text="a batch of")
    torch.cuda.synchronize()
    assert bool((out == -77).all())
    again = tsg.Attention(ctx, 4, 2, 64, 16, "e4m3", window=40, scale=c.scale, k_scale=c.k_scale,
                          v_scale=c.v_scale)
    again.encode_decode(cache, batch, d["q"], out)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(out, want, tol)


def test_norm_weights_on_another_device(tsg, ctx):  # noqa: F811
    weight, inv = torch.ones(64, device="cuda").bfloat16(), torch.ones(32)
    refused(tsg, tsg.HeadNormRope, weight, weight, inv, text="two devices")
    c = Case([1], [20], 2, 1, 64, seed=73)
    d = c.to_device()
    attn, rope = plan(tsg, ctx, c), tsg.HeadNormRope(weight, weight)
    rope.device = 1  # as of weights on a second card
    rows = torch.zeros(1, 64, dtype=torch.float16, device="cuda")
    refused(tsg, attn.encode_append, attn.cache(d["k"], d["v"]),
            attn.batch(d["table"], d["lengths"], 1), d["q"], rows, rows, rope, d["q"],
            text="context's device")


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_one_plan_on_two_streams(tsg, ctx, op):  # noqa: F811
    """Calls of one plan on streams in turn, with no event between: they share its scratch,
    and each waits for the last. The long call comes first, so that the next would overlap it."""
    cases = [Case([1, 1], [20000, 30000], 8, 2, 128, page=64, seed=74),
             Case([1] * 3, [900, 4000, 777], 8, 2, 128, page=64, seed=75)]
    devices = [c.to_device() for c in cases]
    want = [launch(tsg, ctx, c, op, d=d, uniform=True) for c, d in zip(cases, devices)]
    attn = plan(tsg, ctx, cases[0])
    calls = [(attn.cache(d["k"], d["v"]), attn.batch(d["table"], d["lengths"], c.total), d["q"])
             for c, d in zip(cases, devices)]
    call = attn.encode_decode if op == "decode" else attn.encode_prefill
    outs = [[torch.full_like(w, -77.0) for w in want] for _ in range(10)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for pair in outs:
        call(*calls[0], pair[0])  # on the default stream
        for args, out, stream in zip(calls, pair, streams):
            call(*args, out, stream=stream)
    torch.cuda.synchronize()
    ctx.synchronize()
    for pair in outs:
        assert all(torch.equal(out, w) for out, w in zip(pair, want))


def test_plan_captured_between_eager_calls(tsg, ctx):  # noqa: F811
    """A capture takes no event of the eager stream, and the eager calls after it none of its
    stream; replays and eager calls in turn on one stream agree."""
    c = Case([1, 1], [3000, 5000], 8, 2, 64, page=64, seed=76)
    d = c.to_device()
    attn = plan(tsg, ctx, c)
    cache, batch = attn.cache(d["k"], d["v"]), attn.batch(d["table"], d["lengths"], 2)
    outs = [torch.full_like(d["q"], -77.0) for _ in range(3)]
    attn.encode_decode(cache, batch, d["q"], outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.encode_decode(cache, batch, d["q"], outs[1])
    for _ in range(3):
        outs[1].fill_(-77.0)
        graph.replay()
        attn.encode_prefill(cache, batch, d["q"], outs[2])
        attn.encode_decode(cache, batch, d["q"], outs[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
    ctx.synchronize()
    want, tol = c.attention()
    for out in outs:
        assert_near(out, want, tol)


# rows of each sequence as the right starts have them, starts as given, the first sequence
# behind the last wrong one
BAD_STARTS = [([5, 4], [0, 9, 5], 2), ([5, 4], [0, 5, 99], 2), ([5, 4], [0, -1, 9], 2),
              ([8, 3, 4], [0, 8, 4, 15], 2), ([8, 2, 3, 4], [0, 8, 2, 5, 15], 2),
              ([300, 40, 200, 8], [0, 300, 280, 540, 548], 2), ([3, 4, 2], [7, 3, 7, 8], 1)]


@pytest.mark.parametrize("rows,starts,good", BAD_STARTS)
@pytest.mark.parametrize("op", ["prefill", "append"])
def test_bad_row_starts(tsg, ctx, op, rows, starts, good):  # noqa: F811
    """Starts that fall or pass the rows, two sequences that claim a row among them: the
    sequences behind the last such one are right, every row before them is NaN, and appending
    writes nothing of them to the cache."""
    c = Case(rows, [r + 9 * i for i, r in enumerate(rows)], 4, 2, 64, seed=77)
    c.k.nan_to_num_(0.5)  # recycled pages, comparable
    c.v.nan_to_num_(0.5)
    d = c.to_device()
    before = d["k"].clone(), d["v"].clone()
    d["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    lo, end = (starts[good], starts[-1]) if good < len(rows) else (c.total, c.total)
    counts = [0] * good + [starts[i + 1] - starts[i] for i in range(good, len(rows))]
    out = torch.full((c.total, 4, 64), -77.0, dtype=torch.float16, device="cuda")
    if op == "prefill":
        launch(tsg, ctx, c, op, d=d, out=out, uniform=False)
    else:
        attn = plan(tsg, ctx, c)
        kv = torch.randn(c.total, 2, 64, device="cuda").half()
        attn.encode_append(attn.cache(d["k"], d["v"]),
                           attn.batch(d["table"], d["lengths"], c.total, d["starts"]), d["q"], kv, kv,
                           tsg.HeadNormRope(), out)
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert e.value.status == 1 and "row starts" in str(e.value)
    ctx.synchronize()
    assert bool(torch.isnan(out[:lo]).all())
    assert bool((out[end:] == -77).all())
    if op == "prefill":
        c.rows, c.starts = counts, torch.tensor(starts)
        want, tol = c.attention()
        assert_near(out[lo:end], want[lo:end], tol[lo:end])
        return
    same = torch.ones(before[0].shape[0], 16, dtype=torch.bool)
    for s, n in enumerate(counts):
        for i in range(n):
            row, pos = starts[s] + i, c.lengths[s] - n + i
            assert torch.equal(out[row], d["q"][row] if pos >= 0 else torch.zeros_like(out[row]))
            if pos >= 0:
                page, slot = c.slot(s, pos)
                same[page, slot] = False
                assert torch.equal(d["k"][page, :, slot], kv[row])
    where = same.cuda()[:, None, :, None].expand_as(before[0])
    assert torch.equal(d["k"][where], before[0][where])
    assert torch.equal(d["v"][where], before[1][where])


@pytest.mark.parametrize("op", ["prefill", "append"])
def test_bad_row_starts_far_back(tsg, ctx, op):  # noqa: F811
    """The fall lies more than 64 sequences before the last; a row behind that belongs to none."""
    c = Case([1] * 200, [4] * 200, 2, 1, 32, seed=78)
    d = c.to_device()
    d["starts"] = torch.arange(0, 201, dtype=torch.int32, device="cuda").clamp(max=199)
    d["starts"][50] = 48
    out = torch.full((200, 2, 32), -77.0, dtype=torch.float16, device="cuda")
    if op == "prefill":
        launch(tsg, ctx, c, op, d=d, out=out, uniform=False)
    else:
        attn = plan(tsg, ctx, c)
        kv = torch.zeros(200, 32, dtype=torch.float16, device="cuda")
        attn.encode_append(attn.cache(d["k"], d["v"]),
                           attn.batch(d["table"], d["lengths"], 200, d["starts"]), d["q"], kv, kv,
                           tsg.HeadNormRope(), out)
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert "row starts" in str(e.value)
    assert bool((out[199] == -77).all()) and bool(torch.isfinite(out[48:199]).all())
    assert bool(torch.isnan(out[:48]).all())


def test_outputs_that_share_elements_with_inputs(tsg, ctx):  # noqa: F811
    """q itself is taken; q at another stride, its later rows, columns that reach into it and,
    appending, the keys' or values' columns are refused. Columns beside q are not shared."""
    c = Case([3], [60], 4, 2, 64, seed=79)
    d = c.to_device()
    attn = plan(tsg, ctx, c)
    cache, batch = attn.cache(d["k"], d["v"]), attn.batch(d["table"], d["lengths"], 3)
    wide = torch.zeros(8, 1024, dtype=torch.float16, device="cuda")
    wide[:3, 256:512] = d["q"].view(3, 256)
    q, k, v = wide[:3, 256:512], wide[:3, 512:640], wide[:3, 640:768]
    other_stride = wide.view(-1)[256:].as_strided((3, 256), (512, 1))
    for call in (attn.encode_decode, attn.encode_prefill):
        for out in (wide[1:4, 256:512], wide[:3, 8:264], wide[:3, 504:760], other_stride):
            refused(tsg, call, cache, batch, q, out, text="shares elements")
    for out in (wide[1:4, 256:512], wide[:3, 384:640], wide[:3, 752:1008], other_stride):
        refused(tsg, attn.encode_append, cache, batch, q, k, v, tsg.HeadNormRope(), out,
                text="shares elements")
    before = wide.clone()
    torch.cuda.synchronize()
    want, tol = c.attention()
    for out in (wide[:3, :256], wide[:3, 768:], wide[3:6, 512:768], q):
        for call in (attn.encode_decode, attn.encode_prefill)[out is q:]:
            call(cache, batch, q, out)
            ctx.synchronize()
            assert_near(out.reshape(3, 4, 64), want, tol)
    assert torch.equal(wide[:3, 512:768], before[:3, 512:768])


def test_append_to_one_pool_for_both(tsg, ctx):  # noqa: F811
    """Rotated keys and plain values would go to the same slots; reading it as both is fine."""
    c = Case([1], [40], 2, 1, 64, seed=80)
    c.v = c.k
    d = c.to_device()
    attn = plan(tsg, ctx, c)
    cache, batch = attn.cache(d["k"], d["k"]), attn.batch(d["table"], d["lengths"], 1)
    out = torch.empty_like(d["q"])
    attn.encode_decode(cache, batch, d["q"], out)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(out, want, tol)
    rows = torch.zeros(1, 64, dtype=torch.float16, device="cuda")
    refused(tsg, attn.encode_append, cache, batch, d["q"], rows, rows, tsg.HeadNormRope(), out,
            text="two pools")


def test_one_row_in_place_at_two_strides(tsg, ctx):  # noqa: F811
    """A single row has no second one that its stride could place in q."""
    c = Case([1], [60], 4, 2, 64, seed=81)
    d = c.to_device()
    attn = plan(tsg, ctx, c)
    cache, batch = attn.cache(d["k"], d["v"]), attn.batch(d["table"], d["lengths"], 1)
    want, tol = c.attention()
    wide = torch.zeros(4, 1024, dtype=torch.float16, device="cuda")
    for call in (attn.encode_decode, attn.encode_prefill):
        wide[0, :256] = d["q"].view(256)
        call(cache, batch, wide[:, :256], wide.view(-1)[:512].view(2, 256))
        ctx.synchronize()
        assert_near(wide[:1, :256].reshape(1, 4, 64), want, tol)
