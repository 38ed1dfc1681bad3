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
