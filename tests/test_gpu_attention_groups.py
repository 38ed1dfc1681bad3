"""Groups of a batch that share nothing (of no sequence, of one, of padding) take nothing from those
that do: neither their splits nor their sharing."""
from __future__ import annotations

import gc

import pytest
import torch

from tests.attention_ref import Case
from tests.test_gpu_attention import ctx, launch, tsg  # noqa: F401 (fixtures)
from tests.test_gpu_attention_shared import call, check, share

pytestmark = pytest.mark.gpu

# query heads, key heads, head size, sequences that share, their rows
LAYOUTS = [(8, 2, 64, 8, 1), (32, 8, 128, 8, 2), (16, 8, 256, 16, 1), (16, 2, 256, 4, 1),
           (8, 1, 512, 5, 3)]


def batch(q_heads, kv_heads, dim, seqs, rows, more=3, prefix=2048, kv="f16"):
    """`seqs` sequences behind one prefix, and `more` with a few keys of their own."""
    lengths = [prefix + rows + 7 * s for s in range(seqs)] + [40 + 30 * s for s in range(more)]
    c = Case([rows] * (seqs + more), lengths, q_heads, kv_heads, dim, page=64, kv=kv, seed=dim)
    return share(c, [0, seqs], [prefix])


def groups(c, seqs, more):
    """One group in different company."""
    n = seqs + more
    yield [0, seqs] + list(range(seqs + 1, n + 1)), [c.shared[0]] + [64] * more       # of one
    yield [0, seqs] + [seqs] * 63, c.shared + [c.shared[0]] * 63                      # of none, behind
    yield [0] * 64 + [seqs], [128] * 63 + c.shared                                    # before
    yield [0] * 1024 + [seqs] * 1025, [640] * 1023 + c.shared + [64] * 1024           # on both sides
    yield [0, seqs, n], c.shared + [0]                                                # of no tokens


@pytest.mark.parametrize("layout", LAYOUTS)
def test_company_changes_no_bit(tsg, ctx, layout):  # noqa: F811
    c = batch(*layout)
    d = c.to_device()
    alone = check(tsg, ctx, c, d=d)
    decode = launch(tsg, ctx, c, "decode", d=d)
    assert not torch.equal(alone, decode)  # it is read once: other sums
    for starts, shared in groups(c, layout[3], 3):
        d["groups"], d["shared"] = (torch.tensor(t, dtype=torch.int32, device="cuda")
                                    for t in (starts, shared))
        assert torch.equal(call(tsg, ctx, c, d=d), alone), len(shared)
    ctx.synchronize()


def test_padding_changes_no_bit(tsg, ctx):  # noqa: F811
    """Sequences of no tokens in groups of their own, as a batch of fixed size has."""
    c = batch(32, 8, 128, 6, 1, more=10)
    c.lengths[6:] = [0] * 10
    d = c.to_device()
    alone = check(tsg, ctx, c, d=d)
    d["groups"], d["shared"] = (torch.tensor(t, dtype=torch.int32, device="cuda")
                                for t in ([0, 6, 11, 16], [2048, 2048, 64]))
    assert torch.equal(call(tsg, ctx, c, d=d), alone)
    ctx.synchronize()


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("seqs,prefix,once", [
    (7, 9024, False), (8, 8128, False), (8, 8192, True), (15, 9024, True), (15, 4032, False),
    (16, 512, True)])
def test_wide_heads_share_from_so_many_rows(tsg, ctx, kv, seqs, prefix, once):  # noqa: F811
    """Either side of the rule for heads over 128: 32 rows of a group's heads, or 8 sequences and
    8192 tokens."""
    c = batch(4, 2, 256, seqs, 1, more=0, prefix=prefix, kv=kv)
    d = c.to_device()
    got = check(tsg, ctx, c, d=d)
    assert torch.equal(got, launch(tsg, ctx, c, "decode", d=d)) != once


@pytest.mark.parametrize("dim,heads", [(64, (8, 2)), (256, (16, 2))])
def test_groups_of_both_sides(tsg, ctx, dim, heads):  # noqa: F811
    """Groups with enough rows beside ones with few, empty ones, and sequences of none."""
    lengths = [700 + 5 * s for s in range(6)] + [330, 340] + [90, 80, 70] + [1200 + s for s in range(7)]
    c = Case([2] * 18, lengths, *heads, dim, seed=3)
    check(tsg, ctx, share(c, [0, 6, 6, 8, 9, 11, 11, 18], [640, 320, 320, 64, 64, 10, 1152]))


def test_wrong_starts_among_many(tsg, ctx):  # noqa: F811
    c = batch(8, 2, 64, 8, 1)
    for at in (0, 70, 2047):
        starts = [8] * 2048 + [11]
        starts[at] = 12
        c.groups, c.shared = starts, [64] * 2048
        got = call(tsg, ctx, c)
        with pytest.raises(tsg.TsgError) as e:
            ctx.synchronize()
        assert e.value.status == 1 and "group starts" in str(e.value)
        assert bool(torch.isnan(got).all())


def test_more_tiles_than_the_card_holds(tsg, ctx):  # noqa: F811
    """Many groups that share: a tile each, one split."""
    seqs = 600
    lengths = [129 + s % 37 for s in range(seqs)]
    c = Case([1] * seqs, lengths, 4, 1, 32, seed=5)
    share(c, list(range(0, seqs + 1, 2)), [128] * (seqs // 2))
    check(tsg, ctx, c)


@pytest.mark.parametrize("dim", [128, 512])
def test_layers_with_a_window_hold_no_scratch_for_prefixes(tsg, ctx, dim):  # noqa: F811
    """Their scratch is a prefill call's partial sums: 65,536 rows (whole in 2 MiB, and so allocated)."""
    def held(window, plans=6):
        gc.collect()
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        keep = [tsg.Attention(ctx, 8, 1, dim, 16, window=window) for _ in range(plans)]
        used = before - torch.cuda.mem_get_info()[0]
        del keep
        return used / plans

    rows = 4 * (dim + 2)
    assert 65536 * rows <= held(1024) <= 65536 * rows + 2 ** 22
    assert 98304 * rows <= held(0) <= 98304 * rows + 2 ** 22
