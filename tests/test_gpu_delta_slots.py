"""Slots of many sequences: those that clash are found wherever they are, and no others."""
from __future__ import annotations

import pytest

from tests.delta_ref import NONE, Case
from tests.test_gpu_delta import check, ctx, tsg  # noqa: F401 (fixtures)
from tests.test_gpu_delta_calls import only_sequence_is_bad

pytestmark = pytest.mark.gpu


def case(op, seqs, kept):
    rows = [kept] * seqs if op != "prefill" else [1 + s % 3 for s in range(seqs)]
    return Case(rows, 1, 1, 16, 16, seed=70, every=kept > 1)


SIZES = [("conv", 300, 1), ("conv", 150, 8), ("decode", 300, 1), ("decode", 130, 2),
         ("decode", 70, 8), ("prefill", 300, 1)]


@pytest.mark.parametrize("op,seqs,kept", SIZES)
def test_far_apart(tsg, ctx, op, seqs, kept):  # noqa: F811
    """The first and the last slot of a list, in passes of 64 and of 256 and behind them; one that
    clashes with itself does not."""
    c = case(op, seqs, kept)
    d = c.to_device()
    bad = [3, 65, seqs - 1]
    d["outs"][3 * kept] = d["outs"][65 * kept + kept - 1]
    d["outs"][(seqs - 1) * kept + kept - 1] = d["ins"][0]
    if kept > 1:
        c.outs[10 * kept] = c.outs[10 * kept + 1]
        d["outs"][10 * kept] = c.outs[10 * kept + 1]
    only_sequence_is_bad(tsg, ctx, c, op, d, bad)


@pytest.mark.parametrize("op,seqs,kept", SIZES)
def test_no_slot_clashes_with_none(tsg, ctx, op, seqs, kept):  # noqa: F811
    """Sequences without a slot to read and to write, beside some with."""
    c = case(op, seqs, kept)
    for s in range(0, seqs, 3):
        c.ins[s] = NONE
    for i in range(len(c.outs)):
        if i % 5 in (0, 3):
            c.outs[i] = NONE
    c.outs[:kept] = [NONE] * kept
    check(tsg, ctx, c, op)


@pytest.mark.parametrize("op,seqs,kept", [SIZES[0], SIZES[4], SIZES[5]])
def test_all_write_one_slot(tsg, ctx, op, seqs, kept):  # noqa: F811
    c = case(op, seqs, kept)
    d = c.to_device()
    d["outs"].fill_(c.outs[0])
    only_sequence_is_bad(tsg, ctx, c, op, d, list(range(seqs)))
