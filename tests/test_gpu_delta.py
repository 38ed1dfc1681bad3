"""The gated delta rule and its convolution on the GPU against their definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

from tests.attention_ref import assert_near
from tests.delta_ref import NONE, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tsg():
    import tsugumi_amd
    return tsugumi_amd


@pytest.fixture(scope="module")
def ctx(tsg):
    return tsg.Context(0)


def check(tsg, ctx, c, op, **launch):
    """A call against the reference: outputs and written states within their tolerance, every
    other row and slot as it was."""
    d = c.launch(tsg, ctx, op, **launch)
    ctx.synchronize()
    mine = c.used()
    if op == "conv":
        out, tol, pool = c.convolution()
        got, kept = d["conv_out"].cpu()[:c.total], d["conv"].cpu()
        assert torch.equal(kept, pool)
        assert torch.equal(d["s"].cpu(), c.s)
    else:
        out, tol, pool, pool_tol = c.rule(op == "prefill")
        got = d["out"].cpu()[:c.total]
        assert torch.equal(d["conv"].cpu(), c.conv)
        assert_near(d["s"], pool, pool_tol, "states")
    assert_near(got[mine], out[mine], tol[mine], op)
    assert bool((got[~mine] == -77).all())
    return d


# ------------------------------------------------------------------ convolution

@pytest.mark.parametrize("width", [2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("rows", [[1], [1, 1, 1], [15, 16, 17, 1, 40], [3, 0, 33, 2], [0, 0, 7]])
def test_convolution(tsg, ctx, width, rows):
    check(tsg, ctx, Case(rows, 2, 4, 48, 80, width=width, seed=width, slots="apart"), "conv")


@pytest.mark.parametrize("slots", ["place", "fresh", "fork"])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [5, 2, 1, 21]])
def test_convolution_slots(tsg, ctx, slots, rows):
    check(tsg, ctx, Case(rows, 1, 2, 64, 64, seed=20, slots=slots), "conv")


def test_convolution_padding_and_strides(tsg, ctx):
    """Rows before the first sequence and behind the last stay as they were; x lies in wider
    rows."""
    check(tsg, ctx, Case([9, 30], 1, 1, 16, 16, seed=21, spare=5, lead=3, row_pad=24), "conv")


@pytest.mark.parametrize("width,rows", [(4, 3), (4, 1), (8, 8), (2, 5)])
@pytest.mark.parametrize("slots", ["apart", "place", "fresh"])
def test_convolution_keeps_every_state(tsg, ctx, width, rows, slots):
    check(tsg, ctx, Case([rows] * 3, 1, 3, 32, 48, width=width, seed=22, slots=slots, every=True),
          "conv")


def test_convolution_without_kept_states(tsg, ctx):
    c = Case([4, 20], 1, 1, 16, 32, seed=23)
    c.outs[0] = NONE
    check(tsg, ctx, c, "conv")


def test_convolution_large_prompt(tsg, ctx):
    check(tsg, ctx, Case([700, 301], 4, 8, 64, 64, seed=24), "conv")


def test_convolution_of_more_than_a_million_rows(tsg, ctx):
    """More row tiles than 65536: the reference at the sequences' ends and past that tile."""
    n = 16 * 65536 + 300
    c = Case([n - 37, 37], 1, 1, 16, 16, seed=26)
    d = c.launch(tsg, ctx, "conv")
    ctx.synchronize()
    w, x = c.weight.double().T, c.x.double()
    for s, first, last in ((0, 0, n - 38), (1, n - 37, n - 1)):
        assert torch.equal(d["conv"][c.outs[s]].cpu(), c.x[last - 2:last + 1])
        old = c.conv[c.ins[s]].double()
        for row in (first, first + 1, first + 36, last, max(first, 16 * 65536 + 5)):
            rows = torch.stack([x[row - j] if row - j >= first else old[row - j - first + 3]
                                for j in (3, 2, 1, 0)])
            y, size = (rows * w).sum(0), (rows * w).abs().sum(0)
            want = y * torch.sigmoid(y)
            tol = 5.5 * 2.0 ** -24 * size + want.abs() * (2.0 ** -11 + 2.0 ** -21
                                                          + y.abs() * 2.0 ** -22) + 2.0 ** -25
            assert_near(d["conv_out"][row], want, tol)


def test_convolution_extremes(tsg, ctx):
    """Sums far on either side of zero, and an infinity that only the rows that it reaches take."""
    c = Case([40], 1, 1, 16, 16, seed=25, size=300.0)
    check(tsg, ctx, c, "conv")
    c.x[11, 5] = float("inf")
    c.weight[5] = torch.tensor([0.5, 1.0, 0.25, 2.0]).bfloat16()
    d = c.launch(tsg, ctx, "conv")
    ctx.synchronize()
    out, tol, pool = c.convolution()
    got = d["conv_out"].cpu()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[11:15, 5] = True
    assert bool((got[bad] == float("inf")).all())
    assert_near(got[~bad], out[~bad], tol[~bad])


# ------------------------------------------------------------------ row by row

DIMS = [(16, 16), (48, 64), (64, 80), (80, 32), (128, 128), (144, 48), (192, 192), (256, 512)]


@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("rows", [1, 2, 8])
def test_decode(tsg, ctx, dk, dv, rows):
    check(tsg, ctx, Case([rows] * 3, 2, 4, dk, dv, seed=30 + rows), "decode")


@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 5), (3, 3), (2, 8), (16, 32)])
def test_decode_heads(tsg, ctx, hk, hv):
    check(tsg, ctx, Case([2, 2], hk, hv, 64, 48, seed=31), "decode")


@pytest.mark.parametrize("slots", ["place", "fresh", "fork"])
@pytest.mark.parametrize("every", [False, True])
def test_decode_slots(tsg, ctx, slots, every):
    check(tsg, ctx, Case([3] * 5, 1, 2, 64, 64, seed=32, slots=slots, every=every), "decode")


@pytest.mark.parametrize("rows", [1, 2, 7, 8])
def test_decode_keeps_every_state(tsg, ctx, rows):
    check(tsg, ctx, Case([rows] * 4, 2, 2, 128, 64, seed=33, every=True), "decode")


def test_decode_slots_twice_and_not_kept(tsg, ctx):
    """The later row's state stays in a slot that a list names twice; NONE keeps nothing."""
    c = Case([4, 4], 1, 1, 32, 32, seed=34, every=True)
    c.outs[1], c.outs[5] = c.outs[3], NONE
    check(tsg, ctx, c, "decode")


def test_decode_many_sequences(tsg, ctx):
    check(tsg, ctx, Case([1] * 300, 1, 2, 32, 32, seed=35), "decode")


def test_decode_large_batch_of_large_states(tsg, ctx):
    check(tsg, ctx, Case([1] * 20, 4, 8, 128, 128, seed=36), "decode")


EXTREMES = {
    "forgets": dict(gate=40.0),          # decays of 0 and of 1, steps of 0 and of 1
    "large": dict(size=3000.0, state=1e6),
    "small": dict(size=1e-3, state=1e-6),
    "scale": dict(scale=-3.5),
    "eps": dict(eps=0.5),
}


@pytest.mark.parametrize("what", EXTREMES)
def test_decode_extremes(tsg, ctx, what):
    check(tsg, ctx, Case([8, 8], 1, 2, 64, 64, seed=37, **EXTREMES[what]), "decode")


def test_decode_zero_rows_of_keys(tsg, ctx):
    c = Case([6], 1, 2, 64, 64, seed=38)
    c.qkv[2] = 0
    c.qkv[4, :128] = 0
    check(tsg, ctx, c, "decode")


# ------------------------------------------------------------------ any number of rows

@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("rows", [[1], [63, 64, 65], [130, 1, 2]])
def test_prefill(tsg, ctx, dk, dv, rows):
    check(tsg, ctx, Case(rows, 1, 2, dk, dv, seed=40), "prefill")


@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 5), (3, 3), (2, 8)])
def test_prefill_heads(tsg, ctx, hk, hv):
    check(tsg, ctx, Case([70, 20], hk, hv, 64, 48, seed=41), "prefill")


@pytest.mark.parametrize("slots", ["place", "fresh", "fork"])
@pytest.mark.parametrize("rows", [[100, 100], [5, 0, 129, 64]])
def test_prefill_slots(tsg, ctx, slots, rows):
    check(tsg, ctx, Case(rows, 1, 2, 64, 64, seed=42, slots=slots), "prefill")


def test_prefill_padding_and_strides(tsg, ctx):
    check(tsg, ctx, Case([70, 3, 66], 1, 2, 32, 48, seed=43, spare=70, lead=9, row_pad=40),
          "prefill")


def test_prefill_without_kept_states(tsg, ctx):
    c = Case([80, 65], 1, 1, 64, 32, seed=44)
    c.outs[1] = NONE
    check(tsg, ctx, c, "prefill")


@pytest.mark.parametrize("what", EXTREMES)
@pytest.mark.parametrize("dk", [64, 128])
def test_prefill_extremes(tsg, ctx, what, dk):
    check(tsg, ctx, Case([200, 70], 1, 2, dk, 48, seed=45, **EXTREMES[what]), "prefill")


def test_prefill_equal_keys(tsg, ctx):
    """All rows have one key: the triangle that is inverted is full of ones."""
    c = Case([150], 1, 2, 64, 64, seed=46, gate=3.0)
    c.qkv[:, 64:128] = c.qkv[0, 64:128]
    check(tsg, ctx, c, "prefill")


def test_prefill_zero_rows_of_keys(tsg, ctx):
    c = Case([100], 1, 2, 64, 64, seed=47)
    c.qkv[5] = 0
    c.qkv[64:70, :128] = 0
    check(tsg, ctx, c, "prefill")


def test_prefill_long(tsg, ctx):
    check(tsg, ctx, Case([1500], 1, 2, 128, 32, seed=48), "prefill")


def test_prefill_many_sequences(tsg, ctx):
    rows = [(7 * i) % 40 for i in range(150)]
    check(tsg, ctx, Case(rows, 1, 1, 32, 32, seed=49), "prefill")


@pytest.mark.parametrize("rows,heads,dk", [([64] * 32, (16, 64), 16), ([130] * 12, (32, 64), 64)])
def test_prefill_with_a_full_card(tsg, ctx, rows, heads, dk):
    """More workgroups than the card holds at once: their waves drift apart."""
    check(tsg, ctx, Case(rows, *heads, dk, 16, seed=52), "prefill")


def test_prefill_columns_of_different_sizes(tsg, ctx):
    """Value elements and states from 1e-6 to 1e4 side by side: each column is held to its own
    size."""
    c = Case([140], 1, 1, 128, 64, seed=50)
    size = torch.logspace(-6, 4, 64)
    c.qkv[:, 256:320] = (c.qkv[:, 256:320].float() * size.clamp(1e-3)).half()
    c.s *= size
    check(tsg, ctx, c, "prefill")


def test_prefill_is_decode_in_parts(tsg, ctx):
    """A prompt at once, as two chunks and row by row leads to the same states within what the
    forms may be off."""
    c = Case([96], 2, 4, 64, 64, seed=51)
    whole = check(tsg, ctx, c, "prefill")
    _, _, pool, tol = c.rule(True)
    delta = c.plan(tsg, ctx)
    d = c.to_device()
    states, gates = delta.states(d["s"]), tsg.DeltaGates(d["a_log"], d["dt_bias"])
    q, k, v = c.split(d["qkv"])
    a, b = d["ab"].split(c.hv, 1)
    slot = torch.tensor(c.outs, dtype=torch.int32, device="cuda")
    scratch = torch.empty(delta.scratch_bytes(70, 1), dtype=torch.uint8, device="cuda")
    first = True
    for lo, hi in ((0, 70), (70, 88), (88, 96)):
        batch = delta.batch(d["ins"] if first else slot, slot, hi - lo)
        rows = [t[lo:hi] for t in (q, k, v, a, b)]
        if hi < 96:
            delta.encode_prefill(states, batch, *rows, gates, d["out"][lo:hi], scratch)
        else:
            delta.encode_decode(states, batch, *rows, gates, d["out"][lo:hi])
        first = False
    ctx.synchronize()
    assert_near(d["s"], pool, 2 * tol)
    out, out_tol, _, _ = c.rule(True)
    assert_near(d["out"][:96], out, 2 * out_tol)
    assert whole["s"].shape == d["s"].shape
