"""Gated delta rule calls as programs make them: bad device data, refusals, infinities, graphs
and streams."""
from __future__ import annotations

import pytest
import torch

from tests.attention_ref import assert_near
from tests.delta_ref import NONE, Case
from tests.test_gpu_delta import check, ctx, tsg  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

OPS = ["conv", "decode", "prefill"]


def case(op, seqs=3, **more):
    rows = [2] * seqs if op == "decode" else [20, 70, 3, 1, 64][:seqs]
    return Case(rows, 1, 2, 64, 32, seed=60, **more)


def outputs(c, op, d):
    got = d["conv_out" if op == "conv" else "out"].cpu()[:c.total]
    return got, d["conv" if op == "conv" else "s"].cpu()


def reference(c, op):
    if op == "conv":
        out, tol, pool = c.convolution()
        return out, tol, pool, torch.zeros_like(pool, dtype=torch.float64)
    return c.rule(op == "prefill")


def reported(tsg, ctx, text):  # noqa: F811
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert e.value.status == 1 and text in str(e.value)
    ctx.synchronize()  # reported once


def only_sequence_is_bad(tsg, ctx, c, op, d, bad):  # noqa: F811
    c.launch(tsg, ctx, op, d=d)
    reported(tsg, ctx, "slot")
    got, pool = outputs(c, op, d)
    bad_rows = torch.zeros(c.total, dtype=torch.bool)
    for s in bad:
        bad_rows[c.starts[s]:c.starts[s + 1]] = True
        for i in range(c.kept):
            c.outs[s * c.kept + i] = NONE
    assert bool(torch.isnan(got[bad_rows]).all())
    out, tol, want, want_tol = reference(c, op)
    assert_near(got[~bad_rows], out[~bad_rows], tol[~bad_rows])
    assert_near(pool, want.double(), want_tol)


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("which", ["in", "out"])
@pytest.mark.parametrize("value", [10 ** 6, -2, 8])
def test_slot_past_the_pool(tsg, ctx, op, which, value):  # noqa: F811
    c = case(op)
    assert c.s.shape[0] == 8
    d = c.to_device()
    d["ins" if which == "in" else "outs"][1] = value
    only_sequence_is_bad(tsg, ctx, c, op, d, [1])


@pytest.mark.parametrize("op", OPS)
def test_out_slot_of_another_sequence(tsg, ctx, op):  # noqa: F811
    """Two sequences that write one slot are both refused; one that writes what another reads is."""
    c = case(op, seqs=5)
    d = c.to_device()
    d["outs"][3] = d["outs"][1]
    d["outs"][4] = d["ins"][0]
    only_sequence_is_bad(tsg, ctx, c, op, d, [1, 3, 4])


@pytest.mark.parametrize("op", ["conv", "decode"])
def test_out_slot_in_another_sequences_list(tsg, ctx, op):  # noqa: F811
    c = Case([3] * 4, 1, 2, 64, 32, seed=61, every=True)
    d = c.to_device()
    d["outs"][7] = d["outs"][0]   # the second sequence's second row, the first's first
    only_sequence_is_bad(tsg, ctx, c, op, d, [0, 2])


@pytest.mark.parametrize("op", ["conv", "prefill"])
@pytest.mark.parametrize("starts", [[0, 30, 20, 93], [0, 20, 90, 94], [5, 4, 3, 2],
                                    [0, 20, 90, -1]])
def test_wrong_row_starts(tsg, ctx, op, starts):  # noqa: F811
    c = case(op)
    d = c.to_device()
    d["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    c.launch(tsg, ctx, op, d=d, uniform=False)
    reported(tsg, ctx, "row starts")
    got, pool = outputs(c, op, d)
    assert bool(torch.isnan(got).all())
    assert torch.equal(pool, c.conv if op == "conv" else c.s)


@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("where", ["q", "k", "v", "a", "b", "state"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinities_reach_no_row_before(tsg, ctx, op, where, value):  # noqa: F811
    """An infinity or NaN in a row's operands reaches neither the rows before it nor another
    sequence nor the other key head's value heads; in q only its own row; in v, its own column at
    least from there on."""
    c = Case([8, 8] if op == "decode" else [75, 70], 2, 2, 64, 32, seed=62)
    d = c.to_device()
    at = 3 if op == "decode" else 41
    row = c.starts[1] + at
    if where in "qkv":
        first = {"q": 0, "k": 128, "v": 256}[where]
        d["qkv"][row, first + 3] = value
    elif where == "state":
        d["s"][c.ins[1], 0, 4, 3] = value
        row = c.starts[1]
    else:
        d["ab"][row, 0 if where == "a" else 2] = value
    c.launch(tsg, ctx, op, d=d)
    ctx.synchronize()
    out, tol, pool, pool_tol = c.rule(op == "prefill")
    got, states = outputs(c, op, d)
    apart = torch.ones_like(out, dtype=torch.bool)
    end = row + 1 if where == "q" else c.starts[2]
    apart[row:end, 0] = False
    assert_near(got[apart], out[apart], tol[apart])
    finite_gate = where == "b" and value == value or where == "a" and value == float("-inf")
    if where == "q":
        assert not bool(torch.isfinite(got[row, 0]).any())
    elif where in ("v", "state"):
        assert not bool(torch.isfinite(got[row:end, 0, 3]).any())
        assert not bool(torch.isfinite(states[c.outs[1], 0, :, 3]).any())
    elif not finite_gate and not (where == "a" and value == float("inf")):
        assert not bool(torch.isfinite(got[row:end, 0]).any())
        assert not bool(torch.isfinite(states[c.outs[1], 0]).any())
    untouched = torch.ones_like(pool, dtype=torch.bool)
    untouched[c.outs[1], 0] = where == "q"
    if where == "state":
        untouched[c.ins[1], 0, 4, 3] = False
    assert_near(states[untouched], pool[untouched], pool_tol[untouched])


@pytest.mark.parametrize("where", ["a", "b"])
def test_a_gates_nan_stays_in_its_value_head(tsg, ctx, where):  # noqa: F811
    """Three value heads share a key head; the first's gate is NaN at a row, the others are right."""
    c = Case([90], 1, 3, 64, 32, seed=68)
    d = c.to_device()
    d["ab"][41, 0 if where == "a" else 3] = float("nan")
    c.launch(tsg, ctx, "prefill", d=d)
    ctx.synchronize()
    out, tol, pool, pool_tol = c.rule(True)
    assert bool(torch.isnan(d["out"][41:90, 0]).all())
    assert_near(d["out"][:41], out[:41], tol[:41])
    assert_near(d["out"][:90, 1:], out[:, 1:], tol[:, 1:])
    assert_near(d["s"][:, 1:], pool[:, 1:], pool_tol[:, 1:])


@pytest.mark.parametrize("seqs", [8, 300])
def test_prefill_of_many_chunks(tsg, ctx, seqs):  # noqa: F811
    check(tsg, ctx, Case([64 + 64 * (i % 2) + i % 5 for i in range(seqs)] if seqs < 100 else
                         [2 * (i % 5) for i in range(seqs)], 2, 6, 32, 16, seed=69), "prefill")


def refused(tsg, call, *args, status=1, text=""):  # noqa: F811
    with pytest.raises(tsg.TsgError) as e:
        call(*args)
    assert e.value.status == status and text in str(e.value)


def pieces(tsg, ctx, c, d):  # noqa: F811
    delta = c.plan(tsg, ctx)
    states = delta.states(d["s"], d["conv"])
    batch = delta.batch(d["ins"], d["outs"], c.total, None if c.uniform else d["starts"])
    gates = tsg.DeltaGates(d["a_log"], d["dt_bias"])
    return delta, states, batch, gates, [*c.split(d["qkv"]), *d["ab"].split(c.hv, 1)]


def test_refusals(tsg, ctx):  # noqa: F811
    c = Case([9, 9], 1, 2, 64, 32, seed=63)
    d = c.to_device()
    delta, states, batch, gates, rows = pieces(tsg, ctx, c, d)
    out, scratch = d["out"], torch.empty(delta.scratch_bytes(18, 2), dtype=torch.uint8, device="cuda")
    refused(tsg, delta.encode_decode, states, batch, *rows, gates, out, status=4)
    ragged = delta.batch(d["ins"], d["outs"], c.total, d["starts"])
    refused(tsg, delta.encode_decode, states, ragged, *rows, gates, out, text="row starts")
    refused(tsg, delta.encode_prefill, states, batch, *rows, gates, out, scratch[:-1], text="scratch")
    refused(tsg, delta.encode_prefill, states, batch, *rows, gates, out,
            torch.empty(len(scratch) + 8, dtype=torch.uint8, device="cuda")[8:], status=2)
    refused(tsg, delta.encode_prefill, states, batch, *rows, gates, out, scratch.cpu())
    kept = delta.batch(d["ins"], torch.zeros(16, dtype=torch.int32, device="cuda"), 16)
    refused(tsg, delta.encode_prefill, states, kept, *rows, gates, out, scratch, text="keeps one")
    # operands
    for i in range(5):
        short = list(rows)
        short[i] = rows[i][:-1]
        refused(tsg, delta.encode_prefill, states, batch, *short, gates, out, scratch)
        other = list(rows)
        other[i] = rows[i].float()
        refused(tsg, delta.encode_prefill, states, batch, *other, gates, out, scratch)
    flat = d["qkv"].view(-1)
    for shared in (rows[2], flat[:18 * 64].view(18, 64), flat.as_strided((18, 64), (184, 1), 8)):
        refused(tsg, delta.encode_prefill, states, batch, *rows, gates, shared, scratch, text="shares")
    refused(tsg, delta.encode_prefill, states, batch, *rows, gates, d["ab"].view(-1)[:0].view(0, 64),
            scratch)
    refused(tsg, delta.encode_conv, states, batch, d["x"], d["weight"], d["x"], text="shares")
    refused(tsg, delta.encode_conv, states, batch, d["x"], d["weight"][:, :3], d["conv_out"])
    refused(tsg, delta.encode_conv, delta.states(d["s"]), batch, d["x"], d["weight"], d["conv_out"],
            text="NULL")
    refused(tsg, delta.encode_prefill, delta.states(None, d["conv"]), batch, *rows, gates, out,
            scratch, text="NULL")
    # pools, batches and gates
    refused(tsg, delta.states)
    refused(tsg, delta.states, d["s"], d["conv"][:-1])
    refused(tsg, delta.states, d["s"].half())
    refused(tsg, delta.states, d["s"].transpose(2, 3))
    refused(tsg, delta.states, d["s"].cpu())
    refused(tsg, delta.batch, d["ins"], d["outs"][:1], 18)
    refused(tsg, delta.batch, d["ins"].long(), d["outs"], 18)
    refused(tsg, delta.batch, d["ins"], d["outs"], 17)
    refused(tsg, delta.batch, d["ins"], d["outs"], 18, d["starts"][:2])
    refused(tsg, delta.batch, d["ins"].cpu(), d["outs"], 18)
    refused(tsg, tsg.DeltaGates, d["a_log"], d["dt_bias"][:1])
    refused(tsg, tsg.DeltaGates, d["a_log"].double(), d["dt_bias"].double())
    one = tsg.GatedDelta(ctx, 1, 1, 64, 32)
    refused(tsg, one.encode_conv, states, batch, d["x"], d["weight"], d["conv_out"], text="states of")
    refused(tsg, delta.encode_prefill, states, batch, *rows, tsg.DeltaGates(d["a_log"][:1], d["dt_bias"][:1]),
            out, scratch, text="gates")
    attn = tsg.Attention(ctx, 2, 1, 64, 16)
    other = attn.batch(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), d["ins"], 18)
    refused(tsg, delta.encode_prefill, states, other, *rows, gates, out, scratch, text="a batch of")
    refused(tsg, tsg.GatedDelta, ctx, 1, 2, 40, 32, status=3)
    torch.cuda.synchronize()
    assert bool((out == -77).all()) and torch.equal(d["s"].cpu(), c.s)
    ctx.synchronize()


def test_too_large_for_one_launch(tsg, ctx):  # noqa: F811
    """Refused before anything is launched."""
    seqs, hv, dk, dv = 1040, 256, 16, 512
    delta = tsg.GatedDelta(ctx, 1, hv, dk, dv)
    half = lambda *shape: torch.zeros(*shape, dtype=torch.float16, device="cuda")  # noqa: E731
    none = torch.full((seqs,), NONE, dtype=torch.int32, device="cuda")
    gates = tsg.DeltaGates(torch.zeros(hv, device="cuda"), torch.zeros(hv, device="cuda"))
    out = torch.full((seqs, hv, dv), -77.0, dtype=torch.float16, device="cuda")
    scratch = torch.zeros(delta.scratch_bytes(seqs, seqs), dtype=torch.uint8, device="cuda")
    refused(tsg, delta.encode_prefill, delta.states(torch.zeros(1, hv, dk, dv, device="cuda")),
            delta.batch(none, none, seqs), half(seqs, dk), half(seqs, dk), half(seqs, hv * dv),
            half(seqs, hv), half(seqs, hv), gates, out, scratch, status=3, text="launch")
    torch.cuda.synchronize()
    assert bool((out == -77).all()) and not bool(scratch.any())
    ctx.synchronize()


def test_a_sequence_without_rows_hands_its_state_on(tsg, ctx):  # noqa: F811
    """Bit for bit, whatever the sizes beside each other in a column."""
    c = Case([0, 70, 0], 1, 2, 64, 32, seed=71)
    e = torch.randint(-140, 127, c.s[0].shape, generator=torch.Generator().manual_seed(72))
    c.s[c.ins[0]] = torch.ldexp(c.s[c.ins[0]] + 1, e)
    c.s[c.ins[2], :, ::5] = float("inf")
    c.s[c.ins[2], :, 1::5] = 3e38
    d = c.to_device()
    c.launch(tsg, ctx, "prefill", d=d)
    ctx.synchronize()
    for s in (0, 2):
        assert torch.equal(d["s"][c.outs[s]].cpu(), c.s[c.ins[s]])


def test_closed_context_and_plan(tsg):  # noqa: F811
    c = Case([2], 1, 1, 64, 32, seed=64)
    d = c.to_device()
    own = tsg.Context(0)
    delta, states, batch, gates, rows = pieces(tsg, own, c, d)
    other = c.plan(tsg, own)
    other.close()
    refused(tsg, other.encode_decode, states, batch, *rows, gates, d["out"])
    own.close()
    refused(tsg, delta.encode_decode, states, batch, *rows, gates, d["out"], text="closed")
    refused(tsg, delta.encode_conv, states, batch, d["x"], d["weight"], d["conv_out"], text="closed")
    torch.cuda.synchronize()
    assert bool((d["out"] == -77).all())
    delta.close()


def test_pools_of_wider_slots(tsg, ctx):  # noqa: F811
    """Slots further apart than a state is large, as views of a larger pool."""
    c = Case([2] * 3, 1, 2, 64, 32, seed=65)
    d = c.to_device()
    wide = torch.zeros(c.s.shape[0], 3, 64, 32, device="cuda")
    wide[:, :2] = d["s"]
    wide[:, 2] = 5.0
    d["s"] = wide[:, :2]
    check(tsg, ctx, c, "decode", d=d)
    assert bool((wide[:, 2] == 5).all())


@pytest.mark.parametrize("op", OPS)
def test_far_slots(tsg, ctx, op):  # noqa: F811
    """Slots whose places pass 2^32 elements of the pool."""
    c = Case([1 if op == "decode" else 21] * 9, 1, 2, 64, 32, seed=74)
    d = c.to_device()
    for name, type in (("s", torch.float32), ("conv", torch.float16)):
        shape = d[name].shape
        far = torch.empty_strided(shape, (2 ** 28 - 16, *d[name].stride()[1:]), dtype=type, device="cuda")
        d[name] = far.copy_(d[name])
    assert 2 ** 28 * max(c.ins + c.outs) >= 2 ** 32
    check(tsg, ctx, c, op, d=d)


def test_calls_beside_each_other(tsg, ctx):  # noqa: F811
    """One plan's calls on two streams at once, each with its slots and scratch: as one by one."""
    cases = [(Case([700, 130], 2, 8, 64, 64, seed=75), "prefill"),
             (Case([8] * 40, 2, 8, 64, 64, seed=76), "decode"),
             (Case([500, 333], 2, 8, 64, 64, seed=77), "conv"),
             (Case([411] * 2, 2, 8, 64, 64, seed=78), "prefill")]
    wants = [c.launch(tsg, ctx, op) for c, op in cases]
    ctx.synchronize()
    runs, delta = [], cases[0][0].plan(tsg, ctx)
    for c, op in cases:
        d = c.to_device()
        runs.append((op, d, delta.states(d["s"], d["conv"]), tsg.DeltaGates(d["a_log"], d["dt_bias"]),
                     delta.batch(d["ins"], d["outs"], c.total, None if c.uniform else d["starts"]),
                     [*c.split(d["qkv"]), *d["ab"].split(c.hv, 1)],
                     torch.empty(delta.scratch_bytes(c.total, len(c.rows)), dtype=torch.uint8, device="cuda")))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for turn in range(6):
        for i, (op, d, states, gates, batch, rows, scratch) in enumerate(runs):
            stream = streams[i % 2]
            if op == "conv":
                delta.encode_conv(states, batch, d["x"], d["weight"], d["conv_out"], stream=stream)
            elif op == "decode":
                delta.encode_decode(states, batch, *rows, gates, d["out"], stream=stream)
            else:
                delta.encode_prefill(states, batch, *rows, gates, d["out"], scratch, stream=stream)
    torch.cuda.synchronize()
    ctx.synchronize()
    for (c, op), run, want in zip(cases, runs, wants):
        for got, ref in zip(outputs(c, op, run[1]), outputs(c, op, want)):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("op", OPS)
def test_on_another_stream(tsg, ctx, op):  # noqa: F811
    c = case(op)
    stream = torch.cuda.Stream()
    d = c.to_device()
    stream.wait_stream(torch.cuda.current_stream())
    c.launch(tsg, ctx, op, d=d, stream=stream)
    stream.synchronize()
    want = c.launch(tsg, ctx, op)
    ctx.synchronize()
    for got, ref in zip(outputs(c, op, d), outputs(c, op, want)):
        assert torch.equal(got, ref)


@pytest.mark.parametrize("op", OPS)
def test_captured_and_replayed(tsg, ctx, op):  # noqa: F811
    """A graph replays with the slots, rows and states that its buffers then hold, with eager work
    in between; every replay against the eager result."""
    c = case(op)
    d = c.to_device()
    delta, states, batch, gates, rows = pieces(tsg, ctx, c, d)
    scratch = torch.empty(delta.scratch_bytes(c.total, 3), dtype=torch.uint8, device="cuda")

    def call():
        if op == "conv":
            delta.encode_conv(states, batch, d["x"], d["weight"], d["conv_out"])
        elif op == "decode":
            delta.encode_decode(states, batch, *rows, gates, d["out"])
        else:
            delta.encode_prefill(states, batch, *rows, gates, d["out"], scratch)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for turn in range(4):
        other = Case(c.rows if op == "decode" or turn != 2 else [60, 2, 31], 1, 2, 64, 32,
                     seed=70 + turn, slots="place" if turn % 2 else "apart")
        fresh = other.to_device()
        for name in d:
            d[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        want = other.launch(tsg, ctx, op)
        ctx.synchronize()
        for got, ref in zip(outputs(other, op, d), outputs(other, op, want)):
            assert torch.equal(got, ref)


def test_padded_sequences_of_a_fixed_batch(tsg, ctx):  # noqa: F811
    """A batch of fixed size whose last sequences are padding: no slots, nothing kept."""
    c = Case([1] * 6, 1, 2, 64, 32, seed=66)
    for s in (4, 5):
        c.ins[s] = c.outs[s] = NONE
    check(tsg, ctx, c, "decode")
    check(tsg, ctx, c, "conv")


def test_a_layers_run(tsg, ctx):  # noqa: F811
    """The convolution into the rule, a prompt and then tokens one by one, states in place: every
    step against the reference's on the same inputs."""
    prompt, steps = 70, 3
    c = Case([prompt], 2, 4, 64, 48, seed=67, slots="place")
    d = c.to_device()
    delta = c.plan(tsg, ctx)
    states, gates = delta.states(d["s"], d["conv"]), tsg.DeltaGates(d["a_log"], d["dt_bias"])
    scratch = torch.empty(delta.scratch_bytes(prompt, 1), dtype=torch.uint8, device="cuda")
    for step in range(steps + 1):
        n = prompt if step == 0 else 1
        now = Case([n], 2, 4, 64, 48, seed=67 + step, slots="place")
        now.ins, now.outs = list(c.ins), list(c.outs)
        now.weight, now.a_log, now.dt_bias = c.weight, c.a_log, c.dt_bias
        now.conv, now.s = d["conv"].cpu(), d["s"].cpu()
        x, ab = now.x.cuda(), now.ab.cuda()
        mixed = torch.empty(n, c.channels, dtype=torch.float16, device="cuda")
        out = torch.empty(n, 4, 48, dtype=torch.float16, device="cuda")
        batch = delta.batch(d["ins"], d["outs"], n)
        delta.encode_conv(states, batch, x, d["weight"], mixed)
        rows = [*c.split(mixed), *ab.split(4, 1)]
        if n > 8:
            delta.encode_prefill(states, batch, *rows, gates, out, scratch)
        else:
            delta.encode_decode(states, batch, *rows, gates, out)
        ctx.synchronize()
        want, tol, pool = now.convolution()
        assert_near(mixed, want, tol)
        assert torch.equal(d["conv"].cpu(), pool)
        now.qkv = mixed.cpu()
        want, tol, pool, pool_tol = now.rule(n > 8)
        assert_near(out, want, tol)
        assert_near(d["s"], pool, pool_tol)
