"""Prompts whose rows differ in size by all of fp16's range: what one row holds takes no bits
from the others of its chunk."""
from __future__ import annotations

import pytest
import torch

from tests.attention_ref import assert_near
from tests.delta_ref import E24, HALF, Case
from tests.test_gpu_delta import check, ctx, tsg  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


class Split(Case):
    """The rule with what split operands may be off where their lower halves are kept times 2^11.

    Such a half ends at fp16's least step times 2^-11: half of one is 2^-36 at the most. S, r and u,
    scaled so that a bound on their column lies in 2^13 ... 2^14, are off by `step` = 2^-36 2^-13
    bound at most beside 2^-22 of their own size (the half's rounding; 2^-21 with that of the
    operand's other product, which is left out); T, at 32 for 1, by 2^-41; keys, kept with norms
    of 2 ... 4, by 2^-25 an element, 2^-26 dk^0.5 of a column's sum. The weights of the outputs are
    rounded to fp16 (`weights` of their size, 2^-35 at 1024 for 1). All else as Case has it."""
    weights, weights_least = HALF, 2.0 ** -35

    def _chunk_error(self, q, k, v, decay, beta, m, bound):
        dk, split = self.dk, 2.0 ** -21
        q, k, v = q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1)
        beta, total = beta.T, decay.clamp(min=-1000).T.cumsum(1)
        lower = torch.exp((total[:, :, None] - total[:, None, :]).clamp(max=0)).tril()
        a = (beta[:, :, None] * lower * (k @ k.transpose(1, 2))).tril(-1)
        t = torch.linalg.inv(torch.eye(a.shape[1], dtype=torch.float64) + a)
        p = lower * (q @ k.transpose(1, 2))
        kn, qn, sn, since = k.norm(dim=2), q.norm(dim=2), m.norm(dim=1), total.exp()
        pa = beta[:, :, None] * lower * kn[:, :, None] * kn[:, None, :]
        r = beta[:, :, None] * (v - since[:, :, None] * (k @ m))
        before = dk ** 0.5 * bound * 2.0 ** -49
        bound = 1.01 * dk ** 0.5 * m.abs().amax(1) + 65 * v.abs().amax(1)
        step = (bound * 2.0 ** -49)[:, None]
        low = torch.ones_like(lower).tril()
        from_s = since[:, :, None] * (((dk + 32) * E24 + split) * sn + before)[:, None]
        dr = beta[:, :, None] * (4 * E24 * v.abs() + kn[:, :, None] * from_s) + step
        ta, u = t.abs(), t @ r
        dt = ta @ (pa.tril(-1) * (dk + 24) * E24 + a.abs() * (80 * E24)) @ ta
        du = ta @ dr + dt @ r.abs() + (ta @ r.abs()) * (72 * E24 + 2 * split) \
            + (low @ r.abs()) * 2.0 ** -41
        until = torch.exp(total[:, -1:] - total)[:, :, None] * kn[:, :, None]
        state = (until * du + until * u.abs() * (104 * E24 + 2 * split + dk ** 0.5 * 2.0 ** -26)).sum(1) \
            + sn * 8 * E24 + 4 * k.shape[1] * step[:, 0]
        du = du + step
        outs = p.abs() @ du + (p.abs() @ u.abs()) * (self.weights + split + 72 * E24) \
            + (low @ u.abs()) * self.weights_least + qn[:, :, None] * from_s \
            + (lower * qn[:, :, None] * kn[:, None, :] * (dk + 24) * E24) @ u.abs()
        return state, outs, bound


SIZES = [(6e4, 1e-2), (6e4, 1e-4), (1e3, 1e-3), (1.0, 1e-4), (6e4, 6e4)]


def of_sizes(kind, dk, slots, large, small, at, rows=(64,)):
    """Rows of `small` values, and row `at` (of every chunk) of `large` ones."""
    c = kind(list(rows), 1, 2, dk, 32, seed=90, slots=slots, state=0.3 * small)
    v = c.split()[2]
    size = torch.full((c.total, 1), small)
    for s, n in enumerate(c.rows):
        size[c.starts[s] + at:c.starts[s] + n:64] = large
    scaled = torch.randn(v.shape, generator=torch.Generator().manual_seed(91)).clamp(-1, 1) * size
    c.qkv[:, 2 * c.dk:c.channels] = scaled.half()
    return c


@pytest.mark.parametrize("kind", [Case, Split])
@pytest.mark.parametrize("slots", ["fresh", "apart"])
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("large,small", SIZES)
def test_large_row_behind_small_ones(tsg, ctx, kind, slots, dk, large, small):  # noqa: F811
    check(tsg, ctx, of_sizes(kind, dk, slots, large, small, 63), "prefill")


@pytest.mark.parametrize("at", [0, 17, 40])
@pytest.mark.parametrize("large,small", SIZES)
def test_large_row_among_small_ones(tsg, ctx, large, small, at):  # noqa: F811
    """Also in several chunks, the last one short."""
    check(tsg, ctx, of_sizes(Split, 128, "apart", large, small, at, rows=(150, 64)), "prefill")


@pytest.mark.parametrize("dk", [64, 128, 256])
def test_state_that_a_chunk_forgets(tsg, ctx, dk):  # noqa: F811
    """A state of 1e4 that decays to less than the rows' values of 1e-3."""
    c = Split([70], 1, 2, dk, 32, seed=92, state=1e4, gate=4.0)
    c.qkv[:, 2 * dk:] = (c.qkv[:, 2 * dk:].float() * 1e-3).half()
    check(tsg, ctx, c, "prefill")


def test_causal_up_to_its_bits(tsg, ctx):  # noqa: F811
    """Rows before a large one are what they are without it, up to fp16's rounding."""
    a, b = (of_sizes(Split, 128, "apart", large, 1e-3, 63) for large in (6e4, 1e-3))
    got = [c.launch(tsg, ctx, "prefill")["out"].cpu()[:63].double() for c in (a, b)]
    ctx.synchronize()
    _, tol, _, _ = a.rule(True)
    assert_near(got[0], got[1], 2 * tol[:63])


class Fine(Split):
    """Weights split as the rest: rounded by 2^-22 of their size, 2^-22 more for the lower halves'
    product, which is left out; half a least step, times 2^-11, 2^-46 at 1024 for 1."""
    weights, weights_least = 2.0 ** -21, 2.0 ** -46


@pytest.mark.parametrize("slots", ["fresh", "apart"])
@pytest.mark.parametrize("dk,dv", [(16, 16), (64, 80), (128, 128), (192, 64), (256, 512)])
def test_outputs_are_rounded_once(tsg, ctx, dk, dv, slots):  # noqa: F811
    """A prompt's outputs are as far off as a token's: what their own rounding and fp32's sums
    leave, also where a row's parts cancel."""
    check(tsg, ctx, Fine([150, 64, 7], 1, 2, dk, dv, seed=93, slots=slots, gate=2.0), "prefill")


@pytest.mark.parametrize("large,small", SIZES)
def test_outputs_are_rounded_once_at_any_size(tsg, ctx, large, small):  # noqa: F811
    check(tsg, ctx, of_sizes(Fine, 128, "apart", large, small, 30, rows=(100,)), "prefill")
