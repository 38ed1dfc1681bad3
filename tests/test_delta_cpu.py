"""What the gated delta rule's entry points refuse, checked without a GPU (tsg_delta_check
makes the checks that the launches make), and the test reference's own definitions."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from tests.delta_ref import CHUNK, NONE, Case

INVALID, ALIGNMENT, UNSUPPORTED = 1, 2, 3


@pytest.fixture(scope="module")
def abi():
    from tsugumi_amd import _abi
    _abi.load()
    return _abi


def config(abi, **over):
    c = abi.DeltaConfig(2, 4, 64, 32, 4, 0.125, 1e-6)
    for name, value in over.items():
        setattr(c, name, value)
    return c


def states(abi, **over):
    p = abi.DeltaStates(1 << 20, 1 << 24, 4 * 64 * 32, 3 * 384, 5)
    for name, value in over.items():
        setattr(p, name, value)
    return p


def batch(abi, **over):
    b = abi.DeltaBatch(None, 1 << 12, 1 << 13, 2, 6, 1)
    for name, value in over.items():
        setattr(b, name, value)
    return b


def rows(abi, **over):
    r = abi.DeltaRows(1 << 16, 1 << 17, 1 << 18, 1 << 19, 1 << 21, 128, 128, 128, 4, 4)
    for name, value in over.items():
        setattr(r, name, value)
    return r


def status(abi, c, p=None, b=None, r=None):
    return abi.load().tsg_delta_check(*[None if x is None else C.addressof(x)
                                        for x in (c, p, b, r)])


def test_accepts(abi):
    assert status(abi, config(abi), states(abi), batch(abi), rows(abi)) == 0
    assert status(abi, config(abi, key_dim=256, value_dim=512, conv_width=8, value_heads=256)) == 0
    assert status(abi, config(abi), states(abi, s=None), batch(abi, row_starts=1 << 14, rows=7)) == 0
    assert status(abi, config(abi), states(abi, num_slots=1, slot_stride=0, conv_stride=0),
                  batch(abi, kept=3)) == 0


@pytest.mark.parametrize("over,want", [
    (dict(key_heads=0), INVALID), (dict(value_heads=0), INVALID), (dict(value_heads=3), INVALID),
    (dict(key_heads=8, value_heads=4), INVALID), (dict(value_heads=512), INVALID),
    (dict(key_dim=0), UNSUPPORTED), (dict(key_dim=72), UNSUPPORTED), (dict(key_dim=272), UNSUPPORTED),
    (dict(value_dim=0), UNSUPPORTED), (dict(value_dim=40), UNSUPPORTED),
    (dict(value_dim=528), UNSUPPORTED), (dict(conv_width=1), UNSUPPORTED),
    (dict(conv_width=9), UNSUPPORTED), (dict(scale=math.nan), INVALID),
    (dict(scale=math.inf), INVALID), (dict(scale=1e7), INVALID), (dict(eps=0.0), INVALID),
    (dict(eps=math.nan), INVALID), (dict(eps=2.0), INVALID),
])
def test_config_refusals(abi, over, want):
    assert status(abi, config(abi, **over)) == want
    assert len(abi.load().tsg_last_error()) > 0


@pytest.mark.parametrize("over,want", [
    (dict(num_slots=0), INVALID), (dict(num_slots=0xFFFFFFFF), INVALID),
    (dict(s=(1 << 20) + 4), ALIGNMENT), (dict(conv=(1 << 24) + 8), ALIGNMENT),
    (dict(slot_stride=4 * 64 * 32 + 2), ALIGNMENT), (dict(conv_stride=3 * 384 + 4), ALIGNMENT),
    (dict(slot_stride=4 * 64 * 32 - 4), INVALID), (dict(conv_stride=3 * 384 - 8), INVALID),
    (dict(slot_stride=1 << 30), INVALID), (dict(conv_stride=1 << 30), INVALID),
])
def test_state_refusals(abi, over, want):
    assert status(abi, config(abi), states(abi, **over)) == want


@pytest.mark.parametrize("over,want", [
    (dict(num_seqs=0), INVALID), (dict(num_seqs=(1 << 16) + 1, rows=(1 << 16) + 1), INVALID),
    (dict(rows=0), INVALID), (dict(rows=(1 << 22) + 2), INVALID), (dict(rows=7), INVALID),
    (dict(in_slots=None), INVALID), (dict(out_slots=None), INVALID),
    (dict(in_slots=(1 << 12) + 2), ALIGNMENT), (dict(out_slots=(1 << 13) + 1), ALIGNMENT),
    (dict(row_starts=(1 << 14) + 2), ALIGNMENT), (dict(kept=0), INVALID), (dict(kept=2), INVALID),
    (dict(kept=3, row_starts=1 << 14), INVALID), (dict(kept=9, rows=18), INVALID),
])
def test_batch_refusals(abi, over, want):
    assert status(abi, config(abi), None, batch(abi, **over)) == want


@pytest.mark.parametrize("over,want", [
    *[({n: None}, INVALID) for n in "qkvab"],
    *[({n: 8 + (1 << 16)}, ALIGNMENT) for n in "qkv"], *[({n: 1 + (1 << 16)}, ALIGNMENT) for n in "ab"],
    *[({n + "_stride": 120}, INVALID) for n in "qkv"], *[({n + "_stride": 132}, ALIGNMENT) for n in "qkv"],
    (dict(a_stride=3), INVALID), (dict(b_stride=0), INVALID),
    *[({n + "_stride": (1 << 27) + 8}, UNSUPPORTED) for n in "qkv"],
])
def test_row_refusals(abi, over, want):
    assert status(abi, config(abi), None, None, rows(abi, **over)) == want


def test_null_arguments(abi):
    lib = abi.load()
    assert lib.tsg_delta_check(None, None, None, None) == INVALID
    out = C.c_void_p(1)
    assert lib.tsg_delta_create(None, C.addressof(config(abi)), C.byref(out)) == INVALID
    assert not out.value
    assert lib.tsg_delta_create(None, C.addressof(config(abi)), None) == INVALID
    assert lib.tsg_delta_conv(*[None] * 5, 0, None, None, 0) == INVALID
    assert lib.tsg_delta_decode(*[None] * 8, 0) == INVALID
    assert lib.tsg_delta_prefill(*[None] * 8, 0, None, 0) == INVALID
    assert lib.tsg_delta_prefill_scratch_bytes(None, 5, 5) == 0
    lib.tsg_delta_destroy(None)


def test_reference_rule_is_its_chunked_form():
    """The reference's rows, one after another, against the products over 64 rows at once that
    a prompt may take, in 64 bits: one formula, computed apart."""
    c = Case([150], 1, 2, 32, 16, seed=3, gate=2.0)
    out, _, pool, _ = c.rule()
    q, k, v = (t.double().reshape(150, -1, d) for t, d in zip(c.split(), (32, 32, 16)))
    q, k = (x / (x.square().sum(-1, keepdim=True) + c.eps).sqrt() for x in (q, k))
    for h in range(2):
        x = c.ab[:, h].double() + c.dt_bias[h].double()
        g = -torch.exp(c.a_log[h].double()) * torch.nn.functional.softplus(x)
        beta = torch.sigmoid(c.ab[:, 2 + h].double())
        s = c.s[c.ins[0], h].double()
        for i in range(0, 150, CHUNK):
            r = slice(i, min(150, i + CHUNK))
            G = g[r].cumsum(0)
            w = torch.exp((G[:, None] - G).clamp(max=0)).tril()
            kk, qq = k[r, 0], q[r, 0]
            a = (beta[r, None] * w * (kk @ kk.T)).tril(-1)
            u = torch.linalg.solve(torch.eye(len(G), dtype=torch.float64) + a,
                                   beta[r, None] * (v[r, h] - G.exp()[:, None] * (kk @ s)))
            o = c.scale * (G.exp()[:, None] * (qq @ s) + (w * (qq @ kk.T)) @ u)
            assert torch.allclose(o, out[r, h], rtol=1e-11, atol=1e-12)
            s = G[-1].exp() * s + (kk * (G[-1] - G).exp()[:, None]).T @ u
        assert torch.allclose(s, pool[c.outs[0], h], rtol=1e-11, atol=1e-12)


def test_reference_convolution_is_torchs():
    c = Case([5, 1, 9], 1, 1, 16, 16, width=4, seed=4)
    c.ins[1] = NONE
    out, _, pool = c.convolution()
    for s, n in enumerate(c.rows):
        old = torch.zeros(3, c.channels) if c.ins[s] == NONE else c.conv[c.ins[s]].float()
        x = torch.cat((old, c.x[c.starts[s]:c.starts[s] + n].float())).double()
        y = torch.nn.functional.conv1d(x.T[None], c.weight.double()[:, None], groups=c.channels)
        assert torch.allclose(out[c.starts[s]:c.starts[s] + n],
                              torch.nn.functional.silu(y[0].T), rtol=1e-12, atol=1e-12)
        assert torch.equal(pool[c.outs[s]].double(), x[-3:])
