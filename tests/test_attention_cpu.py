"""What the attention entry points refuse, checked without a GPU (tsg_attn_check
makes the checks that the launches make), and the test reference's own definitions."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from tests.attention_ref import Case, append_reference

INVALID, ALIGNMENT, UNSUPPORTED, DECLINED = 1, 2, 3, 4


@pytest.fixture(scope="module")
def abi():
    from tsugumi_amd import _abi
    _abi.load()
    return _abi


def config(abi, **over):
    c = abi.AttnConfig(8, 2, 64, 16, 0, 0, 0, 0.125, 1.0, 1.0)
    for name, value in over.items():
        setattr(c, name, value)
    return c


def pages(abi, c, **over):
    p = abi.KVPages(1 << 20, 1 << 24, 10, c.head_dim, c.head_dim * c.page_tokens,
                    c.head_dim * c.page_tokens * c.kv_heads)
    for name, value in over.items():
        setattr(p, name, value)
    return p


def batch(abi, **over):
    b = abi.AttnBatch(1 << 12, 1 << 13, None, 4, 2, 6)
    for name, value in over.items():
        setattr(b, name, value)
    return b


def status(abi, c, p=None, b=None):
    ref = [None if x is None else C.addressof(x) for x in (c, p, b)]
    return abi.load().tsg_attn_check(*ref)


def test_accepts(abi):
    c = config(abi)
    assert status(abi, c, pages(abi, c), batch(abi)) == 0
    c = config(abi, kv_type=1, head_dim=512, page_tokens=4096, window=1024, sinks=4, k_scale=0.01)
    assert status(abi, c, pages(abi, c), batch(abi, row_starts=1 << 14, rows=7)) == 0


@pytest.mark.parametrize("over,want", [
    (dict(q_heads=0), INVALID), (dict(kv_heads=0), INVALID), (dict(q_heads=7), INVALID),
    (dict(q_heads=2048, kv_heads=1024), INVALID), (dict(kv_type=2), INVALID),
    (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=60), UNSUPPORTED),
    (dict(head_dim=520), UNSUPPORTED), (dict(head_dim=72, kv_type=1), UNSUPPORTED),
    (dict(page_tokens=0), UNSUPPORTED), (dict(page_tokens=8), UNSUPPORTED),
    (dict(page_tokens=48), UNSUPPORTED), (dict(page_tokens=8192), UNSUPPORTED),
    (dict(sinks=4), INVALID), (dict(window=1 << 31), INVALID),
    (dict(scale=math.nan), INVALID), (dict(scale=math.inf), INVALID), (dict(scale=1e7), INVALID),
    (dict(k_scale=2.0), INVALID), (dict(kv_type=1, k_scale=0.0), INVALID),
    (dict(kv_type=1, v_scale=-1.0), INVALID), (dict(kv_type=1, v_scale=math.nan), INVALID),
])
def test_config_refusals(abi, over, want):
    assert status(abi, config(abi, **over)) == want
    assert len(abi.load().tsg_last_error()) > 0


@pytest.mark.parametrize("over,want", [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(num_pages=0), INVALID),
    (dict(k=(1 << 20) + 8), ALIGNMENT), (dict(v=(1 << 24) + 2), ALIGNMENT),
    (dict(token_stride=68), ALIGNMENT), (dict(head_stride=1028), ALIGNMENT),
    (dict(page_stride=2052), ALIGNMENT), (dict(token_stride=56), INVALID),
    (dict(head_stride=1016), INVALID), (dict(head_stride=0), INVALID),
    (dict(page_stride=2040), INVALID), (dict(page_stride=0), INVALID),
    (dict(head_stride=64, token_stride=120), INVALID),
    (dict(page_stride=1 << 45), INVALID),
    (dict(token_stride=1 << 30, head_stride=1 << 35, page_stride=1 << 40), UNSUPPORTED),
])
def test_page_refusals(abi, over, want):
    c = config(abi)
    assert status(abi, c, pages(abi, c, **over)) == want


def test_page_layouts(abi):
    c = config(abi)
    assert status(abi, c, pages(abi, c, head_stride=64, token_stride=128)) == 0
    assert status(abi, c, pages(abi, c, num_pages=1, page_stride=0)) == 0
    one = config(abi, q_heads=8, kv_heads=1)
    assert status(abi, one, pages(abi, one, head_stride=0)) == 0
    # rows of 8 elements are 16 bytes of fp16 and 8 of e4m3
    e4m3 = config(abi, kv_type=1)
    assert status(abi, e4m3, pages(abi, e4m3, token_stride=72, page_stride=1 << 20)) == ALIGNMENT


@pytest.mark.parametrize("over,want", [
    (dict(num_seqs=0), INVALID), (dict(rows=0), INVALID), (dict(rows=7), INVALID),
    (dict(rows=1 << 30), INVALID), (dict(num_seqs=1 << 30, rows=1 << 30), INVALID),
    (dict(page_table=None), INVALID), (dict(lengths=None), INVALID),
    (dict(table_stride=0), INVALID), (dict(table_stride=1 << 27), INVALID),
    (dict(lengths=(1 << 13) + 2), ALIGNMENT), (dict(page_table=(1 << 12) + 1), ALIGNMENT),
    (dict(row_starts=(1 << 14) + 3, rows=7), ALIGNMENT),
])
def test_batch_refusals(abi, over, want):
    assert status(abi, config(abi), None, batch(abi, **over)) == want


def test_null_objects(abi):
    lib, c = abi.load(), config(abi)
    assert lib.tsg_attn_check(None, None, None) == INVALID
    handle = C.c_void_p(1)
    assert lib.tsg_attn_create(None, C.addressof(c), C.byref(handle)) == INVALID
    assert handle.value is None
    assert lib.tsg_attn_create(None, C.addressof(c), None) == INVALID
    for call in (lib.tsg_attn_decode, lib.tsg_attn_prefill):
        assert call(None, None, None, None, None, 0, None, 0) == INVALID
    assert lib.tsg_attn_append(None, None, None, None, None, None, None, 0) == INVALID
    lib.tsg_attn_destroy(None)


# ---------------------------------------------------------- the test reference

def test_reference_attention_against_a_full_softmax():
    c = Case([6, 4], [40, 9], 4, 2, 16, window=12, sinks=3, seed=1)
    want, _ = c.attention()
    for s in range(2):
        n, length, first = c.rows[s], c.lengths[s], int(c.starts[s])
        k = c.tokens("k", s).repeat_interleave(2, 1)
        v = c.tokens("v", s).repeat_interleave(2, 1)
        q = c.q[first:first + n].double()
        logits = torch.einsum("ihd,jhd->hij", q, k) / 4
        i, j = torch.arange(length - n, length)[:, None], torch.arange(length)[None]
        logits[:, (j > i) | ((i - j >= 12) & (j >= 3))] = -math.inf
        out = torch.einsum("hij,jhd->ihd", logits.softmax(-1), v)
        assert torch.allclose(out, want[first:first + n], atol=1e-12)


def test_reference_rotation_is_by_relative_position():
    g = torch.Generator().manual_seed(2)
    q, k = torch.randn(1, 1, 32, generator=g), torch.randn(1, 1, 32, generator=g)
    inv = (100.0 ** (-torch.arange(0, 32, 2).double() / 32)).float()
    for interleaved in (False, True):
        dots = []
        for a, b in ((5, 2), (1005, 1002)):
            (qr, _), _, _ = append_reference(q, k, k, torch.tensor([a]), None, None, inv, 32,
                                             interleaved, 0.0, False)
            _, (kr, _), _ = append_reference(q, k, k, torch.tensor([b]), None, None, inv, 32,
                                             interleaved, 0.0, False)
            dots.append(float((qr * kr).sum()))
        assert abs(dots[0] - dots[1]) < 1e-9


# ------------------------------------------- what the Python classes refuse

def bare_plan(tsg):
    """An Attention of 8 query and 2 key heads of 64 without a device behind it."""
    attn = tsg.Attention.__new__(tsg.Attention)
    attn.handle, attn._half, attn._device = None, (torch.float16,), -1  # as of meta tensors
    return attn


def test_python_refuses_values_past_32_bits():
    """What ctypes would cut off to 32 bits: 2^32 sinks are none, 2^32 + 8 heads are eight."""
    import tsugumi_amd as tsg

    class NoContext:
        lib, handle, device = tsg.load(), None, 0

    fine = dict(q_heads=8, kv_heads=2, head_dim=64, page_tokens=16, window=64, sinks=1)
    for name in fine:
        for value in (fine[name] + (1 << 32), -1):
            with pytest.raises(tsg.TsgError) as e:
                tsg.Attention(NoContext(), **{**fine, name: value})
            assert e.value.status == INVALID and name in str(e.value)
    attn = bare_plan(tsg)
    for stride, status in ((512, None), ((1 << 32) + 512, INVALID)):
        rows = torch.empty_strided((2, 512), (stride, 1), dtype=torch.float16, device="meta")
        if status is None:
            assert attn._rows(rows, 2, 8, 512) == (0, 512)
            continue
        with pytest.raises(tsg.TsgError) as e:
            attn._rows(rows, 2, 8, 512)
        assert e.value.status == status
