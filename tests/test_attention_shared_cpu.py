"""What decode attention over shared prefixes refuses, checked without a GPU."""
from __future__ import annotations

import ctypes as C

import pytest

from tests.test_attention_cpu import ALIGNMENT, DECLINED, INVALID, abi, batch, config  # noqa: F401


def prefixes(abi, **over):  # noqa: F811
    x = abi.AttnPrefixes(1 << 12, 1 << 13, 2)
    for name, value in over.items():
        setattr(x, name, value)
    return x


def status(abi, c, b, x):  # noqa: F811
    return abi.load().tsg_attn_prefixes_check(*[None if v is None else C.addressof(v)
                                                for v in (c, b, x)])


def test_accepts(abi):  # noqa: F811
    assert status(abi, config(abi), None, prefixes(abi)) == 0
    assert status(abi, config(abi), batch(abi), prefixes(abi)) == 0
    assert status(abi, config(abi), batch(abi, num_seqs=2048, rows=2048 * 8), prefixes(abi)) == 0


@pytest.mark.parametrize("over,want", [
    (dict(num_groups=0), INVALID), (dict(num_groups=2049), INVALID),
    (dict(group_starts=None), INVALID), (dict(shared=None), INVALID),
    (dict(group_starts=(1 << 12) + 2), ALIGNMENT), (dict(shared=(1 << 13) + 1), ALIGNMENT),
])
def test_prefix_refusals(abi, over, want):  # noqa: F811
    assert status(abi, config(abi), batch(abi), prefixes(abi, **over)) == want


def test_other_refusals(abi):  # noqa: F811
    c, x = config(abi), prefixes(abi)
    assert status(abi, None, None, x) == INVALID
    assert status(abi, c, None, None) == INVALID
    assert status(abi, config(abi, window=16), batch(abi), x) == DECLINED
    assert status(abi, c, batch(abi, row_starts=1 << 14), x) == INVALID
    assert status(abi, c, batch(abi, num_seqs=2, rows=18), x) == DECLINED
    assert status(abi, c, batch(abi, num_seqs=2049, rows=2049), x) == DECLINED
    assert status(abi, c, batch(abi, num_seqs=0), x) == INVALID
    assert abi.load().tsg_attn_decode_shared(*[None] * 6, 0, None, 0) == INVALID
