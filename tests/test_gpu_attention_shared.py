"""Decode attention of batches that share prefixes, against the definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from tests.attention_ref import E4M3, Case, assert_near
from tests.test_gpu_attention import ctx, launch, plan, tsg  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

DIMS = [(4, 2, 64), (8, 1, 80), (6, 3, 128), (2, 2, 128), (16, 2, 136), (4, 2, 256), (8, 1, 272), (4, 1, 512)]


def share(c, starts, shared):
    """Gives the sequences of a group the pages of its first for the tokens that they share (the
    last of these pages whole), and NaN to the slots that no sequence then has written."""
    for g, tokens in enumerate(shared):
        first, end = starts[g], starts[g + 1]
        pages = min(-(-tokens // c.page), c.table.shape[1])
        for s in range(first + 1, end):
            c.table[s, :pages] = c.table[first, :pages]
    written = torch.zeros(c.k.shape[0], c.page, dtype=torch.bool)
    for s, n in enumerate(c.lengths):
        t = torch.arange(n)
        written[c.table[s, t // c.page].long(), t % c.page] = True
    for x, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        y = torch.randn(x.shape, generator=c.g)
        y = y.half() if c.kv == "f16" else (y / scale).to(E4M3)
        view = (lambda t: t) if c.kv == "f16" else (lambda t: t.view(torch.uint8))
        view(x).copy_(view(y))
        where = ~written[:, None, :, None].expand(x.shape)
        view(x).masked_fill_(where, math.nan if c.kv == "f16" else 0x7F)
    c.groups, c.shared = list(starts), list(shared)
    return c


def call(tsg, ctx, c, d=None, attn=None, out=None, stream=None):  # noqa: F811
    d = c.to_device() if d is None else d
    attn = plan(tsg, ctx, c) if attn is None else attn
    for name in ("groups", "shared"):
        if name not in d:
            d[name] = torch.tensor(getattr(c, name), dtype=torch.int32, device="cuda")
    out = torch.full_like(d["q"], -77.0) if out is None else out
    attn.encode_decode_shared(attn.cache(d["k"], d["v"]),
                              attn.batch(d["table"], d["lengths"], c.total),
                              attn.prefixes(d["groups"], d["shared"]), d["q"], out, stream=stream)
    return out


def check(tsg, ctx, c, **more):  # noqa: F811
    got = call(tsg, ctx, c, **more)
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(got, want, tol)
    return got


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("q_heads,kv_heads,dim", DIMS)
def test_head_layouts(tsg, ctx, q_heads, kv_heads, dim, kv):  # noqa: F811
    if kv == "e4m3" and dim % 16:
        dim += 8
    c = Case([2] * 5, [200, 211, 192, 250, 193], q_heads, kv_heads, dim, kv=kv, seed=dim)
    check(tsg, ctx, share(c, [0, 3, 5], [192, 128]))


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
@pytest.mark.parametrize("q_heads,kv_heads,dim", [(4, 2, 256), (8, 1, 272), (16, 2, 144), (4, 1, 512)])
@pytest.mark.parametrize("prefix", [64, 1600])
def test_wide_heads_of_many_rows(tsg, ctx, q_heads, kv_heads, dim, kv, prefix):  # noqa: F811
    """On the side of the rule where heads over 128 share: also rows inside the prefix, and over
    several splits."""
    seqs = -(-64 * kv_heads // (2 * q_heads)) + 2
    lengths = [prefix + 40 + 9 * s for s in range(seqs)]
    lengths[1] = prefix - 20
    c = Case([2] * seqs, lengths, q_heads, kv_heads, dim, kv=kv, seed=dim)
    check(tsg, ctx, share(c, [0, seqs // 2, seqs], [prefix, prefix]))


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("heads", [(1, 1), (7, 1), (16, 2), (40, 1)])
def test_blocks_of_rows(tsg, ctx, rows, heads):  # noqa: F811
    """Groups whose rows end inside a tile of 128, and pass several."""
    c = Case([rows] * 6, [140, 170, 150, 139, 201, 144], *heads, 64, seed=rows)
    check(tsg, ctx, share(c, [0, 4, 6], [130, 100]))


@pytest.mark.parametrize("shared", [0, 1, 63, 64, 65, 127, 128, 500, 10 ** 6])
def test_shared_lengths(tsg, ctx, shared):  # noqa: F811
    """From nothing to more than the sequences (and their page tables) have."""
    c = Case([1] * 3, [531, 530, 560], 4, 2, 64, seed=3)
    share(c, [0, 3], [min(shared, 528)])
    c.shared = [shared if shared <= 500 else 528]
    check(tsg, ctx, c)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_page_sizes(tsg, ctx, page):  # noqa: F811
    """Pages smaller and larger than a key tile: a prefix may end inside one."""
    c = Case([2] * 4, [300, 310, 260, 301], 4, 2, 64, page=page, seed=page)
    check(tsg, ctx, share(c, [0, 4], [256 // page * page or 200]))


@pytest.mark.parametrize("starts,shared", [
    ([0, 8], [128]), ([2, 5], [128]), ([0, 1, 8], [128, 64]), ([0, 4, 4, 8], [128, 64, 192]),
    ([0, 2, 4, 6, 8], [64, 128, 192, 70]), ([3, 3], [64]), ([8, 8, 8], [64, 64]),
    ([1, 2, 3, 4, 5, 6, 7, 8], [64] * 7), ([0] * 40 + [8], [64] * 39 + [128]),
    ([0] * 2047 + [5, 8], [0] * 2046 + [192, 64])])
def test_groups(tsg, ctx, starts, shared):  # noqa: F811
    """Sequences before, between and behind groups; groups of one sequence and of none, these
    also more than there are sequences."""
    c = Case([1] * 8, [200, 230, 199, 300, 195, 210, 222, 201], 6, 2, 64, seed=4)
    check(tsg, ctx, share(c, starts, shared))


def test_sequences_shorter_than_what_they_share(tsg, ctx):  # noqa: F811
    """Rows inside the prefix see a part of it only; a padded sequence is zeros, also as the first
    of its group (whose pages then are not read)."""
    c = Case([3] * 8, [400, 130, 2, 0, 390, 0, 200, 180], 4, 2, 64, seed=5)
    got = check(tsg, ctx, share(c, [0, 5, 8], [384, 128]))
    assert bool((got[9:12] == 0).all()) and bool((got[15:18] == 0).all())
    assert bool((got[6] == 0).all())


def test_first_sequence_shorter_than_the_others(tsg, ctx):  # noqa: F811
    """What is read of the first's pages ends with its length."""
    c = Case([1] * 3, [100, 400, 300], 4, 2, 64, seed=6)
    share(c, [0, 3], [96])
    c.shared = [290]
    check(tsg, ctx, c)


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
def test_long_prefix_over_splits(tsg, ctx, kv):  # noqa: F811
    c = Case([1] * 5, [9100, 9001, 9400, 12000, 9064], 8, 2, 128, page=64, kv=kv, seed=7)
    check(tsg, ctx, share(c, [0, 5], [8999 // 64 * 64]))


def test_long_own_parts(tsg, ctx):  # noqa: F811
    c = Case([2] * 3, [300, 7000, 3000], 4, 1, 64, page=64, seed=8)
    check(tsg, ctx, share(c, [0, 3], [192]))


@pytest.mark.parametrize("seqs", [1, 70, 300])
def test_many_sequences(tsg, ctx, seqs):  # noqa: F811
    """More sequences than a wave has lanes, and than runs are balanced over."""
    lengths = [100 + (37 * s) % 90 for s in range(seqs)]
    c = Case([1] * seqs, lengths, 2, 1, 32, seed=9)
    starts = list(range(0, seqs, 11)) + [seqs]
    check(tsg, ctx, share(c, starts, [64 + 32 * (g % 2) for g in range(len(starts) - 1)]))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_values_that_a_row_does_not_see(tsg, ctx, value, which):  # noqa: F811
    """In the prefix behind a short sequence's last token: the rows that see it take it, the
    others nothing."""
    c = Case([2] * 3, [300, 170, 310], 4, 2, 64, seed=10)
    share(c, [0, 3], [256])
    c.put(which, 0, 180, 1, value)
    want, tol = c.attention()
    got = call(tsg, ctx, c)
    ctx.synchronize()
    if which == "k" and value != value:
        want[[0, 1, 4, 5], 2:] = math.nan
    if which == "k" and value == value:  # NaN, or an infinite logit of either sign
        want[[0, 1, 4, 5], 2:] = got[[0, 1, 4, 5], 2:].double().cpu()
    if which == "v":
        assert not bool(torch.isfinite(got[[0, 1, 4, 5], 2:]).any())
        want[[0, 1, 4, 5], 2:] = got[[0, 1, 4, 5], 2:].double().cpu()
    assert_near(got, want, tol)


def test_far_apart_logits(tsg, ctx):  # noqa: F811
    """The own part's logits far above the prefix's and far below."""
    for size in (0.01, 60.0):
        c = Case([1] * 3, [200, 220, 240], 4, 2, 64, seed=11)
        share(c, [0, 3], [192])
        for s in range(3):
            for t in range(192, c.lengths[s]):
                i, j = c.slot(s, t)
                c.k[i, :, j] *= size
        check(tsg, ctx, c)


def test_equals_decode_and_itself(tsg, ctx):  # noqa: F811
    """The same bits each time; those of decode up to its own tolerance; without groups that share,
    decode's bits."""
    c = Case([4] * 6, [2000, 2100, 2050, 1990, 2300, 2001], 8, 2, 128, page=64, seed=12)
    share(c, [0, 6], [1984])
    d = c.to_device()
    got = [call(tsg, ctx, c, d=d) for _ in range(3)]
    ctx.synchronize()
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    decode = launch(tsg, ctx, c, "decode", d=d)
    want, tol = c.attention()
    assert_near(decode, got[0].double().cpu(), 2 * tol)
    d["shared"].zero_()
    alone = call(tsg, ctx, c, d=d)
    ctx.synchronize()
    assert torch.equal(alone, decode)


def test_strided_rows_and_in_place(tsg, ctx):  # noqa: F811
    c = Case([2, 2], [150, 131], 4, 2, 64, seed=13)
    share(c, [0, 2], [128])
    d = c.to_device()
    wide = torch.randn(4, 4 * 64 + 128, device="cuda").half()
    wide[:, 64:320] = d["q"].view(4, 256)
    d["q"] = wide[:, 64:320]
    before = wide.clone()
    call(tsg, ctx, c, d=d, out=d["q"])
    ctx.synchronize()
    want, tol = c.attention()
    assert_near(wide[:, 64:320].reshape(4, 4, 64), want, tol)
    assert torch.equal(wide[:, :64], before[:, :64]) and torch.equal(wide[:, 320:], before[:, 320:])


def test_tokens_outside_heads(tsg, ctx):  # noqa: F811
    c = Case([3, 3], [150, 231], 6, 3, 64, layout="tokens", seed=14)
    check(tsg, ctx, share(c, [0, 2], [144]))


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
def test_far_pages(tsg, ctx, kv):  # noqa: F811
    """Shared and own pages whose places pass 2^32 elements of the pool."""
    c = share(Case([2] * 4, [300, 311, 290, 333], 8, 2, 128, kv=kv, seed=10), [0, 4], [256])
    d = c.to_device()
    pages = c.k.shape[0]
    stride = -(-(2 ** 33) // pages) // 16 * 16
    shared = c.table[0, :16].long()  # at the pool's end, where their places are the farthest
    order = torch.cat([torch.tensor([i for i in range(pages) if i not in shared.tolist()]), shared])
    for name in ("k", "v"):
        x = d[name].view(torch.uint8 if kv == "e4m3" else torch.int16)
        far = torch.empty_strided(x.shape, (stride, *x.stride()[1:]), dtype=x.dtype, device="cuda")
        far.copy_(x[order.cuda()])
        d[name] = far.view(d[name].dtype)
    place = torch.empty(pages, dtype=torch.int32)
    place[order] = torch.arange(pages, dtype=torch.int32)
    d["table"] = place[c.table.long()].cuda()
    assert int(d["table"][0, 0]) * stride > 2 ** 32
    check(tsg, ctx, c, d=d)


def reported(tsg, ctx, text):  # noqa: F811
    with pytest.raises(tsg.TsgError) as e:
        ctx.synchronize()
    assert e.value.status == 1 and text in str(e.value)
    ctx.synchronize()


@pytest.mark.parametrize("starts", [[0, 3, 2], [0, 2, 5], [0, -1, 4], [7, 8, 9]])
def test_wrong_group_starts(tsg, ctx, starts):  # noqa: F811
    c = share(Case([1] * 4, [150, 160, 170, 180], 4, 2, 64, seed=15), [0, 2, 4], [128, 64])
    c.groups = starts
    got = call(tsg, ctx, c)
    reported(tsg, ctx, "group starts")
    assert bool(torch.isnan(got).all())


def test_bad_page_and_length(tsg, ctx):  # noqa: F811
    """The first sequence's bad page reaches its group, another's its own rows; a sequence longer
    than its table is NaN and harms no other."""
    base = share(Case([1] * 4, [150, 160, 170, 180], 4, 2, 64, seed=16), [0, 2, 4], [128, 64])
    want, tol = base.attention()
    for s, page, bad in ((0, 3, [0, 1]), (1, 9, [1]), (1, 3, []), (3, 10, [3])):
        d = base.to_device()
        d["table"][s, page] = 10 ** 6
        got = call(tsg, ctx, base, d=d)
        if bad:
            reported(tsg, ctx, "page table entry")
        else:
            ctx.synchronize()  # not its own: the first sequence's is read there
        fine = [i for i in range(4) if i not in bad]
        assert bool(torch.isnan(got[bad]).all())
        assert_near(got[fine], want[fine], tol[fine])
    for s in (0, 3):
        d = base.to_device()
        d["lengths"][s] = 10 ** 6
        got = call(tsg, ctx, base, d=d)
        reported(tsg, ctx, "longer than its page table")
        fine = [i for i in range(4) if i != s]
        assert bool(torch.isnan(got[s]).all())
        assert_near(got[fine], want[fine], tol[fine])


def test_call_refusals(tsg, ctx):  # noqa: F811
    c = share(Case([1] * 3, [150, 160, 170], 4, 2, 64, seed=17), [0, 3], [128])
    d = c.to_device()
    attn = plan(tsg, ctx, c)
    cache, out = attn.cache(d["k"], d["v"]), torch.full_like(d["q"], -77.0)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    good = attn.prefixes(ints(0, 3), ints(128))
    batch = attn.batch(d["table"], d["lengths"], 3)

    def refused(status, f, *args):
        with pytest.raises(tsg.TsgError) as e:
            f(*args)
        assert e.value.status == status

    refused(1, attn.prefixes, ints(0, 3), ints(128, 5))
    refused(1, attn.prefixes, ints(0), ints())
    refused(1, attn.prefixes, ints(0, 3).long(), ints(128))
    refused(1, attn.prefixes, ints(0, 3).cpu(), ints(128))
    refused(4, tsg.Attention(ctx, 4, 2, 64, 16, window=64).prefixes, ints(0, 3), ints(128))
    shared = attn.encode_decode_shared
    refused(1, shared, cache, attn.batch(d["table"], d["lengths"], 3, ints(0, 1, 2, 3)), good, d["q"], out)
    refused(1, shared, cache, batch, good, d["q"][:2], out)
    refused(1, shared, cache, batch, good, d["q"], d["q"].view(-1)[64:].as_strided((2, 256), (256, 1)))
    many = torch.zeros(27, 4, 64, dtype=torch.float16, device="cuda")
    refused(4, shared, cache, attn.batch(d["table"], d["lengths"], 27), good, many, many)
    lengths = torch.ones(2049, dtype=torch.int32, device="cuda")
    table = torch.zeros(2049, 1, dtype=torch.int32, device="cuda")
    many = torch.zeros(2049, 4, 64, dtype=torch.float16, device="cuda")
    refused(4, shared, cache, attn.batch(table, lengths, 2049), good, many, many)
    big = tsg.Attention(ctx, 32, 1, 64, 16)
    many = torch.zeros(2047, 32, 64, dtype=torch.float16, device="cuda")
    refused(4, big.encode_decode_shared, big.cache(d["k"][:, :1], d["v"][:, :1]),
            big.batch(table[:2047], lengths[:2047], 2047), good, many, many)
    torch.cuda.synchronize()
    assert bool((out == -77).all())
    ctx.synchronize()


def test_captured_and_replayed(tsg, ctx):  # noqa: F811
    """A graph replays with the groups, shared lengths, tables and lengths that its buffers then
    hold, beside eager calls of the plan in between."""
    make = [([0, 4], [128], [150, 160, 170, 180]), ([0, 2, 4], [64, 128], [200, 190, 180, 170]),
            ([1, 4], [192], [20, 200, 220, 230]), ([0, 4], [0], [150, 160, 170, 180])]
    cases = []
    for i, (starts, shared, lengths) in enumerate(make):
        if len(starts) == 2:  # two groups always
            starts, shared = starts + starts[-1:], shared + [0]
        c = Case([2] * 4, lengths, 4, 2, 64, seed=80 + i)
        if c.table.shape[1] < 15:
            c = Case([2] * 4, lengths[:3] + [230], 4, 2, 64, seed=80 + i)
        cases.append(share(c, starts, shared))
    d = cases[0].to_device()
    attn = plan(tsg, ctx, cases[0])
    out = call(tsg, ctx, cases[0], d=d, attn=attn)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(tsg, ctx, cases[0], d=d, attn=attn, out=out)
    for c in cases + cases[:1]:
        e = c.to_device()
        eager = call(tsg, ctx, c, d=e, attn=attn)
        for name in d:
            d[name].copy_(e[name])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        want, tol = c.attention()
        assert_near(out, want, tol)
    ctx.synchronize()


def test_on_two_streams(tsg, ctx):  # noqa: F811
    """Calls of one plan on streams in turn wait for each other: they share its scratch."""
    c = share(Case([1] * 4, [9000, 9100, 9200, 9300], 8, 2, 128, page=64, seed=90), [0, 4], [8960])
    d = c.to_device()
    attn = plan(tsg, ctx, c)
    want = call(tsg, ctx, c, d=d, attn=attn)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.full_like(want, -77.0) for _ in range(12)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        call(tsg, ctx, c, d=d, attn=attn, out=out, stream=streams[i % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)
    ctx.synchronize()
