"""A hybrid decoder's token mixers together: a prompt run once, its pages shared and its state
read by every sequence that goes on from it, and their tokens as one captured step."""
from __future__ import annotations

import pytest
import torch

from tests import attention_ref, delta_ref
from tests.attention_ref import assert_near
from tests.test_gpu_attention import ctx, tsg  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

SEQS, PROMPT, PAGE, STEPS = 4, 70, 16, 4
HK, HV, DK, DV = 2, 4, 64, 48           # the rule's layer
QH, KH, DIM = 8, 2, 64                  # the attention's


def half(g, *shape):
    return torch.randn(*shape, generator=g).half()


def test_sequences_from_one_prompt(tsg, ctx):  # noqa: F811
    g = torch.Generator().manual_seed(101)
    ints = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    device = lambda *shape: torch.zeros(*shape, dtype=torch.float16, device="cuda")  # noqa: E731

    # slot 0 holds the prompt's state, 1..4 the sequences'; pages 0..4 the prompt's tokens
    layer = delta_ref.Case([PROMPT], HK, HV, DK, DV, seed=102)
    delta = layer.plan(tsg, ctx)
    weight = layer.weight.cuda()
    s = torch.full((SEQS + 1, HV, DK, DV), float("nan"), device="cuda")
    conv = torch.full((SEQS + 1, layer.width - 1, layer.channels), float("nan"), device="cuda").half()
    states, gates = delta.states(s, conv), tsg.DeltaGates(layer.a_log.cuda(), layer.dt_bias.cuda())
    attn = tsg.Attention(ctx, QH, KH, DIM, PAGE)
    full = PROMPT // PAGE
    table = torch.tensor([[*range(full), *(full + 2 * i + j for j in (0, 1))] for i in range(SEQS)],
                         dtype=torch.int32)
    k, v = device(2, full + 2 * SEQS, KH, PAGE, DIM)
    cache, rope = attn.cache(k, v), tsg.HeadNormRope()
    tokens = torch.arange(full * PAGE, PROMPT) % PAGE

    def rule_is_right(now, x, ab, mixed, out, prefill):
        now.x, now.ab, now.qkv = x.cpu(), ab.cpu(), mixed.cpu()
        now.weight, now.a_log, now.dt_bias = layer.weight, layer.a_log, layer.dt_bias
        want, tol, pool = now.convolution()
        assert_near(mixed, want, tol)
        assert torch.equal(conv.cpu()[now.outs], pool[now.outs])
        want, tol, pool, pool_tol = now.rule(prefill)
        assert_near(out, want, tol)
        assert_near(s[now.outs], pool[now.outs], pool_tol[now.outs])

    # the prompt, once
    x, ab = half(g, PROMPT, layer.channels).cuda(), half(g, PROMPT, 2 * HV).cuda()
    mixed, out = device(PROMPT, layer.channels), device(PROMPT, HV, DV)
    batch = delta.batch(ints([-1]), ints([0]), PROMPT)
    scratch = torch.empty(delta.scratch_bytes(PROMPT, 1), dtype=torch.uint8, device="cuda")
    delta.encode_conv(states, batch, x, weight, mixed)
    delta.encode_prefill(states, batch, *layer.split(mixed), *ab.split(HV, 1), gates, out, scratch)
    q, kv = half(g, PROMPT, QH, DIM).cuda(), half(g, 2, PROMPT, KH, DIM).cuda()
    attn.encode_append(cache, attn.batch(table[:1].cuda(), ints([PROMPT]), PROMPT), q, kv[0], kv[1],
                       rope, q)
    ctx.synchronize()
    layer.ins, layer.outs = [delta_ref.NONE], [0]
    layer.conv, layer.s = conv.cpu(), s.cpu()
    rule_is_right(layer, x, ab, mixed, out, True)
    for t in (k, v):  # what the prompt has of its last page is every sequence's own
        for i in range(1, SEQS):
            t[int(table[i, full]), :, tokens] = t[int(table[0, full]), :, tokens]

    # a token of every sequence: both layers' calls as one graph
    x, ab = device(SEQS, layer.channels), device(SEQS, 2 * HV)
    mixed, out = device(SEQS, layer.channels), device(SEQS, HV, DV)
    q, kv, q_out, seen = device(SEQS, QH, DIM), device(2, SEQS, KH, DIM), device(SEQS, QH, DIM), device(SEQS, QH, DIM)
    ins, outs, lengths = ints([0] * SEQS), ints(range(1, SEQS + 1)), ints([PROMPT] * SEQS)
    batch = delta.batch(ins, outs, SEQS)
    pages = attn.batch(table.cuda(), lengths, SEQS)
    shared = attn.prefixes(ints([0, SEQS]), ints([full * PAGE]))

    def step():
        lengths.add_(1)
        delta.encode_conv(states, batch, x, weight, mixed)
        delta.encode_decode(states, batch, *layer.split(mixed), *ab.split(HV, 1), gates, out)
        attn.encode_append(cache, pages, q, kv[0], kv[1], rope, q_out)
        attn.encode_decode_shared(cache, pages, shared, q_out, seen)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for turn in range(STEPS):
        for t in (x, ab, q, kv):
            t.copy_(half(g, *t.shape))
        now = delta_ref.Case([1] * SEQS, HK, HV, DK, DV)
        now.ins, now.outs = ins.tolist(), outs.tolist()
        now.conv, now.s = conv.cpu(), s.cpu()
        graph.replay()
        ctx.synchronize()
        torch.cuda.synchronize()
        rule_is_right(now, x, ab, mixed, out, False)
        length = PROMPT + turn + 1
        assert lengths.tolist() == [length] * SEQS
        c = attention_ref.Case([1] * SEQS, [length] * SEQS, QH, KH, DIM, PAGE)
        c.table, c.k, c.v, c.q = table, k.cpu(), v.cpu(), q_out.cpu()
        for i in range(SEQS):
            assert torch.equal(c.tokens("v", i)[-1], kv[1, i].cpu().double())
        want, tol = c.attention()
        assert_near(seen, want, tol)
        ins.copy_(outs)  # from now on in place
