"""The token mixers of a hybrid decoder for serving, as cases that can be timed.

Layers that mix tokens by the gated delta rule make two calls between their projections,
with a recurrent state for every sequence in a slot of a pool:

  conv     the short causal convolution of the projected rows, with SiLU
           (GatedDelta.encode_conv)
  decode   the rule for 1..8 new tokens of each sequence (GatedDelta.encode_decode)
  prefill  the rule over a prompt's rows, or the next chunk's (GatedDelta.encode_prefill)

and the attention layers between them, where sequences of a batch begin alike:

  shared   attention of 1..8 new tokens of each sequence, the keys of the common prefix
           read once for all of a group's sequences (Attention.encode_decode_shared)

A case's `rows` are the new tokens of a sequence; `rows_lo` makes a batch ragged, `spare`
rows behind the last sequence belong to none. A state is read from one slot and written
to another, as for sequences that fork a prefix's; a sequence whose case says `fresh` (the
odd ones) starts without one. `every` keeps the state after each row, as a speculative
block needs that may be taken in part. For `shared`, `groups` of the sequences share
`shared` tokens (`shared_lo` of the first group), and each has up to `own` more, its new
rows among them.
"""
import functools
import math

import torch

own = False

HYBRID = {"key_heads": 16, "value_heads": 32, "key_dim": 128, "value_dim": 128, "width": 4}
WIDE = {"key_heads": 4, "value_heads": 4, "key_dim": 256, "value_dim": 512, "width": 4}
GROUP4 = {"q_heads": 32, "kv_heads": 8, "dim": 128}
HEADS = {"q_heads": 16, "kv_heads": 8, "dim": 256}
EPS = 1e-6
CHUNK = 64
NONE = -1  # no slot


def listed():
    return [
        # one decoded token: the smallest call
        {"name": "conv_token", "op": "conv", "seqs": 1, "rows": 1, **HYBRID},
        # prompts of a serving step, ragged, with padding behind the last
        {"name": "conv_prompts", "op": "conv", "seqs": 7, "rows": 3001, "rows_lo": 201,
         "spare": 37, "fresh": True, **HYBRID},
        # one decoded token: latency
        {"name": "delta_token", "op": "decode", "seqs": 1, "rows": 1, **HYBRID},
        # a serving batch: every sequence's state is read and written
        {"name": "delta_batch", "op": "decode", "seqs": 64, "rows": 1, **HYBRID},
        # speculative blocks of three, whose states are kept after each row
        {"name": "delta_block3", "op": "decode", "seqs": 24, "rows": 3, "every": True, **HYBRID},
        # a short chat turn after a longer one
        {"name": "delta_67", "op": "prefill", "seqs": 1, "rows": 67, **HYBRID},
        # prompts of a serving step, ragged, with padding behind the last
        {"name": "delta_prompts", "op": "prefill", "seqs": 7, "rows": 3001, "rows_lo": 201,
         "spare": 37, "fresh": True, **HYBRID},
        # a long prompt
        {"name": "delta_long", "op": "prefill", "seqs": 1, "rows": 8192, "fresh": True, **HYBRID},
        # a layer of few wide heads
        {"name": "delta_wide", "op": "prefill", "seqs": 2, "rows": 2011, **WIDE},
        # several answers to one conversation: latency
        {"name": "shared_few", "op": "shared", "seqs": 4, "rows": 1, "groups": 1, "shared": 2017,
         "own": 60, "own_lo": 7, "page": 16, "kv": "f16", **HEADS},
        # a serving batch behind one long system prompt
        {"name": "shared_batch", "op": "shared", "seqs": 64, "rows": 1, "groups": 1,
         "shared": 16011, "own": 501, "own_lo": 11, "page": 16, "kv": "f16", **GROUP4},
        # speculative blocks over an 8-bit cache, three prompts in the batch
        {"name": "shared_block5_e4m3", "op": "shared", "seqs": 30, "rows": 5, "groups": 3,
         "shared": 9001, "shared_lo": 4001, "own": 801, "own_lo": 40, "page": 64, "kv": "e4m3",
         **GROUP4},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("conv", "decode", "prefill", "prefill", "shared"))
    c = {"op": op}
    if op == "shared":
        kv_heads = rng.choice((1, 2, 4, 8))
        c.update(q_heads=kv_heads * rng.choice((1, 2, 3, 4, 8)), kv_heads=kv_heads,
                 dim=rng.choice((64, 80, 128, 128, 192, 256, 512)),
                 page=rng.choice((16, 32, 64, 128)), kv=rng.choice(("f16", "f16", "e4m3")),
                 rows=rng.choice((1, 1, 1, rng.randint(2, 8))))
        # what a token costs, against 32 query and 8 key heads of 128
        wide = max(1.0, c["q_heads"] * c["dim"] / 4096, c["kv_heads"] * c["dim"] / 1024)
        c["seqs"] = _log_int(rng, 1, int(64 / wide / (1 if c["rows"] == 1 else 2)) + 1)
        c["groups"] = rng.randint(1, max(1, c["seqs"] // 4))
        c["shared"] = _log_int(rng, 1, int(16000 / wide / (1 if c["rows"] == 1 else 2)))
        c["shared_lo"] = rng.randint(c["shared"] // 4, c["shared"])
        c["own"] = c["rows"] - 1 + _log_int(rng, 1, 500)
        c["own_lo"] = rng.randint(c["rows"], c["own"])
        return c
    c["key_heads"] = rng.choice((1, 2, 4, 8, 16))
    c["value_heads"] = c["key_heads"] * rng.choice((1, 2, 2, 3, 4))
    c["key_dim"] = rng.choice((48, 64, 80, 128, 128, 128, 192, 256))
    c["value_dim"] = rng.choice((64, 80, 128, 128, 128, 192, 256, 512))
    c["width"] = rng.choice((2, 3, 4, 4, 4, 8))
    # what a token costs, against the listed cases' heads
    wide = max(c["value_heads"] * c["key_dim"] * c["value_dim"] / (32 * 128 * 128),
               c["value_heads"] * c["value_dim"] / 4096, c["key_heads"] * c["key_dim"] / 2048)
    if op == "decode":
        c["rows"] = rng.choice((1, 1, 1, rng.randint(2, 8)))
        c["every"] = rng.random() < 0.4
        kept = c["rows"] if c["every"] else 1
        c["seqs"] = _log_int(rng, 1, max(1, min(512, int(128 / wide / (1 + kept)))))
    else:
        longest = 11000 if op == "conv" else 8192
        most = min(longest, int(longest / max(0.25, wide)))
        c["seqs"] = _log_int(rng, 1, max(1, int(16 / max(1.0, wide))))
        c["rows"] = _log_int(rng, 1, max(2, int(most / c["seqs"])))
        if c["seqs"] > 1:
            c["rows_lo"] = rng.randint(max(1, c["rows"] // 8), c["rows"])
            c["spare"] = rng.choice((0, rng.randint(1, 40)))
    c["fresh"] = rng.random() < 0.5
    return c


# ------------------------------------------------------------------ the batch

def _spread(lo, hi, n):
    """n whole numbers from lo to hi, both among them, in a mixed order."""
    if n == 1:
        return [hi]
    step = next(s for s in (5, 7, 11, 13, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _rows(case):
    return _spread(case.get("rows_lo", case["rows"]), case["rows"], case["seqs"])


def _starts(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def _channels(case):
    return 2 * case["key_heads"] * case["key_dim"] + case["value_heads"] * case["value_dim"]


def _has_state(case):
    return [not (case.get("fresh") and (s % 2 == 1 or case["seqs"] == 1))
            for s in range(case["seqs"])]


def _prefixes(case):
    """First sequence of every group (and the end), and the tokens that each group shares:
    whole pages."""
    n, page = case["groups"], case["page"]
    starts = [case["seqs"] * g // n for g in range(n + 1)]
    shared = _spread(case.get("shared_lo", case["shared"]), case["shared"], n)
    return starts, [t // page * page for t in shared]


def _lengths(case):
    starts, shared = _prefixes(case)
    more = _spread(case["own_lo"], case["own"], case["seqs"])
    return [shared[g] + more[s] for g in range(case["groups"])
            for s in range(starts[g], starts[g + 1])]


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_shared(case, g) if case["op"] == "shared" else _prepare_delta(case, g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_delta(case, g):
    counts = _rows(case)
    starts = _starts(counts)
    hk, hv, dk, dv = (case[n] for n in ("key_heads", "value_heads", "key_dim", "value_dim"))
    channels, width, seqs = _channels(case), case["width"], case["seqs"]
    rows = starts[-1] + case.get("spare", 0)

    def normal(*shape, dtype=torch.float16):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    kept = case["rows"] if case.get("every") else 1
    slots = seqs * (1 + kept) + 2
    order = torch.randperm(slots, generator=g, device="cuda").to(torch.int32)
    first = order[:seqs].clone()
    first[~torch.tensor(_has_state(case), device="cuda")] = NONE
    st = {"case": case, "rows": rows, "used": starts[-1], "starts": _ints(starts),
          "uniform": len(set(counts)) == 1 and not case.get("spare"), "most": max(counts),
          "in_slots": first, "out_slots": order[seqs:seqs * (1 + kept)].clone()}
    if case["op"] == "conv":
        st["x"] = normal(rows, channels)
        st["weight"] = (0.4 * normal(channels, width, dtype=torch.float32)).to(torch.bfloat16)
        st["conv_states"] = normal(slots, width - 1, channels)
        st["out"] = torch.zeros(rows, channels, device="cuda", dtype=torch.float16)
    else:
        # rows as the convolution leaves them, and the two gates' projections in one buffer
        x = normal(rows, channels, dtype=torch.float32)
        st["qkv"] = (1.5 * x * torch.sigmoid(1.5 * x)).half()
        st["ab"] = normal(rows, 2 * hv)
        uniform = torch.rand(2, hv, generator=g, device="cuda", dtype=torch.float64)
        # decays of 1..16 a unit of time, steps of 0.001..0.1
        st["a_log"] = torch.log(1 + 15 * uniform[0]).float()
        step = torch.exp(math.log(1e-3) + uniform[1] * math.log(100))
        st["dt_bias"] = torch.log(torch.expm1(step)).float()
        st["states"] = 0.3 * normal(slots, hv, dk, dv, dtype=torch.float32)
        st["out"] = torch.zeros(rows, hv, dv, device="cuda", dtype=torch.float16)
    if own:
        import tsugumi_amd as tsg
        delta = st["delta"] = tsg.GatedDelta(_context(), hk, hv, dk, dv, conv_width=width, eps=EPS)
        st["pool"] = delta.states(st.get("states"), st.get("conv_states"))
        st["batch"] = delta.batch(st["in_slots"], st["out_slots"], rows,
                                  None if st["uniform"] else st["starts"])
        if case["op"] != "conv":
            st["gates"] = tsg.DeltaGates(st["a_log"], st["dt_bias"])
        if case["op"] == "prefill":
            st["scratch"] = torch.empty(delta.scratch_bytes(rows, seqs), dtype=torch.uint8,
                                        device="cuda")
    return st


def _prepare_shared(case, g):
    lengths, (groups, shared) = _lengths(case), _prefixes(case)
    page, hq, hk, d = case["page"], case["q_heads"], case["kv_heads"], case["dim"]
    e4m3 = case["kv"] == "e4m3"
    seqs, rows = case["seqs"], case["rows"]
    per = -(-max(lengths) // page)
    # a page of a group's prefix is the same for its sequences, every other one its own
    ids, pages = [], 0
    for first, end, tokens in zip(groups, groups[1:], shared):
        common = list(range(pages, pages + tokens // page))
        pages += len(common)
        for s in range(first, end):
            mine = -(-lengths[s] // page) - len(common)
            ids.append(common + list(range(pages, pages + mine)))
            ids[-1] += [0] * (per - len(ids[-1]))
            pages += mine
    pages += 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    st = {"case": case, "table": order[torch.tensor(ids, device="cuda")],
          "lengths": _ints(lengths), "longest": max(lengths), "rows": seqs * rows,
          "groups": _ints(groups), "shared": _ints(shared),
          "k_scale": 1 / 64 if e4m3 else 1.0, "v_scale": 1 / 32 if e4m3 else 1.0}

    def pool(scale):
        t = torch.randn(pages, hk, page, d, generator=g, device="cuda", dtype=torch.float16)
        return (t / scale).to(torch.float8_e4m3fn) if e4m3 else t

    st["k_pages"], st["v_pages"] = pool(st["k_scale"]), pool(st["v_scale"])
    # slots that no token has been written to hold NaN, as recycled memory may
    slot = torch.arange(per * page, device="cuda").view(1, per, page)
    written = torch.zeros(pages, page, dtype=torch.int32, device="cuda")
    live = (slot < st["lengths"].view(-1, 1, 1)).to(torch.int32)
    written.index_put_((st["table"].long().flatten(),), live.flatten(0, 1), accumulate=True)
    where = (written == 0)[:, None, :, None]
    for name in ("k_pages", "v_pages"):
        st[name] = (st[name].view(torch.uint8).masked_fill_(where, 0x7F).view(torch.float8_e4m3fn)
                    if e4m3 else st[name].masked_fill_(where, math.nan))
    st["q"] = 1.5 * torch.randn(seqs * rows, hq, d, generator=g, device="cuda",
                                dtype=torch.float16)
    st["out"] = torch.zeros(seqs * rows, hq, d, device="cuda", dtype=torch.float16)
    if own:
        import tsugumi_amd as tsg
        attn = st["attn"] = tsg.Attention(_context(), hq, hk, d, page, kv_type=case["kv"],
                                          k_scale=st["k_scale"], v_scale=st["v_scale"])
        st["cache"] = attn.cache(st["k_pages"], st["v_pages"])
        st["batch"] = attn.batch(st["table"], st["lengths"], seqs * rows)
        st["prefixes"] = attn.prefixes(st["groups"], st["shared"])
    return st


@functools.lru_cache(maxsize=None)
def _context():
    import tsugumi_amd as tsg
    return tsg.Context(0)


# ------------------------------------------------------------------ one pass

def run(st):
    c = st["case"]
    if c["op"] == "conv":
        if own:
            st["delta"].encode_conv(st["pool"], st["batch"], st["x"], st["weight"], st["out"])
        else:
            _conv(st)
        return {"out": st["out"], "conv_states": st["conv_states"]}
    if c["op"] == "shared":
        if own:
            st["attn"].encode_decode_shared(st["cache"], st["batch"], st["prefixes"], st["q"],
                                            st["out"])
        else:
            _attention(st)
        return st["out"]
    kw, vw = c["key_heads"] * c["key_dim"], c["value_heads"] * c["value_dim"]
    q, k, v = st["qkv"].split((kw, kw, vw), dim=1)
    a, b = st["ab"].split(c["value_heads"], dim=1)
    if own and c["op"] == "decode":
        st["delta"].encode_decode(st["pool"], st["batch"], q, k, v, a, b, st["gates"], st["out"])
    elif own:
        st["delta"].encode_prefill(st["pool"], st["batch"], q, k, v, a, b, st["gates"], st["out"],
                                   st["scratch"])
    elif c["op"] == "decode":
        _recurrent(st, q, k, v, a, b)
    else:
        _chunked(st, q, k, v, a, b)
    return {"out": st["out"], "states": st["states"]}


def _loaded(pool, slots):
    """The slots' contents in 32 bits, zeros for a sequence that has none."""
    x = pool[slots.long().clamp(min=0)].float()
    return torch.where((slots == NONE).view(-1, *[1] * (x.dim() - 1)), 0.0, x)


def _turns(st, most):
    """Rows of every sequence's first `most` turns (clamped to the buffer), and which it has."""
    starts, turn = st["starts"].long(), torch.arange(most, device="cuda")
    rows = starts[:-1, None] + turn
    return rows.clamp(max=st["rows"] - 1), rows < starts[1:, None]


def _conv(st):
    width, n = st["case"]["width"], st["used"]
    rows, mine = _turns(st, st["most"])
    # every sequence's inputs behind those that its slot keeps
    x = torch.cat((_loaded(st["conv_states"], st["in_slots"]),
                   st["x"][rows].float().masked_fill_(~mine[..., None], 0.0)), 1)
    weight = st["weight"].float()
    y = torch.zeros_like(x[:, width - 1:])
    for j in range(width):
        y += x[:, j:j + st["most"]] * weight[:, j]
    st["out"][:n] = (y / (1 + torch.exp(-y)))[mine].half()
    count = mine.sum(1)
    last = count[:, None] + torch.arange(width - 1, device="cuda")
    kept = x.gather(1, last[..., None].expand(-1, -1, x.shape[2]))
    st["conv_states"][st["out_slots"].long()] = kept.half()


def _gates(st, a, b):
    """Logarithm of a row's decay, in 64 bits for its long sums, and its step's size."""
    x = a.double() + st["dt_bias"].double()
    soft = x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))
    return -torch.exp(st["a_log"].double()) * soft, 1 / (1 + torch.exp(-b.float()))


def _keys(st, q, k):
    """Normed queries and keys, for every value head."""
    c = st["case"]
    each = c["value_heads"] // c["key_heads"]

    def normed(x):
        x = x.float().unflatten(-1, (c["key_heads"], c["key_dim"]))
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)
        return x.repeat_interleave(each, -2)

    return normed(q) * c["key_dim"] ** -0.5, normed(k)


def _recurrent(st, q, k, v, a, b):
    """A row of every sequence at a time."""
    c, n = st["case"], st["case"]["rows"]
    s = _loaded(st["states"], st["in_slots"])
    q, k = _keys(st, q, k)
    decay, beta = _gates(st, a, b)
    decay = torch.exp(decay).float()
    v = v.float().unflatten(1, (c["value_heads"], c["value_dim"]))
    slots = st["out_slots"].long().view(c["seqs"], -1)
    for i in range(n):
        s = s * decay[i::n, :, None, None]
        u = (v[i::n] - (k[i::n, :, None] @ s)[:, :, 0]) * beta[i::n, :, None]
        s = s + k[i::n, :, :, None] * u[:, :, None]
        st["out"][i::n] = (q[i::n, :, None] @ s)[:, :, 0].half()
        if c.get("every"):
            st["states"][slots[:, i]] = s
    if not c.get("every"):
        st["states"][slots[:, 0]] = s


def _inverse(a):
    """(1 + a)^-1 of strictly lower triangles, by halves."""
    n = a.shape[-1]
    if n == 1:
        return torch.ones_like(a)
    h = n // 2
    top, low = _inverse(torch.stack((a[..., :h, :h], a[..., h:, h:])))
    corner = -(low @ a[..., h:, :h] @ top)
    return torch.cat((torch.cat((top, torch.zeros_like(top)), -1),
                      torch.cat((corner, low), -1)), -2)


def _chunked(st, q, k, v, a, b):
    """All chunks' triangles at once, then the state from chunk to chunk."""
    c = st["case"]
    chunks = -(-st["most"] // CHUNK)
    rows, mine = _turns(st, chunks * CHUNK)

    def cut(x):  # [sequence, chunk, head, row, ..]
        x = x[rows].masked_fill_(~mine.view(*mine.shape, *[1] * (x.dim() - 1)), 0.0)
        return x.unflatten(1, (chunks, CHUNK)).transpose(2, 3)

    q, k = (cut(x) for x in _keys(st, q, k))
    v = cut(v.float().unflatten(1, (c["value_heads"], c["value_dim"])))
    log_decay, beta = (cut(x) for x in _gates(st, a, b))
    total = log_decay.cumsum(-1)
    apart = (total[..., :, None] - total[..., None, :]).clamp(max=0)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda").tril()
    weight = torch.where(lower, torch.exp(apart).float(), 0.0)
    tri = _inverse((beta[..., None] * weight * (k @ k.transpose(-1, -2))).tril(-1))
    scores = weight * (q @ k.transpose(-1, -2))
    since = torch.exp(total).float()[..., None]
    until = torch.exp(total[..., -1:] - total).float()[..., None]
    s = _loaded(st["states"], st["in_slots"])
    out = []
    for i in range(chunks):
        u = tri[:, i] @ (beta[:, i, ..., None] * (v[:, i] - since[:, i] * (k[:, i] @ s)))
        out.append(since[:, i] * (q[:, i] @ s) + scores[:, i] @ u)
        s = since[:, i, :, -1:] * s + (until[:, i] * k[:, i]).transpose(-1, -2) @ u
    out = torch.stack(out, 1).transpose(2, 3).flatten(1, 2)
    st["out"][:st["used"]] = out[mine].half()
    st["states"][st["out_slots"].long()] = s


def _attention(st):
    """Every sequence's rows against all of its pages, padded to the longest."""
    c = st["case"]
    n, hk, d, lengths = c["rows"], c["kv_heads"], c["dim"], st["lengths"].long()
    group = c["q_heads"] // hk
    key = torch.arange(st["longest"], device="cuda")

    def tokens(pages, scale):
        x = pages.view(torch.uint8)[st["table"].long()].view(pages.dtype) if c["kv"] == "e4m3" \
            else pages[st["table"].long()]
        x = x.float().transpose(2, 3).flatten(1, 2)[:, :st["longest"]] * scale
        x.masked_fill_((key >= lengths[:, None])[..., None, None], 0.0)
        return x.transpose(1, 2)

    q = st["q"].float().view(-1, n, hk, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    keys = tokens(st["k_pages"], st["k_scale"])
    scores = (q @ keys.transpose(-1, -2) * d ** -0.5).unflatten(2, (group, n))
    del keys
    at = (lengths - n)[:, None] + torch.arange(n, device="cuda")
    scores.masked_fill_((key > at[..., None])[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    values = tokens(st["v_pages"], st["v_scale"])
    out = (scores.flatten(2, 3) @ values).unflatten(2, (group, n)) / total
    st["out"].copy_(out.permute(0, 3, 1, 2, 4).reshape(st["out"].shape))


# ------------------------------------------------------------------ work

def work(case):
    if case["op"] == "shared":
        (groups, shared), lengths = _prefixes(case), _lengths(case)
        hq, hk, d, n = case["q_heads"], case["kv_heads"], case["dim"], case["rows"]
        cell = 1 if case["kv"] == "e4m3" else 2
        keys = sum(lengths) - sum(t * (b - a - 1) for t, a, b in zip(shared, groups, groups[1:]))
        seen = sum(n * t - n * (n - 1) // 2 for t in lengths)
        return {"bytes": 4 * case["seqs"] * n * hq * d + keys * 2 * hk * d * cell,
                "flops": 4 * d * hq * seen}
    n, channels, hv = sum(_rows(case)), _channels(case), case["value_heads"]
    kept = case["rows"] if case.get("every") else 1
    read, written = sum(_has_state(case)), case["seqs"] * kept
    if case["op"] == "conv":
        w = case["width"]
        return {"bytes": 4 * n * channels + 2 * w * channels
                + 2 * (w - 1) * channels * (read + written), "flops": n * channels * (2 * w + 4)}
    cells = hv * case["key_dim"] * case["value_dim"]
    return {"bytes": 2 * n * (channels + 2 * hv + hv * case["value_dim"]) + 8 * hv
            + 4 * cells * (read + written), "flops": 7 * n * cells}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    """The definitions in 64 bits, a sequence at a time."""
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    return {"conv": _exact_conv, "shared": _exact_shared}.get(case["op"], _exact_delta)(case, st)


def _exact_conv(case, st):
    out, pool, w = st["out"].double(), st["conv_states"].double(), case["width"]
    kernel = st["weight"].double().T
    starts = _starts(_rows(case))
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        slot = int(st["in_slots"][s])
        before = torch.zeros_like(pool[0]) if slot == NONE else st["conv_states"][slot].double()
        x = torch.cat((before, st["x"][a:b].double()))
        y = (x.unfold(0, w, 1).transpose(1, 2) * kernel).sum(1)
        out[a:b] = y * torch.sigmoid(y)
        pool[int(st["out_slots"][s])] = x[len(x) - (w - 1):]
    return {"out": out, "conv_states": pool}


def _exact_delta(case, st):
    """One token after another, on the state itself."""
    hk, hv, dk, dv = (case[n] for n in ("key_heads", "value_heads", "key_dim", "value_dim"))
    out, pool = st["out"].double(), st["states"].double()
    n = st["rows"]
    qkv = st["qkv"].double()
    q, k = qkv[:, :2 * hk * dk].view(n, 2, hk, dk).unbind(1)
    v = qkv[:, 2 * hk * dk:].view(n, hv, dv)
    q, k = ((x / torch.sqrt(x.square().sum(2, keepdim=True) + EPS))
            .repeat_interleave(hv // hk, 1) for x in (q, k))
    rate = torch.nn.functional.softplus(st["ab"][:, :hv].double() + st["dt_bias"].double())
    decay = torch.exp(-torch.exp(st["a_log"].double()) * rate)
    beta = torch.sigmoid(st["ab"][:, hv:].double())
    starts = _starts(_rows(case))
    slots = st["out_slots"].view(case["seqs"], -1).tolist()
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        slot = int(st["in_slots"][s])
        m = torch.zeros(hv, dk, dv, dtype=torch.float64, device="cuda") if slot == NONE \
            else st["states"][slot].double()
        for r in range(a, b):
            m = m * decay[r, :, None, None]
            seen = (m * k[r, :, :, None]).sum(1)
            m = m + k[r, :, :, None] * (beta[r, :, None] * (v[r] - seen))[:, None]
            out[r] = (m * q[r, :, :, None]).sum(1) / math.sqrt(dk)
            if case.get("every"):
                pool[slots[s][r - a]] = m
        if not case.get("every"):
            pool[slots[s][0]] = m
    return {"out": out, "states": pool}


def _exact_shared(case, st):
    page, hk, d, n = case["page"], case["kv_heads"], case["dim"], case["rows"]
    group = case["q_heads"] // hk
    out = torch.zeros(st["rows"], case["q_heads"], d, device="cuda", dtype=torch.float64)
    for s, length in enumerate(_lengths(case)):
        ids = st["table"][s, :-(-length // page)].long()
        hidden = torch.arange(length, device="cuda") > torch.arange(
            length - n, length, device="cuda")[:, None]
        for h in range(hk):
            k = st["k_pages"][ids, h].reshape(-1, d)[:length].double() * st["k_scale"]
            v = st["v_pages"][ids, h].reshape(-1, d)[:length].double() * st["v_scale"]
            q = st["q"][s * n:s * n + n, h * group:h * group + group].double()
            logit = (q.transpose(0, 1) @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            out[s * n:s * n + n, h * group:h * group + group] = \
                (torch.softmax(logit, -1) @ v).transpose(0, 1)
    return out
