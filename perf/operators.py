"""The attention half of a decoder layer, as cases that can be timed.

Between the Q, K and V projections and the O projection a decoder makes two calls
for a layer, over a paged key/value cache:

  append   the norms of the query and key heads and the position rotation, with the
           keys and values going into the cache (Attention.encode_append)
  decode   attention of 1..8 new tokens of each sequence (Attention.encode_decode)
  prefill  attention of a prompt's rows, or of the next chunk of one
           (Attention.encode_prefill)

A case's `rows` are the new tokens of a sequence, `length` the tokens it has in the
cache with them; `length_lo` and `rows_lo` make a batch ragged. `spare` rows behind
the last sequence belong to no sequence. Head layouts, windows and sinks are the
layer's; `kv` is the cache's type. Keys, values and queries are N(0, 1) as the heads'
norms leave them; slots of the cache that no token has been written to hold NaN for
the attention, as recycled memory may. Pages lie in the pool in a random order.
"""
import functools
import math

import torch

own = False

HEADS = {"q_heads": 16, "kv_heads": 8, "dim": 256}       # queries of 4096, keys of 2048
GROUP4 = {"q_heads": 32, "kv_heads": 8, "dim": 128}
GLOBAL = {"q_heads": 16, "kv_heads": 2, "dim": 512}
FULL = {"window": 0, "sinks": 0}
LOCAL = {"window": 1024, "sinks": 0}


def listed():
    return [
        # one decoded token: the smallest call
        {"name": "append_token", "op": "append", "seqs": 1, "rows": 1, "length": 1001, "page": 16,
         "kv": "f16", "rot": 256, "pairs": "half", **HEADS},
        # speculative blocks of five in a batch, 8-bit cache, a quarter of each head rotated
        {"name": "append_block5_e4m3", "op": "append", "seqs": 32, "rows": 5, "length": 8011,
         "length_lo": 40, "page": 64, "kv": "e4m3", "rot": 64, "pairs": "interleaved", **HEADS},
        # prompts of a serving step, ragged, with padding behind the last
        {"name": "append_prompts", "op": "append", "seqs": 7, "rows": 3001, "rows_lo": 201,
         "length": 3001, "length_lo": 201, "spare": 37, "page": 16, "kv": "f16", "rot": 128,
         "pairs": "half", **GROUP4},
        # one decoded token on a sliding-window layer: latency
        {"name": "decode_token", "op": "decode", "seqs": 1, "rows": 1, "length": 1001, "page": 16,
         "kv": "f16", **HEADS, **LOCAL},
        # one long conversation: the length has to be split over the card
        {"name": "decode_long", "op": "decode", "seqs": 1, "rows": 1, "length": 131001, "page": 64,
         "kv": "f16", **GROUP4, **FULL},
        # a serving batch of ragged lengths over an 8-bit cache
        {"name": "decode_batch_e4m3", "op": "decode", "seqs": 64, "rows": 1, "length": 16001,
         "length_lo": 301, "page": 64, "kv": "e4m3", **GROUP4, **FULL},
        # speculative blocks on a global layer of wide heads
        {"name": "decode_block5", "op": "decode", "seqs": 6, "rows": 5, "length": 6007,
         "length_lo": 77, "page": 16, "kv": "f16", **GLOBAL, **FULL},
        # a short chat turn after a longer one
        {"name": "prefill_67", "op": "prefill", "seqs": 1, "rows": 67, "length": 967, "page": 16,
         "kv": "f16", **HEADS, **LOCAL},
        # the next chunk of a long document over an 8-bit cache
        {"name": "prefill_chunk_e4m3", "op": "prefill", "seqs": 1, "rows": 512, "length": 16896,
         "page": 64, "kv": "e4m3", **GROUP4, **FULL},
        # ragged prompts on a sliding-window layer whose first tokens stay visible
        {"name": "prefill_window", "op": "prefill", "seqs": 3, "rows": 4501, "rows_lo": 901,
         "length": 4501, "length_lo": 901, "spare": 19, "page": 16, "kv": "f16", **HEADS,
         "window": 1024, "sinks": 4},
        # a long prompt on a global layer
        {"name": "prefill_long", "op": "prefill", "seqs": 1, "rows": 8192, "length": 8192,
         "page": 64, "kv": "f16", **GROUP4, **FULL},
        # a prompt on a global layer of wide heads
        {"name": "prefill_wide", "op": "prefill", "seqs": 1, "rows": 2011, "length": 2011,
         "page": 16, "kv": "f16", **GLOBAL, **FULL},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "decode", "prefill"))
    kv_heads = rng.choice((1, 2, 4, 8))
    q_heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    dim = rng.choice((64, 80, 96, 128, 128, 192, 256, 256, 512))
    c = {"op": op, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
         "page": rng.choice((16, 32, 64, 128)), "kv": rng.choice(("f16", "f16", "e4m3"))}
    # what a token costs, against 32 query and 8 key heads of 128
    wide = max(1.0, q_heads * dim / 4096, kv_heads * dim / 1024)
    if op == "append":
        c["rot"] = rng.choice((dim, dim // 2 // 16 * 16, dim // 4 // 16 * 16))
        c["pairs"] = rng.choice(("half", "half", "interleaved"))
        c["seqs"] = _log_int(rng, 1, 64)
        c["rows"] = _log_int(rng, 1, max(1, int(11000 / wide / c["seqs"])))
        c["length"] = c["rows"] + rng.choice((0, _log_int(rng, 1, 20000 // c["seqs"] + 1)))
    else:
        local = rng.random() < 0.5
        c["window"] = _log_int(rng, 16, 2048) if local else 0
        c["sinks"] = rng.choice((0, 4, rng.randint(1, 100))) if local else 0
        c["seqs"] = _log_int(rng, 1, 64 if op == "decode" else 8)
        if op == "decode":
            c["rows"] = rng.choice((1, 1, 1, rng.randint(2, 8)))
            most = 500000 / wide / c["seqs"] / (1 if c["rows"] == 1 else 2)
            c["length"] = max(c["rows"], _log_int(rng, 1, int(min(131072, most))))
        else:
            most = 4600 / math.sqrt(wide * c["seqs"])
            c["rows"] = _log_int(rng, 1, max(2, int(most)))
            c["length"] = c["rows"] + rng.choice((0, 0, _log_int(rng, 1, max(2, int(most)))))
    if c["seqs"] > 1:
        c["length_lo"] = rng.randint(c["length"] // 8, c["length"])
        if op != "decode":
            c["rows_lo"] = rng.randint(max(1, c["rows"] // 8), c["rows"])
            c["length_lo"] = max(c["length_lo"], c["rows_lo"])
            c["spare"] = rng.choice((0, rng.randint(1, 40)))
    return c


# ------------------------------------------------------------------ the batch

def _spread(lo, hi, n):
    """n whole numbers from lo to hi, both among them, in a mixed order."""
    if n == 1:
        return [hi]
    step = next(s for s in (5, 7, 11, 13, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _batch(case):
    """Every sequence's new rows and its length in the cache."""
    n = case["seqs"]
    rows = _spread(case.get("rows_lo", case["rows"]), case["rows"], n)
    lengths = _spread(case.get("length_lo", case["length"]), case["length"], n)
    return rows, [max(r, length) for r, length in zip(rows, lengths)]


def _visible(case, rows, length):
    """Pairs of a new row and a key that it sees, and the keys that any row sees."""
    window, sinks = case["window"], case["sinks"]
    pairs = 0
    for p in range(length - rows, length):
        if not window or p < window:
            pairs += p + 1
        else:
            pairs += window + min(sinks, p + 1 - window)
    first = max(0, length - rows - window + 1) if window else 0
    return pairs, length - first + min(sinks, first)


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, lengths = _batch(case)
    page, hq, hk, d = case["page"], case["q_heads"], case["kv_heads"], case["dim"]
    e4m3 = case["kv"] == "e4m3"
    per = -(-max(lengths) // page)
    pages = len(rows) * per + 3
    order = torch.randperm(pages, generator=g, device="cuda")[:len(rows) * per]
    table = order.view(len(rows), per).to(torch.int32)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    total = starts[-1] + case.get("spare", 0)
    st = {"case": case, "table": table,
          "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
          "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
          "uniform": len(set(rows)) == 1 and not case.get("spare"),
          "rows": total, "used": starts[-1], "most": max(rows), "longest": max(lengths),
          "k_scale": 1 / 64 if e4m3 else 1.0, "v_scale": 1 / 32 if e4m3 else 1.0}

    def half(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)

    def pool(scale):
        t = half(pages, hk, page, d)
        return (t / scale).to(torch.float8_e4m3fn) if e4m3 else t

    st["k_pages"], st["v_pages"] = pool(st["k_scale"]), pool(st["v_scale"])
    if case["op"] == "append":
        # the rows of one fused projection: a query part, a key part, a value part
        st["qkv"] = half(total, (hq + 2 * hk) * d) * 1.7
        st["q_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
        st["k_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
        exponent = torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64)
        st["inv_freq"] = (1e6 ** (-exponent / max(1, case["rot"]))).to(torch.float32)
        st["q_out"] = torch.zeros(total, hq, d, device="cuda", dtype=torch.float16)
    else:
        slot = torch.arange(per * page, device="cuda").view(1, per, page)
        unwritten = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        unwritten[table.long()] = slot >= st["lengths"].view(-1, 1, 1)
        where = unwritten[:, None, :, None]
        for name in ("k_pages", "v_pages"):
            st[name] = (st[name].view(torch.uint8).masked_fill_(where, 0x7F)
                        .view(torch.float8_e4m3fn) if e4m3
                        else st[name].masked_fill_(where, math.nan))
        st["q"] = half(total, hq, d) * 1.5
        st["out"] = torch.zeros(total, hq, d, device="cuda", dtype=torch.float16)
    if own:
        import tsugumi_amd as tsg
        st["attn"] = tsg.Attention(_context(), hq, hk, d, page, kv_type=case["kv"],
                                   window=case.get("window", 0), sinks=case.get("sinks", 0),
                                   k_scale=st["k_scale"], v_scale=st["v_scale"])
        st["cache"] = st["attn"].cache(st["k_pages"], st["v_pages"])
        st["batch"] = st["attn"].batch(table, st["lengths"], total,
                                       None if st["uniform"] else st["starts"])
        if case["op"] == "append":
            st["rope"] = tsg.HeadNormRope(st["q_weight"], st["k_weight"], st["inv_freq"],
                                          interleaved=case["pairs"] == "interleaved", eps=1e-6)
    return st


@functools.lru_cache(maxsize=None)
def _context():
    import tsugumi_amd as tsg
    return tsg.Context(0)


# ------------------------------------------------------------------ one pass

def run(st):
    c = st["case"]
    if c["op"] == "append":
        hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
        q, k, v = st["qkv"].split((hq * d, hk * d, hk * d), dim=1)
        if own:
            st["attn"].encode_append(st["cache"], st["batch"], q, k, v, st["rope"], st["q_out"])
        else:
            _append(st, q, k, v)
        return {"q": st["q_out"], "k": st["k_pages"], "v": st["v_pages"]}
    if own:
        call = st["attn"].encode_decode if c["op"] == "decode" else st["attn"].encode_prefill
        call(st["cache"], st["batch"], st["q"], st["out"])
    else:
        _attention(st)
    return st["out"]


def _row_places(st):
    """Sequence, turn in it and position of every row that a sequence has."""
    row, starts = torch.arange(st["used"], device="cuda"), st["starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, row - starts[seq], st["lengths"].long()[seq] - starts[seq + 1] + row


def _append(st, q, k, v):
    c = st["case"]
    d, rot = c["dim"], c["rot"]
    n = st["used"]
    seq, _, pos = _row_places(st)

    def normed(x, weight):
        x = x[:n].view(n, -1, d).float()
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()

    # far positions: the angle in 64 bits
    angle = pos.double()[:, None, None] * st["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def rotated(x):
        if c["pairs"] == "half":
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), -1)
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((turned, x[..., rot:]), -1)

    st["q_out"][:n] = rotated(normed(q, st["q_weight"])).half()
    page, slot = st["table"].long()[seq, pos // c["page"]], pos % c["page"]
    for pages, x, scale in ((st["k_pages"], rotated(normed(k, st["k_weight"])), st["k_scale"]),
                            (st["v_pages"], v[:n].view(n, -1, d).float(), st["v_scale"])):
        if c["kv"] == "e4m3":
            x = (x / scale).clamp(-448, 448).to(torch.float8_e4m3fn)
            pages.view(torch.uint8)[page, :, slot] = x.view(torch.uint8)
        else:
            pages[page, :, slot] = x.half()


def _attention(st):
    """Every sequence's rows against all of its pages, padded to the longest."""
    c = st["case"]
    hk, d, group = c["kv_heads"], c["dim"], c["q_heads"] // c["kv_heads"]
    n, lengths, starts = st["most"], st["lengths"].long(), st["starts"].long()
    count = starts[1:] - starts[:-1]
    turn = torch.arange(n, device="cuda")
    rows = (starts[:-1, None] + turn).clamp(max=st["rows"] - 1)
    pos = (lengths - count)[:, None] + turn

    def tokens(pages, scale):
        x = pages.view(torch.uint8)[st["table"].long()].view(pages.dtype) if c["kv"] == "e4m3" \
            else pages[st["table"].long()]
        x = x.float().transpose(2, 3).flatten(1, 2)[:, :st["longest"]]
        written = torch.arange(x.shape[1], device="cuda") < lengths[:, None]
        return torch.where(written[..., None, None], x * scale, 0.0).transpose(1, 2)

    keys, values = tokens(st["k_pages"], st["k_scale"]), tokens(st["v_pages"], st["v_scale"])
    q = st["q"][rows].float().view(-1, n, hk, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = q @ keys.transpose(-1, -2) * d ** -0.5
    key = torch.arange(st["longest"], device="cuda")
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= (pos[..., None] - key < c["window"]) | (key < c["sinks"])
    scores = scores.view(len(lengths), hk, group, n, -1)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=-1e30)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ values).view(len(lengths), hk, group, n, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)
    seq, at, _ = _row_places(st)
    st["out"][:st["used"]] = out[seq, at].half()


# ------------------------------------------------------------------ work

def work(case):
    rows, lengths = _batch(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    cell = 1 if case["kv"] == "e4m3" else 2
    n = sum(rows)
    if case["op"] == "append":
        read = n * (hq + 2 * hk) * d * 2 + case["rot"] * 2 + 4 * d
        return {"bytes": read + n * hq * d * 2 + n * 2 * hk * d * cell,
                "flops": n * (hq + hk) * (4 * d + 3 * case["rot"])}
    seen = [_visible(case, r, length) for r, length in zip(rows, lengths)]
    return {"bytes": 2 * n * hq * d * 2 + sum(k for _, k in seen) * 2 * hk * d * cell,
            "flops": 4 * d * hq * sum(p for p, _ in seen)}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    """The definition in 64 bits, a sequence (and a head) at a time."""
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    rows, lengths = _batch(case)
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    group, first = case["q_heads"] // hk, 0
    if case["op"] == "append":
        hq, rot = case["q_heads"], case["rot"]
        q_out = st["q_out"].double()
        pages = {"k": st["k_pages"].double(), "v": st["v_pages"].double()}
        for s, (n, length) in enumerate(zip(rows, lengths)):
            x = st["qkv"][first:first + n].double().view(n, hq + 2 * hk, d)
            rms = x.pow(2).mean(2, keepdim=True).add(1e-6).sqrt()
            at = torch.arange(length - n, length, device="cuda")
            turn = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64),
                               at.double()[:, None] * st["inv_freq"].double())[:, None]

            def turned(y):
                y = y.clone()
                if case["pairs"] == "half":
                    re, im = slice(0, rot // 2), slice(rot // 2, rot)
                else:
                    re, im = slice(0, rot, 2), slice(1, rot, 2)
                z = torch.complex(y[..., re].contiguous(), y[..., im].contiguous()) * turn
                y[..., re], y[..., im] = z.real, z.imag
                return y

            q_out[first:first + n] = turned(x[:, :hq] / rms[:, :hq] * st["q_weight"].double())
            heads = slice(hq, hq + hk)
            new = {"k": turned(x[:, heads] / rms[:, heads] * st["k_weight"].double())
                   / st["k_scale"], "v": x[:, hq + hk:] / st["v_scale"]}
            for name, y in new.items():
                if case["kv"] == "e4m3":
                    y = y.clamp(-448, 448)
                pages[name].index_put_((st["table"].long()[s, at // page], torch.arange(
                    hk, device="cuda")[:, None], at % page), y.transpose(0, 1))
            first += n
        return {"q": q_out, **pages}
    out = torch.zeros(st["rows"], case["q_heads"], d, device="cuda", dtype=torch.float64)
    for s, (n, length) in enumerate(zip(rows, lengths)):
        ids = st["table"][s].long()
        at = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None]
        hidden = key > at
        if case["window"]:
            hidden |= (key <= at - case["window"]) & (key >= case["sinks"])
        for h in range(hk):
            k = st["k_pages"][ids, h].reshape(-1, d)[:length].double() * st["k_scale"]
            v = st["v_pages"][ids, h].reshape(-1, d)[:length].double() * st["v_scale"]
            for i in range(h * group, h * group + group):
                logit = st["q"][first:first + n, i].double() @ k.T / math.sqrt(d)
                p = torch.softmax(logit.masked_fill_(hidden, -math.inf), 1)
                out[first:first + n, i] = p @ v
        first += n
    return out
