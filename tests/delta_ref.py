"""The gated delta rule and its convolution in 64 bits, from their definitions, with what
the kernels may be off, and batches for their tests."""
from __future__ import annotations

import math

import torch

NONE = -1
HALF = 2.0 ** -11   # half a step of fp16
TINY = 2.0 ** -25   # half of its smallest
E24 = 2.0 ** -24    # half a step of fp32
CHUNK = 64


class Case:
    """Sequences of `rows` rows (a list) with their pools on the CPU (`to_device` moves them).
    `slots`: "apart" reads and writes slots of their own, "place" one slot a sequence, "fresh"
    starts without a state, "fork" lets all read one. `every`: the state behind each row."""

    def __init__(self, rows, key_heads, value_heads, key_dim, value_dim, width=4, seed=0, spare=0,
                 slots="apart", every=False, lead=0, gate=1.0, state=0.3, size=1.0, scale=None,
                 eps=1e-6, row_pad=0):
        self.rows, self.hk, self.hv, self.dk, self.dv = list(rows), key_heads, value_heads, key_dim, value_dim
        self.width, self.every, self.eps = width, every, eps
        self.scale = key_dim ** -0.5 if scale is None else scale
        self.channels = 2 * key_heads * key_dim + value_heads * value_dim
        g = torch.Generator().manual_seed(seed)
        n = len(self.rows)
        self.kept = self.rows[0] if every else 1
        self.starts = [lead]
        for r in self.rows:
            self.starts.append(self.starts[-1] + r)
        self.total = self.starts[-1] + spare
        self.uniform = len(set(self.rows)) == 1 and not spare and not lead
        pool = n * (1 + self.kept) + 2
        order = torch.randperm(pool, generator=g).tolist()
        self.ins = {"apart": order[:n], "place": order[:n], "fresh": [NONE] * n,
                    "fork": order[:1] * n}[slots]
        self.outs = order[n:n + n * self.kept]
        if slots == "place":
            for s in range(n):
                self.outs[(s + 1) * self.kept - 1] = order[s]
        rn = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
        m = max(1, self.total)
        self.x = (rn(m, self.channels + row_pad) * size).half()
        self.weight = (0.4 * rn(self.channels, width)).bfloat16()
        self.conv = rn(pool, width - 1, self.channels).half()
        x = rn(m, self.channels + row_pad) * 1.5
        self.qkv = (size * x * torch.sigmoid(x)).half()
        self.ab = (gate * rn(m, 2 * value_heads)).half()
        self.a_log = torch.log(1 + 15 * torch.rand(value_heads, generator=g))
        step = torch.exp(math.log(1e-3) + torch.rand(value_heads, generator=g) * math.log(100))
        self.dt_bias = torch.log(torch.expm1(step))
        self.s = state * rn(pool, value_heads, key_dim, value_dim)

    def split(self, t=None):
        t = self.qkv if t is None else t
        kw = self.hk * self.dk
        return (t[:, :kw], t[:, kw:2 * kw], t[:, 2 * kw:self.channels])

    def convolution(self):
        """Outputs, what they may be off, and the pool behind the call."""
        w = self.weight.double()
        out = torch.zeros(self.total, self.channels, dtype=torch.float64)
        tol, pool = torch.zeros_like(out), self.conv.clone()
        for s, n in enumerate(self.rows):
            a = self.starts[s]
            old = torch.zeros_like(self.conv[0]) if self.ins[s] == NONE else self.conv[self.ins[s]]
            x = torch.cat((old, self.x[a:a + n, :self.channels]))
            for i in range(n):
                prod = x[i:i + self.width].double() * w.T
                y, size = prod.sum(0), prod.abs().sum(0)
                out[a + i] = y * torch.sigmoid(y)
                # the products' sum in fp32 (silu's slope is at most 1.1), the exponential and
                # the reciprocal (2^-21 of the result; the exponent's own rounding is y * 2^-23
                # of it), the result's rounding
                tol[a + i] = 1.1 * (self.width + 1) * E24 * size + out[a + i].abs() * (
                    HALF + 2.0 ** -21 + y.abs() * 2.0 ** -22) + TINY
            for i in (range(n) if self.every else [n - 1]):
                slot = self.outs[s * self.kept + i] if self.every else self.outs[s]
                if slot != NONE:
                    pool[slot] = x[i + 1:i + self.width]
        return out, tol, pool

    def rule(self, chunked=False):
        """Outputs and states, row after row, each with what the kernels may be off.

        A row takes a state's column to (1 - beta k k^T) e S + beta k v, which does not lengthen
        a difference between two columns: so the errors' 2-norms of a column only add up. What
        one row adds, in fp32: the products over the key elements (dk + 16 roundings of at
        most |S|, the norm of k (dk / 2 + 8) in them and in k u twice, the decay's exponent
        (8 of its size), and the update's roundings. `chunked` bounds add what 64 rows at a
        time bring (see _chunk_error)."""
        q, k, v = (t.double() for t in self.split())
        n = q.shape[0]
        norm = lambda x: x / (x.square().sum(-1, keepdim=True) + self.eps).sqrt()  # noqa: E731
        each = self.hv // self.hk
        q = norm(q.reshape(n, self.hk, self.dk)).repeat_interleave(each, 1)
        k = norm(k.reshape(n, self.hk, self.dk)).repeat_interleave(each, 1)
        v = v.reshape(n, self.hv, self.dv)
        x = self.ab[:, :self.hv].double() + self.dt_bias.double()
        soft = x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))
        decay = -torch.exp(self.a_log.double()) * soft
        beta = torch.sigmoid(self.ab[:, self.hv:].double())
        out = torch.zeros(self.total, self.hv, self.dv, dtype=torch.float64)
        tol, pool = torch.zeros_like(out), self.s.double()
        pool_tol = torch.zeros_like(pool)
        dk = self.dk
        for i, rows in enumerate(self.rows):
            first = self.starts[i]
            m = torch.zeros(self.hv, dk, self.dv, dtype=torch.float64) \
                if self.ins[i] == NONE else self.s[self.ins[i]].double()
            err = torch.zeros(self.hv, self.dv, dtype=torch.float64)
            bound = m.abs().amax(1)
            for j in range(rows):
                r = first + j
                if chunked and j % CHUNK == 0:
                    span = slice(r, first + min(rows, j + CHUNK))
                    state_err, out_err, bound = self._chunk_error(
                        q[span], k[span], v[span], decay[span], beta[span], m, bound)
                e = decay[r].exp()
                before = m.norm(dim=1)
                m = m * e[:, None, None]
                u = beta[r][:, None] * (v[r] - (m * k[r][:, :, None]).sum(1))
                m = m + k[r][:, :, None] * u[:, None]
                g = decay[r].abs().clamp(max=100)[:, None]
                err = e[:, None] * err + E24 * (
                    before * e[:, None] * (3 * dk + 40 + 8 * g) + u.abs() * (dk + 40)
                    + beta[r][:, None] * v[r].abs() * 4)
                out[r] = self.scale * (m * q[r][:, :, None]).sum(1)
                reach = q[r].norm(dim=1)[:, None] * abs(self.scale)
                tol[r] = reach * (err + E24 * (2 * dk + 40 + 8 * g) * (before + u.abs())) \
                    + HALF * out[r].abs() + TINY
                if chunked:
                    tol[r] += abs(self.scale) * out_err[:, j % CHUNK]
                    if j % CHUNK == CHUNK - 1 or j == rows - 1:  # the chunk's state is formed
                        err = err + state_err
                if self.every:
                    self._put(pool, pool_tol, self.outs[i * self.kept + j], m, err)
            if not self.every:
                self._put(pool, pool_tol, self.outs[i], m, err)
        out[out.abs() >= 65520] *= math.inf  # what fp16 rounds to infinity
        return out, tol, pool, pool_tol

    @staticmethod
    def _put(pool, pool_tol, slot, m, err):
        if slot != NONE:
            pool[slot] = m
            pool_tol[slot] = (err[:, None] + E24 * m.abs()).expand_as(m)

    def _chunk_error(self, q, k, v, decay, beta, m, bound):
        """What a chunk of rows adds to the error of a state's columns (2-norm) and of its
        outputs, per head. With A_ij = beta_i e^(Gi - Gj) k_i.k_j below the diagonal, T = (1 + A)^-1
        and u = T r, r = beta (v - e^G K S): the products over the key elements are sums in
        fp32 of operands split in two halves of fp16 (2^-21 of the sizes' products); T is off
        by |T| |A| |T| times the roundings of A (dk + 24) and of the substitution (64 + 16);
        u by |T| times r's error, T's times |r| and its own sum's. The state's columns take K^T u,
        the outputs the weights e^(Gi - Gj) q_i.k_j, rounded to fp16 as u may be for them.

        Halves of fp16 end at steps of 2^-24, half of one off at most: S, r and u, scaled so
        that a bound on their column lies in 2^13 ... 2^14, by `step` = 2^-25 2^-14 2 bound
        (`before` for S, by the last chunk's bound); T and the weights, at 1024 for 1, by 2^-35;
        u times the rows' factors by step, times keys kept with norms under 4."""
        dk = self.dk
        q, k, v = q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1)
        beta, total = beta.T, decay.clamp(min=-1000).T.cumsum(1)
        apart = (total[:, :, None] - total[:, None, :]).clamp(max=0)
        lower = torch.exp(apart).tril()
        a = (beta[:, :, None] * lower * (k @ k.transpose(1, 2))).tril(-1)
        t = torch.linalg.inv(torch.eye(a.shape[1], dtype=torch.float64) + a)
        p = lower * (q @ k.transpose(1, 2))
        kn, qn = k.norm(dim=2), q.norm(dim=2)
        pa = beta[:, :, None] * lower * kn[:, :, None] * kn[:, None, :]
        sn = m.norm(dim=1)
        since = total.exp()
        r = beta[:, :, None] * (v - since[:, :, None] * (k @ m))
        split = 2.0 ** -21
        before = bound * 2.0 ** -38
        bound = 1.01 * dk ** 0.5 * m.abs().amax(1) + 65 * v.abs().amax(1)
        step = (bound * 2.0 ** -38)[:, None]
        low = torch.ones_like(lower).tril()
        ds = dk ** 0.5 * before[:, None]
        dr = beta[:, :, None] * (4 * E24 * v.abs() + ((dk + 32) * E24 + split)
                                 * since[:, :, None] * kn[:, :, None] * sn[:, None]
                                 + since[:, :, None] * kn[:, :, None] * ds) + step
        ta = t.abs()
        dt = ta @ (pa.tril(-1) * (dk + 24) * E24 + a.abs() * (80 * E24)) @ ta
        u = t @ r
        du = ta @ dr + dt @ r.abs() + (ta @ r.abs()) * (72 * E24 + 2 * split) \
            + (low @ r.abs()) * 2.0 ** -35
        until = torch.exp(total[:, -1:] - total)[:, :, None] * kn[:, :, None]
        state = (until * du + until * u.abs() * (72 * E24 + 2 * split + 32 * E24)).sum(1) \
            + sn * 8 * E24 + 4 * k.shape[1] * step[:, 0]
        outs = p.abs() @ du + (p.abs() @ u.abs()) * (2 * HALF + 72 * E24) + (low @ u.abs()) * 2.0 ** -35 \
            + (lower * qn[:, :, None] * kn[:, None, :] * (dk + 24) * E24) @ u.abs() \
            + ((dk + 32) * E24 + split) * (since * qn)[:, :, None] * sn[:, None] \
            + (since * qn)[:, :, None] * ds + p.abs().sum(2, keepdim=True) * step
        return state, outs, bound

    def to_device(self):
        ints = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
        d = {n: getattr(self, n).cuda()
             for n in ("x", "weight", "conv", "qkv", "ab", "a_log", "dt_bias", "s")}
        d.update(ins=ints(self.ins), outs=ints(self.outs), starts=ints(self.starts))
        d["conv_out"] = torch.full((max(1, self.total), self.channels), -77.0, dtype=torch.float16,
                                   device="cuda")
        d["out"] = torch.full((max(1, self.total), self.hv, self.dv), -77.0, dtype=torch.float16,
                              device="cuda")
        return d

    def plan(self, tsg, ctx):
        return tsg.GatedDelta(ctx, self.hk, self.hv, self.dk, self.dv, conv_width=self.width,
                              scale=self.scale, eps=self.eps)

    def launch(self, tsg, ctx, op, d=None, uniform=None, stream=None):
        """One call; returns its device buffers."""
        d = self.to_device() if d is None else d
        delta = self.plan(tsg, ctx)
        states = delta.states(d["s"], d["conv"])
        starts = None if (self.uniform if uniform is None else uniform) else d["starts"]
        batch = delta.batch(d["ins"], d["outs"], self.total, starts)
        if op == "conv":
            delta.encode_conv(states, batch, d["x"][:, :self.channels], d["weight"], d["conv_out"],
                              stream=stream)
            return d
        q, k, v = self.split(d["qkv"])
        a, b = d["ab"].split(self.hv, 1)
        args = (states, batch, q, k, v, a, b, tsg.DeltaGates(d["a_log"], d["dt_bias"]), d["out"])
        if op == "decode":
            delta.encode_decode(*args, stream=stream)
        else:
            d["scratch"] = torch.empty(delta.scratch_bytes(self.total, len(self.rows)),
                                       dtype=torch.uint8, device="cuda")
            delta.encode_prefill(*args, d["scratch"], stream=stream)
        return d

    def used(self):
        """Which rows are some sequence's."""
        mine = torch.zeros(self.total, dtype=torch.bool)
        mine[self.starts[0]:self.starts[-1]] = True
        return mine
