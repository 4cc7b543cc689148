"""64-bit references of the paged HCA cache's operators and pools to run them on.

``Pool`` lays sequences out in shuffled pages whose unused bytes are a sentinel;
the references go token by token and sequence by sequence in float64 numpy.
"""

from __future__ import annotations

import numpy as np
import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
STORE = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SENTINEL = 0x5b


def unit(x):
    return x / np.maximum(np.linalg.norm(x, axis=-1, keepdims=True), 1e-12)


def quantise(x, store):
    """Rows of numbers (numpy) -> (torch codes, uint8 scale codes or None)."""
    x = torch.from_numpy(np.ascontiguousarray(x, np.float64))
    if store == "bf16":
        return x.to(torch.bfloat16), None
    amax = x.abs().amax(-1)
    e = torch.ceil(torch.log2(amax.clamp_min(1e-300) / TOP[store]))
    e = torch.where(amax < 2.0 ** -100, torch.zeros_like(e), e)
    y = (x * torch.exp2(-e)[..., None]).float()
    codes = y.round().to(torch.int8) if store == "int8" else y.to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def values(codes, scales):
    """Codes (and scale codes) -> float64 numpy."""
    x = codes.float().cpu().double().numpy()
    if scales is None:
        return x
    s = scales.cpu().numpy().astype(np.int64)
    return np.where((s == 255)[..., None], np.nan, np.ldexp(x, (s - 127)[..., None]))


def half_step(x, scales, store):
    """Largest rounding error of values x held in a format (numpy; scales: 2^e)."""
    x = np.abs(x)
    if store == "bf16":
        return x * 2.0 ** -8
    if store == "int8":
        return np.broadcast_to(0.5 * scales[..., None], x.shape)
    return np.maximum(x * 2.0 ** -4, 2.0 ** -10 * scales[..., None])


class Pool:
    """Pages for S sequences (slot i holds sequence i), filled with the sentinel."""

    def __init__(self, S, nbp, nrp, page, c, store, seed=0, spare=3, device="cuda", high=0):
        g = np.random.default_rng(seed)
        self.S, self.nbp, self.nrp, self.page, self.c, self.store = S, nbp, nrp, page, c, store
        n = S * (nbp + nrp) + spare
        es = 2 if store == "bf16" else 1
        raw = torch.full((n + high, page, c * es), SENTINEL, dtype=torch.uint8, device=device)
        self.rows = raw.view(STORE[store])
        self.scales = None if store == "bf16" else \
            torch.full((n + high, page), 126, dtype=torch.uint8, device=device)
        order = high + g.permutation(n)[:S * (nbp + nrp)].reshape(S, nbp + nrp)
        ints = lambda a: torch.tensor(np.ascontiguousarray(a), dtype=torch.int32, device=device)  # noqa: E731
        self.blocks, self.ring = ints(order[:, :nbp]), ints(order[:, nbp:])
        self.state = torch.full((S, 3, c), 7.0, device=device)
        self.device = device

    @property
    def cap(self):
        return self.nrp * self.page

    def _at(self, table, slot, index):
        index = torch.as_tensor(np.atleast_1d(index), device=self.device).long()
        return table[slot].long()[index // self.page], index % self.page

    def put(self, table, slot, index, x):
        """Rows x (numpy) quantised into a slot's rows `index`."""
        if len(np.atleast_1d(index)) == 0:
            return
        codes, sc = quantise(x, self.store)
        pg, ln = self._at(table, slot, index)
        es = 2 if self.store == "bf16" else 1
        raw = self.rows.view(torch.uint8).view(-1, self.page, self.c * es)
        raw[pg, ln] = codes.contiguous().view(torch.uint8).view(-1, self.c * es).to(self.device)
        if sc is not None:
            self.scales[pg, ln] = sc.to(self.device)

    def get(self, table, slot, index):
        if len(np.atleast_1d(index)) == 0:
            return np.zeros((0, self.c))
        pg, ln = self._at(table, slot, index)
        raw = self.rows.view(torch.uint8).view(self.rows.shape[0], self.page, -1)[pg, ln]
        return values(raw.view(STORE[self.store]), None if self.scales is None else self.scales[pg, ln])

    def get_scale(self, table, slot, index):
        if self.scales is None:
            return np.ones(len(np.atleast_1d(index)))
        pg, ln = self._at(table, slot, index)
        return np.exp2(self.scales[pg, ln].cpu().numpy().astype(np.float64) - 127)


def step(lens, ctx, slots, device="cuda"):
    """(slots, cu, ctx) on the device and the packed offsets."""
    cu = np.concatenate([[0], np.cumsum(lens)])
    ints = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=device)  # noqa: E731
    return ints(slots), ints(cu), ints(ctx), cu


def attention(pool, q, lens, ctx, slots, *, m2, win, sink, scale, normalize_q=True):
    """float64 outputs and, per element, sum_j p_j |k_j| (what weight errors can move)."""
    outs, mags, at = [], [], 0
    for slot, n, x in zip(slots, lens, ctx):
        qs = q[at:at + n].astype(np.float64)
        at += n
        if normalize_q:
            qs = unit(qs)
        nb = min((x + n) // m2, pool.nbp * pool.page)
        kb = pool.get(pool.blocks, slot, np.arange(nb))
        w0 = max(0, x - win + 1) if win else x + n
        pos = np.arange(w0, x + n)
        kw = pool.get(pool.ring, slot, pos % pool.cap) if win and n else np.zeros((0, pool.c))
        keys = np.concatenate([kb, kw])
        for i in range(n):
            t = x + i
            ok = np.concatenate([(np.arange(nb) + 1) * m2 <= t + 1, (pos <= t) & (pos > t - win)])
            k = keys[ok]
            s = scale * qs[i] @ k.T
            if not len(k):
                outs.append(np.zeros_like(qs[i]))
                mags.append(np.zeros_like(qs[i]))
                continue
            extra = np.full((len(s), 0), 0.0) if sink is None else sink.astype(np.float64)[:, None]
            m = np.max(np.concatenate([s, extra], 1), 1, keepdims=True)
            e = np.exp(s - m)
            p = e / (e.sum(1, keepdims=True) + np.exp(extra - m).sum(1, keepdims=True))
            outs.append(p @ k)
            mags.append(p @ np.abs(k))
    shape = (0,) + q.shape[1:]
    return (np.stack(outs), np.stack(mags)) if outs else (np.zeros(shape), np.zeros(shape))


def append(C, Z, B_pos, lens, ctx, slots, state, *, m2, normalize=True):
    """What a chunk leaves, in float64: {(slot, block): row}, {(slot, position): window
    row}, {slot: [3, c] sums of the open block}."""
    rows, wins, sums, at = {}, {}, {}, 0
    for slot, n, x in zip(slots, lens, ctx):
        m = l = a = None
        if x % m2:
            m, l, a = (v.astype(np.float64) for v in state[slot])
        for i in range(n):
            p = x + i
            c, z = C[at + i].astype(np.float64), Z[at + i].astype(np.float64) + B_pos[p % m2]
            wins[slot, p] = unit(c) if normalize else c
            if p % m2 == 0:
                m, l, a = np.full_like(z, -np.inf), np.zeros_like(z), np.zeros_like(z)
            mn = np.maximum(m, z)
            safe = np.where(np.isfinite(mn), mn, 0.0)
            f, e = np.exp(m - safe), np.exp(z - safe)
            l, a, m = l * f + e, a * f + np.where(e > 0, e * c, 0.0), mn
            if (p + 1) % m2 == 0:
                r = np.where(l > 0, a / np.where(l > 0, l, 1.0), 0.0)
                rows[slot, p // m2] = unit(r) if normalize else r
        if n and (x + n) % m2:
            sums[slot] = np.stack([m, l, a])
        at += n
    return rows, wins, sums
