"""The serving operators of the paged HCA cache and of 4-bit weights, as cases to time and compare.

``attention``  a chunk of new tokens per sequence over the pages of its cache: compressed rows,
               window rows and a sink in one softmax (single tokens are chunks of one)
``append``     a chunk's tokens into the cache: compression of the blocks they end, the window
               rows, both quantised as they are written, and the open block's running sums
``read``       cached rows back out of their pages, packed, as numbers
``w4``         few rows times a matrix of 4-bit weights with group scales

Sizes are those of ``bench.py`` (16 heads of 128, blocks of 128 tokens, a window of 128, d_model
2048, contexts of 128K tokens and more) and of the default ``HybridConfig`` (4 heads of 64,
blocks of 64, a window of 16); ``draw`` spreads further cases over the same ranges.

The plain forms below are elementary torch in 32 bits over the same page tables; ``exact`` goes
sequence by sequence in 64 bits.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_STORE = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_TOP = {"e4m3": 448.0, "int8": 127.0}
_D64 = torch.float64


def _chunk(name, kind, S, ctx, length, ragged, m2, win, nh, c, page, store, dtype):
    """S sequences of about ctx cached tokens, chunks of up to `length` new ones."""
    return {"name": name, "kind": kind, "S": S, "ctx": ctx, "len": length, "ragged": ragged,
            "m2": m2, "win": win, "nh": nh, "c": c, "page": page, "store": store, "dtype": dtype}


def _read(name, S, n, c, page, store, dtype):
    return {"name": name, "kind": "read", "S": S, "rows": n, "c": c, "page": page,
            "store": store, "dtype": dtype}


def _w4(name, M, N, K, group, zeros, residual, dtype):
    return {"name": name, "kind": "w4", "M": M, "N": N, "K": K, "group": group, "zeros": zeros,
            "residual": residual, "dtype": dtype}


def listed():
    return [
        # the next token of one short conversation: latency
        _chunk("attention_token", "attention", 1, 5003, 1, False, 128, 128, 16, 128, 16, "bf16", "bf16"),
        # one token for each of a batch of unequal contexts of up to 1M tokens
        _chunk("attention_batch", "attention", 128, 1048576, 1, True, 128, 128, 16, 128, 64, "e4m3", "bf16"),
        # guesses to verify, one to eight tokens a sequence, at the default configuration's heads
        _chunk("attention_verify", "attention", 37, 8190, 8, True, 64, 16, 4, 64, 32, "int8", "fp16"),
        # the next pieces of eight long prompts
        _chunk("attention_prefill", "attention", 8, 131072, 2048, True, 128, 128, 16, 128, 64, "e4m3", "bf16"),
        # one token into the cache of each sequence of a batch
        _chunk("append_batch", "append", 64, 131072, 1, True, 128, 128, 16, 128, 64, "e4m3", "bf16"),
        # the pieces of sixteen prompts
        _chunk("append_prefill", "append", 16, 131072, 2048, True, 128, 128, 16, 128, 64, "e4m3", "bf16"),
        # short prompts at the default configuration's sizes, 16-bit pages
        _chunk("append_short", "append", 9, 0, 333, True, 64, 16, 4, 64, 16, "bf16", "fp16"),
        # a batch of caches of 1M tokens out of their pages, to move or to keep
        _read("read_back", 16, 8192, 128, 64, "e4m3", "bf16"),
        # a few short ones, for a computation in fp32
        _read("read_short", 5, 211, 64, 16, "int8", "fp32"),
        # the query projection of one token
        _w4("w4_token", 1, 2048, 2048, 128, False, False, "bf16"),
        # the output projection of a small batch with the residual stream added, odd sizes
        _w4("w4_rows", 5, 2072, 1056, 32, True, True, "fp16"),
        # a large matrix for sixteen sequences
        _w4("w4_large", 16, 16384, 8192, 128, True, False, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "append", "read", "w4"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "w4":
        M = _log_int(rng, 1, 16)
        K = 32 * _log_int(rng, 4, 256)
        N = _log_int(rng, 40, 16384)
        group = rng.choice([32, 64, 128])
        K -= K % group
        return _anon(_w4("", M, N, K, group, rng.random() < 0.5, rng.random() < 0.4, dtype))
    c = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    store = rng.choice(["bf16", "e4m3", "e4m3", "int8"])
    if kind == "read":
        n = _log_int(rng, 3, 8192)
        S = _log_int(rng, 1, max(1, min(64, 131072 // n)))
        return _anon(_read("", S, n, c, page, store, rng.choice(["bf16", "fp16", "fp32"])))
    m2 = rng.choice([16, 64, 128])
    win = rng.choice([1, 16, 77, 128])
    nh = rng.choice([1, 4, 6, 16, 16])
    ctx = rng.choice([0, _log_int(rng, 1, 8192 * m2), _log_int(rng, 1, 8192 * m2)])
    if kind == "append":
        # an 8-bit row is compared as float8 values; int8 codes have no such type
        store = rng.choice(["bf16", "e4m3"])
        length = _log_int(rng, 1, 2048)
        S = _log_int(rng, 1, max(1, min(64, 32768 // length, (1 << 17) * m2 // (ctx + 1))))
    else:
        length = rng.choice([1, _log_int(rng, 2, 16), _log_int(rng, 2, 2048)])
        if length > 16:
            ctx //= 8
        cost = length * nh * (ctx // m2 + length // m2 + length + win)
        S = _log_int(rng, 1, max(1, min(128, (1 << 28) // cost, (1 << 20) * m2 // (ctx + 1))))
    return _anon(_chunk("", kind, S, ctx, length, rng.random() < 0.7, m2, win, nh, c, page, store, dtype))


def _anon(case):
    case.pop("name")
    return case


# --------------------------------------------------------------------------- inputs

def _lens(case):
    """Chunk lengths and cached tokens of the sequences: by the case alone."""
    S, ctx, n = case["S"], case["ctx"], case["len"]
    if not case["ragged"]:
        return [n] * S, [ctx] * S
    lens = [n - (i * 7919) % max(1, n - n // 8) if i else n for i in range(S)]
    return lens, [ctx - (i * 104729) % (ctx // 2 + 1) for i in range(S)]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-12)


def _quantise(x, store):
    """Rows of fp32 values -> (codes, E8M0 codes of the rows' scales or None)."""
    if store == "bf16":
        return x.to(torch.bfloat16), None
    amax = x.abs().amax(-1)
    frac, expo = torch.frexp(amax)  # amax = frac 2^expo, frac in [1/2, 1)
    tfrac, texpo = math.frexp(_TOP[store])
    e = expo - texpo + (frac > tfrac)
    e = torch.where(amax < 2.0 ** -100, torch.zeros_like(e), e)
    v = torch.ldexp(x, -e[..., None])
    codes = v.round().to(torch.int8) if store == "int8" else v.to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, scales):
    """Codes and E8M0 codes -> fp32 values."""
    x = codes.float()
    return x if scales is None else torch.ldexp(x, scales.to(torch.int32)[..., None] - 127)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool(g, n_pages, page, c, store):
    """Pages of unit rows, as a cache holds them, in random order of use."""
    x = _unit(torch.randn(n_pages, page, c, device="cuda", generator=g))
    rows, scales = _quantise(x, store)
    return rows, scales, torch.randperm(n_pages, device="cuda", generator=g).int()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    dt = _DTYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    st = dict(case)
    if kind == "w4":
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        st["x"] = rnd(M, K).to(dt)
        st["packed"] = torch.randint(0, 256, (N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
        # steps of a group: spread about those of a matrix of variance 1 / K
        st["scales"] = (0.37 * K ** -0.5 * (0.5 + torch.rand(K // G, N, device="cuda", generator=g))).to(dt)
        st["zeros"] = (torch.randint(4, 12, (K // G, N), device="cuda", generator=g, dtype=torch.uint8)
                       if case["zeros"] else None)
        st["residual"] = rnd(M, N).to(dt) if case["residual"] else None
        return st
    S, page, c, store = case["S"], case["page"], case["c"], case["store"]
    if kind == "read":
        n = case["rows"]
        counts = [n - (i * 31) % max(1, n // 3) for i in range(S)]
        first = [(i * 5) % 9 for i in range(S)]
        nbp = -(-(n + 8) // page)
        st["rows_"], st["scales"], order = _pool(g, S * nbp, page, c, store)
        st["table"] = order.view(S, nbp)
        st["slots"] = torch.randperm(S, device="cuda", generator=g).int()
        cu = [0]
        for k in counts:
            cu.append(cu[-1] + k)
        st |= {"cu": _ints(cu), "first": _ints(first), "total": cu[-1], "out_dtype": dt}
        return st
    lens, ctx = _lens(case)
    m2, win = case["m2"], case["win"]
    nbp = -(-max(1, max((x + n) // m2 for x, n in zip(ctx, lens))) // page)
    nrp = -(-(win + case["len"] - 1) // page)
    st["rows_"], st["scales"], order = _pool(g, S * (nbp + nrp), page, c, store)
    order = order.view(S, nbp + nrp)
    st["blocks"], st["ring"] = order[:, :nbp].contiguous(), order[:, nbp:].contiguous()
    st["slots"] = torch.randperm(S, device="cuda", generator=g).int()
    cu = [0]
    for k in lens:
        cu.append(cu[-1] + k)
    st |= {"cu": _ints(cu), "ctx_": _ints(ctx), "total": cu[-1], "max_ctx": max(ctx)}
    if kind == "attention":
        st["q"] = rnd(cu[-1], case["nh"], c).to(dt)
        st["sink"] = rnd(case["nh"])
        # scores of unit vectors, spread as a trained temperature spreads them
        st["scale"] = c ** 0.5
        return st
    both = rnd(cu[-1], 2 * c).to(dt)  # the two projections, one output
    st["C"], st["Z"] = both[:, :c], both[:, c:]
    st["B_pos"] = 0.02 * rnd(m2, c)
    # an open block's sums, as the tokens before the chunk leave them
    m, l = 1.0 + rnd(S, c).abs(), 1.0 + rnd(S, c).abs()
    st["state"] = torch.stack([m, l, 0.3 * l * rnd(S, c)], 1)
    return st


# --------------------------------------------------------------------------- one pass

def run(s):
    kind = s["kind"]
    if own:
        return _own(s)
    return {"attention": _plain_attention, "append": _plain_append, "read": _plain_read,
            "w4": _plain_w4}[kind](s)


def _own(s):
    import os
    import sys
    pkg = os.path.abspath("kda-csa-hca-fusion_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import kch
    kind = s["kind"]
    if kind == "w4":
        return kch.linear_w4(s["x"], s["packed"], s["scales"], s["zeros"], residual=s["residual"])
    if kind == "read":
        return kch.paged_read(s["rows_"], s["scales"], s["table"], s["slots"], s["cu"],
                              total=s["total"], first=s["first"], dtype=s["out_dtype"])
    if kind == "attention":
        return kch.hca_paged_attention(
            s["q"], s["rows_"], s["scales"], s["blocks"], s["ring"], s["slots"], s["cu"], s["ctx_"],
            m2=s["m2"], sliding_window=s["win"], max_len=s["len"], max_ctx=s["max_ctx"],
            sink_logits=s["sink"], scale=s["scale"])
    kch.hca_paged_append(
        s["C"], s["Z"], s["B_pos"], s["rows_"], s["scales"], s["state"], s["blocks"], s["ring"],
        s["slots"], s["cu"], s["ctx_"], m2=s["m2"], max_len=s["len"])
    return _append_outputs(s)


def _append_outputs(s):
    out = {"rows": s["rows_"], "state": s["state"]}
    if s["scales"] is not None:
        out["scales"] = s["scales"].view(torch.float8_e8m0fnu)
    return out


def _owner(s):
    """Of every packed token: its sequence, its place in the chunk, its position."""
    cu = s["cu"].long()
    at = torch.arange(s["total"], device=cu.device)
    seq = torch.searchsorted(cu, at, right=True) - 1
    i = at - cu[seq]
    return seq, i, s["ctx_"].long()[seq] + i


def _plain_attention(s):
    S, L, m2, win, page, c, nh = s["S"], s["len"], s["m2"], s["win"], s["page"], s["c"], s["nh"]
    seq, i, _ = _owner(s)
    q = _unit(s["q"].float())
    qp = q.new_zeros(S, L, nh, c)
    qp[seq, i] = q
    slot = s["slots"].long()
    ctx = s["ctx_"].long()
    # every sequence's compressed rows, then its window rows from position ctx - win + 1 on
    nb = max(1, (s["max_ctx"] + L) // m2)
    b = torch.arange(nb, device=q.device)
    bp = s["blocks"].long()[slot][:, b // page]
    pos = ctx[:, None] - win + 1 + torch.arange(win + L - 1, device=q.device)
    R = s["ring"].shape[1] * page
    r = pos % R
    rp = torch.gather(s["ring"].long()[slot], 1, r // page)
    pages = torch.cat([bp, rp], 1)
    lines = torch.cat([(b % page).expand(S, nb), r % page], 1)
    keys = _values(s["rows_"][pages, lines], None if s["scales"] is None else s["scales"][pages, lines])
    t = ctx[:, None] + torch.arange(L, device=q.device)
    seen_b = b < ((t + 1) // m2)[..., None]
    seen_w = (pos[:, None] >= 0) & (pos[:, None] <= t[..., None]) & (pos[:, None] > t[..., None] - win)
    seen = torch.cat([seen_b, seen_w], -1)[:, :, None]
    sc = torch.matmul(qp.view(S, L * nh, c), keys.transpose(1, 2).contiguous()).view(S, L, nh, -1)
    sc = torch.where(seen, s["scale"] * sc, float("-inf"))
    top = sc.amax(-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(sc - top)
    den = e.sum(-1, keepdim=True) + torch.exp(s["sink"].view(nh, 1) - top)
    out = torch.matmul((e / den).view(S, L * nh, -1), keys).view(S, L, nh, c)
    return out[seq, i].to(s["q"].dtype)


def _put(s, table, index, x, where):
    """Rows x (fp32) quantised into their pages where `where` holds."""
    page = s["page"]
    codes, e8 = _quantise(x, s["store"])
    pages = torch.gather(table, -1, (index // page).clamp(0, table.shape[-1] - 1))
    at = (pages * page + index % page)[where]
    flat = s["rows_"].view(-1, s["c"])
    if s["store"] == "e4m3":
        flat.view(torch.uint8)[at] = codes.view(torch.uint8)[where]
    else:
        flat[at] = codes[where]
    if e8 is not None:
        s["scales"].view(-1)[at] = e8[where]


def _plain_append(s):
    S, L, m2, c = s["S"], s["len"], s["m2"], s["c"]
    seq, i, pos = _owner(s)
    slot, ctx, lens = s["slots"].long(), s["ctx_"].long(), s["cu"].long().diff()
    C, Z = s["C"].float(), s["Z"].float()
    # window rows
    R = s["ring"].shape[1] * s["page"]
    ring = s["ring"].long()[slot]
    _put(s, ring[seq], (pos % R)[:, None], _unit(C)[:, None], torch.ones_like(pos, dtype=torch.bool)[:, None])
    # blocks: [S, blocks the chunk touches, m2, c], the open block's sums as one more entry
    nb = (L + m2 - 2) // m2 + 1
    j = pos % m2
    k = pos // m2 - (ctx // m2)[seq]
    z = C.new_full((S, nb, m2, c), float("-inf"))
    v = C.new_zeros(S, nb, m2, c)
    z[seq, k, j] = Z + s["B_pos"][j]
    v[seq, k, j] = C
    old = s["state"][slot]
    carry = torch.zeros(S, nb, dtype=torch.bool, device=C.device)
    carry[:, 0] = ctx % m2 > 0
    om = torch.where(carry[..., None], old[:, None, 0], float("-inf"))
    top = torch.maximum(z.amax(2), om)
    safe = top.clamp_min(-3e38)
    e = torch.exp(z - safe[:, :, None])
    w = torch.exp(om - safe)
    l = e.sum(2) + w * torch.where(carry[..., None], old[:, None, 1], 0.0)
    a = (e * v).sum(2) + w * torch.where(carry[..., None], old[:, None, 2], 0.0)
    row = torch.where(l > 0, a / l.clamp_min(1e-38), 0.0)
    b = ctx[:, None] // m2 + torch.arange(nb, device=C.device)
    ends = (b + 1) * m2 <= (ctx + lens)[:, None]
    _put(s, s["blocks"].long()[slot], b, _unit(row), ends)
    last = (ctx + lens) // m2 - ctx // m2
    open_ = (ctx + lens) % m2 > 0
    sel = last.clamp_max(nb - 1)
    one = torch.arange(S, device=C.device)
    new = torch.stack([top[one, sel], l[one, sel], a[one, sel]], 1)
    keep = open_ & (lens > 0)
    s["state"][slot[keep]] = new[keep]
    return _append_outputs(s)


def _plain_read(s):
    page = s["page"]
    cu = s["cu"].long()
    at = torch.arange(s["total"], device=cu.device)
    seq = torch.searchsorted(cu, at, right=True) - 1
    r = (s["first"].long()[seq] + at - cu[seq]) % (s["table"].shape[1] * page)
    pages = s["table"].long()[s["slots"].long()[seq], r // page]
    x = _values(s["rows_"][pages, r % page], None if s["scales"] is None else s["scales"][pages, r % page])
    return x.to(s["out_dtype"])


def _plain_w4(s):
    N, K, G = s["N"], s["K"], s["group"]
    p = s["packed"]
    codes = torch.stack([p & 15, p >> 4], -1).view(N, K // G, G).float()
    z = 8.0 if s["zeros"] is None else s["zeros"].t().float()[..., None]
    W = ((codes - z) * s["scales"].t().float()[..., None]).view(N, K)
    y = s["x"].float() @ W.t()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


# --------------------------------------------------------------------------- bytes and operations

def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if kind == "w4":
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        b = N * K / 2 + N * K / G * (3 if case["zeros"] else 2) + 2 * M * (K + N)
        return {"bytes": b + (2 * M * N if case["residual"] else 0), "flops": 2.0 * M * N * K}
    c = case["c"]
    row = 2 * c if case["store"] == "bf16" else c + 1
    if kind == "read":
        n = sum(case["rows"] - (i * 31) % max(1, case["rows"] // 3) for i in range(case["S"]))
        return {"bytes": n * (row + c * size), "flops": 0.0}
    lens, ctx = _lens(case)
    m2, win = case["m2"], case["win"]
    if kind == "append":
        n = sum(lens)
        ends = sum((x + k) // m2 - x // m2 for x, k in zip(ctx, lens))
        return {"bytes": n * (2 * c * size + row) + ends * row + 24 * c * case["S"] + 4 * m2 * c,
                "flops": 10.0 * n * c}
    nbytes = flops = 0.0
    for x, k in zip(ctx, lens):
        nbytes += ((x + k) // m2 + min(win + k - 1, x + k)) * row + 2 * k * case["nh"] * c * size
        lo, hi = x + 1, x + k  # tokens that a query has seen, itself among them
        blocks = (sum(t // m2 for t in range(lo, hi + 1)))
        near = sum(min(t, win) for t in range(lo, hi + 1))
        flops += 4.0 * case["nh"] * c * (blocks + near)
    return {"bytes": nbytes, "flops": flops}


# --------------------------------------------------------------------------- 64 bits

def _row64(s, page, line):
    x = s["rows_"][page, line].to(_D64)
    if s["scales"] is None:
        return x
    return x * torch.pow(torch.tensor(2.0, dtype=_D64, device=x.device),
                         s["scales"][page, line].to(_D64) - 127.0).unsqueeze(-1)


def _quant64(x, store):
    """The values that rows of 64-bit numbers are held as."""
    if store == "bf16":
        return x.to(torch.bfloat16), None
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / _TOP[store]))
    e = torch.where(amax < 2.0 ** -100, torch.zeros_like(e), e)
    y = x * torch.exp2(-e)
    return y.float().to(torch.float8_e4m3fn), (e[..., 0] + 127).to(torch.uint8)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "w4":
        lo, hi = (s["packed"] & 15).to(_D64), (s["packed"] >> 4).to(_D64)
        W = torch.empty(case["N"], case["K"], dtype=_D64, device="cuda")
        W[:, 0::2], W[:, 1::2] = lo, hi
        W -= 8.0 if s["zeros"] is None else s["zeros"].to(_D64).repeat_interleave(case["group"], 0).t()
        W *= s["scales"].to(_D64).repeat_interleave(case["group"], 0).t()
        y = torch.matmul(s["x"].to(_D64), W.t())
        return y if s["residual"] is None else y + s["residual"].to(_D64)
    page, slots = case["page"], s["slots"].tolist()
    if kind == "read":
        cu, first, out = s["cu"].tolist(), s["first"].tolist(), []
        cap = s["table"].shape[1] * page
        for k, slot in enumerate(slots):
            r = (first[k] + torch.arange(cu[k + 1] - cu[k], device="cuda")) % cap
            out.append(_row64(s, s["table"][slot].long()[r // page], r % page))
        return torch.cat(out)
    lens, ctx = _lens(case)
    m2, win, c = case["m2"], case["win"], case["c"]
    R = s["ring"].shape[1] * page
    start, out = 0, []
    if kind == "attention":
        sink = s["sink"].to(_D64)
        for slot, n, x in zip(slots, lens, ctx):
            q = s["q"][start:start + n].to(_D64)
            q = q / q.norm(dim=-1, keepdim=True).clamp_min(1e-12)
            nb, w0 = (x + n) // m2, max(0, x - win + 1)
            bi = torch.arange(nb, device="cuda")
            wi = torch.arange(w0, x + n, device="cuda")
            kb = _row64(s, s["blocks"][slot].long()[bi // page], bi % page)
            kw = _row64(s, s["ring"][slot].long()[wi % R // page], wi % R % page)
            keys = torch.cat([kb, kw])
            t = x + torch.arange(n, device="cuda")[:, None]
            ok = torch.cat([(bi + 1) * m2 <= t + 1, (wi <= t) & (wi >= t - win + 1)], 1)
            z = s["scale"] * (q.reshape(-1, c) @ keys.t()).view(n, case["nh"], -1)
            z = z.masked_fill(~ok[:, None], -math.inf)
            z = torch.cat([z, sink.view(1, -1, 1).expand(n, -1, 1)], -1)
            p = torch.softmax(z, -1)[..., :-1]
            out.append((p.reshape(n * case["nh"], -1) @ keys).view(n, case["nh"], c))
            start += n
        return torch.cat(out)
    rows, scales, state = s["rows_"], s["scales"], s["state"].to(_D64)

    def put(table, index, x):
        y, e = _quant64(x, case["store"])
        pages = table.long()[index // page]
        if e is None:
            rows[pages, index % page] = y
        else:
            rows.view(torch.uint8)[pages, index % page] = y.view(torch.uint8)
            scales[pages, index % page] = e

    for slot, n, x in zip(slots, lens, ctx):
        C, Z = s["C"][start:start + n].to(_D64), s["Z"][start:start + n].to(_D64)
        p = torch.arange(x, x + n, device="cuda")
        put(s["ring"][slot], p % R, C / C.norm(dim=-1, keepdim=True).clamp_min(1e-12))
        z = Z + s["B_pos"].to(_D64)[p % m2]
        at = 0
        while at < n:
            b = (x + at) // m2
            to = min(n, (b + 1) * m2 - x)
            zb, vb = z[at:to], C[at:to]
            m = zb.amax(0)
            if at == 0 and x % m2:
                m = torch.maximum(m, state[slot, 0])
            l = torch.exp(zb - m).sum(0)
            a = (torch.exp(zb - m) * vb).sum(0)
            if at == 0 and x % m2:
                f = torch.exp(state[slot, 0] - m)
                l, a = l + f * state[slot, 1], a + f * state[slot, 2]
            if (x + to) % m2 == 0:
                row = (a / l)[None]
                put(s["blocks"][slot], torch.tensor([b], device="cuda"),
                    row / row.norm(dim=-1, keepdim=True).clamp_min(1e-12))
            else:
                new = torch.stack([m, l, a])
                state[slot] = new
            at = to
        start += n
    got = {"rows": rows.to(_D64), "state": state}
    if scales is not None:
        got["scales"] = scales.view(torch.float8_e8m0fnu).to(_D64)
    return got
