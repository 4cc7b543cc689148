"""The paged HCA cache on the GPU against 64-bit references (tests/paged_ref.py).

Tolerances. A rounding to bf16 is off by at most u = 2^-8 of the value. The
attention rounds the query (score error at most |scale| u |q||k| = |scale| u for
unit vectors, which moves each weight by a factor of at most e^(2 |scale| u)) and
the weights (u), so an output is off by at most (e^(2 |scale| u) - 1 + u) sum p |k|, times a
half step of its own type; fp32 sums and exponentials are a few 2^-22 beside it (1e-5
is allowed). A quantised row is within half a step of the 64-bit row, where the fp32
row that is rounded differs from it by a few 2^-22 (1e-5 allowed).
"""

from __future__ import annotations

import numpy as np
import paged_ref as ref
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def f64(t):
    return t.detach().float().cpu().double().numpy()


def attn_tol(out, mag, scale, dtype, knorm=1.0):
    w = np.expm1(2 * abs(scale) * 2.0 ** -8 * knorm) + 2.0 ** -8
    return w * mag * (1 + HALF[dtype]) + HALF[dtype] * np.abs(out) + 1e-5


def fill(pool, lens, ctx, slots, m2, win, rng, scale_rows=1.0):
    """Random unit rows for everything the chunk's queries may see."""
    for slot, n, x in zip(slots, lens, ctx):
        nb = min((x + n) // m2, pool.nbp * pool.page)
        pool.put(pool.blocks, slot, np.arange(nb), scale_rows * ref.unit(rng.standard_normal((nb, pool.c))))
        if win:
            pos = np.arange(max(0, x - win + 1), x + n)
            pool.put(pool.ring, slot, pos % pool.cap,
                     scale_rows * ref.unit(rng.standard_normal((len(pos), pool.c))))


def pages_for(lens, ctx, m2, win, page):
    nbp = -(-max(1, max((x + n) // m2 for x, n in zip(ctx, lens))) // page)
    nrp = -(-(win + max(lens) - 1) // page) if win else 0
    return nbp, nrp


def run_attention(pool, q, lens, ctx, slots, m2, win, sink, scale, normalize_q=True, max_ctx=None, out=None,
                  max_len=None):
    import kch
    s, cu, cx, _ = ref.step(lens, ctx, slots)
    return kch.hca_paged_attention(
        q, pool.rows, pool.scales, pool.blocks, pool.ring if win else None, s, cu, cx, m2=m2,
        sliding_window=win, max_len=max(lens) if max_len is None else max_len,
        max_ctx=max(ctx) if max_ctx is None else max_ctx,
        sink_logits=None if sink is None else torch.from_numpy(sink).float().cuda(), scale=scale,
        normalize_q=normalize_q, out=out)


ATTN = [
    # lens, ctx, m2, win, nh, c, page, store, dtype, sink, scale
    ([1], [0], 16, 16, 16, 128, 16, "bf16", "bf16", True, 1.0),             # the first token
    ([1], [5003], 128, 128, 16, 128, 16, "bf16", "bf16", True, 11.3),
    ([1, 1, 1], [40, 4095, 16383], 4, 77, 16, 128, 64, "e4m3", "bf16", True, 11.3),  # key ranges, joined
    ([1, 1], [70000, 12], 4, 0, 4, 64, 32, "int8", "fp16", False, 1.0),      # no window, a sequence of few rows
    ([8, 1, 3, 5], [100, 0, 63, 8190], 64, 16, 4, 64, 32, "int8", "fp16", True, 8.0),
    ([2, 7], [15, 16], 16, 1, 16, 128, 1, "e4m3", "fp32", True, 1.0),       # pages of one row, a window of one
    ([5], [333], 1, 128, 6, 128, 128, "bf16", "bf16", True, 11.3),          # heads that do not fill a tile, m2 = 1
    ([130, 1, 77], [0, 3000, 512], 16, 128, 16, 128, 32, "e4m3", "bf16", True, 11.3),
    ([300], [10], 64, 5, 1, 64, 16, "bf16", "fp16", False, -8.0),           # one head, a negative scale
    ([3, 0, 2], [50, 60, 70], 16, 16, 33, 64, 16, "e4m3", "bf16", True, 8.0),  # an empty chunk, 33 heads
    ([40, 17], [9000, 20000], 8, 0, 2, 128, 256, "int8", "bf16", True, 5.0),
    ([16], [30], 16, 16, 4, 128, 16, "bf16", "fp32", False, 1.0),
]


@pytest.mark.parametrize("i", range(len(ATTN)))
def test_attention(dev, i):
    lens, ctx, m2, win, nh, c, page, store, dtype, sink, scale = ATTN[i]
    rng = np.random.default_rng(100 + i)
    slots = list(rng.permutation(len(lens)))
    pool = ref.Pool(len(lens), *pages_for(lens, ctx, m2, win, page), page, c, store, seed=i)
    fill(pool, lens, ctx, slots, m2, win, rng)
    q = torch.from_numpy(rng.standard_normal((sum(lens), nh, c))).to("cuda", DT[dtype])
    snk = rng.standard_normal(nh).astype(np.float32) if sink else None
    out = run_attention(pool, q, lens, ctx, slots, m2, win, snk, scale)
    want, mag = ref.attention(pool, f64(q), lens, ctx, slots, m2=m2, win=win, sink=snk, scale=scale)
    assert out.dtype == q.dtype and out.shape == q.shape
    # stored keys are unit rows up to their own rounding (at most 2^-4)
    tol = attn_tol(want, mag, scale, dtype, knorm=1 + 2.0 ** -4)
    assert (np.abs(f64(out) - want) <= tol).all(), np.abs(f64(out) - want).max()
    # (a first token of a block size 16 cache sees its window only, and itself alone at position 0)
    if ctx == [0] and lens == [1]:
        assert np.abs(want).max() > 0


def test_attention_without_keys_is_zero(dev):
    rng = np.random.default_rng(3)
    pool = ref.Pool(2, 1, 0, 16, 64, "e4m3")
    q = torch.from_numpy(rng.standard_normal((20, 4, 64))).cuda().bfloat16()
    fill(pool, [15, 5], [0, 14], [0, 1], 16, 0, rng)
    for snk in (None, np.ones(4, np.float32)):
        out = run_attention(pool, q, [15, 5], [0, 14], [0, 1], 16, 0, snk, 1.0)
        assert (out[:15] == 0).all() and (out[15] == 0).all()
        assert (out[16:].float().abs().amax(-1) > 0).all()  # position 15 on sees block 0


def test_attention_raw_queries_and_rows(dev):
    rng = np.random.default_rng(4)
    lens, ctx, m2, win, c = [3, 9], [200, 77], 16, 32, 128
    pool = ref.Pool(2, *pages_for(lens, ctx, m2, win, 16), 16, c, "int8")
    fill(pool, lens, ctx, [1, 0], m2, win, rng, scale_rows=3.0)
    q = torch.from_numpy(0.7 * rng.standard_normal((12, 16, c))).cuda().bfloat16()
    out = run_attention(pool, q, lens, ctx, [1, 0], m2, win, None, c ** -0.5, normalize_q=False)
    want, mag = ref.attention(pool, f64(q), lens, ctx, [1, 0], m2=m2, win=win, sink=None, scale=c ** -0.5,
                              normalize_q=False)
    # the queries are bf16 already: their rounding is exact
    assert (np.abs(f64(out) - want) <= attn_tol(want, mag, 0.0, "bf16")).all()


@pytest.mark.parametrize("max_ctx", [0, 30000, 2 ** 31 - 1])
def test_attention_bounds_only_lay_out(dev, max_ctx):
    """max_ctx and max_len change the split, not the answer."""
    rng = np.random.default_rng(5)
    lens, ctx, m2, win = [1, 2], [30000, 123], 4, 16
    pool = ref.Pool(2, *pages_for(lens, ctx, m2, win, 64), 64, 128, "e4m3")
    fill(pool, lens, ctx, [0, 1], m2, win, rng)
    q = torch.from_numpy(rng.standard_normal((3, 16, 128))).cuda().bfloat16()
    want, mag = ref.attention(pool, f64(q), lens, ctx, [0, 1], m2=m2, win=win, sink=None, scale=4.0)
    for max_len in (2, 40):
        out = run_attention(pool, q, lens, ctx, [0, 1], m2, win, None, 4.0, max_ctx=max_ctx, max_len=max_len)
        assert (np.abs(f64(out) - want) <= attn_tol(want, mag, 4.0, "bf16", 1 + 2.0 ** -4)).all()


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_attention_rows_not_seen_do_not_matter(dev, store):
    """NaN rows reach exactly the queries that see them; masked, unused and other sequences' rows none."""
    rng = np.random.default_rng(6)
    lens, ctx, m2, win, c, nh = [12, 4], [28, 50], 16, 8, 64, 4
    pool = ref.Pool(2, *pages_for(lens, ctx, m2, win, 16), 16, c, store)
    # every byte of the pool is NaN until written: unused lines and spare pages
    nan_byte = {"bf16": 0xff, "e4m3": 0x7f, "int8": 0x55}[store]
    pool.rows.view(torch.uint8).fill_(nan_byte)
    if pool.scales is not None:
        pool.scales.fill_(255)
    fill(pool, lens, ctx, [0, 1], m2, win, rng)
    q = torch.from_numpy(rng.standard_normal((16, nh, c))).cuda().bfloat16()
    clean = run_attention(pool, q, lens, ctx, [0, 1], m2, win, None, 8.0)
    assert torch.isfinite(clean).all()
    # sequence 0: the window row of position 33 (seen by 33 .. 40) and block 1 (from position 31 on)
    def poison(table, index):
        pg, ln = pool._at(table, 0, index)
        if pool.scales is None:
            pool.rows[pg, ln, 5] = float("nan")
        else:
            pool.scales[pg, ln] = 255
    poison(pool.ring, 33 % pool.cap)
    out = run_attention(pool, q, lens, ctx, [0, 1], m2, win, None, 8.0)
    pos = 28 + np.arange(12)
    sees = torch.from_numpy((pos >= 33) & (pos < 33 + win)).cuda()
    assert torch.isnan(out[:12][sees]).all()
    assert torch.equal(out[:12][~sees], clean[:12][~sees]) and torch.equal(out[12:], clean[12:])
    poison(pool.blocks, 1)
    out = run_attention(pool, q, lens, ctx, [0, 1], m2, win, None, 8.0)
    sees = torch.from_numpy(pos >= 31).cuda()
    assert torch.isnan(out[:12][sees]).all() and torch.equal(out[:12][~sees], clean[:12][~sees])
    assert torch.equal(out[12:], clean[12:])


def test_rows_behind_the_last_sequence(dev):
    rng = np.random.default_rng(7)
    lens, ctx = [2, 1], [100, 50]
    pool = ref.Pool(2, 2, 2, 16, 128, "e4m3")
    fill(pool, lens, ctx, [0, 1], 16, 16, rng)
    q = torch.from_numpy(rng.standard_normal((70, 16, 128))).cuda().bfloat16()
    q[3:] = float("nan")
    a = run_attention(pool, q, lens, ctx, [0, 1], 16, 16, None, 1.0)
    assert (a[3:] == 0).all() and torch.isfinite(a).all()
    mine = torch.full_like(q, 3.0)
    b = run_attention(pool, q, lens, ctx, [0, 1], 16, 16, None, 1.0, out=mine)
    assert b is mine and (b[3:] == 3.0).all() and torch.equal(a[:3], b[:3])


def test_what_the_tables_do_not_hold(dev):
    """Entries that name no page read as zero rows and are not written; sequences that are not described
    rightly are passed over."""
    import kch
    rng = np.random.default_rng(8)
    lens, ctx, m2, win, c = [1, 1, 1, 1], [100, 100, 100, 100], 16, 16, 64
    pool = ref.Pool(4, 1, 1, 16, c, "int8")
    fill(pool, lens, ctx, range(4), m2, win, rng)
    q = torch.from_numpy(rng.standard_normal((4, 4, c))).cuda().bfloat16()
    clean = run_attention(pool, q, lens, ctx, range(4), m2, win, None, 1.0)
    pool.blocks[0, 0], pool.ring[1, 0] = -1, pool.rows.shape[0]
    out = run_attention(pool, q, lens, ctx, range(4), m2, win, None, 1.0)
    assert torch.equal(out[2:], clean[2:])
    # rows of zeros: score 0, value 0
    k = pool.get(pool.ring, 0, np.arange(85, 101) % pool.cap)
    qn = ref.unit(f64(q[0]))
    e = np.exp(qn @ k.T)
    want = e @ k / (e.sum(1, keepdims=True) + 6)
    assert np.abs(f64(out[0]) - want).max() < 3 * 2.0 ** -8 * np.abs(k).max()
    before = pool.rows.view(torch.uint8).clone(), pool.scales.clone(), pool.state.clone()
    s, cu, cx, _ = ref.step(lens, [111] * 4, [0, 1, 2, 3])
    s[2], cx[3] = 9, -5
    C = torch.from_numpy(rng.standard_normal((4, c))).cuda()
    kch.hca_paged_append(C.float(), C.float(), torch.zeros(m2, c).cuda(), pool.rows, pool.scales, pool.state,
                         pool.blocks, pool.ring, s, cu, cx, m2=m2, max_len=1)
    wrote = (pool.rows.view(torch.uint8) != before[0]).any(-1)
    # sequence 0 its window row alone, sequence 1 its block alone
    pg0, ln0 = pool._at(pool.ring, 0, 111 % 16)
    pg1, ln1 = pool._at(pool.blocks, 1, 111 // m2)
    assert wrote.sum() == 2 and wrote[pg0, ln0].all() and wrote[pg1, ln1].all()
    assert torch.equal(pool.state, before[2])  # both blocks ended: no open block to write


APPEND = [
    # lens, ctx, m2, win, c, page, store, dtype, normalize
    ([1, 1, 1], [0, 127, 255], 128, 128, 128, 16, "e4m3", "bf16", True),
    ([1], [7], 8, 0, 64, 16, "int8", "fp16", True),
    ([77, 1, 0, 30], [100, 0, 5, 31], 16, 16, 64, 32, "bf16", "fp16", True),
    ([300, 5], [1000, 60], 64, 128, 128, 64, "e4m3", "fp32", True),
    ([130], [0], 128, 1, 128, 1, "int8", "bf16", True),
    ([40, 64], [3, 64], 1, 8, 128, 16, "e4m3", "bf16", True),        # every token a block
    ([50], [10], 20, 4, 64, 8, "int8", "fp32", False),               # raw rows, a block of no power of two
    ([9, 500], [130, 5], 300, 77, 128, 128, "bf16", "bf16", False),
]


def check_rows(pool, table, slot, index, want, store):
    got = pool.get(table, slot, index)
    sc = pool.get_scale(table, slot, index)
    tol = ref.half_step(want, sc, store) * (1 + 1e-4) + 1e-5 * np.abs(want).max(-1, keepdims=True)
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    if store != "bf16":
        # the least power of two that holds the row (either side of it where the largest channel is on the border)
        top = np.abs(want).max(-1) / ref.TOP[store]
        assert (top <= sc * (1 + 1e-5)).all() and (top >= sc / 2 * (1 - 1e-5)).all()


@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append(dev, i):
    import kch
    lens, ctx, m2, win, c, page, store, dtype, norm = APPEND[i]
    rng = np.random.default_rng(200 + i)
    S = len(lens)
    slots = list(rng.permutation(S))
    pool = ref.Pool(S, *pages_for(lens, ctx, m2, win, page), page, c, store, seed=i)
    both = torch.from_numpy(rng.standard_normal((sum(lens), 2 * c + 8))).to("cuda", DT[dtype])
    C, Z = both[:, :c], both[:, c:2 * c]
    Bp = torch.from_numpy(0.3 * rng.standard_normal((m2, c))).float().cuda()
    l0 = 1 + rng.random((S, c))
    st = np.stack([rng.standard_normal((S, c)), l0, l0 * rng.standard_normal((S, c))], 1).astype(np.float32)
    pool.state.copy_(torch.from_numpy(st))
    before = pool.rows.view(torch.uint8).clone()
    s, cu, cx, _ = ref.step(lens, ctx, slots)
    kch.hca_paged_append(C, Z, Bp, pool.rows, pool.scales, pool.state, pool.blocks, pool.ring if win else None,
                         s, cu, cx, m2=m2, max_len=max(lens), normalize=norm)
    rows, wins, sums = ref.append(f64(C), f64(Z), f64(Bp), lens, ctx, slots, st, m2=m2, normalize=norm)
    for (slot, b), row in rows.items():
        check_rows(pool, pool.blocks, slot, b, row[None], store)
    if win:
        for (slot, p), row in wins.items():
            check_rows(pool, pool.ring, slot, p % pool.cap, row[None], store)
    for slot in range(S):
        got = f64(pool.state[slot])
        if slot in sums:
            # sums of positive weights, m exact to fp32: each a few 2^-22 of its magnitude
            scale = np.stack([np.abs(sums[slot][0]), sums[slot][1], sums[slot][1] * 4])
            assert (np.abs(got - sums[slot]) <= 2e-5 * scale + 1e-6).all()
        else:
            assert (got == st[slot]).all()
    # nothing else of the pool
    changed = (pool.rows.view(torch.uint8) != before).any(-1)
    mine = torch.zeros_like(changed)
    for slot, b in rows:
        mine[pool._at(pool.blocks, slot, b)] = True
    if win:
        for slot, p in wins:
            mine[pool._at(pool.ring, slot, p % pool.cap)] = True
    assert not (changed & ~mine).any()


def test_append_masked_and_bad_tokens(dev):
    """Gates of -inf leave a token out, a block of such tokens is zeros; a NaN channel makes the rows NaN."""
    import kch
    rng = np.random.default_rng(9)
    c, m2 = 64, 8
    pool = ref.Pool(1, 1, 2, 16, c, "e4m3")
    C = torch.from_numpy(rng.standard_normal((24, c))).float().cuda()
    Z = torch.from_numpy(rng.standard_normal((24, c))).float().cuda()
    Z[3], C[3] = float("-inf"), float("inf")    # a padded token: its value does not matter
    Z[8:16] = float("-inf")                     # a whole block of them
    C[20, 7] = float("nan")
    s, cu, cx, _ = ref.step([24], [0], [0])
    args = (torch.zeros(m2, c).cuda(), pool.rows, pool.scales, pool.state, pool.blocks, pool.ring, s, cu, cx)
    kch.hca_paged_append(C, Z, *args, m2=m2, max_len=24)
    Cn, Zn = f64(C), f64(Z)
    Cn[3] = 0
    Cn[20] = 0
    rows, wins, _ = ref.append(Cn, Zn, np.zeros((m2, c)), [24], [0], [0], np.zeros((1, 3, c)), m2=m2)
    check_rows(pool, pool.blocks, 0, 0, rows[0, 0][None], "e4m3")
    assert (pool.get(pool.blocks, 0, 1) == 0).all()
    assert np.isnan(pool.get(pool.blocks, 0, 2)).all()
    assert np.isnan(pool.get(pool.ring, 0, [3, 20])).all()
    check_rows(pool, pool.ring, 0, 19, wins[0, 19][None], "e4m3")


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("c", [64, 128])
def test_read_gives_the_values(dev, store, c):
    import kch
    rng = np.random.default_rng(10)
    pool = ref.Pool(3, 5, 3, 8, c, store)
    for s in range(3):
        pool.put(pool.blocks, s, np.arange(40), rng.standard_normal((40, c)) * 10.0 ** rng.integers(-3, 3, (40, 1)))
        pool.put(pool.ring, s, np.arange(24), rng.standard_normal((24, c)))
    if pool.scales is not None:
        pool.scales[pool._at(pool.blocks, 2, 1)] = 255
    counts, first = [40, 0, 33], [0, 3, 35]
    s, cu, f, _ = ref.step(counts, first, [2, 0, 1])
    for dt in ("fp32", "bf16", "fp16"):
        out = kch.paged_read(pool.rows, pool.scales, pool.blocks, s, cu, total=80, first=f, dtype=DT[dt])
        want = np.concatenate([pool.get(pool.blocks, 2, np.arange(40)),
                               pool.get(pool.blocks, 1, (35 + np.arange(33)) % 40), np.zeros((7, c))])
        want = torch.from_numpy(want).float().to(DT[dt])
        assert torch.equal(torch.nan_to_num(out.cpu(), nan=99.0), torch.nan_to_num(want, nan=99.0))
    keep = torch.full((80, c), 5.0, device="cuda")
    kch.paged_read(pool.rows, pool.scales, pool.ring, s, cu, total=80, out=keep)
    assert (keep[73:] == 5.0).all() and not (keep[:73] == 5.0).any()


def test_many_sequences_are_found(dev):
    """More sequences than a wave's lanes, empty ones among them."""
    import kch
    rng = np.random.default_rng(11)
    S = 200
    counts = [int(k) for k in rng.integers(0, 4, S)]
    pool = ref.Pool(S, 1, 0, 4, 64, "int8")
    for s in range(S):
        pool.put(pool.blocks, s, np.arange(4), rng.standard_normal((4, 64)))
    s, cu, _, _ = ref.step(counts, [0] * S, range(S))
    out = kch.paged_read(pool.rows, pool.scales, pool.blocks, s, cu, total=sum(counts), dtype=torch.float32)
    want = np.concatenate([pool.get(pool.blocks, i, np.arange(n)) for i, n in enumerate(counts) if n])
    assert np.array_equal(out.cpu().double().numpy(), want)


@pytest.mark.parametrize("store", ["e4m3", "bf16"])
def test_pool_past_32_bit_offsets(dev, store):
    """Pages whose bytes lie beyond 2^31 (e4m3) and 2^32 (bf16) of the pool's start."""
    import kch
    rng = np.random.default_rng(12)
    c, page, m2, win = 128, 64, 16, 32
    high = 2 ** 31 // (c * page) + 5
    pool = ref.Pool(1, 2, 1, page, c, store, high=high)
    assert int(pool.blocks.min()) >= high
    C = torch.from_numpy(rng.standard_normal((1, 2 * c))).cuda().bfloat16()
    fill(pool, [1], [1007], [0], m2, win, rng)
    s, cu, cx, _ = ref.step([1], [1007], [0])
    st = f64(pool.state)
    Bp = torch.zeros(m2, c).cuda()
    kch.hca_paged_append(C[:, :c], C[:, c:], Bp, pool.rows, pool.scales, pool.state, pool.blocks, pool.ring, s, cu,
                         cx, m2=m2, max_len=1)
    rows, wins, _ = ref.append(f64(C[:, :c]), f64(C[:, c:]), f64(Bp), [1], [1007], [0], st, m2=m2)
    check_rows(pool, pool.blocks, 0, 62, rows[0, 62][None], store)
    check_rows(pool, pool.ring, 0, 1007 % pool.cap, wins[0, 1007][None], store)
    q = torch.from_numpy(rng.standard_normal((1, 16, c))).cuda().bfloat16()
    out = run_attention(pool, q, [1], [1007], [0], m2, win, None, 8.0)
    want, mag = ref.attention(pool, f64(q), [1], [1007], [0], m2=m2, win=win, sink=None, scale=8.0)
    assert (np.abs(f64(out) - want) <= attn_tol(want, mag, 8.0, "bf16", 1 + 2.0 ** -4)).all()
    got = kch.paged_read(pool.rows, pool.scales, pool.blocks, s, torch.tensor([0, 63], dtype=torch.int32).cuda(),
                         total=63, dtype=torch.float32)
    assert np.array_equal(got.cpu().double().numpy(), pool.get(pool.blocks, 0, np.arange(63)))


def test_captured_step_replays_with_new_contents(dev):
    """One captured append + attention, replayed on other slots, lengths and positions, beside eager calls."""
    import kch
    rng = np.random.default_rng(13)
    m2, win, c, nh, page, S, N = 16, 16, 64, 4, 16, 3, 6
    pool = ref.Pool(4, 8, 2, page, c, "e4m3")
    for s in range(4):
        pool.put(pool.blocks, s, np.arange(128), ref.unit(rng.standard_normal((128, c))))
        pool.put(pool.ring, s, np.arange(32), ref.unit(rng.standard_normal((32, c))))
    pool.state.zero_()
    Bp = torch.from_numpy(rng.standard_normal((m2, c))).float().cuda()
    C, Z = torch.zeros(N, c, device="cuda"), torch.zeros(N, c, device="cuda")
    q = torch.zeros(N, nh, c, device="cuda", dtype=torch.bfloat16)
    s, cu, cx, _ = ref.step([1, 1, 1], [5, 6, 7], [0, 1, 2])
    out = torch.zeros_like(q)

    def go(pl, o):
        kch.hca_paged_append(C, Z, Bp, pl.rows, pl.scales, pl.state, pl.blocks, pl.ring, s, cu, cx, m2=m2, max_len=4)
        return kch.hca_paged_attention(q, pl.rows, pl.scales, pl.blocks, pl.ring, s, cu, cx, m2=m2, max_len=4,
                                       sliding_window=win, max_ctx=2000, scale=8.0, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(pool, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(pool, out)
    for lens, ctx, slots in (([1, 4, 1], [5, 14, 2000], [3, 0, 1]), ([0, 2, 4], [9, 100, 47], [2, 1, 0]),
                             ([2, 2, 2], [63, 0, 1], [0, 3, 2])):
        C.copy_(torch.from_numpy(rng.standard_normal((N, c))))
        Z.copy_(torch.from_numpy(rng.standard_normal((N, c))))
        q.copy_(torch.from_numpy(rng.standard_normal((N, nh, c))))
        a, b, d, _ = ref.step(lens, ctx, slots)
        s.copy_(a), cu.copy_(b), cx.copy_(d)
        twin = ref.Pool(4, 8, 2, page, c, "e4m3")
        twin.rows, twin.scales, twin.state = (t.clone() for t in (pool.rows.view(torch.uint8), pool.scales,
                                                                  pool.state))
        twin.rows = twin.rows.view(torch.float8_e4m3fn)
        twin.blocks, twin.ring = pool.blocks, pool.ring
        out.fill_(-1.0)
        graph.replay()
        eager = go(twin, torch.full_like(q, -1.0))
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(pool.rows.view(torch.uint8), twin.rows.view(torch.uint8))
        assert torch.equal(pool.state, twin.state) and torch.equal(pool.scales, twin.scales)
        want, mag = ref.attention(pool, f64(q[:sum(lens)]), lens, ctx, slots, m2=m2, win=win, sink=None, scale=8.0)
        assert (np.abs(f64(out[:sum(lens)]) - want) <= attn_tol(want, mag, 8.0, "bf16", 1 + 2.0 ** -4)).all()
        assert (out[sum(lens):] == -1.0).all()


def test_two_streams_at_once(dev):
    rng = np.random.default_rng(14)
    lens, ctx, m2, win = [1], [60000], 4, 64
    pools, qs, alone = [], [], []
    for i in range(2):
        p = ref.Pool(1, *pages_for(lens, ctx, m2, win, 64), 64, 128, "int8", seed=i)
        fill(p, lens, ctx, [0], m2, win, rng)
        pools.append(p)
        qs.append(torch.from_numpy(rng.standard_normal((1, 16, 128))).cuda().bfloat16())
        alone.append(run_attention(p, qs[-1], lens, ctx, [0], m2, win, None, 8.0))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run_attention(pools[i], qs[i], lens, ctx, [0], m2, win, None, 8.0))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i in range(2) for o in got[i])


# --------------------------------------------------------------------------- the cache object

@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("c", [64, 48])
def test_cache_of_sequences_that_come_and_go(dev, kv, c):
    """Chunks of several sequences through the cache against the whole history in 64 bits."""
    import kch
    rng = np.random.default_rng(15)
    m2, win, nh = 8, 12, 4
    cache = kch.HCAPagedCache(64, c, m2, win, max_seqs=4, max_tokens=200, max_chunk=40, page=8, kv_dtype=kv,
                              device="cuda")
    Bp = torch.from_numpy(0.3 * rng.standard_normal((m2, c))).float().cuda()
    sink = torch.from_numpy(rng.standard_normal(nh)).float().cuda()
    hist, free = {}, cache.n_free_pages
    store = {torch.bfloat16: "bf16", torch.float8_e4m3fn: "e4m3", torch.int8: "int8"}[kv]

    def step(slots, lens):
        N = sum(lens)
        x = torch.from_numpy(rng.standard_normal((N, 2 * c))).cuda().bfloat16()
        q = torch.from_numpy(rng.standard_normal((N, nh, c))).cuda().bfloat16()
        cache.append_step(slots, x[:, :c], x[:, c:], Bp, lens)
        out = cache.forward_step(q, scale=6.0, sink_logits=sink)
        at = 0
        for s, n in zip(slots, lens):
            hist[s] = np.concatenate([hist[s], f64(x[at:at + n])])
            h = hist[s]
            rows, wins, _ = ref.append(h[:, :c], h[:, c:], f64(Bp), [len(h)], [0], [0], np.zeros((1, 3, c)), m2=m2)
            kb, kw = f64(cache.read_blocks(s, torch.float32)), f64(cache.read_window(s, torch.float32))
            assert kb.shape == (len(h) // m2, c) and kw.shape == (min(win, len(h)), c)
            for b in range(len(kb)):
                amax = np.abs(rows[0, b]).max()
                sc = np.array([2.0 ** np.ceil(np.log2(amax / ref.TOP.get(store, 1.0)))])
                assert (np.abs(kb[b] - rows[0, b]) <= 2 * ref.half_step(rows[0, b][None], sc, store)[0] + 1e-5).all()
            for i in range(n):
                # the values that the cache holds, seen from this token (window rows older than the last win ones
                # are gone by now: the tokens that saw them are skipped)
                t = len(h) - n + i
                lo = max(0, t - win + 1)
                if lo < len(h) - len(kw):
                    continue
                keys = np.concatenate([kb[:(t + 1) // m2], kw[lo - (len(h) - len(kw)):t + 1 - (len(h) - len(kw))]])
                sc = 6.0 * ref.unit(f64(q[at + i])) @ keys.T
                e = np.exp(sc)
                p = e / (e.sum(1, keepdims=True) + np.exp(f64(sink))[:, None])
                want, mag = p @ keys, p @ np.abs(keys)
                assert (np.abs(f64(out[at + i]) - want) <= attn_tol(want, mag, 6.0, "bf16", 1 + 2.0 ** -4)).all()
            at += n

    a, b = cache.add(), cache.add()
    hist[a] = hist[b] = np.zeros((0, 2 * c))
    step([a, b], [37, 1])
    step([b, a], [9, 1])
    step([a], [1])
    d = cache.add()
    hist[d] = np.zeros((0, 2 * c))
    step([d, a, b], [3, 1, 22])
    cache.release(a)
    e = cache.add()
    hist[e] = np.zeros((0, 2 * c))
    for _ in range(9):
        step([e, b, d], [1, 1, 1])
    step([e], [40])
    for s in (b, d, e):
        cache.release(s)
    assert cache.n_free_pages == free


def test_cache_matches_the_decoding_cache(dev):
    """Equally long sequences in 16 bits: the same tokens through HCADecodingCache."""
    import kch
    torch.manual_seed(0)
    B, c, m2, win, nh, T = 3, 128, 16, 32, 16, 70
    old = kch.HCADecodingCache(B, c, m2, win, "cuda", torch.bfloat16)
    new = kch.HCAPagedCache(32, c, m2, win, max_seqs=B, max_tokens=256, max_chunk=T, page=16, kv_dtype=torch.bfloat16)
    slots = [new.add() for _ in range(B)]
    Bp = 0.1 * torch.randn(m2, c, device="cuda")
    sink = torch.randn(nh, device="cuda")
    for n in (T, 1, 1, 1):
        x = torch.randn(B, n, 2 * c, device="cuda").bfloat16()
        C, Z = x[..., :c], x[..., c:]
        old.append_step(C, Z, Bp)
        new.append_step(slots, C.reshape(-1, c), Z.reshape(-1, c), Bp, [n] * B)
        q = torch.randn(B, n, nh, c, device="cuda").bfloat16()
        out = new.forward_step(q.reshape(-1, nh, c), sink_logits=sink).view(B, n, nh, c)
    want = old.forward_step(torch.nn.functional.normalize(q.float(), dim=-1), nh=nh, sink_logits=sink)
    # both within 3 u + u of the softmax over the same rows (the older cache rounds a raw row first: u more)
    assert (out.float() - want).abs().max() <= 10 * 2.0 ** -8 * want.abs().max()


def test_cache_refuses(dev):
    import kch
    mk = lambda **k: kch.HCAPagedCache(8, 64, 8, 8, max_seqs=2, max_tokens=64, max_chunk=4, page=8, **k)  # noqa: E731
    cache = mk()
    x, Bp = torch.randn(4, 64, device="cuda"), torch.zeros(8, 64, device="cuda")
    a = cache.add()
    with pytest.raises(ValueError, match="append_step first"):
        cache.forward_step(torch.zeros(1, 4, 64, device="cuda"))
    for args, msg in ((([a, a], x[:2], x[:2], Bp), "each slot once"), (([a], x[:2], x[:2], Bp), r"must be \[1, 64\]"),
                      (([1], x[:1], x[:1], Bp), "holds no sequence"), (([a], x, x, Bp, [5]), "max_chunk"),
                      (([a], x[:1], x[:1], Bp[:4]), "B_pos"), (([a], x, x, Bp, [-1]), "chunk of -1")):
        with pytest.raises(ValueError, match=msg):
            cache.append_step(*args)
    with pytest.raises(RuntimeError, match="GPU"):
        cache.append_step([a], x[:1].cpu(), x[:1].cpu(), Bp)
    for _ in range(16):
        cache.append_step([a], x, x, Bp, [4])
    with pytest.raises(ValueError, match="max_tokens"):
        cache.append_step([a], x[:1], x[:1], Bp)
    assert cache.n_tokens(a) == 64
    cache.add()
    with pytest.raises(RuntimeError, match="every slot"):
        cache.add()
    small = kch.HCAPagedCache(3, 64, 8, 8, max_seqs=2, max_tokens=640, max_chunk=64, page=8)
    y = torch.randn(64, 64, device="cuda")
    with pytest.raises(RuntimeError, match="pages needed"):
        small.add()  # its ring alone has 9
    assert small.n_free_pages == 3
    small2 = kch.HCAPagedCache(10, 64, 8, 8, max_seqs=1, max_tokens=640, max_chunk=64, page=8)
    s = small2.add()
    small2.append_step([s], y, y, Bp, [64])
    with pytest.raises(RuntimeError, match="pages needed"):
        small2.append_step([s], y, y, Bp, [64])
    assert small2.n_tokens(s) == 64


def test_operators_refuse(dev):
    import kch
    pool = ref.Pool(1, 1, 1, 16, 64, "int8")
    s, cu, cx, _ = ref.step([1], [3], [0])
    q, C, Bp = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 64, device="cuda"), torch.zeros(8, 64, device="cuda")

    def attn(**k):
        a = dict(q=q, rows=pool.rows, scales=pool.scales, block_table=pool.blocks, ring_table=pool.ring, slots=s,
                 cu_seqlens=cu, ctx_lens=cx, m2=8, sliding_window=8, max_len=1, max_ctx=3)
        a.update(k)
        return kch.hca_paged_attention(**a)

    attn()
    for k, msg in ((dict(scales=None), "scales"), (dict(q=q[..., :32]), "q must be"), (dict(slots=s.long()), "slots"),
                   (dict(cu_seqlens=cu[:1]), "cu_seqlens has"), (dict(max_len=10), "need a ring"), (dict(m2=0), "m2"),
                   (dict(sink_logits=torch.zeros(3)), "sink_logits"), (dict(ring_table=None), "need a ring"),
                   (dict(out=torch.zeros(1, 4, 64)), "out must"), (dict(max_ctx=-1), "max_ctx")):
        with pytest.raises(ValueError, match=msg):
            attn(**k)
    with pytest.raises(TypeError, match="rows must be"):
        attn(rows=pool.rows.float())
    with pytest.raises(NotImplementedError, match="float64"):
        attn(q=q.double())
    with pytest.raises(RuntimeError, match="GPU"):
        attn(q=q.cpu())
    with pytest.raises(NotImplementedError, match="no gradients"):
        attn(q=q.clone().requires_grad_())
    with torch.no_grad():
        attn(q=q.clone().requires_grad_())

    def app(**k):
        a = dict(C=C, Z=C, B_pos=Bp, rows=pool.rows, scales=pool.scales, state=pool.state, block_table=pool.blocks,
                 ring_table=pool.ring, slots=s, cu_seqlens=cu, ctx_lens=cx, m2=8, max_len=1)
        a.update(k)
        kch.hca_paged_append(**a)

    app()
    for k, msg in ((dict(Z=C.half()), "one dtype"), (dict(B_pos=Bp[:3]), "B_pos"), (dict(max_len=17), "max_len"),
                   (dict(state=pool.state[:, :2]), "state")):
        with pytest.raises(ValueError, match=msg):
            app(**k)
    with pytest.raises(NotImplementedError, match="no gradients"):
        app(Z=C.clone().requires_grad_())
    with pytest.raises(ValueError, match="total"):
        kch.paged_read(pool.rows, pool.scales, pool.blocks, s, cu, total=-1)


def test_no_sequences_at_all(dev):
    """S = 0: every row lies behind the last sequence; an empty pool is not read."""
    import kch
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = torch.zeros(0, 16, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.ones(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    out = kch.hca_paged_attention(q, rows, None, z(1, 1), z(1, 1), z(0), z(1), z(0), m2=8, sliding_window=8,
                                  max_len=1, max_ctx=0)
    assert (out == 0).all()
    for dt in (torch.float32, torch.bfloat16):
        assert (kch.paged_read(rows, None, z(1, 1), z(0), z(1), total=5, dtype=dt) == 0).all()
    kch.hca_paged_append(q[:, 0], q[:, 0], torch.zeros(8, 64, device="cuda"), rows, None,
                         torch.zeros(1, 3, 64, device="cuda"), z(1, 1), z(1, 1), z(0), z(1), z(0), m2=8, max_len=1)
    with pytest.raises(RuntimeError, match="without pages"):
        kch.hca_paged_attention(q, rows, None, z(1, 1), z(1, 1), z(1), z(2), z(1), m2=8, sliding_window=8, max_len=1)


def test_chunks_longer_than_max_len(dev):
    """max_len is a promise: what a chunk has past it is zeros (left as it was in out), the rest is right."""
    rng = np.random.default_rng(21)
    m2, win = 16, 16
    for nh, lens in ((16, [5, 2]), (4, [40, 3])):
        cut = 1 if nh == 16 else 20
        pool = ref.Pool(2, *pages_for(lens, [100, 50], m2, win, 16), 16, 64, "e4m3")
        fill(pool, lens, [100, 50], [0, 1], m2, win, rng)
        q = torch.from_numpy(rng.standard_normal((sum(lens), nh, 64))).cuda().bfloat16()
        whole = run_attention(pool, q, lens, [100, 50], [0, 1], m2, win, None, 8.0)
        out = run_attention(pool, q, lens, [100, 50], [0, 1], m2, win, None, 8.0, max_len=cut)
        got = torch.zeros(sum(lens), dtype=torch.bool)
        got[:cut] = True
        got[lens[0]:lens[0] + min(cut, lens[1])] = True
        assert (out[~got] == 0).all() and (out[got].float() - whole[got].float()).abs().max() <= 2.0 ** -6
        mine = torch.full_like(q, 9.0)
        run_attention(pool, q, lens, [100, 50], [0, 1], m2, win, None, 8.0, max_len=cut, out=mine)
        assert (mine[~got] == 9.0).all() and torch.equal(mine[got], out[got])


def test_parameters_that_ask_for_gradients_are_refused(dev):
    import kch
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = torch.zeros(2, 16, 64, device="cuda", dtype=torch.bfloat16)
    x = torch.ones(1, 64, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    at = (z(1, 1), torch.ones(1, 1, dtype=torch.int32, device="cuda"), z(1), cu, z(1))
    with pytest.raises(NotImplementedError, match="no gradients"):
        kch.hca_paged_append(x, x, torch.zeros(8, 64, device="cuda", requires_grad=True), rows, None,
                             torch.zeros(1, 3, 64, device="cuda"), *at, m2=8, max_len=1)
    with pytest.raises(NotImplementedError, match="no gradients"):
        kch.hca_paged_attention(x[:, None], rows, None, *at, m2=8, sliding_window=8, max_len=1,
                                sink_logits=torch.zeros(1, device="cuda", requires_grad=True))


def test_cache_refuses_capture(dev, monkeypatch):
    """The cache's counts come from the host: a graph would replay this step's."""
    import kch
    cache = kch.HCAPagedCache(4, 64, 8, 8, max_seqs=2, max_tokens=64, page=16)
    s = cache.add()
    x = torch.ones(1, 64, device="cuda", dtype=torch.bfloat16)
    Bp = torch.zeros(8, 64, device="cuda")
    cache.append_step([s], x, x, Bp)
    out = cache.forward_step(x[:, None])
    free, n = cache.n_free_pages, cache.n_tokens(s)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for f in (cache.add, lambda: cache.append_step([s], x, x, Bp), lambda: cache.forward_step(x[:, None]),
                  lambda: cache.read_blocks(s), lambda: cache.read_window(s)):
            with pytest.raises(RuntimeError, match="graph"):
                f()
    assert cache.n_free_pages == free and cache.n_tokens(s) == n
    assert torch.equal(cache.forward_step(x[:, None]), out)


# fp16 queries: both products in fp16, its half step u = 2^-11. Below its normal range a
# rounding is off by at most 2^-25 instead (of a key at a quarter 2^-23, of a bf16 key, cut,
# 2^-24): of the query sqrt(c) 2^-25 <= 2^-21 in a score of unit vectors, of the keys sqrt(c)
# 2^-23 <= 2^-19, of each weight 2^-25 beside a sum of at least 1, and of the keys 2^-23 in the output.
FP16 = [
    ([1], [5003], 128, 128, 16, 128, 16, "bf16", 11.3),
    ([1, 1, 1], [40, 4095, 16383], 4, 77, 16, 128, 64, "e4m3", 11.3),
    ([8, 1, 3, 5], [100, 0, 63, 8190], 64, 16, 4, 64, 32, "int8", 8.0),
    ([2, 7], [15, 16], 16, 1, 16, 128, 1, "e4m3", 1.0),
    ([130, 1, 77], [0, 3000, 512], 16, 128, 16, 128, 32, "bf16", 11.3),
    ([40, 170], [9000, 20000], 8, 0, 2, 64, 64, "e4m3", 5.0),
    ([64], [700], 4, 33, 1, 128, 16, "int8", -11.3),
]


def fp16_tol(out, mag, scale, keys, kmax, knorm):
    u = 2.0 ** -11
    w = np.expm1(2 * abs(scale) * knorm * (u + 2.0 ** -18)) + u
    return (w * mag + keys * 2.0 ** -25 * kmax + 2.0 ** -23) * (1 + u) + u * np.abs(out) + 1e-5


@pytest.mark.parametrize("i", range(len(FP16)))
def test_attention_fp16_products(dev, i):
    lens, ctx, m2, win, nh, c, page, store, scale = FP16[i]
    rng = np.random.default_rng(500 + i)
    slots = list(rng.permutation(len(lens)))
    pool = ref.Pool(len(lens), *pages_for(lens, ctx, m2, win, page), page, c, store, seed=i)
    fill(pool, lens, ctx, slots, m2, win, rng)
    q = torch.from_numpy(rng.standard_normal((sum(lens), nh, c))).to("cuda", torch.float16)
    snk = rng.standard_normal(nh).astype(np.float32)
    out = run_attention(pool, q, lens, ctx, slots, m2, win, snk, scale)
    want, mag = ref.attention(pool, f64(q), lens, ctx, slots, m2=m2, win=win, sink=snk, scale=scale)
    keys = max((x + n) // m2 for x, n in zip(ctx, lens)) + win
    tol = fp16_tol(want, mag, scale, keys, 1.0, 1 + 2.0 ** -4)
    assert (np.abs(f64(out) - want) <= tol).all(), np.abs(f64(out) - want).max()


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("n", [1, 20])
def test_attention_fp16_rows_at_the_edge_of_its_range(dev, store, n):
    """Rows of fp16 values up to its largest are answered, rows past it are NaN to those that see them."""
    rng = np.random.default_rng(9)
    m2, win, c, nh, ctx = 4, 16, 64, 4, 100
    pool = ref.Pool(1, *pages_for([n], [ctx], m2, win, 32), 32, c, store)
    nb = (ctx + n) // m2
    big = 65504.0 * rng.choice([-1.0, 1.0, 0.999, 0.5, 2.0 ** -9], (nb, c))
    pool.put(pool.blocks, 0, np.arange(nb), big)
    pos = np.arange(ctx - win + 1, ctx + n)
    pool.put(pool.ring, 0, pos % pool.cap, 65504.0 * rng.uniform(-1, 1, (len(pos), c)))
    q = torch.from_numpy(rng.standard_normal((n, nh, c))).to("cuda", torch.float16)
    scale = 2.0 ** -19
    out = run_attention(pool, q, [n], [ctx], [0], m2, win, None, scale, normalize_q=False)
    want, mag = ref.attention(pool, f64(q), [n], [ctx], [0], m2=m2, win=win, sink=None, scale=scale,
                              normalize_q=False)
    # fp16 queries are exact; a bf16 row's 65536 is taken as 65504, 2^-11 of it, which moves its
    # score by at most |scale| 2^5 sum |q|
    u, moved = 2.0 ** -11, scale * 2.0 ** 5 * np.abs(f64(q)).sum(-1).max()
    tol = (np.expm1(2 * moved) + 2 * u) * mag * (1 + u) + u * np.abs(want) + (nb + win) * 2.0 ** -25 * 65536 + 1e-5
    assert (np.abs(want) <= 65504).all()
    assert (np.abs(f64(out) - want) <= tol).all(), np.abs(f64(out) - want).max()
    if store == "bf16":
        b = (ctx + n) // m2 - 1  # the last block's row, which only the last queries see
        pool.put(pool.blocks, 0, np.array([b]), np.full((1, c), 2.0 ** 17))
    else:
        b = (ctx + n) // m2 - 1
        pool.put(pool.blocks, 0, np.array([b]), np.full((1, c), 2.0 ** 19))
    poisoned = run_attention(pool, q, [n], [ctx], [0], m2, win, None, scale, normalize_q=False)
    sees = torch.from_numpy((ctx + np.arange(n) + 1) // m2 > b).cuda()
    assert sees.any() and torch.isnan(poisoned[sees]).all()
    assert torch.equal(poisoned[~sees], out[~sees])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [4, 40])
def test_attention_nan_codes_reach_only_who_sees_them(dev, dtype, n):
    """An e4m3 NaN in one channel of a row: NaN for the queries that see it, nothing for the others."""
    rng = np.random.default_rng(11)
    m2, win, c, nh, ctx = 4, 8, 64, 4, 61
    pool = ref.Pool(1, *pages_for([n], [ctx], m2, win, 32), 32, c, "e4m3")
    fill(pool, [n], [ctx], [0], m2, win, rng)
    q = torch.from_numpy(rng.standard_normal((n, nh, c))).to("cuda", DT[dtype])
    clean = run_attention(pool, q, [n], [ctx], [0], m2, win, None, 8.0)
    b = (ctx + n) // m2 - 1
    pos = ctx + np.arange(n)
    raw = pool.rows.view(torch.uint8)
    for table, at, sees in ((pool.blocks, b, (pos + 1) // m2 > b),
                            (pool.ring, (ctx + 2) % pool.cap, (pos >= ctx + 2) & (pos < ctx + 2 + win))):
        page, line = int(table[0, at // 32]), at % 32
        held = int(raw[page, line, c - 3])
        raw[page, line, c - 3] = 0xff
        out = run_attention(pool, q, [n], [ctx], [0], m2, win, None, 8.0)
        raw[page, line, c - 3] = held
        sees = torch.from_numpy(sees).cuda()
        assert sees.any() and (~sees).any()
        assert torch.isnan(out[sees]).all() and torch.equal(out[~sees], clean[~sees])
