"""Edges of the serving operators on the GPU: steps that say nothing or too much, masks of the type's
lowest value, rows that are not finite, and how many bits the products keep."""

from __future__ import annotations

import copy

import numpy as np
import paged_ref as ref
import pytest
import torch
from test_paged_gpu import DT, f64, fill, pages_for, run_attention

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- rows that nothing answers

@pytest.mark.parametrize("nh,lens,max_len", [
    (4, [3, 2, 4, 1], 4), (16, [2, 1, 2, 1], 2), (16, [3, 40, 30, 5], 40), (4, [3, 40, 90, 5], 20), (16, [1, 1, 9, 1], 1),
])
def test_rows_of_sequences_passed_over_are_zeros(dev, nh, lens, max_len, monkeypatch):
    """A fresh result holds zeros, never what its memory held before: rows ahead of the first sequence, of slots
    outside the table, of a negative context and behind the last sequence. A given one keeps them."""
    import kch
    rng = np.random.default_rng(31)
    m2, win, c = 16, 16, 64
    ctx = [100, 90, 80, 70]
    pool = ref.Pool(4, *pages_for(lens, ctx, m2, win, 16), 16, c, "e4m3")
    fill(pool, lens, ctx, [0, 1, 2, 3], m2, win, rng)
    n = sum(lens)
    q = torch.from_numpy(rng.standard_normal((2 + n + 5, nh, c))).cuda().bfloat16()
    s, cu, cx, _ = ref.step(lens, ctx, [0, 1, 2, 3])

    def go(out=None):
        return kch.hca_paged_attention(q, pool.rows, pool.scales, pool.blocks, pool.ring, s, cu + 2, cx, m2=m2,
                                       sliding_window=win, max_len=max_len, max_ctx=200, scale=8.0, out=out)

    whole = go().clone()
    monkeypatch.setattr(torch, "empty_like", lambda t: torch.full_like(t, float("nan")))
    first = go()
    assert (first[:2] == 0).all() and (first[2 + n:] == 0).all() and torch.equal(first[2:2 + n], whole[2:2 + n])
    at = 2 + np.concatenate([[0], np.cumsum(lens)])
    for bad, how in ((1, "slot"), (2, "slots"), (3, "ctx"), (0, "ctx")):
        keep = s.clone(), cx.clone()
        if how == "ctx":
            cx[bad] = -5
        else:
            s[bad] = -1 if how == "slot" else 4
        out, mine = go(), go(torch.full_like(q, 9.0))
        s.copy_(keep[0]), cx.copy_(keep[1])
        for i in range(4):
            a, b = at[i], at[i + 1]
            if i == bad:
                assert (out[a:b] == 0).all() and (mine[a:b] == 9.0).all()
            else:
                assert torch.equal(out[a:b], whole[a:b])
        assert (out[:2] == 0).all() and (out[2 + n:] == 0).all()
        assert (mine[:2] == 9.0).all() and (mine[2 + n:] == 9.0).all()
    # the last sequence says it has more rows than there are
    cu[4] = 1000
    out = go()
    assert (out[at[3]:] == 0).all() and torch.equal(out[2:at[3]], whole[2:at[3]])


@pytest.mark.parametrize("lens", [[0, 0], [3, 2]])
def test_no_token_of_any_chunk(dev, lens):
    """max_len = 0: no row is answered, whatever the contexts' bound."""
    import kch
    rng = np.random.default_rng(32)
    pool = ref.Pool(2, 1, 1, 16, 128, "int8")
    fill(pool, [3, 2], [50, 60], [0, 1], 16, 8, rng)
    q = torch.from_numpy(rng.standard_normal((7, 16, 128))).cuda().bfloat16()
    s, cu, cx, _ = ref.step(lens, [50, 60], [0, 1])
    for max_ctx in (60, 10 ** 6, None):
        args = (pool.rows, pool.scales, pool.blocks, pool.ring, s, cu, cx)
        kw = dict(m2=16, sliding_window=8, max_len=0, max_ctx=max_ctx)
        assert (kch.hca_paged_attention(q, *args, **kw) == 0).all()
        mine = torch.full_like(q, 3.0)
        assert kch.hca_paged_attention(q, *args, out=mine, **kw) is mine and (mine == 3.0).all()


@pytest.mark.parametrize("top", [1, 30])
def test_captured_padded_step(dev, top):
    """A captured call that makes its own result, replayed on steps with padding entries: what it held in the replay
    before does not show, eager work and synchronisations between the replays."""
    import kch
    rng = np.random.default_rng(37)
    S, N, nh, c, m2, win = 4, 3 * top + 5, 16, 64, 16, 16
    ctx = [9000, 40, 3000, 500]
    pool = ref.Pool(S, *pages_for([top] * S, ctx, m2, win, 32), 32, c, "int8")
    fill(pool, [top] * S, ctx, range(S), m2, win, rng)
    q = torch.zeros(N, nh, c, device="cuda", dtype=torch.bfloat16)
    s, cu, cx, _ = ref.step([top] * S, ctx, range(S))

    def go():
        return kch.hca_paged_attention(q, pool.rows, pool.scales, pool.blocks, pool.ring, s, cu, cx, m2=m2,
                                       sliding_window=win, max_len=top, max_ctx=9000, scale=8.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    for lead, lens, slots in ((0, [top, 1, top, 1], [0, 1, 2, 3]), (2, [top, 1, 1, top], [-1, 1, -1, 3]),
                              (0, [1, 0, 1, 1], [0, -1, 2, 7]), (1, [top] * 3 + [0], [-1] * 4), (0, [1] * 4, [3, 2, 1, 0])):
        q.copy_(torch.from_numpy(rng.standard_normal(q.shape)))
        at = lead + np.concatenate([[0], np.cumsum(lens)])
        s.copy_(torch.tensor(slots)), cu.copy_(torch.tensor(at))
        cx.copy_(torch.tensor([ctx[k] if 0 <= k < S else 3 for k in slots]))
        graph.replay()
        eager = go()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        answered = torch.zeros(N, dtype=torch.bool, device="cuda")
        for i, k in enumerate(slots):
            answered[at[i]:at[i + 1]] = 0 <= k < S
        assert (out[~answered] == 0).all() and (out[answered].float().abs().amax(-1) > 0).all()


# --------------------------------------------------------------------------- masks and rows that are not finite

@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_blocks_masked_with_the_lowest_value(dev, dtype, store):
    """Gates of the type's lowest value: alone in a block they weigh alike (its plain mean), beside others nothing,
    and they outweigh -inf; the sums that a chunk leaves and the next one takes up as well."""
    import kch
    rng = np.random.default_rng(33)
    c, m2 = 64, 8
    low = torch.finfo(DT[dtype]).min
    pool = ref.Pool(1, 1, 4, 16, c, store)
    C = torch.from_numpy(rng.standard_normal((40, c))).to("cuda", DT[dtype])
    Z = torch.from_numpy(rng.standard_normal((40, c))).to("cuda", DT[dtype])
    Z[0:8] = low                     # a whole block
    Z[8:11] = low                    # some of one
    Z[16:24], Z[18] = float("-inf"), low   # one weight left
    Z[24:40, ::2] = low              # every other channel of two blocks
    Bp = torch.zeros(m2, c).cuda()
    for cut in (40, 5, 27, 16):      # ends of the first chunk
        pool.state.fill_(7.0)
        for a, b in ((0, cut), (cut, 40)):
            if a == b:
                continue
            s, cu, cx, _ = ref.step([b - a], [a], [0])
            kch.hca_paged_append(C[a:b], Z[a:b], Bp, pool.rows, pool.scales, pool.state, pool.blocks, pool.ring, s, cu,
                                 cx, m2=m2, max_len=b - a)
        rows, _, _ = ref.append(f64(C), f64(Z), f64(Bp), [40], [0], [0], np.zeros((1, 3, c)), m2=m2)
        want = np.stack([rows[0, b] for b in range(5)])
        got, sc = pool.get(pool.blocks, 0, np.arange(5)), pool.get_scale(pool.blocks, 0, np.arange(5))
        tol = ref.half_step(want, sc, store) * (1 + 1e-4) + 1e-5 * np.abs(want).max(-1, keepdims=True)
        assert (np.abs(got - want) <= tol).all(), (cut, np.abs(got - want).max())


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_with_a_channel_that_is_not_finite(dev, store, normalize, bad):
    """They read as NaN in every channel, in each format, the rows beside them as they are."""
    import kch
    rng = np.random.default_rng(34)
    for c, n in ((64, 24), (128, 24), (128, 1)):
        m2 = 8
        pool = ref.Pool(1, 1, 2, 16, c, store)
        C = torch.from_numpy(rng.standard_normal((24, c))).float().cuda()
        Z = torch.zeros_like(C)
        C[20, 7], C[5, c - 1] = bad, bad
        Bp = torch.zeros(m2, c).cuda()
        for a in range(0, 24, n):
            s, cu, cx, _ = ref.step([n], [a], [0])
            kch.hca_paged_append(C[a:a + n], Z[a:a + n], Bp, pool.rows, pool.scales, pool.state, pool.blocks, pool.ring,
                                 s, cu, cx, m2=m2, max_len=n, normalize=normalize)
        s, cu, _, _ = ref.step([3], [0], [0])
        keys = kch.paged_read(pool.rows, pool.scales, pool.blocks, s, cu, total=3, dtype=torch.float32)
        s, cu, _, _ = ref.step([24], [0], [0])
        win = kch.paged_read(pool.rows, pool.scales, pool.ring, s, cu, total=24, dtype=torch.float32)
        assert torch.isnan(keys[[0, 2]]).all() and torch.isfinite(keys[1]).all() and keys[1].abs().max() > 0
        ok = torch.ones(24, dtype=torch.bool)
        ok[20] = ok[5] = False
        assert torch.isnan(win[~ok]).all() and torch.isfinite(win[ok]).all() and (win[ok].abs().amax(-1) > 0).all()


# --------------------------------------------------------------------------- bits kept

# A rounding to a type whose half step is u is off by u / sqrt(3) sqrt(3 / (8 ln 2)) = 0.425 u of the value in the root
# mean square (values spread evenly over their logarithm). An output has two of them, its own and those of
# its weights, which for keys of random directions add up in norm as the weighted keys themselves do: 0.601 u
# of the output's norm, 2.35e-3 in bf16 and 2.94e-4 in fp16. A query of 16 bits has none: one rounded once more
# would move scores by 0.425 u |scale| / sqrt(c) in the root mean square, at |scale| = 64 and c = 128 seven
# times those bounds (c = 64: ten times). fp32 queries: what is left are fp32 sums of at most c products and
# the exponentials, a few 2^-24 of the scores' |scale| log2 e <= 93 and of the output: 16 2^-24 |scale| allowed.
def rms_bound(dtype, scale):
    u = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}.get(dtype)
    return 1.05 * 0.601 * u if u else 16 * 2.0 ** -24 * abs(scale)


BITS = [
    # lens, ctx, m2, win, nh, c, page, store
    ([1], [5003], 128, 128, 16, 128, 16, "bf16"),
    ([1, 1, 1], [40, 4095, 16383], 4, 77, 16, 128, 64, "e4m3"),
    ([8, 1, 3, 5], [100, 0, 63, 8190], 64, 16, 4, 64, 32, "int8"),
    ([4], [600], 16, 64, 16, 128, 64, "bf16"),
    ([90, 17], [9000, 3000], 8, 33, 2, 128, 64, "e4m3"),
    ([130, 1], [2000, 600], 16, 128, 16, 64, 32, "int8"),
    ([30], [50000], 16, 128, 16, 128, 64, "bf16"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -12, 37.0])
@pytest.mark.parametrize("i", range(len(BITS)))
def test_queries_keep_their_bits(dev, i, size, dtype):
    """Normalised queries of any length, at a scale where a rounding of theirs would show."""
    lens, ctx, m2, win, nh, c, page, store = BITS[i]
    rng = np.random.default_rng(600 + i)
    slots = list(rng.permutation(len(lens)))
    pool = ref.Pool(len(lens), *pages_for(lens, ctx, m2, win, page), page, c, store, seed=i)
    fill(pool, lens, ctx, slots, m2, win, rng)
    q = torch.from_numpy(size * rng.standard_normal((sum(lens), nh, c))).to("cuda", DT[dtype])
    for scale in (64.0, -64.0):
        out = run_attention(pool, q, lens, ctx, slots, m2, win, None, scale)
        want, _ = ref.attention(pool, f64(q), lens, ctx, slots, m2=m2, win=win, sink=None, scale=scale)
        err = np.linalg.norm(f64(out) - want) / np.linalg.norm(want)
        assert err <= rms_bound(dtype, scale), err


@pytest.mark.parametrize("n", [1, 40])
def test_fp32_queries_that_are_not_normalised(dev, n):
    rng = np.random.default_rng(35)
    m2, win, c, nh = 16, 32, 128, 16
    pool = ref.Pool(1, *pages_for([n], [700], m2, win, 32), 32, c, "bf16")
    fill(pool, [n], [700], [0], m2, win, rng, scale_rows=3.0)
    q = torch.from_numpy(rng.standard_normal((n, nh, c))).float().cuda()
    snk = rng.standard_normal(nh).astype(np.float32)
    out = run_attention(pool, q, [n], [700], [0], m2, win, snk, c ** -0.5, normalize_q=False)
    want, _ = ref.attention(pool, f64(q), [n], [700], [0], m2=m2, win=win, sink=snk, scale=c ** -0.5,
                            normalize_q=False)
    # scores of up to 3 |q| / sqrt(c) = 4: as |scale| = 4 of unit vectors
    assert np.linalg.norm(f64(out) - want) <= 16 * 2.0 ** -24 * 4 * np.linalg.norm(want)


def test_lengths_of_queries_past_the_sums(dev):
    """Queries of zeros, of an infinite sum of squares (normalised to zeros, as F.normalize in fp32) and NaN."""
    rng = np.random.default_rng(36)
    m2, win, c, nh = 16, 32, 128, 4
    for n in (4, 40):
        pool = ref.Pool(1, *pages_for([n], [300], m2, win, 32), 32, c, "e4m3")
        fill(pool, [n], [300], [0], m2, win, rng)
        for dtype in ("bf16", "fp32"):
            q = torch.from_numpy(rng.standard_normal((n, nh, c))).to("cuda", DT[dtype])
            q[0] = 0.0
            zero = run_attention(pool, q, [n], [300], [0], m2, win, None, 8.0)
            q[0] = 1e30
            big = run_attention(pool, q, [n], [300], [0], m2, win, None, 8.0)
            assert torch.equal(big, zero) and torch.isfinite(big).all()
            q[0, :, 3] = float("inf")
            q[1, 2, 5] = float("nan")
            out = run_attention(pool, q, [n], [300], [0], m2, win, None, 8.0)
            assert torch.isnan(out[0]).all() and torch.isnan(out[1, 2]).all()
            assert torch.equal(out[2:], big[2:]) and torch.equal(out[1, :2], big[1, :2])


# --------------------------------------------------------------------------- long contexts

LONG = [
    # lens, ctx, m2, win, nh, c, page, store
    ([1, 1, 1], [40, 4095, 7003], 1, 77, 16, 128, 64, "e4m3"),
    ([1], [49999], 4, 128, 16, 128, 16, "bf16"),
    ([2, 1], [7999, 6001], 1, 5, 16, 128, 32, "int8"),
    ([3, 1], [24003, 100], 4, 16, 4, 64, 1, "int8"),
    ([4], [12001], 1, 33, 16, 128, 64, "e4m3"),
    ([130, 7], [9001, 3000], 1, 128, 1, 128, 32, "bf16"),
    ([40, 30], [48000, 9], 4, 7, 4, 128, 64, "e4m3"),
    ([17], [6200], 1, 16, 6, 64, 128, "int8"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("i", range(len(LONG)))
def test_every_key_counts_once(dev, i, dtype):
    """Keys that are one unit vector each and queries of zeros: every channel of an output is how many keys have it
    over how many there are, at most 110 here: a key left out or taken twice, at a border of ranges, steps, tiles
    or pages, shows (one in 110 against half a step of 2^-8 and the fp32 sums)."""
    lens, ctx, m2, win, nh, c, page, store = LONG[i]
    rng = np.random.default_rng(700 + i)
    slots = list(rng.permutation(len(lens)))
    pool = ref.Pool(len(lens), *pages_for(lens, ctx, m2, win, page), page, c, store, seed=i)
    most = 0
    for slot, n, x in zip(slots, lens, ctx):
        nb, pos = (x + n) // m2, np.arange(max(0, x - win + 1), x + n)
        for table, at in ((pool.blocks, np.arange(nb)), (pool.ring, pos % pool.cap)):
            # channels in turn, the turn's start by the slot
            pool.put(table, slot, at, np.eye(c)[(np.arange(len(at)) * 7 + slot + (table is pool.ring)) % c])
        most = max(most, -(-nb // c) + -(-win // c))
    assert most <= 110
    q = torch.zeros(sum(lens), nh, c, device="cuda", dtype=DT[dtype])
    out = f64(run_attention(pool, q, lens, ctx, slots, m2, win, None, 8.0))
    want, _ = ref.attention(pool, np.zeros(q.shape), lens, ctx, slots, m2=m2, win=win, sink=None, scale=8.0)
    pos = np.concatenate([x + np.arange(n) for n, x in zip(lens, ctx)])
    seen = ((pos + 1) // m2 + np.minimum(pos + 1, win))[:, None, None]
    assert (np.abs(want * seen - np.rint(want * seen)) < 1e-6).all()
    assert (np.abs(out * seen - want * seen) < 0.45).all(), np.abs(out * seen - want * seen).max()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("i", range(len(LONG)))
def test_long_contexts_in_norm(dev, i, dtype):
    """Random keys, the error against the output's norm: a step of keys left out would be several per cent."""
    lens, ctx, m2, win, nh, c, page, store = LONG[i]
    rng = np.random.default_rng(800 + i)
    slots = list(rng.permutation(len(lens)))
    pool = ref.Pool(len(lens), *pages_for(lens, ctx, m2, win, page), page, c, store, seed=i)
    fill(pool, lens, ctx, slots, m2, win, rng)
    q = torch.from_numpy(rng.standard_normal((sum(lens), nh, c))).to("cuda", DT[dtype])
    snk = rng.standard_normal(nh).astype(np.float32)
    out = run_attention(pool, q, lens, ctx, slots, m2, win, snk, 11.3)
    want, _ = ref.attention(pool, f64(q), lens, ctx, slots, m2=m2, win=win, sink=snk, scale=11.3)
    err = np.linalg.norm(f64(out) - want) / np.linalg.norm(want)
    assert err <= rms_bound(dtype, 11.3), err


# --------------------------------------------------------------------------- the class and the layer

def test_class_and_layer_refuse_inputs_that_ask_for_gradients(dev):
    import kch
    cache = kch.HCAPagedCache(8, 64, 8, 8, max_seqs=1, max_tokens=64, max_chunk=4, page=16)
    s = cache.add()
    x, Bp = torch.ones(1, 64, device="cuda"), torch.zeros(8, 64, device="cuda")
    ask = lambda t: t.clone().requires_grad_()  # noqa: E731
    for args in ((ask(x), x, Bp), (x, ask(x), Bp), (x, x, ask(Bp))):
        with pytest.raises(NotImplementedError, match="no gradients"):
            cache.append_step([s], *args)
    assert cache.n_tokens(s) == 0
    with torch.no_grad():
        cache.append_step([s], ask(x), x, ask(Bp))
        want = cache.forward_step(ask(x)[:, None])
    with pytest.raises(NotImplementedError, match="no gradients"):
        cache.forward_step(ask(x)[:, None])
    with pytest.raises(NotImplementedError, match="no gradients"):
        cache.forward_step(x[:, None], sink_logits=torch.zeros(1, device="cuda", requires_grad=True))
    assert torch.equal(cache.forward_step(x[:, None]), want)

    cfg = kch.HybridConfig(d_model=128, hca_m2=16, hca_nh=2, hca_c=64, hca_dc=64, hca_sliding_window=24)
    layer = kch.HCAHybridLayer(cfg).cuda().bfloat16()
    served = layer.paged_cache(8, max_seqs=1, max_tokens=64, max_chunk=4, page=16)
    t = served.add()
    x = torch.randn(1, 128, device="cuda").bfloat16()
    for group in (0, 64):
        for kw in (dict(x=ask(x)), dict(x=x, residual=ask(x))):
            with pytest.raises(NotImplementedError, match="no gradients"):
                layer.forward_paged(kw.pop("x"), served, [t], weight_group=group, **kw)
        assert served.n_tokens(t) == 0
    # the layer's own weights are constants to it
    assert not layer.forward_paged(x, served, [t]).requires_grad
    with torch.no_grad():
        layer.forward_paged(ask(x), served, [t], residual=ask(x))
    assert served.n_tokens(t) == 2


def test_layer_refuses_a_cache_of_another_kind(dev):
    """A window or rows of another kind than its forward's would answer something else."""
    import kch
    cfg = kch.HybridConfig(d_model=128, hca_m2=16, hca_nh=2, hca_c=64, hca_dc=64, hca_sliding_window=24)
    layer = kch.HCAHybridLayer(cfg).cuda().bfloat16()
    x = torch.randn(1, 128, device="cuda").bfloat16()
    for c, m2, win, kw in ((64, 16, 8, {}), (64, 16, 0, {}), (64, 8, 24, {}), (32, 16, 24, {}),
                           (64, 16, 24, dict(normalize_qk=False))):
        cache = kch.HCAPagedCache(8, c, m2, win, max_seqs=1, max_tokens=64, page=32, **kw)
        s = cache.add()
        with pytest.raises(ValueError, match="forward_paged: the cache"):
            layer.forward_paged(x, cache, [s])
        assert cache.n_tokens(s) == 0
    cache = kch.HCAPagedCache(8, 64, 16, 24, max_seqs=1, max_tokens=64, page=32)
    assert layer.forward_paged(x, cache, [cache.add()]).shape == x.shape


def test_layer_refuses_before_the_tokens_are_appended(dev):
    """A call that fails leaves the sequences as they were: the same tokens can be sent again."""
    import kch
    cfg = kch.HybridConfig(d_model=128, hca_m2=16, hca_nh=2, hca_c=64, hca_dc=64, hca_sliding_window=24)
    layer = kch.HCAHybridLayer(cfg).cuda().bfloat16()
    cache = layer.paged_cache(8, max_seqs=1, max_tokens=64, max_chunk=4, page=32)
    s = cache.add()
    x = torch.randn(2, 128, device="cuda").bfloat16()
    for group, res in ((0, x[:, :64]), (0, x[None, :1, :64]), (0, x.repeat(2, 1)), (0, x.cpu()), (64, x[:1]), (64, x.float()),
                       (64, x.cpu())):
        with pytest.raises((ValueError, TypeError), match="residual"):
            layer.forward_paged(x, cache, [s], [2], residual=res, weight_group=group)
        assert cache.n_tokens(s) == 0, (group, res.shape)
    with pytest.raises(TypeError, match="weights"):
        layer.forward_paged(x.half(), cache, [s], [2])
    with pytest.raises(TypeError, match="bfloat16"):
        layer.forward_paged(x.float(), cache, [s], [2], weight_group=64)
    assert cache.n_tokens(s) == 0
    a = layer.forward_paged(x, cache, [s], [2], residual=x[:1])   # (broadcasts where no kernel adds it)
    assert a.shape == x.shape and cache.n_tokens(s) == 2


def test_four_bit_serving_holds_no_16_bit_copies(dev):
    import kch
    cfg = kch.HybridConfig(d_model=1024, hca_m2=16, hca_nh=16, hca_c=64, hca_dc=512, hca_sliding_window=24)
    layer = kch.HCAHybridLayer(cfg).cuda().bfloat16()
    cache = layer.paged_cache(8, max_seqs=1, max_tokens=64, page=32)
    s = cache.add()
    x = torch.randn(1, 1024, device="cuda").bfloat16()
    layer.forward_paged(x, cache, [s], weight_group=64)   # (the codes are made here)
    layer.invalidate_weight_cache()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    layer.forward_paged(x, cache, [s], weight_group=64)
    held = torch.cuda.memory_allocated() - before
    n = sum(p.numel() for p in (layer.W_KV.weight, layer.W_Z.weight, layer.W_DQ.weight, layer.W_UQ.weight,
                                layer.o_proj.weight))
    # codes, 16-bit scales and zero points a group, small vectors and the allocator's steps
    assert held <= n / 2 + 3 * n / 64 + 2 ** 18, (held, n)


@pytest.mark.parametrize("group", [0, 64])
def test_weights_put_where_freed_ones_were(dev, group):
    """A parameter replaced twice between two calls lies where the first one was: its copies are made anew."""
    import kch
    cfg = kch.HybridConfig(d_model=1024, hca_m2=16, hca_nh=16, hca_c=64, hca_dc=512, hca_sliding_window=24)
    layer = kch.HCAHybridLayer(cfg).cuda().bfloat16()
    x = torch.randn(1, 1024, device="cuda").bfloat16()

    def first_token():
        cache = layer.paged_cache(8, max_seqs=1, max_tokens=64, page=32)
        return layer.forward_paged(x, cache, [cache.add()], weight_group=group)

    def fresh():
        return torch.nn.Parameter(torch.randn(layer.W_KV.weight.shape, device="cuda", dtype=torch.bfloat16))

    layer.W_KV.weight = fresh()
    first_token()
    for _ in range(2):
        layer.W_KV.weight = fresh()
    got = first_token()
    layer.invalidate_weight_cache()
    assert torch.equal(got, first_token())
    twin = copy.deepcopy(layer)  # makes its own copies
    assert all(f._w is None for f in [twin._fused, twin._fused_step, *twin._fused_w4.values()])


# --------------------------------------------------------------------------- 4-bit weights

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K,G,zeros", [
    (1, 64, 256, 64, False), (5, 100, 96, 32, True), (16, 250, 512, 128, True), (3, 8212, 160, 32, True),
    (16, 16404, 192, 64, False), (33, 40, 128, 128, True),
])
def test_linear_w4_of_rows_that_are_not_finite(dev, dtype, M, N, K, G, zeros):
    """An infinite x gives the infinity of its weight's sign (NaN where the weight is zero or two of them differ), NaN
    gives NaN, values whose sums pass fp32 on the way what their weights make of them; other rows nothing."""
    import kch
    from test_w4_gpu import make, weights
    packed, scales, zp = make(N, K, G, zeros, dtype, M)
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(M, K, device="cuda", generator=g).to(DT[dtype])
    res = torch.randn(M, N, device="cuda", generator=g).to(DT[dtype])
    clean = kch.linear_w4(x, packed, scales, zp, residual=res)
    W = weights(packed, scales, zp, G)
    inf = float("inf")
    rows = [{0: inf}, {K - 1: -inf}, {3: inf, K // 2: inf}, {7: float("nan")}]
    if dtype == "bf16":
        rows += [{1: 3e38, 2: -3e38}, {K - 2: 1.5e37, 40: -2e37}]
    for at in rows:
        m = M - 1
        y = x.clone()
        for k, v in at.items():
            y[m, k] = v
        out = kch.linear_w4(y, packed, scales, zp, residual=res)
        assert torch.equal(out[:m], clean[:m]) if m else True
        with np.errstate(invalid="ignore", over="ignore"):
            xs = f64(y[m])
            want = np.array([sum(xs[k] * W[:, k] for k in at)]) + f64(res[m])
            rest = xs.copy()
            rest[list(at)] = 0.0
            want = torch.from_numpy(want[0] + W @ rest).to(DT[dtype]).float()
        got = out[m].float().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        assert (torch.sign(got) == torch.sign(want))[torch.isinf(want)].all()
        ok = torch.isfinite(want)
        # two roundings (this reference's and the operator's): a step apart at most. Where two terms past fp32's
        # sums cancel (equal weights), what was added between them is gone: a 64-bit sum of K terms is off by up to
        # K 2^-53 of the sum of their magnitudes, in whatever order
        with np.errstate(invalid="ignore", over="ignore"):
            lost = torch.from_numpy(K * 2.0 ** -53 * (np.abs(W) @ np.abs(xs)))
        tol = 2 * torch.finfo(DT[dtype]).eps * want.abs() + 1e-2 + torch.nan_to_num(lost, nan=0.0, posinf=0.0)
        assert ((got - want).abs() <= tol)[ok].all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,N,K,G,zeros", [
    # 512 tiles of 16 x 16 and more: two and four of them a workgroup, N no multiple of theirs, tails of K
    (3, 8212, 160, 32, True), (16, 8196, 256, 128, False), (33, 8212, 256, 128, True), (7, 8180, 192, 64, True),
    (16, 16404, 96, 32, True), (5, 16404, 192, 64, False), (1, 16388, 160, 32, False), (20, 8260, 224, 32, True),
    (9, 16372, 384, 128, True), (2, 8191, 160, 32, True),
])
def test_linear_w4_of_many_tiles(dev, dtype, residual, M, N, K, G, zeros):
    import kch
    from test_w4_gpu import check, make
    w = make(N, K, G, zeros, dtype, M + N)
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(M, K, device="cuda", generator=g).to(DT[dtype])
    res = torch.randn(M, N, device="cuda", generator=g).to(DT[dtype]) if residual else None
    check(kch.linear_w4(x, *w, residual=res), x, *w, G, dtype, res)
