"""The HCA layer served from a paged cache (4-bit projections, quantised append, chunk attention, output
projection with the residual) against its own forward over the whole sequences."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(dtype):
    import kch
    torch.manual_seed(3)
    cfg = kch.HybridConfig(d_model=256, hca_m2=16, hca_nh=4, hca_c=64, hca_dc=128, hca_sliding_window=24)
    layer = kch.HCAHybridLayer(cfg).cuda().to(dtype).eval()
    with torch.no_grad():
        layer.sink.normal_()
        for lin in (layer.W_KV, layer.W_Z, layer.W_DQ, layer.W_UQ, layer.o_proj):
            lin.weight.normal_(std=lin.weight.shape[1] ** -0.5)
        layer.B_pos.normal_(std=0.3)
    return cfg, layer


def serve(layer, cache, X, residual, group, plan):
    """The packed steps of a plan [(sequences, lengths)] over whole sequences X, answers by sequence."""
    slots, at, out = [cache.add() for _ in X], [0] * len(X), [[] for _ in X]
    for seqs, lens in plan:
        pick = lambda Y: torch.cat([Y[s][at[s]:at[s] + n] for s, n in zip(seqs, lens)])  # noqa: E731
        y = layer.forward_paged(pick(X), cache, [slots[s] for s in seqs], lens,
                                residual=None if residual is None else pick(residual), weight_group=group)
        for s, n, part in zip(seqs, lens, y.split(list(lens))):
            out[s].append(part)
            at[s] += n
    return [torch.cat(o) for o in out]


PLAN = [([0, 1, 2], [40, 1, 17]), ([2, 0], [3, 1]), ([1], [50]), ([0, 1, 2], [1, 1, 1]), ([2, 1, 0], [30, 1, 8])]


# e4m3 rows are off by up to 2^-4 of a value, int8 ones by half a step of 1/127 of their largest, bf16 ones 2^-8:
# the output is a weighted mean of such rows (and the weights move by the same relative error at most twice), so it
# is within 3 such errors of the largest output, with the 16-bit roundings of q, P and the projections beside it
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv,tol", [(torch.bfloat16, 3e-2), (torch.float8_e4m3fn, 3 * 2.0 ** -4), (torch.int8, 6e-2)])
def test_layer_over_a_paged_cache(dev, dtype, kv, tol):
    cfg, layer = make(dtype)
    total = [sum(n for q, ns in PLAN for i, n in zip(q, ns) if i == s) for s in range(3)]
    X = [torch.randn(n, cfg.d_model, device="cuda").to(dtype) for n in total]
    res = [torch.randn_like(x) for x in X]
    cache = layer.paged_cache(40, max_seqs=3, max_tokens=128, max_chunk=50, page=16, kv_dtype=kv)
    got = serve(layer, cache, X, res, 0, PLAN)
    for x, r, y in zip(X, res, got):
        want, _ = layer(x[None])
        assert y.dtype == dtype
        err = (y.float() - r.float() - want[0].float()).abs().max()
        assert err <= tol * want.float().abs().max() + 2.0 ** -7 * 4, err


def test_four_bit_projections(dev):
    """With 4-bit weights: the same as the layer whose weights are the 4-bit ones' values."""
    import kch
    cfg, layer = make(torch.bfloat16)
    X = [torch.randn(n, cfg.d_model, device="cuda").bfloat16() for n in (50, 71, 51)]
    plan = [([0, 1, 2], [40, 60, 17]), ([2, 0, 1], [33, 9, 10]), ([0, 1, 2], [1, 1, 1])]
    run = lambda g: serve(layer, layer.paged_cache(40, max_seqs=3, max_tokens=128, max_chunk=60, page=16,  # noqa: E731
                                                   kv_dtype=torch.bfloat16), X, None, g, plan)
    got = run(64)
    again = run(64)
    assert all(torch.equal(a, b) for a, b in zip(got, again))

    def values(w):
        p, s, z = kch.quantize_w4(w, 64, dtype=torch.bfloat16)
        q = torch.stack([p & 15, p >> 4], -1).flatten(1).float()
        return (q - z.t().float().repeat_interleave(64, 1)) * s.t().float().repeat_interleave(64, 1)

    with torch.no_grad():
        proj = values(torch.cat([layer.W_KV.weight, layer.W_Z.weight, layer.W_DQ.weight]))
        for lin, w in zip((layer.W_KV, layer.W_Z, layer.W_DQ), proj.split([64, 64, 128])):
            lin.weight.copy_(w)
        layer.W_UQ.weight.copy_(values(layer.W_UQ.weight))
        layer.o_proj.weight.copy_(values(layer.o_proj.weight))
    # the values are rounded to bf16 in the layer (2^-8 each), in linear_w4 they are not
    for a, b in zip(got, run(0)):
        assert (a.float() - b.float()).abs().max() <= 4e-2 * b.float().abs().max()
    # changed weights are quantised anew
    layer.o_proj.weight.data.mul_(2.0)
    layer.invalidate_weight_cache()
    assert (run(64)[0].float() - 2 * got[0].float()).abs().max() <= 8e-2 * got[0].float().abs().max()


def test_layer_refuses(dev):
    cfg, layer = make(torch.bfloat16)
    cache = layer.paged_cache(8, max_seqs=1, max_tokens=64, max_chunk=4, page=16)
    s = cache.add()
    x = torch.randn(1, cfg.d_model, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="x must be"):
        layer.forward_paged(x[None], cache, [s])
    with pytest.raises(ValueError, match="group_size"):
        layer.forward_paged(x, cache, [s], weight_group=48)
    with pytest.raises(ValueError, match="must be"):
        layer.forward_paged(x, cache, [s], [2])
    assert cache.n_tokens(s) == 0
    assert layer.forward_paged(x, cache, [s]).shape == x.shape and cache.n_tokens(s) == 1
