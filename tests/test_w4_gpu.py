"""Linear maps with 4-bit weights on the GPU against 64-bit references.

Tolerance: half a step of the output's type (u = 2^-8 bf16, 2^-11 fp16) of the value,
and the fp32 sums. Within a group of G columns the kernel sums x (o + q) and x with o
= 128 (bf16) or 1024 (fp16): at most G + 2 roundings of 2^-24 of (o + 15) sum |x| each, times the
scale; the groups' results add K / G roundings of 2^-24 of the sum of their magnitudes.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
OFFSET = {"bf16": 128.0, "fp16": 1024.0}


def f64(t):
    return t.detach().float().cpu().double().numpy()


def make(N, K, G, zeros, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    packed = torch.randint(0, 256, (N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = (0.02 * (0.5 + torch.rand(K // G, N, device="cuda", generator=g))).to(DT[dtype])
    zp = torch.randint(0, 16, (K // G, N), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    return packed, scales, zp


def weights(packed, scales, zeros, G):
    p = packed.cpu().numpy()
    q = np.stack([p & 15, p >> 4], -1).reshape(p.shape[0], -1).astype(np.float64)
    z = 8.0 if zeros is None else f64(zeros).repeat(G, 0).T
    return f64(scales).repeat(G, 0).T * (q - z)


def check(y, x, packed, scales, zeros, G, dtype, res=None):
    xs = f64(x)
    want = xs @ weights(packed, scales, zeros, G).T
    ax = np.abs(xs).reshape(xs.shape[0], -1, G).sum(-1)            # [M, K / G]
    raw = (OFFSET[dtype] + 15) * ax @ f64(scales)                   # sum_g s_g (o + 15) sum |x|
    tol = 2.0 ** -24 * (G + 2 + ax.shape[1]) * raw
    if res is not None:
        want = want + f64(res)
    tol = tol + HALF[dtype] * (np.abs(want) + tol)
    err = np.abs(f64(y) - want)
    assert (err <= tol).all(), (err / tol).max()
    # roundings of independent signs: far below the sum of their bounds
    assert np.linalg.norm(err) <= 1.05 * HALF[dtype] * np.linalg.norm(want) + 1e-12


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K,G,zeros", [
    (1, 16, 32, 32, False), (1, 1, 64, 64, True), (3, 17, 96, 32, True), (16, 250, 128, 128, True),
    (5, 2072, 1056, 32, True), (1, 2048, 2048, 128, False), (16, 512, 4096, 64, True), (7, 48, 8192, 128, True),
    (17, 33, 320, 64, True), (50, 40, 384, 128, False), (2, 1030, 192, 64, False), (9, 4100, 640, 128, True),
])
def test_linear_w4(dev, dtype, M, N, K, G, zeros):
    import kch
    w = make(N, K, G, zeros, dtype, M + N)
    x = torch.randn(M, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(K)).to(DT[dtype])
    y = kch.linear_w4(x, *w)
    assert y.shape == (M, N) and y.dtype == x.dtype
    check(y, x, *w, G, dtype)
    res = torch.randn(M, N, device="cuda").to(DT[dtype])
    check(kch.linear_w4(x, *w, residual=res), x, *w, G, dtype, res)


def test_extreme_codes_are_exact(dev):
    """Codes 0 and 15 with zero points 0 and 15 on one-hot rows: single products, no rounding."""
    import kch
    N, K, G = 32, 128, 32
    packed = torch.randint(0, 256, (N, K // 2), device="cuda", dtype=torch.uint8)
    scales = torch.full((K // G, N), 0.5, device="cuda", dtype=torch.bfloat16)
    zeros = torch.tensor([0, 15, 8, 3], dtype=torch.uint8, device="cuda")[:, None].expand(4, N).contiguous()
    x = torch.zeros(16, K, device="cuda", dtype=torch.bfloat16)
    cols = [0, 1, 2, 3, 4, 5, 6, 7, 31, 32, 63, 64, 95, 96, 126, 127]
    x[range(16), cols] = 2.0
    y = kch.linear_w4(x, packed, scales, zeros)
    assert np.array_equal(f64(y), 2.0 * weights(packed, scales, zeros, G).T[cols])


def test_rows_of_other_layouts(dev):
    """Strided and misaligned rows, leading dimensions, no rows at all."""
    import kch
    N, K, G = 40, 256, 64
    w = make(N, K, G, True, "bf16", 1)
    big = torch.randn(4, K + 24, device="cuda").bfloat16()
    for x in (big[:, 8:8 + K], big[:, 3:3 + K], big[1:2, 5:5 + K], big.t().contiguous().t()[:, :K],
              big[::2, :K], big[:1, :K].expand(4, K)):
        check(kch.linear_w4(x, *w), x, *w, G, "bf16")
    y = kch.linear_w4(big[:, :K].reshape(2, 2, K), *w)
    assert y.shape == (2, 2, N)
    assert torch.equal(y.view(4, N), kch.linear_w4(big[:, :K], *w))
    wide = torch.randn(4, N + 7, device="cuda").bfloat16()
    for res in (wide[:, 3:3 + N], wide[:1, :N].expand(4, N)):
        check(kch.linear_w4(big[:, :K], *w, residual=res), big[:, :K], *w, G, "bf16", res)
    off = torch.zeros(N * K // 2 + 1, dtype=torch.uint8, device="cuda")[1:].view(N, K // 2)
    off.copy_(w[0])
    assert torch.equal(kch.linear_w4(big[:, :K], off, *w[1:]), kch.linear_w4(big[:, :K], *w))
    assert kch.linear_w4(big[:0, :K], *w).shape == (0, N)


@pytest.mark.parametrize("zero_points", [True, False])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_quantize_and_module(dev, zero_points, G):
    import kch
    torch.manual_seed(1)
    lin = torch.nn.Linear(256, 72, bias=False).cuda().bfloat16()
    with torch.no_grad():
        lin.weight[3] = 0.0
        lin.weight[4] = lin.weight[4].abs()
    m = kch.W4Linear.from_linear(lin, G, zero_points=zero_points)
    W = weights(m.packed, m.scales, m.zeros, G)
    # within half a step of the weight; a bf16 scale is off by 2^-8, which reaches 15 (7.5) codes of
    # the group's end: clamped there, at most 16 2^-8 of a step more
    step = f64(m.scales).repeat(G, 0).T
    assert (np.abs(W - f64(lin.weight)) <= (0.5 + (1.0 if zero_points else 0.0) * 2.0 ** -4 + 2.0 ** -3) * step + 1e-9).all()
    assert (W[3] == 0).all()
    x, res = torch.randn(2, 3, 256, device="cuda").bfloat16(), torch.randn(2, 3, 72, device="cuda").bfloat16()
    y = m(x, res)
    check(y.view(6, 72), x.view(6, 256), m.packed, m.scales, m.zeros, G, "bf16", res.view(6, 72))
    twin = kch.W4Linear(*[None if t is None else torch.zeros_like(t) for t in (m.packed, m.scales, m.zeros)])
    twin.load_state_dict(m.state_dict())
    assert torch.equal(twin(x, res), y) and (m.in_features, m.out_features) == (256, 72)


def test_captured_and_on_another_stream(dev):
    import kch
    w = make(96, 512, 128, True, "fp16", 2)
    x = torch.randn(4, 512, device="cuda").half()
    want = kch.linear_w4(x, *w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(kch.linear_w4(x, *w), want)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = kch.linear_w4(x, *w)
    for i in range(3):
        x.copy_(torch.randn(4, 512, device="cuda"))
        g.replay()
        assert torch.equal(y, kch.linear_w4(x, *w))


def test_refusals(dev):
    import kch
    N, K, G = 32, 128, 64
    packed, scales, zeros = make(N, K, G, True, "bf16", 3)
    x = torch.zeros(2, K, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        kch.linear_w4(x.float(), packed, scales, zeros)
    for args, msg in (((x[:, :64], packed, scales, zeros), "columns"), ((x, packed.int(), scales, zeros), "packed"),
                      ((x, packed, scales.half(), zeros), "scales"), ((x, packed, scales[:, :8], zeros), "scales"),
                      ((x, packed, scales, zeros.int()), "zeros"), ((x, packed, scales, zeros[:1]), "zeros"),
                      ((x, packed, scales.repeat(4, 1), None), "rows of scales"),
                      ((x, packed, scales[:1].contiguous().repeat(1, 1)[:0], None), "rows of scales")):
        with pytest.raises(ValueError, match=msg):
            kch.linear_w4(*args)
    with pytest.raises(ValueError, match="residual"):
        kch.linear_w4(x, packed, scales, zeros, residual=x)
    with pytest.raises(NotImplementedError, match="no gradients"):
        kch.linear_w4(x.clone().requires_grad_(), packed, scales, zeros)
    with pytest.raises(RuntimeError, match="GPU"):
        kch.linear_w4(x.cpu(), packed, scales, zeros)
    for w, g, msg in ((x, 48, "group_size"), (x[:, :100], 64, "group_size"), (x[0], 64, "weight")):
        with pytest.raises(ValueError, match=msg):
            kch.quantize_w4(w, g)
    with pytest.raises(ValueError, match="bias"):
        kch.W4Linear.from_linear(torch.nn.Linear(64, 8))


def test_scales_that_ask_for_gradients_are_refused(dev):
    import kch
    packed, scales, zeros = make(32, 128, 64, True, "bf16", 3)
    x = torch.zeros(2, 128, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="no gradients"):
        kch.linear_w4(x, packed, scales.clone().requires_grad_(), zeros)
