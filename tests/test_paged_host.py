"""The paged cache's and the 4-bit weights' C entry points refuse before any HIP call
(no GPU), and the layout queries."""

from __future__ import annotations

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from kch import _lib
    return _lib.load()


FAKE = 0x10000  # an aligned address that no refused call reads


def attn(lib, **k):
    a = dict(q=FAKE, sink=None, out=FAKE, rows=FAKE, scales=FAKE, bt=FAKE, rt=FAKE, slots=FAKE, cu=FAKE, ctx=FAKE,
             S=1, N=1, nh=4, c=64, m2=8, win=8, P=4, page=16, nbp=1, nrp=1, n_slots=1, max_len=1, max_ctx=8,
             scale=1.0, norm=1, tail=0, fmt=2, dt=1, ws=None, nbytes=0, stream=None)
    a.update(k)
    rc = lib.kch_hca_paged_attn(*a.values())
    return rc, lib.kch_last_error().decode()


@pytest.mark.parametrize("k,code,msg", [
    (dict(fmt=3), 1, "format"), (dict(fmt=-1), 1, "format"), (dict(c=96), 2, "c=96"), (dict(S=-1), 1, "bad sizes"),
    (dict(S=65535), 2, "65534"), (dict(page=24), 2, "power of two"), (dict(page=2048), 2, "power of two"),
    (dict(page=0), 2, "power of two"), (dict(dt=3), 1, "dtype"), (dict(m2=0), 1, "m2=0"), (dict(win=-1), 1, "win=-1"),
    (dict(nh=0), 1, "nh=0"), (dict(max_ctx=-1), 1, "max_ctx"), (dict(win=17), 1, "ring"),
    (dict(max_len=10), 1, "ring"), (dict(nrp=0, rt=None), 1, "without a ring"), (dict(q=None), 1, "null"),
    (dict(rows=None), 1, "null pool"), (dict(scales=None), 1, "null pool"), (dict(slots=None), 1, "null"),
    (dict(bt=None), 1, "null table"), (dict(q=FAKE + 8), 1, "aligned"), (dict(rows=FAKE + 4), 1, "aligned"),
    (dict(N=2 ** 29, nh=4), 1, "below 2^30"), (dict(nbp=2 ** 27, page=1024), 2, "table"),
    (dict(max_ctx=10 ** 6), 1, "workspace of"),
    (dict(max_ctx=10 ** 6, ws=FAKE + 64, nbytes=1 << 40), 1, "256-byte"),
])
def test_attention_refuses(lib, k, code, msg):
    rc, err = attn(lib, **k)
    assert rc == code and msg in err and err.startswith("kch_hca_paged_attn"), err


def test_nothing_to_do_is_fine(lib):
    assert attn(lib, N=0, q=None, out=None)[0] == 0
    assert attn(lib, S=0, q=None, slots=None, cu=None)[0] == 0
    assert attn(lib, max_len=0, q=None)[0] == 0


def test_append_refuses(lib):
    def app(**k):
        a = dict(C=FAKE, ldc=64, Z=FAKE, ldz=64, B=FAKE, rows=FAKE, scales=FAKE, state=FAKE, bt=FAKE, rt=FAKE,
                 slots=FAKE, cu=FAKE, ctx=FAKE, S=1, N=1, c=64, m2=8, P=4, page=16, nbp=1, nrp=1, n_slots=1,
                 max_len=1, norm=1, fmt=1, dt=1, stream=None)
        a.update(k)
        return lib.kch_hca_paged_append(*a.values()), lib.kch_last_error().decode()

    for k, code, msg in ((dict(m2=0), 1, "m2=0"), (dict(max_len=17), 1, "ring"), (dict(max_len=-1), 1, "max_len"),
                         (dict(C=None), 1, "null"), (dict(state=None), 1, "null"), (dict(ctx=None), 1, "null"),
                         (dict(ldc=63), 1, "aligned"), (dict(ldz=68), 1, "aligned"), (dict(C=FAKE + 2), 1, "aligned"),
                         (dict(dt=7), 1, "dtype"), (dict(c=32), 2, "c=32")):
        rc, err = app(**k)
        assert rc == code and msg in err, err
    assert app(S=0)[0] == 0 and app(N=0)[0] == 0 and app(max_len=0)[0] == 0


def test_read_and_w4_refuse(lib):
    def read(**k):
        a = dict(rows=FAKE, scales=FAKE, t=FAKE, slots=FAKE, cu=FAKE, first=None, out=FAKE, S=1, N=1, c=64, P=4,
                 page=16, nbp=1, n_slots=1, tail=1, fmt=1, dt=1, stream=None)
        a.update(k)
        return lib.kch_paged_read(*a.values()), lib.kch_last_error().decode()

    for k, code, msg in ((dict(dt=9), 1, "dtype"), (dict(out=None), 1, "null"), (dict(out=FAKE + 8), 1, "aligned"),
                         (dict(fmt=5), 1, "format"), (dict(N=-1), 1, "bad sizes")):
        rc, err = read(**k)
        assert rc == code and msg in err, err
    assert read(N=0)[0] == 0

    def w4(**k):
        a = dict(x=FAKE, ldx=64, codes=FAKE, s=FAKE, z=None, res=None, ldr=0, y=FAKE, ldy=8, M=1, N=8, K=64, G=32,
                 dt=1, stream=None)
        a.update(k)
        return lib.kch_linear_w4(*a.values()), lib.kch_last_error().decode()

    for k, code, msg in ((dict(dt=0), 2, "dtype"), (dict(G=48), 2, "group"), (dict(K=80, ldx=80), 2, "multiple"),
                         (dict(K=0), 2, "multiple"), (dict(M=-1), 1, "sizes"), (dict(x=None), 1, "null"),
                         (dict(s=None), 1, "null"), (dict(ldx=63), 1, "strides"), (dict(ldy=7), 1, "strides"),
                         (dict(res=FAKE, ldr=7), 1, "strides"), (dict(ldx=68), 2, "aligned"),
                         (dict(codes=FAKE + 8), 2, "aligned"), (dict(M=2 ** 21), 2, "rows")):
        rc, err = w4(**k)
        assert rc == code and msg in err, err
    assert w4(M=0, x=None)[0] == 0 and w4(N=0, y=None)[0] == 0


def test_workspace_query(lib):
    q = lib.kch_hca_paged_attn_ws_bytes
    assert q(1, 1, 16, 128, 128, 128, 1, 100) == 0          # one range of keys
    long = q(1, 1, 16, 128, 128, 128, 1, 10 ** 6)
    assert long > 0 and long % (16 * 130 * 4) == 0          # ranges times rows times (c + 2) floats
    assert q(1, 1, 16, 100, 128, 128, 1, 10 ** 6) == 0 and q(0, 0, 16, 128, 128, 128, 1, 10 ** 6) == 0
    assert q(4, 8192, 16, 128, 128, 128, 2048, 131072) == 0  # query tiles fill the device


def test_no_cpu_path():
    import kch
    z = torch.zeros(1, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kch.paged_read(z, None, i[None], i, torch.zeros(2, dtype=torch.int32), total=1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kch.linear_w4(z[0], torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(1, 8, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="kv_dtype"):
        kch.HCAPagedCache(4, 64, 8, 8, max_seqs=1, max_tokens=64, kv_dtype=torch.float16, device="cpu")
    for k, msg in ((dict(n_pages=0), "n_pages"), (dict(page=12), "power of two"), (dict(max_tokens=2 ** 31), "2\\*\\*31"),
                   (dict(max_chunk=0), "max_chunk"), (dict(win=-1), "win")):
        a = dict(n_pages=4, c=64, m2=8, win=8, max_seqs=1, max_tokens=64, device="cpu")
        a.update(k)
        with pytest.raises(ValueError, match=msg):
            kch.HCAPagedCache(a.pop("n_pages"), a.pop("c"), a.pop("m2"), a.pop("win"), **a)


def test_quantize_w4_on_the_cpu():
    import kch
    torch.manual_seed(0)
    w = torch.randn(24, 256)
    packed, scales, zeros = kch.quantize_w4(w, 64)
    assert packed.shape == (24, 128) and scales.shape == zeros.shape == (4, 24) and scales.dtype == torch.bfloat16
    p = packed.numpy()
    q = np.stack([p & 15, p >> 4], -1).reshape(24, 256).astype(np.float64)
    W = scales.float().double().numpy().repeat(64, 0).T * (q - zeros.numpy().repeat(64, 0).T)
    step = scales.float().double().numpy().repeat(64, 0).T
    assert (np.abs(W - w.double().numpy()) <= (0.5 + 2.0 ** -4 + 2.0 ** -3) * step).all()


def test_references_agree_with_the_oracle():
    """tests/paged_ref.py against the oracle's HCA cache, one token at a time."""
    import paged_ref as ref

    from oracle.caches import HCACacheOracle
    rng = np.random.default_rng(0)
    c, m2, win, nh, T = 64, 8, 12, 3, 30
    orc = HCACacheOracle(1, c, m2, win, "fp32")
    C, Z = rng.standard_normal((T, c)).astype(np.float32), rng.standard_normal((T, c)).astype(np.float32)
    Bp = rng.standard_normal((m2, c)).astype(np.float32)
    q = ref.unit(rng.standard_normal((T, nh, c)))
    sink = rng.standard_normal(nh).astype(np.float32)
    want = []
    for t in range(T):
        orc.append_step(C[None, t:t + 1], Z[None, t:t + 1], Bp)
        want.append(orc.forward_step(q[None, t:t + 1].astype(np.float32), sink_logits=sink)[0, 0])
    rows, wins, sums = ref.append(C, Z, Bp, [T], [0], [0], np.zeros((1, 3, c)), m2=m2)

    class Held:
        page, nbp, nrp = 8, 1, 8
        cap = 64
        blocks, ring = "blocks", "ring"

        def get(self, table, slot, index):
            src = rows if table == "blocks" else wins
            return np.array([src[slot, int(i)] for i in index]).reshape(-1, c)

    Held.c = c
    got, _ = ref.attention(Held(), q, [T], [0], [0], m2=m2, win=win, sink=sink, scale=1.0)
    assert np.abs(got - np.array(want)).max() < 1e-5
    # the sums left open give the block's row once it ends
    more = ref.append(C[:2], Z[:2], Bp, [2], [T], [0], {0: sums[0]}, m2=m2)[0]
    Cn, Zn = np.concatenate([C, C[:2]]), np.concatenate([Z, Z[:2]])
    whole = ref.append(Cn, Zn, Bp, [T + 2], [0], [0], np.zeros((1, 3, c)), m2=m2)[0]
    assert np.abs(more[0, T // m2] - whole[0, T // m2]).max() < 1e-12


def test_quantize_w4_of_a_transposed_weight():
    import kch
    torch.manual_seed(1)
    w = torch.randn(128, 24)
    for a, b in zip(kch.quantize_w4(w.t(), 32), kch.quantize_w4(w.t().contiguous(), 32)):
        assert torch.equal(a, b)
