"""Host side of the serving operators: layouts (no GPU)."""

from __future__ import annotations

import pytest
import torch
from test_paged_host import FAKE, attn


@pytest.fixture(scope="module")
def lib():
    from kch import _lib
    return _lib.load()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls would launch on addresses that are none")
@pytest.mark.parametrize("max_len", [0, 1, 2, 5])
@pytest.mark.parametrize("tail", [0, 1])
@pytest.mark.parametrize("max_ctx", [8, 10 ** 6, 2 ** 31 - 1])
def test_the_query_covers_what_the_call_takes(lib, max_len, tail, max_ctx):
    """A call with the workspace that the query says is not refused for it (it fails at its launch here)."""
    for N in (1, 3):
        n = lib.kch_hca_paged_attn_ws_bytes(1, N, 16, 128, 128, 8, max_len, max_ctx)
        rc, err = attn(lib, N=N, nh=16, c=128, m2=128, max_len=max_len, max_ctx=max_ctx, tail=tail,
                       ws=FAKE if n else None, nbytes=n)
        assert "workspace" not in err or rc == 0, err
        if max_len == 0:
            assert n == 0
