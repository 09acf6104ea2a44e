"""What the block-sparse entry points refuse before they enqueue anything (CPU: a launch would give
a CUDA error, not the refusal that is expected here)."""

import ctypes

import pytest

from h3b200 import _lib
from test_attention_abi import BF16, P, _expect, sparse


def block_sparse(**kw):
    a = dict(q=P, q_st=256, q_sh=128, k=P, k_st=256, k_sh=128, v=P, v_st=256, v_sh=128, blocks=P, top_k=8, block=64,
             out=P, o_st=256, o_sh=128, lse=None, l_st=2, l_sh=1, queries=300, keys=900, heads=2, kv_heads=2,
             scale=0.1, causal=0, dtype=BF16, workspace=P, nbytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().h3b200_block_sparse_attention(*a.values())


@pytest.mark.parametrize("address", [256 + 16, 256 + 48, 256 + 8, 256 + 4])
@pytest.mark.parametrize("top_k", [1, 2, 64])
def test_workspace_alignment(address, top_k):
    """Split lists store their rows 32 bytes at a time: an address that is 16 modulo 32 is refused."""
    ws = ctypes.c_void_p(address)
    _expect(block_sparse(workspace=ws, top_k=top_k), _lib.ERR_INVALID, "misaligned")
    _expect(sparse(workspace=ws, top_k=top_k), _lib.ERR_INVALID, "misaligned")
