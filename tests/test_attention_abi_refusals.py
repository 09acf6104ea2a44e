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


NOT_SPARSE = [
    (dict(block=96), _lib.ERR_UNSUPPORTED, "64 or 128"),
    (dict(block=256), _lib.ERR_UNSUPPORTED, "64 or 128"),
    (dict(scale=float("nan")), _lib.ERR_INVALID, "scale"),
    (dict(scale=-1.0), _lib.ERR_INVALID, "scale"),
    (dict(keys=1 << 31), _lib.ERR_INVALID, "2^30"),
    (dict(queries=1 << 31), _lib.ERR_INVALID, "2^30"),
    (dict(top_k=1 << 25), _lib.ERR_INVALID, "keys"),
    (dict(top_k=1 << 62), _lib.ERR_INVALID, "keys"),
    (dict(q=ctypes.c_void_p(264)), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(out=ctypes.c_void_p(264)), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(o_sh=100), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(v_st=100), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(k_st=0), _lib.ERR_UNSUPPORTED, "stride"),      # broadcast dims have no tensor map
    (dict(k_sh=0), _lib.ERR_UNSUPPORTED, "stride"),
    (dict(v_sh=0), _lib.ERR_UNSUPPORTED, "stride"),
    (dict(q_sh=0), _lib.ERR_UNSUPPORTED, "stride"),
    (dict(q_st=-256), _lib.ERR_UNSUPPORTED, "stride"),
    (dict(v_st=1 << 39), _lib.ERR_UNSUPPORTED, "stride"),
]


@pytest.mark.parametrize("kw,code,text", NOT_SPARSE)
@pytest.mark.parametrize("call", [block_sparse, sparse])
def test_refused_before_any_launch(call, kw, code, text):
    """h3b200_sparse_attention launches the means and the selection first: what its attention refuses has to be
    refused before them."""
    _expect(call(**kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(keys=64 * 30000), _lib.ERR_UNSUPPORTED, "key blocks"),
    (dict(top_k=(1 << 24) + 1, block=64), _lib.ERR_INVALID, "keys"),
    (dict(k_means=P, km_sb=130, km_sh=1300), _lib.ERR_UNSUPPORTED, "stride"),
    (dict(k_means=ctypes.c_void_p(264), km_sb=128, km_sh=640), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(queries=1, scale=0.0, k_means=P, km_sb=128, km_sh=640), _lib.ERR_INVALID, "scale"),
    (dict(queries=1, v_st=100, k_means=P, km_sb=128, km_sh=640), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(blocks=None), _lib.ERR_INVALID, "NULL"),
])
def test_combined_call_refused_before_any_launch(kw, code, text):
    _expect(sparse(**kw), code, text)
