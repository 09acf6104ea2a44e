"""Contract checks of the attention entry points, on the host: no launch, no GPU (CPU)."""

import ctypes

import pytest
import torch

import h3b200
from h3b200 import _lib

P = ctypes.c_void_p(256)     # any aligned address: the checks come before any use
BF16 = _lib.DTYPE_BF16


def _expect(rc, code, text):
    assert rc == code, _lib.load().h3b200_last_error()
    assert text in _lib.load().h3b200_last_error().decode()


def append(**kw):
    a = dict(q=P, q_st=256, q_sh=128, q_out=P, qo_st=256, qo_sh=128, q_weight=None, k=P, k_st=256, k_sh=128,
             k_weight=None, v=P, v_st=256, v_sh=128, k_cache=P, kc_sp=4096, kc_sh=2048, kc_sr=128, v_cache=P,
             vc_sp=4096, vc_sh=2048, vc_sr=128, pages=4, page_size=16, slots=P, slots_dtype=1, positions=P,
             positions_dtype=1, freqs=P, freqs_dtype=0, freqs_rows=64, f_st=256, rot_dim=128, eps=1e-6, dtype=BF16,
             tokens=3, heads=2, kv_heads=2, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().h3b200_append_paged_kv(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=0), _lib.ERR_INVALID, "dtype code"),
    (dict(page_size=12), _lib.ERR_INVALID, "page_size"),
    (dict(page_size=0), _lib.ERR_INVALID, "page_size"),
    (dict(pages=-1), _lib.ERR_INVALID, "page_size"),
    (dict(tokens=-1), _lib.ERR_INVALID, "bad shape"),
    (dict(kv_heads=0), _lib.ERR_INVALID, "bad shape"),
    (dict(heads=0), _lib.ERR_INVALID, "bad shape"),
    (dict(rot_dim=24), _lib.ERR_INVALID, "rot_dim"),
    (dict(rot_dim=144), _lib.ERR_INVALID, "rot_dim"),
    (dict(freqs_dtype=7), _lib.ERR_INVALID, "freqs dtype"),
    (dict(slots_dtype=2), _lib.ERR_INVALID, "int64"),
    (dict(positions=None, freqs_rows=2), _lib.ERR_INVALID, "rotation rows"),
    (dict(k_cache=None), _lib.ERR_INVALID, "NULL"),
    (dict(slots=None), _lib.ERR_INVALID, "NULL"),
    (dict(q_out=None), _lib.ERR_INVALID, "NULL"),
    (dict(k_st=100), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(k=ctypes.c_void_p(258)), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(vc_sr=4), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(f_st=255), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(freqs=ctypes.c_void_p(260)), _lib.ERR_UNSUPPORTED, "alignment"),
])
def test_append_refusals(kw, code, text):
    _expect(append(**kw), code, text)


def test_append_of_nothing():
    assert append(tokens=0, k=None, slots=None) == _lib.OK


def decode(**kw):
    a = dict(q=P, q_sb=256, q_sh=128, k=P, kc_sp=4096, kc_sh=2048, kc_sr=128, v=P, vc_sp=4096, vc_sh=2048, vc_sr=128,
             pages=4, page_size=16, table=P, pt_sb=4, width=4, lengths=P, out=P, o_sb=256, o_sh=128, lse=None, l_sb=2,
             l_sh=1, batch=1, heads=2, kv_heads=2, scale=0.1, dtype=BF16, workspace=P, nbytes=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().h3b200_paged_decode_attention(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=5), _lib.ERR_INVALID, "dtype code"),
    (dict(page_size=20), _lib.ERR_INVALID, "page_size"),
    (dict(heads=3), _lib.ERR_INVALID, "multiple of kv_heads"),
    (dict(kv_heads=0), _lib.ERR_INVALID, "multiple of kv_heads"),
    (dict(batch=-1), _lib.ERR_INVALID, "bad shape"),
    (dict(width=1 << 28), _lib.ERR_INVALID, "2^30"),
    (dict(scale=0.0), _lib.ERR_INVALID, "scale"),
    (dict(scale=float("nan")), _lib.ERR_INVALID, "scale"),
    (dict(scale=float("inf")), _lib.ERR_INVALID, "scale"),
    (dict(lengths=None), _lib.ERR_INVALID, "NULL"),
    (dict(table=None), _lib.ERR_INVALID, "NULL"),
    (dict(batch=64, width=1024, workspace=None), _lib.ERR_INVALID, "workspace"),
    (dict(batch=64, width=1024, workspace=ctypes.c_void_p(264), nbytes=1 << 40), _lib.ERR_INVALID, "workspace"),
    (dict(kc_sr=130), _lib.ERR_UNSUPPORTED, "alignment"),
    (dict(out=ctypes.c_void_p(264)), _lib.ERR_UNSUPPORTED, "alignment"),
])
def test_decode_refusals(kw, code, text):
    _expect(decode(**kw), code, text)


def test_decode_workspace():
    """One split or a cluster needs none; split sequences need their rows and statistics."""
    size = _lib.load().h3b200_paged_decode_workspace_bytes
    assert decode(batch=0, q=None) == _lib.OK
    assert size(0, 8, 8, 4, 16) == 0 and size(1, 3, 2, 4, 16) == 0
    assert size(1, 8, 8, 1, 16) == 0
    assert size(1, 8, 8, 64, 64) == 0                        # 8 heads x 8 splits: one cluster each
    long_one = size(1, 32, 4, 2000, 128)
    assert long_one > 0 and long_one % (8 * 520) == 0        # rows of 128 fp32 and (m, l), tiles of 8 heads
    assert size(64, 64, 8, 141, 64) % (8 * 520) == 0


def sparse(**kw):
    a = dict(q=P, q_st=256, q_sh=128, k=P, k_st=256, k_sh=128, v=P, v_st=256, v_sh=128, k_means=None, km_sh=0, km_sb=0,
             top_k=2, block=64, blocks=P, out=P, o_st=256, o_sh=128, lse=None, l_st=2, l_sh=1, queries=300, keys=300,
             heads=2, kv_heads=2, scale=0.1, causal=0, dtype=BF16, workspace=P, nbytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().h3b200_sparse_attention(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(heads=3), _lib.ERR_INVALID, "multiple of kv_heads"),
    (dict(queries=-1), _lib.ERR_INVALID, "bad shape"),
    (dict(keys=0), _lib.ERR_INVALID, "bad shape"),
    (dict(top_k=0), _lib.ERR_INVALID, "bad shape"),
    (dict(block=0), _lib.ERR_INVALID, "bad shape"),
    (dict(nbytes=100), _lib.ERR_INVALID, "workspace"),
    (dict(workspace=None), _lib.ERR_INVALID, "workspace"),
    (dict(dtype=0), _lib.ERR_INVALID, "dtype code"),
    (dict(v=None), _lib.ERR_INVALID, "NULL"),
    (dict(q_st=100), _lib.ERR_UNSUPPORTED, "alignment"),
])
def test_sparse_refusals(kw, code, text):
    _expect(sparse(**kw), code, text)


def test_block_sparse_refusals():
    lib = _lib.load()

    def call(block=64, top_k=2, keys=300, scale=0.1, queries=300, nbytes=1 << 40):
        return lib.h3b200_block_sparse_attention(P, 256, 128, P, 256, 128, P, 256, 128, P, top_k, block, P, 256, 128,
                                                 None, 2, 1, queries, keys, 2, 2, scale, 0, BF16, P, nbytes, None)

    _expect(call(block=96), _lib.ERR_UNSUPPORTED, "64 or 128")
    _expect(call(block=256), _lib.ERR_UNSUPPORTED, "64 or 128")
    _expect(call(top_k=1 << 25), _lib.ERR_INVALID, "top_k")
    _expect(call(keys=1 << 31), _lib.ERR_INVALID, "2^30")
    _expect(call(scale=-1.0), _lib.ERR_INVALID, "scale")
    _expect(call(nbytes=8), _lib.ERR_INVALID, "workspace")
    assert call(queries=0) == _lib.OK


def test_select_refusals():
    lib = _lib.load()

    def call(heads=2, kv=2, queries=300, keys=300, block=64, top_k=2):
        return lib.h3b200_select_key_blocks(P, P, 1280, 128, heads, kv, queries, keys, block, top_k, 0, P, None)

    _expect(call(heads=3), _lib.ERR_INVALID, "multiple of kv_heads")
    _expect(call(top_k=0), _lib.ERR_INVALID, "bad shape")
    _expect(call(block=0), _lib.ERR_INVALID, "bad shape")
    _expect(call(keys=64 * 30000), _lib.ERR_UNSUPPORTED, "key blocks")
    assert call(queries=0) == _lib.OK


def test_cpu_tensors_are_refused():
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    c = torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int64)
    t = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: h3b200.append_paged_kv(k, k, c, c, i),
                 lambda: h3b200.paged_decode_attention(k, c, c, t, t[:, 0].contiguous()),
                 lambda: h3b200.sparse_attention(k, k, k, 1),
                 lambda: h3b200.attention_block_means(k, 64),
                 lambda: h3b200.block_sparse_attention(k, k, k, torch.zeros(2, 1, 1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()
