"""Attention after the Q/K/V build: paged key / value cache and block-sparse attention.

The tensors that :func:`h3b200.qkv_qknorm_rope` and the QK-norm-RoPE operators write are
read here. Like ``ops.py``: CUDA tensors only, outputs allocated with torch, work enqueued
on the current stream of the tensors' device, ``ValueError`` for arguments outside the
contract, ``NotImplementedError`` for valid ones that are not built, no fallback. Elements
are bf16 or fp16 (one type for all tensors of a call), the head dim is 128. The operators
are for inference: they record nothing for autograd.
"""

from __future__ import annotations

import contextlib
import math

import torch

from . import _lib
from .ops import _TABLE_DTYPE_CODES, _need_cuda, _stream

__all__ = [
    "append_paged_kv",
    "paged_decode_attention",
    "attention_block_means",
    "select_key_blocks",
    "block_sparse_attention",
    "sparse_attention",
]

HEAD_DIM = 128
QUERY_BLOCK = 128   # query rows that share a selection of key blocks
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_INDEX_CODES = {torch.int64: 1, torch.int32: 0}
_SCALE = 1.0 / math.sqrt(HEAD_DIM)


def _same_device(first: torch.Tensor, *ts):
    _need_cuda(first, *ts)
    for t in ts:
        if t is not None and t.device != first.device:
            raise ValueError(f"all tensors must be on one device, got {first.device} and {t.device}")


def _on(t: torch.Tensor):
    """The tensors' device for the launch (nothing to do when it is the current one)."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _dtype_code(t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"attention operators take bf16 or fp16 tensors, got {t.dtype}")
    return code


def _thd(t: torch.Tensor, name: str, dtype: torch.dtype) -> torch.Tensor:
    """[1, T, H, 128] / [T, H, 128] with unit stride on the head dim -> [T, H, 128] view."""
    if t.dim() == 4:
        if t.shape[0] != 1:
            raise ValueError(f"{name}: batch dimension must be 1 (packed token layout)")
        t = t[0]
    if t.dim() != 3 or t.shape[2] != HEAD_DIM:
        raise ValueError(f"{name}: expected [T, H, {HEAD_DIM}] or [1, T, H, {HEAD_DIM}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: head_dim must have unit stride")
    return t


def _cache(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    if t.dim() != 4 or t.shape[3] != HEAD_DIM:
        raise ValueError(f"{name}: expected [pages, kv_heads, page_size, {HEAD_DIM}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.stride(3) != 1:
        raise ValueError(f"{name}: head_dim must have unit stride")


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype) -> None:
    _cache(k_cache, "k_cache", dtype)
    _cache(v_cache, "v_cache", dtype)
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} must have the same shape")


def _groups(heads: int, kv_heads: int) -> None:
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a positive multiple of key heads ({kv_heads})")


def _weight(w: torch.Tensor | None, name: str, like: torch.Tensor) -> torch.Tensor | None:
    if w is None:
        return None
    w = w.detach().to(device=like.device, dtype=like.dtype).reshape(-1).contiguous()
    if w.numel() != HEAD_DIM:
        raise ValueError(f"{name} must have {HEAD_DIM} elements")
    return w


def _index(t: torch.Tensor | None, name: str, tokens: int) -> int:
    if t is None:
        return 1
    code = _INDEX_CODES.get(t.dtype)
    if code is None or t.dim() != 1 or t.shape[0] != tokens or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int64 or int32 tensor of {tokens} elements (one per token), got "
                         f"{t.dtype} {tuple(t.shape)}")
    return code


def append_paged_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    slots: torch.Tensor, frequencies: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                    q: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                    q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """New keys and values into a paged cache, K (and Q) normalised and rotated on the way.

    ``k``, ``v`` [T, kv_heads, 128] (or [1, T, ...]; views of a packed projection work) go to
    row ``slots[t] % page_size`` of page ``slots[t] // page_size`` of ``k_cache`` / ``v_cache``
    [pages, kv_heads, page_size, 128], in place (a cache kept as [pages, page_size, kv_heads,
    128] is passed as its ``transpose(1, 2)``). A token whose slot is -1 (or any value outside
    the pool) is padding: nothing of it is written, its ``q_out`` row included. The slots of
    one call must differ; which token a slot named twice ends up with is not defined.

    With ``k_weight`` [128], K gets per-head RMSNorm first; with ``frequencies`` [P, R / 2, 2,
    2] (or [1, P, 1, R / 2, 2, 2]; fp32, bf16 or fp16), split-half RoPE of its first R dims by
    row ``positions[t]``, or row t without ``positions``. A position outside the table gives
    NaN in the rotated dims. ``q`` [T, heads, 128] is normalised (``q_weight``) and rotated
    the same way into ``q_out`` (default: a new tensor; ``q`` itself works in place).

    Norm and rotation are fp32 and rounded once, at the store (:func:`h3b200.qknorm_rope_strided_`
    also rounds between the two, as the reference it reproduces does). Returns ``q_out``
    (None without ``q``)."""
    _same_device(k, v, k_cache, v_cache, slots, frequencies, positions, q, q_out)
    code = _dtype_code(k)
    k3, v3 = _thd(k, "k", k.dtype), _thd(v, "v", k.dtype)
    if k3.shape != v3.shape:
        raise ValueError(f"k {tuple(k3.shape)} and v {tuple(v3.shape)} must have the same shape")
    t, kv_heads, _ = k3.shape
    _caches(k_cache, v_cache, k.dtype)
    if k_cache.shape[1] != kv_heads:
        raise ValueError(f"the cache holds {k_cache.shape[1]} heads, k has {kv_heads}")
    if kv_heads == 0:
        raise ValueError("k and v need at least one head")
    slot_code = _index(slots, "slots", t)
    position_code = _index(positions, "positions", t)
    rows = stride = rot = table_code = 0
    f = frequencies
    if f is not None:
        if f.dim() == 6 and f.shape[0] == 1 and f.shape[2] == 1:
            f = f[0, :, 0]
        if f.dim() != 4 or f.shape[2] != 2 or f.shape[3] != 2:
            raise ValueError(f"frequencies must be [P, R / 2, 2, 2] or [1, P, 1, R / 2, 2, 2], got "
                             f"{tuple(frequencies.shape)}")
        if f.dtype not in _TABLE_DTYPE_CODES:
            raise ValueError(f"frequencies must be float32, float16 or bfloat16, got {f.dtype}")
        rot = 2 * f.shape[1]
        if rot == 0 or rot > HEAD_DIM or rot % 16:
            raise ValueError(f"frequencies must rotate a multiple of 16 dims, at most {HEAD_DIM}, got {rot}")
        if f.stride(3) != 1 or f.stride(2) != 2 or f.stride(1) != 4:
            f = f.contiguous()
        rows, stride, table_code = f.shape[0], f.stride(0), _TABLE_DTYPE_CODES[f.dtype]
        if positions is None and rows < t:
            raise ValueError(f"frequencies hold {rows} rows for {t} tokens; pass positions to pick rows")
    elif positions is not None:
        raise ValueError("positions need frequencies")
    kw, qw = _weight(k_weight, "k_weight", k3), None
    q3 = qo3 = None
    heads = 0
    if q is not None:
        q3 = _thd(q, "q", k.dtype)
        heads = q3.shape[1]
        if q3.shape[0] != t or heads == 0:
            raise ValueError(f"q must be [{t}, heads, {HEAD_DIM}], got {tuple(q3.shape)}")
        qw = _weight(q_weight, "q_weight", q3)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qo3 = _thd(q_out, "q_out", k.dtype)
        if qo3.shape != q3.shape:
            raise ValueError("q_out must have q's shape")
    elif q_weight is not None or q_out is not None:
        raise ValueError("q_weight and q_out need q")
    with _on(k3):
        _lib.call("h3b200_append_paged_kv", None if q3 is None else q3.data_ptr(), 0 if q3 is None else q3.stride(0),
                  0 if q3 is None else q3.stride(1), None if q3 is None else qo3.data_ptr(),
                  0 if q3 is None else qo3.stride(0), 0 if q3 is None else qo3.stride(1),
                  None if qw is None else qw.data_ptr(), k3.data_ptr(), k3.stride(0), k3.stride(1),
                  None if kw is None else kw.data_ptr(), v3.data_ptr(), v3.stride(0), v3.stride(1),
                  k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), v_cache.data_ptr(),
                  v_cache.stride(0), v_cache.stride(1), v_cache.stride(2), k_cache.shape[0], k_cache.shape[2],
                  slots.data_ptr(), slot_code, None if positions is None else positions.data_ptr(), position_code,
                  None if f is None else f.data_ptr(), table_code, rows, stride, rot, float(eps), code, t, heads,
                  kv_heads, _stream(k3))
    return q_out


def _scale_of(scale) -> float:
    if scale is None:
        return _SCALE
    scale = float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                           lengths: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                           return_lse: bool = False):
    """Attention of one new token per sequence over the pages :func:`append_paged_kv` fills.

    ``q`` [B, heads, 128]; ``k_cache`` / ``v_cache`` [pages, kv_heads, page_size, 128]
    (page_size a multiple of 8, heads a multiple of kv_heads); ``page_table`` int32 [B, width]:
    key j of sequence b is row ``j % page_size`` of page ``page_table[b, j // page_size]``;
    ``lengths`` int32 [B]: keys of each sequence, the new token's own among them (clamped to
    what the table holds). ``scale`` defaults to 1 / sqrt(128).

    A sequence without keys gives zeros (and lse -inf). Page ids outside the pool hold no
    keys. Rows behind a sequence's last key may hold anything. The work of a sequence is
    split over the GPU by its length at run time, so a captured graph stays valid while
    ``lengths`` and ``page_table`` change in place; the same inputs give the same bits.
    Returns ``out`` [B, heads, 128], with ``return_lse`` (out, fp32 [B, heads] log-sum-exp)."""
    _same_device(q, k_cache, v_cache, page_table, lengths, out)
    code = _dtype_code(q)
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or q.stride(2) != 1:
        raise ValueError(f"q must be [B, heads, {HEAD_DIM}] with unit stride on the head dim, got {tuple(q.shape)}")
    b, heads, _ = q.shape
    _caches(k_cache, v_cache, q.dtype)
    pages, kv_heads, page_size, _ = k_cache.shape
    _groups(heads, kv_heads)
    if page_size == 0 or page_size % 8:
        raise ValueError(f"page_size must be a positive multiple of 8, got {page_size}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b or (
            page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"page_table must be int32 [{b}, width] with unit stride, got {page_table.dtype} "
                         f"{tuple(page_table.shape)}")
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (b,) or not lengths.is_contiguous():
        raise ValueError(f"lengths must be a contiguous int32 tensor of {b} elements, got {lengths.dtype} "
                         f"{tuple(lengths.shape)}")
    scale = _scale_of(scale)
    if out is None:
        out = torch.empty((b, heads, HEAD_DIM), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError(f"out must be {q.dtype} {tuple(q.shape)} with unit stride on the head dim")
    lse = torch.empty((b, heads), dtype=torch.float32, device=q.device) if return_lse else None
    width = page_table.shape[1]
    with _on(q):
        nbytes = int(_lib.load().h3b200_paged_decode_workspace_bytes(b, heads, kv_heads, width, page_size))
        work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        _lib.call("h3b200_paged_decode_attention", q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(),
                  k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), v_cache.data_ptr(), v_cache.stride(0),
                  v_cache.stride(1), v_cache.stride(2), pages, page_size, page_table.data_ptr(), page_table.stride(0),
                  width, lengths.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1),
                  None if lse is None else lse.data_ptr(), heads, 1, b, heads, kv_heads, scale, code,
                  None if work is None else work.data_ptr(), nbytes, _stream(q))
    return (out, lse) if return_lse else out


def attention_block_means(x: torch.Tensor, block_size: int) -> torch.Tensor:
    """fp32 [H, ceil(T / block_size), 128] means of the blocks of ``x`` [T, H, 128].

    Summed in 64 bits and rounded once: :func:`select_key_blocks` compares products of
    them. A program that keeps its keys keeps their means too, and passes them to
    :func:`sparse_attention` as ``k_means``."""
    _need_cuda(x)
    code = _dtype_code(x)
    x3 = _thd(x, "x", x.dtype)
    block_size = int(block_size)
    if block_size <= 0 or block_size > 1 << 20:
        raise ValueError(f"block_size must be positive (at most 2^20), got {block_size}")
    t, h, _ = x3.shape
    means = torch.empty((h, -(-t // block_size), HEAD_DIM), dtype=torch.float32, device=x.device)
    with _on(x3):
        _lib.call("h3b200_attention_block_means", x3.data_ptr(), x3.stride(0), x3.stride(1), t, h, block_size, code,
                  means.data_ptr(), _stream(x3))
    return means


def _means(t: torch.Tensor, name: str, heads: int | None, blocks: int) -> None:
    if t.dtype != torch.float32 or t.dim() != 3 or t.shape[1:] != (blocks, HEAD_DIM) or not t.is_contiguous() or (
            heads is not None and t.shape[0] != heads):
        raise ValueError(f"{name} must be contiguous float32 [{heads or 'heads'}, {blocks}, {HEAD_DIM}], got {t.dtype} "
                         f"{tuple(t.shape)}")


def select_key_blocks(q_means: torch.Tensor, k_means: torch.Tensor, top_k: int, queries: int, keys: int,
                      block_size: int = 64, causal: bool = False) -> torch.Tensor:
    """Key blocks each 128-row query block attends to: int32 [kv_heads, query blocks, top_k].

    Row i of a key head holds the ``top_k`` blocks j with the highest ``q_means[h, i] .
    k_means[kv_head, j]``, summed over the query heads h of the group, in ascending order
    (equal scores: the lowest j), and -1 behind them when it can see fewer. Scores are held
    in 64 bits, so that the selection does not depend on a summation order.

    ``causal``: query row r stands at position ``r + keys - queries``. Blocks that start
    behind the query block are never selected, and those that reach into it come first."""
    _same_device(q_means, k_means)
    queries, keys, block_size, top_k = int(queries), int(keys), int(block_size), int(top_k)
    if queries < 0 or keys < 0 or block_size <= 0 or top_k <= 0:
        raise ValueError("top_k and block_size must be positive, queries and keys not negative")
    qb, kb = -(-queries // QUERY_BLOCK), -(-keys // block_size)
    _means(q_means, "q_means", None, qb)
    _means(k_means, "k_means", None, kb)
    heads, kv_heads = q_means.shape[0], k_means.shape[0]
    _groups(heads, kv_heads)
    blocks = torch.empty((kv_heads, qb, top_k), dtype=torch.int32, device=q_means.device)
    with _on(q_means):
        _lib.call("h3b200_select_key_blocks", q_means.data_ptr(), k_means.data_ptr(), heads, kv_heads, queries, keys,
                  block_size, top_k, int(bool(causal)), blocks.data_ptr(), _stream(q_means))
    return blocks


def _qkv(q, k, v):
    _same_device(q, k, v)
    code = _dtype_code(q)
    q3, k3, v3 = _thd(q, "q", q.dtype), _thd(k, "k", q.dtype), _thd(v, "v", q.dtype)
    if k3.shape != v3.shape:
        raise ValueError(f"k {tuple(k3.shape)} and v {tuple(v3.shape)} must have the same shape")
    _groups(q3.shape[1], k3.shape[1])
    if k3.shape[0] == 0:
        raise ValueError("k and v need at least one token")
    return q3, k3, v3, code


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor,
                           block_size: int = 64, scale: float | None = None, causal: bool = False,
                           out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of 128-row query blocks over the key blocks ``blocks`` lists.

    ``q`` [T, heads, 128], ``k`` / ``v`` [S, kv_heads, 128] (any token and head strides, e.g.
    HND-backed views); ``blocks`` int32 [kv_heads, ceil(T / 128), top_k] as
    :func:`select_key_blocks` returns it: ids outside the keys' blocks (-1) name none, an id
    named twice counts twice. ``block_size`` is 64 or 128 keys. With ``causal``, query row r
    sees the listed keys at positions up to ``r + S - T``. A row that sees no key gives
    zeros (and lse -inf). Under ``causal`` all values of a listed block must be finite: those
    a row may not see enter its products with weight zero.
    Returns ``out`` [T, heads, 128], with ``return_lse`` (out, fp32 [T, heads] log-sum-exp)."""
    q3, k3, v3, code = _qkv(q, k, v)
    _same_device(q3, blocks, out)
    t, heads, _ = q3.shape
    s, kv_heads, _ = k3.shape
    block_size = int(block_size)
    if block_size not in (64, 128):
        raise NotImplementedError(f"key blocks of 64 or 128 keys are built, got {block_size}")
    if blocks.dtype != torch.int32 or blocks.dim() != 3 or blocks.shape[:2] != (kv_heads, -(-t // QUERY_BLOCK)) or (
            blocks.shape[2] == 0 or not blocks.is_contiguous()):
        raise ValueError(f"blocks must be contiguous int32 [{kv_heads}, {-(-t // QUERY_BLOCK)}, top_k], got "
                         f"{blocks.dtype} {tuple(blocks.shape)}")
    scale = _scale_of(scale)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    o3 = _thd(out, "out", q.dtype)
    if o3.shape != q3.shape:
        raise ValueError("out must have q's shape")
    lse = torch.empty((t, heads), dtype=torch.float32, device=q.device) if return_lse else None
    top_k = blocks.shape[2]
    with _on(q3):
        nbytes = int(_lib.load().h3b200_block_sparse_workspace_bytes(t, heads, kv_heads, top_k, block_size))
        work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        _lib.call("h3b200_block_sparse_attention", q3.data_ptr(), q3.stride(0), q3.stride(1), k3.data_ptr(),
                  k3.stride(0), k3.stride(1), v3.data_ptr(), v3.stride(0), v3.stride(1), blocks.data_ptr(), top_k,
                  block_size, o3.data_ptr(), o3.stride(0), o3.stride(1), None if lse is None else lse.data_ptr(),
                  heads, 1, t, s, heads, kv_heads, scale, int(bool(causal)), code,
                  None if work is None else work.data_ptr(), nbytes, _stream(q3))
    return (out, lse) if return_lse else out


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, top_k: int, block_size: int = 64,
                     scale: float | None = None, causal: bool = False, k_means: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, return_lse: bool = False, return_blocks: bool = False):
    """Attention over the ``top_k`` key blocks that a cheap score selects for each query block.

    :func:`attention_block_means` of Q (blocks of 128) and K, :func:`select_key_blocks`, then
    :func:`block_sparse_attention`; see those for shapes and masks. ``k_means`` (float32
    [kv_heads, ceil(S / block_size), 128]) replaces the pass over K where a program keeps the
    means of its keys, as it does when it generates one token at a time. ``top_k`` of at
    least the number of key blocks is dense attention.
    Returns ``out``, or a tuple (out, lse, blocks) of what was asked for, in this order."""
    q3, k3, v3, _ = _qkv(q, k, v)
    top_k, block_size = int(top_k), int(block_size)
    if block_size not in (64, 128):
        raise NotImplementedError(f"key blocks of 64 or 128 keys are built, got {block_size}")
    if top_k <= 0:
        raise ValueError(f"top_k must be positive, got {top_k}")
    scale = _scale_of(scale)
    t, s = q3.shape[0], k3.shape[0]
    if k_means is None:
        k_means = attention_block_means(k3, block_size)
    else:
        _same_device(q3, k_means)
        _means(k_means, "k_means", k3.shape[1], -(-s // block_size))
    blocks = select_key_blocks(attention_block_means(q3, QUERY_BLOCK), k_means, top_k, t, s, block_size, causal)
    r = block_sparse_attention(q, k3, v3, blocks, block_size, scale, causal, out, return_lse)
    if not return_blocks:
        return r
    return (*r, blocks) if return_lse else (r, blocks)
