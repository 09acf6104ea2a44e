"""Attention after the Q/K/V build: paged key / value cache and block-sparse attention.

The tensors that :func:`h3b200.qkv_qknorm_rope` and the QK-norm-RoPE operators write are
read here. Like ``ops.py``: CUDA tensors only, outputs allocated with torch, work enqueued
on the current stream of the tensors' device, ``ValueError`` for arguments outside the
contract, ``NotImplementedError`` for valid ones that are not built, no fallback. Elements
are bf16 or fp16 (one type for all tensors of a call), the head dim is 128. The operators
are for inference: they record nothing for autograd.

Scores, sums and softmax statistics of the attention operators are fp32. The softmax
weights are rounded to the element type for the product with V (the tensor core's
operand), beside the rounding of the result: the worst error of a result is about twice
that of one rounding.

A call on one token is bound by the host, so each operator asks a tensor for its shape,
strides and type once and makes one call into the library.
"""

from __future__ import annotations

import contextlib
import math

import torch

from . import _lib
from .ops import _TABLE_DTYPE_CODES

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
_current = contextlib.nullcontext()


def _device(first, *ts) -> int:
    """Index of the CUDA device that holds every given tensor."""
    if not first.is_cuda:
        raise ValueError("h3b200 operators take CUDA tensors only (no CPU fallback)")
    index = first.get_device()
    for t in ts:
        if t is not None and t.get_device() != index:
            raise ValueError(f"all tensors must be on one device, got {[str(x.device) for x in (first, *ts) if x is not None]}")
    return index


def _on(index: int):
    """The tensors' device for the launch (nothing to do when it is the current one)."""
    return _current if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _dtype_code(t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"attention operators take bf16 or fp16 tensors, got {t.dtype}")
    return code


def _thd(t: torch.Tensor, name: str, dtype: torch.dtype):
    """(shape, strides) of [1, T, H, 128] / [T, H, 128] with unit stride on the head dim, as [T, H, 128]."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3 and shape[2] == HEAD_DIM and stride[2] == 1 and t.dtype is dtype:
        return shape, stride
    if len(shape) == 4:
        if shape[0] != 1:
            raise ValueError(f"{name}: batch dimension must be 1 (packed token layout)")
        shape, stride = shape[1:], stride[1:]
    if len(shape) != 3 or shape[2] != HEAD_DIM:
        raise ValueError(f"{name}: expected [T, H, {HEAD_DIM}] or [1, T, H, {HEAD_DIM}], got {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if stride[2] != 1:
        raise ValueError(f"{name}: head_dim must have unit stride")
    return shape, stride


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype):
    """(shape, K strides, V strides) of a paged cache."""
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) != 4 or shape[3] != HEAD_DIM:
        raise ValueError(f"k_cache: expected [pages, kv_heads, page_size, {HEAD_DIM}], got {tuple(shape)}")
    if v_cache.shape != shape:
        raise ValueError(f"k_cache {tuple(shape)} and v_cache {tuple(v_cache.shape)} must have the same shape")
    if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError(f"k_cache and v_cache must be {dtype}, got {k_cache.dtype} and {v_cache.dtype}")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("k_cache and v_cache: head_dim must have unit stride")
    if shape[2] == 0 or shape[2] % 8:
        raise ValueError(f"page_size must be a positive multiple of 8, got {shape[2]}")
    return shape, ks, vs


def _groups(heads: int, kv_heads: int) -> None:
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a positive multiple of key heads ({kv_heads})")


def _weight(w: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    if w.dtype is not like.dtype or w.get_device() != like.get_device() or not w.is_contiguous():
        w = w.detach().to(device=like.device, dtype=like.dtype).contiguous()
    if w.numel() != HEAD_DIM:
        raise ValueError(f"{name} must have {HEAD_DIM} elements")
    return w


def _index(t: torch.Tensor, name: str, tokens: int) -> int:
    code = _INDEX_CODES.get(t.dtype)
    if code is None or t.shape != (tokens,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int64 or int32 tensor of {tokens} elements (one per token), got "
                         f"{t.dtype} {tuple(t.shape)}")
    return code


def _scale_of(scale) -> float:
    if scale is None:
        return _SCALE
    scale = float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def append_paged_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    slots: torch.Tensor, frequencies: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                    q: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                    q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """New keys and values into a paged cache, K (and Q) normalised and rotated on the way.

    ``k``, ``v`` [T, kv_heads, 128] (or [1, T, ...]; views of a packed projection work) go to
    row ``slots[t] % page_size`` of page ``slots[t] // page_size`` of ``k_cache`` / ``v_cache``
    [pages, kv_heads, page_size, 128] (page_size a multiple of 8), in place (a cache kept as
    [pages, page_size, kv_heads, 128] is passed as its ``transpose(1, 2)``). A token whose slot
    is -1 (or any value outside the pool) is padding: nothing of it is written, its row of a
    given ``q_out`` included (a ``q_out`` made here has zeros there). The slots of one call must differ; which token a slot named twice ends up
    with is not defined.

    With ``k_weight`` [128], K gets per-head RMSNorm first; with ``frequencies`` [P, R / 2, 2,
    2] (or [1, P, 1, R / 2, 2, 2]; fp32, bf16 or fp16), split-half RoPE of its first R dims by
    row ``positions[t]``, or row t without ``positions``. A position outside the table gives
    NaN in the rotated dims. ``q`` [T, heads, 128] is normalised (``q_weight``) and rotated
    the same way into ``q_out`` (default: a new tensor, cleared first; ``q`` itself works in place).

    Norm and rotation are fp32 and rounded once, at the store (:func:`h3b200.qknorm_rope_strided_`
    also rounds between the two, as the reference it reproduces does). Returns ``q_out``
    (None without ``q``)."""
    dtype = k.dtype
    code = _dtype_code(k)
    dev = _device(k, v, k_cache, v_cache, slots, frequencies, positions, q, q_out)
    shape, ks = _thd(k, "k", dtype)
    vshape, vs = _thd(v, "v", dtype)
    t, kv_heads, _ = shape
    if vshape != shape or kv_heads == 0:
        raise ValueError(f"k {tuple(shape)} and v {tuple(vshape)} must have the same shape, with at least one head")
    cshape, kcs, vcs = _caches(k_cache, v_cache, dtype)
    if cshape[1] != kv_heads:
        raise ValueError(f"the cache holds {cshape[1]} heads, k has {kv_heads}")
    slot_code = _index(slots, "slots", t)
    position_code, position_ptr = 1, None
    freq_ptr, rows, stride, rot, table_code = None, 0, 0, 0, 0
    if frequencies is not None:
        f = frequencies
        fshape = f.shape
        if len(fshape) == 6 and fshape[0] == 1 and fshape[2] == 1:
            f = f[0, :, 0]
            fshape = f.shape
        if len(fshape) != 4 or fshape[2] != 2 or fshape[3] != 2:
            raise ValueError(f"frequencies must be [P, R / 2, 2, 2] or [1, P, 1, R / 2, 2, 2], got "
                             f"{tuple(frequencies.shape)}")
        table_code = _TABLE_DTYPE_CODES.get(f.dtype)
        if table_code is None:
            raise ValueError(f"frequencies must be float32, float16 or bfloat16, got {f.dtype}")
        rows, rot = fshape[0], 2 * fshape[1]
        if rot == 0 or rot > HEAD_DIM or rot % 16:
            raise ValueError(f"frequencies must rotate a multiple of 16 dims, at most {HEAD_DIM}, got {rot}")
        fs = f.stride()
        if fs[1:] != (4, 2, 1) or fs[0] % 2 or f.data_ptr() % 8:
            f = f.clone(memory_format=torch.contiguous_format)
            fs = f.stride()
        # a table without rows has no address, but is not "no rotation": nothing of it is read
        stride, freq_ptr = fs[0], f.data_ptr() if rows else k.data_ptr()
        if positions is not None:
            position_code, position_ptr = _index(positions, "positions", t), positions.data_ptr()
        elif rows < t:
            raise ValueError(f"frequencies hold {rows} rows for {t} tokens; pass positions to pick rows")
    elif positions is not None:
        raise ValueError("positions need frequencies")
    kw = kw_ptr = qw = qw_ptr = q_ptr = qo_ptr = None
    if k_weight is not None:
        kw = _weight(k_weight, "k_weight", k)
        kw_ptr = kw.data_ptr()
    qs = qos = (0, 0)
    heads = 0
    if q is not None:
        qshape, qs = _thd(q, "q", dtype)
        heads = qshape[1]
        if qshape[0] != t or heads == 0:
            raise ValueError(f"q must be [{t}, heads, {HEAD_DIM}], got {tuple(qshape)}")
        if q_weight is not None:
            qw = _weight(q_weight, "q_weight", q)
            qw_ptr = qw.data_ptr()
        if q_out is None:
            q_out = torch.zeros_like(q)  # the rows of padding tokens stay as they are
        qoshape, qos = _thd(q_out, "q_out", dtype)
        if qoshape != qshape:
            raise ValueError("q_out must have q's shape")
        q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_weight is not None or q_out is not None:
        raise ValueError("q_weight and q_out need q")
    with _on(dev):
        _lib.call("h3b200_append_paged_kv", q_ptr, qs[0], qs[1], qo_ptr, qos[0], qos[1], qw_ptr, k.data_ptr(), ks[0],
                  ks[1], kw_ptr, v.data_ptr(), vs[0], vs[1], k_cache.data_ptr(), kcs[0], kcs[1], kcs[2],
                  v_cache.data_ptr(), vcs[0], vcs[1], vcs[2], cshape[0], cshape[2], slots.data_ptr(), slot_code,
                  position_ptr, position_code, freq_ptr, table_code, rows, stride, rot, eps, code, t, heads, kv_heads,
                  _stream(dev))
    return q_out


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                           lengths: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                           return_lse: bool = False):
    """Attention of one new token per sequence over the pages :func:`append_paged_kv` fills.

    ``q`` [B, heads, 128]; ``k_cache`` / ``v_cache`` [pages, kv_heads, page_size, 128]
    (page_size a multiple of 8, width * page_size at most 2^30, heads a multiple of
    kv_heads); ``page_table`` int32 [B, width]:
    key j of sequence b is row ``j % page_size`` of page ``page_table[b, j // page_size]``;
    ``lengths`` int32 [B]: keys of each sequence, the new token's own among them (clamped to
    what the table holds). ``scale`` defaults to 1 / sqrt(128).

    A sequence without keys gives zeros (and lse -inf). Page ids outside the pool hold no
    keys. Rows behind a sequence's last key may hold anything. The work of a sequence is
    split over the GPU by its length at run time, so a captured graph stays valid while
    ``lengths`` and ``page_table`` change in place; the same inputs give the same bits.
    Returns ``out`` [B, heads, 128], with ``return_lse`` (out, fp32 [B, heads] log-sum-exp)."""
    dtype = q.dtype
    code = _dtype_code(q)
    dev = _device(q, k_cache, v_cache, page_table, lengths, out)
    qshape, qs = q.shape, q.stride()
    if len(qshape) != 3 or qshape[2] != HEAD_DIM or qs[2] != 1:
        raise ValueError(f"q must be [B, heads, {HEAD_DIM}] with unit stride on the head dim, got {tuple(qshape)}")
    b, heads, _ = qshape
    (pages, kv_heads, page_size, _), ks, vs = _caches(k_cache, v_cache, dtype)
    _groups(heads, kv_heads)
    tshape, ts = page_table.shape, page_table.stride()
    if page_table.dtype is not torch.int32 or len(tshape) != 2 or tshape[0] != b or (tshape[1] > 1 and ts[1] != 1):
        raise ValueError(f"page_table must be int32 [{b}, width] with unit stride, got {page_table.dtype} "
                         f"{tuple(tshape)}")
    if lengths.dtype is not torch.int32 or lengths.shape != (b,) or not lengths.is_contiguous():
        raise ValueError(f"lengths must be a contiguous int32 tensor of {b} elements, got {lengths.dtype} "
                         f"{tuple(lengths.shape)}")
    scale = _scale_of(scale)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != qshape or out.dtype is not dtype or out.stride(2) != 1:
        raise ValueError(f"out must be {dtype} {tuple(qshape)} with unit stride on the head dim")
    lse = lse_ptr = work = work_ptr = None
    if return_lse:
        lse = q.new_empty((b, heads), dtype=torch.float32)
        lse_ptr = lse.data_ptr()
    width = tshape[1]
    os = out.stride()
    with _on(dev):
        nbytes = _lib.load().h3b200_paged_decode_workspace_bytes(b, heads, kv_heads, width, page_size)
        if nbytes:
            work = q.new_empty(nbytes, dtype=torch.uint8)
            work_ptr = work.data_ptr()
        _lib.call("h3b200_paged_decode_attention", q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), ks[0], ks[1], ks[2],
                  v_cache.data_ptr(), vs[0], vs[1], vs[2], pages, page_size, page_table.data_ptr(), ts[0], width,
                  lengths.data_ptr(), out.data_ptr(), os[0], os[1], lse_ptr, heads, 1, b, heads, kv_heads, scale, code,
                  work_ptr, nbytes, _stream(dev))
    return (out, lse) if return_lse else out


def attention_block_means(x: torch.Tensor, block_size: int) -> torch.Tensor:
    """fp32 [H, ceil(T / block_size), 128] means of the blocks of ``x`` [T, H, 128].

    Summed in 64 bits and rounded once: :func:`select_key_blocks` compares products of
    them. A program that keeps its keys keeps their means too, and passes them to
    :func:`sparse_attention` as ``k_means``."""
    code = _dtype_code(x)
    dev = _device(x)
    (t, h, _), xs = _thd(x, "x", x.dtype)
    block_size = int(block_size)
    if block_size <= 0 or block_size > 1 << 20:
        raise ValueError(f"block_size must be positive (at most 2^20), got {block_size}")
    means = torch.empty((h, -(-t // block_size), HEAD_DIM), dtype=torch.float32, device=x.device)
    with _on(dev):
        _lib.call("h3b200_attention_block_means", x.data_ptr(), xs[0], xs[1], t, h, block_size, code,
                  means.data_ptr(), _stream(dev))
    return means


def _means(t: torch.Tensor, name: str, heads: int | None, blocks: int) -> None:
    if t.dtype is not torch.float32 or t.dim() != 3 or t.shape[1:] != (blocks, HEAD_DIM) or t.stride(2) != 1 or (
            heads is not None and t.shape[0] != heads):
        raise ValueError(f"{name} must be float32 [{heads or 'heads'}, {blocks}, {HEAD_DIM}] with unit stride on the "
                         f"head dim, got {t.dtype} {tuple(t.shape)}")


def select_key_blocks(q_means: torch.Tensor, k_means: torch.Tensor, top_k: int, queries: int, keys: int,
                      block_size: int = 64, causal: bool = False) -> torch.Tensor:
    """Key blocks each 128-row query block attends to: int32 [kv_heads, query blocks, top_k].

    Row i of a key head holds the ``top_k`` blocks j with the highest ``q_means[h, i] .
    k_means[kv_head, j]``, summed over the query heads h of the group, in ascending order
    (equal scores: the lowest j), and -1 behind them when it can see fewer. Scores are held
    in 64 bits: another summation order changes a selection only where two scores agree to
    about 1e-16 of their terms. At most 24,556 key blocks are built.

    ``causal``: query row r stands at position ``r + keys - queries``. Blocks that start
    behind the query block are never selected, and those that reach into it come first, the
    lowest of them before the others: with ``top_k`` below their number (up to 3 blocks of
    64, 2 of 128) the last rows do not see their own positions."""
    dev = _device(q_means, k_means)
    queries, keys, block_size, top_k = int(queries), int(keys), int(block_size), int(top_k)
    if queries < 0 or keys < 0 or not 0 < block_size <= 1 << 20 or not 0 < top_k <= 1 << 24:
        raise ValueError(f"top_k ({top_k}) and block_size ({block_size}) must be positive (at most 2^24 and 2^20), "
                         "queries and keys not negative")
    qb, kb = -(-queries // QUERY_BLOCK), -(-keys // block_size)
    _means(q_means, "q_means", None, qb)
    _means(k_means, "k_means", None, kb)
    heads, kv_heads = q_means.shape[0], k_means.shape[0]
    _groups(heads, kv_heads)
    q_means = q_means.contiguous()
    blocks = torch.empty((kv_heads, qb, top_k), dtype=torch.int32, device=q_means.device)
    with _on(dev):
        _lib.call("h3b200_select_key_blocks", q_means.data_ptr(), k_means.data_ptr(), k_means.stride(0),
                  k_means.stride(1), heads, kv_heads, queries, keys, block_size, top_k, int(bool(causal)),
                  blocks.data_ptr(), _stream(dev))
    return blocks


def _qkv(q, k, v):
    dtype = q.dtype
    code = _dtype_code(q)
    qshape, qs = _thd(q, "q", dtype)
    kshape, ks = _thd(k, "k", dtype)
    vshape, vs = _thd(v, "v", dtype)
    if kshape != vshape or kshape[0] == 0:
        raise ValueError(f"k {tuple(kshape)} and v {tuple(vshape)} must have the same shape, with at least one token")
    _groups(qshape[1], kshape[1])
    return code, qshape, qs, kshape, ks, vs


def _block_size(block_size) -> int:
    block_size = int(block_size)
    if block_size not in (64, 128):
        raise NotImplementedError(f"key blocks of 64 or 128 keys are built, got {block_size}")
    return block_size


def _out(out, q, qshape):
    """(out, its [T, H] strides)."""
    if out is None:
        out = torch.empty_like(q)
    oshape, os = _thd(out, "out", q.dtype)
    if oshape != qshape:
        raise ValueError("out must have q's shape")
    return out, os


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor,
                           block_size: int = 64, scale: float | None = None, causal: bool = False,
                           out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of 128-row query blocks over the key blocks ``blocks`` lists.

    ``q`` [T, heads, 128], ``k`` / ``v`` [S, kv_heads, 128] (any token and head strides, e.g.
    HND-backed views; expanded dims, of stride 0, are not built for more than one query);
    ``blocks`` int32 [kv_heads, ceil(T / 128), top_k] as
    :func:`select_key_blocks` returns it: ids outside the keys' blocks (-1) name none, an id
    named twice counts twice. ``block_size`` is 64 or 128 keys. With ``causal``, query row r
    sees the listed keys at positions up to ``r + S - T``. A row that sees no key gives
    zeros (and lse -inf). Under ``causal`` all values of a listed block must be finite: those
    a row may not see enter its products with weight zero. ``out`` may be ``q``, but must not
    overlap ``k`` or ``v``.
    Returns ``out`` [T, heads, 128], with ``return_lse`` (out, fp32 [T, heads] log-sum-exp)."""
    dev = _device(q, k, v, blocks, out)
    code, qshape, qs, kshape, ks, vs = _qkv(q, k, v)
    t, heads, _ = qshape
    s, kv_heads, _ = kshape
    block_size = _block_size(block_size)
    bshape = blocks.shape
    if blocks.dtype is not torch.int32 or len(bshape) != 3 or bshape[:2] != (kv_heads, -(-t // QUERY_BLOCK)) or (
            bshape[2] == 0 or not blocks.is_contiguous()):
        raise ValueError(f"blocks must be contiguous int32 [{kv_heads}, {-(-t // QUERY_BLOCK)}, top_k], got "
                         f"{blocks.dtype} {tuple(bshape)}")
    scale = _scale_of(scale)
    out, os = _out(out, q, qshape)
    lse = torch.empty((t, heads), dtype=torch.float32, device=q.device) if return_lse else None
    top_k = bshape[2]
    with _on(dev):
        nbytes = _lib.load().h3b200_block_sparse_workspace_bytes(t, heads, kv_heads, top_k, block_size)
        work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        _lib.call("h3b200_block_sparse_attention", q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1],
                  v.data_ptr(), vs[0], vs[1], blocks.data_ptr(), top_k, block_size, out.data_ptr(), os[0], os[1],
                  None if lse is None else lse.data_ptr(), heads, 1, t, s, heads, kv_heads, scale, int(bool(causal)),
                  code, None if work is None else work.data_ptr(), nbytes, _stream(dev))
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
    dev = _device(q, k, v, k_means, out)
    code, qshape, qs, kshape, ks, vs = _qkv(q, k, v)
    t, heads, _ = qshape
    s, kv_heads, _ = kshape
    top_k, block_size = int(top_k), _block_size(block_size)
    if not 0 < top_k <= 1 << 24:
        raise ValueError(f"top_k must be positive (at most 2^24), got {top_k}")
    scale = _scale_of(scale)
    km_ptr, kms = None, (0, 0)
    if k_means is not None:
        _means(k_means, "k_means", kv_heads, -(-s // block_size))
        km_ptr, kms = k_means.data_ptr(), k_means.stride()
    out, os = _out(out, q, qshape)
    lse = q.new_empty((t, heads), dtype=torch.float32) if return_lse else None
    blocks = q.new_empty((kv_heads, -(-t // QUERY_BLOCK), top_k), dtype=torch.int32)
    with _on(dev):
        nbytes = _lib.load().h3b200_sparse_attention_workspace_bytes(t, s, heads, kv_heads, top_k, block_size,
                                                                     k_means is not None)
        work = q.new_empty(nbytes, dtype=torch.uint8)
        _lib.call("h3b200_sparse_attention", q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(),
                  vs[0], vs[1], km_ptr, kms[0], kms[1], top_k, block_size, blocks.data_ptr(), out.data_ptr(), os[0],
                  os[1], None if lse is None else lse.data_ptr(), heads, 1, t, s, heads, kv_heads, scale,
                  int(bool(causal)), code, work.data_ptr(), nbytes, _stream(dev))
    if return_lse:
        return (out, lse, blocks) if return_blocks else (out, lse)
    return (out, blocks) if return_blocks else out
