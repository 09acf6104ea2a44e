"""Edges of the attention operators on the GPU: weights far below their row's largest one, rotation
tables without rows, outputs made inside a call, captured appends, and lists and grids longer than
what the block-sparse kernel reads of them at once. References and tolerances as in
test_gpu_attention.py, where a test says nothing else.
"""

import math

import pytest
import torch

import h3b200
from test_gpu_attention import (D, F64, _gen, attend64, check_attention, check_decode, half_step, list_mask, randn,
                                table, tiny)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# small weights
# ---------------------------------------------------------------------------


def faint_keys(gen, n, kv, dtype):
    """(k, v) of n keys: the first one outweighs every other by 2^22 to 2^33 for a query of 16 in dim 0 and
    0 elsewhere, and its value is 0, so that the result consists of the faint keys' values alone."""
    k = torch.zeros(n, kv, D, device="cuda")
    fade = 22 + 11 * torch.rand(n, kv, generator=gen, device="cuda")
    k[..., 0] = -fade * math.log(2.0) / (16 * D ** -0.5)
    k[0] = 0.0
    v = 64 * (torch.rand(n, kv, D, generator=gen, device="cuda") + 0.5)
    v[0] = 0.0
    return k.to(dtype), v.to(dtype)


def check_faint(out, lse, q, k, v, smallest):
    """As check_attention, but a weight is held to half of `smallest`, the step of the smallest weights that the
    kernel keeps, relative to the row's largest one."""
    mask = torch.ones(q.shape[0], k.shape[0], dtype=torch.bool, device="cuda")
    o, ls, pv, a, n = attend64(q, k, v, mask, D ** -0.5)
    h = half_step(q.dtype)
    e = (128 * 2.0 ** -24 * a)[:, None]
    tol = pv * (h + 2 * e + 2.0 ** -20 + 2 * k.shape[0] * 2.0 ** -24) + h * o.abs() + tiny(q.dtype) + (
        k.shape[0] * smallest / 2 * float(v.abs().max()))
    off = (out.to(F64) - o).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol).max())} of the tolerance"
    assert bool(((lse.to(F64) - ls).abs() <= e[:, 0] + 2.0 ** -20 + k.shape[0] * 2.0 ** -24 + 2.0 ** -23 * ls.abs()).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,batch,heads,kv", [(777, 1, 8, 8), (3001, 1, 2, 1), (600, 500, 4, 1), (9000, 200, 4, 2),
                                                (60000, 2, 20, 1)])
def test_decode_keeps_faint_weights(dtype, n, batch, heads, kv):
    """fp16 weights keep 39 bits below the largest: 2^15 times as many as fp16 itself has below 1."""
    gen = _gen(n)
    k, v = faint_keys(gen, n, kv, dtype)
    page = 64
    width = -(-n // page)
    pad = torch.zeros(width * page - n, kv, D, dtype=dtype, device="cuda")
    kc, vc = (torch.cat((x, pad)).reshape(width, page, kv, D).transpose(1, 2) for x in (k, v))
    tab = torch.arange(width, dtype=torch.int32, device="cuda").expand(batch, width)
    q = torch.zeros(batch, heads, D, dtype=dtype, device="cuda")
    q[..., 0] = 16.0
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out, lse = h3b200.paged_decode_attention(q, kc, vc, tab, lens, return_lse=True)
    smallest = 2.0 ** -39 if dtype is torch.float16 else 2.0 ** -133
    for b in (0, batch - 1):
        for h in range(heads):
            g = h // (heads // kv)
            check_faint(out[b, h:h + 1], lse[b, h:h + 1], q[b, h:h + 1], k[:, g], v[:, g], smallest)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,n,heads,kv", [(130, 700, 2, 2), (200, 9000, 2, 1), (900, 20000, 24, 2), (900, 60000, 24, 1)])
def test_sparse_keeps_faint_weights(dtype, t, n, heads, kv):
    """Weights count from a maximum that may be 2^8 too low, so fp16 keeps 31 bits below it."""
    gen = _gen(n + t)
    k, v = faint_keys(gen, n, kv, dtype)
    q = torch.zeros(t, heads, D, dtype=dtype, device="cuda")
    q[..., 0] = 16.0
    out, lse = h3b200.sparse_attention(q, k, v, -(-n // 64), return_lse=True)
    smallest = 2.0 ** -31 if dtype is torch.float16 else 2.0 ** -125
    rows = torch.tensor([0, 1, t // 2, t - 1], device="cuda")
    for h in {0, heads - 1}:
        g = h // (heads // kv)
        check_faint(out[rows, h], lse[rows, h], q[rows, h], k[:, g], v[:, g], smallest)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("top", [700.0, 2000.0])
def test_scores_of_many_millions_pick_one_key(dtype, top):
    """Where scores are so large that fp32 holds no fraction of them, a row is its best key's value: off by the
    rounding of one weight and of the result. Every row has another maximum, so that its rounding goes either way."""
    gen = _gen(int(top))
    n, best, rows = 100, 70, 200
    v = randn(gen, n, 1, D, dtype=dtype)
    size = torch.linspace(0.25 * top, top, rows, device="cuda").to(dtype)
    k = (0.9 * top * torch.rand(n, 1, 1, generator=gen, device="cuda")).expand(n, 1, D).to(dtype).contiguous()
    k[best] = top
    q = size[:, None, None].expand(rows, 1, D).contiguous()
    score = D * size.to(F64) * float(k[best, 0, 0]) * D ** -0.5
    page = 8
    pad = torch.zeros(104 - n, 1, D, dtype=dtype, device="cuda")
    kc, vc = (torch.cat((x, pad)).reshape(13, page, 1, D).transpose(1, 2) for x in (k, v))
    tab = torch.arange(13, dtype=torch.int32, device="cuda").expand(rows, 13)
    lens = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    for out, lse in (h3b200.paged_decode_attention(q, kc, vc, tab, lens, return_lse=True),
                     h3b200.sparse_attention(q, k, v, 2, return_lse=True)):
        off = (out[:, 0].to(F64) - v[best, 0].to(F64)).abs()
        assert bool((off <= 2.01 * half_step(dtype) * v[best, 0].to(F64).abs() + tiny(dtype)).all())
        # the fp32 sum of 128 equal products is off by at most 128 * 2^-24 of it
        assert bool(((lse[:, 0].to(F64) - score).abs() <= 130 * 2.0 ** -24 * score).all())


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("tab", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rot", [16, 96, 128])
def test_append_table_without_rows(tab, rot):
    """Every position lies outside a table without rows: NaN in the rotated dims, as for any other such position."""
    gen = _gen(rot)
    t, h, page = 5, 3, 8
    q, k, v = (randn(gen, t, h, D) for _ in range(3))
    kc, vc = (torch.zeros(2, h, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.arange(2, 2 + t, device="cuda")
    f = torch.empty(0, rot // 2, 2, 2, dtype=tab, device="cuda")
    for freqs in (f, f.reshape(1, 0, 1, rot // 2, 2, 2)):
        kc.zero_()
        qo = h3b200.append_paged_kv(k, v, kc, vc, slots, freqs, torch.arange(t, device="cuda"), q=q)
        for got, x in ((qo, q), (kc.transpose(1, 2).reshape(-1, h, D)[2:2 + t], k)):
            assert bool(got[..., :rot].isnan().all()) and torch.equal(got[..., rot:], x[..., rot:])
        assert torch.equal(vc.transpose(1, 2).reshape(-1, h, D)[2:2 + t], v)
    with pytest.raises(ValueError):
        h3b200.append_paged_kv(k, v, kc, vc, slots, f)   # token t would use row t


@pytest.mark.parametrize("tokens,heads", [(9, 4), (700, 24)])
def test_append_made_q_out_is_zero_for_padding(tokens, heads):
    """A q_out made inside the call holds zeros where a token is padding, not what the allocator had there."""
    gen = _gen(tokens)
    qkv = randn(gen, tokens, 3 * heads * D)
    q, k, v = (x.reshape(tokens, heads, D) for x in qkv.split(heads * D, 1))
    page = 16
    pages = tokens // page + 2
    kc, vc = (torch.zeros(pages, heads, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens]
    slots[1], slots[tokens // 2], slots[tokens - 1] = -1, pages * page, -5
    live = (slots >= 0) & (slots < pages * page)
    for shape in ((tokens, heads, D), (1, tokens, heads, D)):
        torch.cuda.synchronize()
        stale = torch.full(shape, float("nan"), dtype=torch.bfloat16, device="cuda")
        del stale
        out = h3b200.append_paged_kv(k, v, kc, vc, slots, table(tokens, 64), q=q.reshape(shape))
        assert out.shape == torch.Size(shape)
        out = out.reshape(tokens, heads, D)
        assert not bool(out[~live].any()) and not bool(out.isnan().any())
        want = torch.zeros(tokens, heads, D, dtype=torch.bfloat16, device="cuda")
        h3b200.append_paged_kv(k, v, kc, vc, slots, table(tokens, 64), q=q, q_out=want)
        assert torch.equal(out, want)


def test_captured_step_follows_slots_tables_and_lengths():
    """One captured step of append and decode attention, replayed while slots, positions, page_table and lengths
    change in place: a batch that grows, one sequence of it into pages it did not have at the capture."""
    gen = _gen(41)
    b, heads, kv, page, pages, dtype = 3, 8, 2, 16, 40, torch.bfloat16
    kc, vc = (torch.zeros(pages, kv, page, D, dtype=dtype, device="cuda") for _ in range(2))
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    tab = torch.full((b, 6), -1, dtype=torch.int32, device="cuda")
    f, kw = table(256, 96), randn(gen, D, std=0.1) + 1
    q, k, v = (randn(gen, b, h, D, dtype=dtype) for h in (heads, kv, kv))
    slots, pos = (torch.full((b,), -1, dtype=torch.int64, device="cuda") for _ in range(2))
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    q_out = torch.zeros_like(q)

    def step():
        h3b200.append_paged_kv(k, v, kc, vc, slots, f, pos, k_weight=kw, q=q, q_weight=kw, q_out=q_out)
        return h3b200.paged_decode_attention(q_out, kc, vc, tab, lens, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()      # padding only: nothing is written
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    assert not bool(kc.any())
    seqs = [[], [], []]
    counts, free = [0, 0, 0], 0
    for n in range(40):
        live = [True, n % 3 != 1, n >= 15]       # a sequence rests now and then, one starts late
        new_slots, new_pos = [-1] * b, [-1] * b
        for i in range(b):
            if not live[i]:
                continue
            if counts[i] % page == 0:
                tab[i, counts[i] // page] = order[free]
                free += 1
            new_slots[i] = int(tab[i, counts[i] // page]) * page + counts[i] % page
            new_pos[i] = counts[i] + 7 * i
            counts[i] += 1
        q.copy_(randn(gen, b, heads, D, dtype=dtype))
        k.copy_(randn(gen, b, kv, D, dtype=dtype))
        v.copy_(randn(gen, b, kv, D, dtype=dtype))
        slots.copy_(torch.tensor(new_slots))
        pos.copy_(torch.tensor(new_pos))
        lens.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        for i in range(b):
            if live[i]:
                at = new_slots[i]
                seqs[i].append((kc[at // page, :, at % page].clone(), vc[at // page, :, at % page].clone()))
                assert torch.equal(seqs[i][-1][1], v[i])
        want, want_lse = h3b200.paged_decode_attention(q_out, kc, vc, tab, lens, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    stacked = [tuple(torch.stack([s[j] for s in seq]) for j in range(2)) for seq in seqs]
    check_decode(q_out, stacked, out, lse, D ** -0.5, dtype)


# ---------------------------------------------------------------------------
# more tiles and items than the block-sparse kernel looks up at once
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries,keys,heads,kv,block,causal", [
    (2000, 6000, 24, 24, 64, False),      # 47 tiles an item
    (1300, 9001, 32, 8, 64, False),       # 71
    (2100, 8500, 20, 4, 128, True),       # up to 67, each query block another count
])
def test_sparse_lists_of_many_tiles(dtype, queries, keys, heads, kv, block, causal):
    """Dense attention through lists of every block: block ids are read 32 tiles at a time."""
    gen = _gen(queries + keys)
    q = randn(gen, queries, heads, D, dtype=dtype, std=1.5)
    k, v = randn(gen, keys, kv, D, dtype=dtype), randn(gen, keys, kv, D, dtype=dtype)
    top_k = -(-keys // block)
    out, lse, blocks = h3b200.sparse_attention(q, k, v, top_k, block, causal=causal, return_lse=True, return_blocks=True)
    for h in (0, heads // 2, heads - 1):
        g = h // (heads // kv)
        mask = list_mask(blocks, g, queries, keys, block, causal)
        ref = attend64(q[:, h], k[:, g], v[:, g], mask, D ** -0.5)
        check_attention(out[:, h], lse[:, h], ref, dtype, float(v.abs().max()), f"head {h}")


@pytest.mark.parametrize("keys,top_k", [(330, 3), (700, 1)])
def test_sparse_more_items_than_a_stream_looks_up(keys, top_k):
    """Over 19,000 items on at most 2 streams of each SM: item counts are read 32 at a time."""
    gen = _gen(keys)
    queries, heads, kv, dtype = 51201, 48, 4, torch.bfloat16
    q = randn(gen, queries, heads, D, dtype=dtype, std=1.5)
    k, v = randn(gen, keys, kv, D, dtype=dtype), randn(gen, keys, kv, D, dtype=dtype)
    blocks = torch.randint(-2, -(-keys // 64) + 1, (kv, -(-queries // 128), top_k), generator=gen, device="cuda",
                           dtype=torch.int32)
    # an id named twice counts twice: the reference's mask cannot say that
    for i in range(1, top_k):
        again = (blocks[..., i:i + 1] == blocks[..., :i]).any(-1)
        blocks[..., i] = torch.where(again, -1, blocks[..., i])
    out, lse = h3b200.block_sparse_attention(q, k, v, blocks, return_lse=True)
    for h in (0, 5, 23, 47):
        g = h // (heads // kv)
        ref = attend64(q[:, h], k[:, g], v[:, g], list_mask(blocks, g, queries, keys, 64, False), D ** -0.5)
        check_attention(out[:, h], lse[:, h], ref, dtype, float(v.abs().max()), f"head {h}")
    out2, lse2 = h3b200.block_sparse_attention(q, k, v, blocks, return_lse=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


# ---------------------------------------------------------------------------
# what the documentation allows
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("queries,keys,heads,kv,top_k,causal", [
    (1, 700, 40, 2, 4, False),         # the decode kernel: two row tiles
    (1, 9000, 8, 2, 141, False),
    (200, 3000, 4, 2, 47, True),       # split lists, joined by a second kernel
    (2500, 2500, 24, 24, 5, True),
])
def test_sparse_output_in_place_of_the_queries(queries, keys, heads, kv, top_k, causal):
    gen = _gen(queries + top_k)
    q = randn(gen, queries, heads, D, std=1.5)
    k, v = randn(gen, keys, kv, D), randn(gen, keys, kv, D)
    want, lse, blocks = h3b200.sparse_attention(q, k, v, top_k, causal=causal, return_lse=True, return_blocks=True)
    mine = q.clone()
    got, lse2, blocks2 = h3b200.sparse_attention(mine, k, v, top_k, causal=causal, out=mine, return_lse=True,
                                                 return_blocks=True)
    assert got is mine and torch.equal(got, want) and torch.equal(lse, lse2) and torch.equal(blocks, blocks2)
    mine = q.clone()
    assert torch.equal(h3b200.block_sparse_attention(mine, k, v, blocks, causal=causal, out=mine), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries", [1, 300, 900])
def test_packed_projection_rows_and_kept_means(dtype, queries):
    """q, k, v as slices of packed projection rows, out as a slice of wider rows, k_means as a slice of a longer
    buffer: the same bits as from tensors of their own."""
    gen = _gen(queries)
    heads, kv, keys = 12, 4, 900
    x = randn(gen, keys, (heads + 2 * kv) * D, dtype=dtype)
    q, k, v = (y.reshape(keys, -1, D) for y in x.split((heads * D, kv * D, kv * D), 1))
    q = q[keys - queries:]
    wide = torch.zeros(queries, 2 * heads * D, dtype=dtype, device="cuda")
    out = wide[:, heads * D:].reshape(queries, heads, D)
    means = torch.full((kv, 40, D), float("nan"), device="cuda")
    means[:, :15] = h3b200.attention_block_means(k, 64)
    got, lse = h3b200.sparse_attention(q, k, v, 6, causal=True, k_means=means[:, :15], out=out, return_lse=True)
    want, lse2, blocks = h3b200.sparse_attention(q.contiguous(), k.contiguous(), v.contiguous(), 6, causal=True,
                                                 return_lse=True, return_blocks=True)
    assert torch.equal(got, want) and torch.equal(lse, lse2) and not bool(wide[:, :heads * D].any())
    for h in (0, heads - 1):
        g = h // (heads // kv)
        ref = attend64(q[:, h], k[:, g], v[:, g], list_mask(blocks, g, queries, keys, 64, True), D ** -0.5)
        check_attention(out[:, h], lse[:, h], ref, dtype, float(v.abs().max()), f"head {h}")


@pytest.mark.parametrize("queries", [1, 260])
@pytest.mark.parametrize("block", [64, 128])
def test_blocks_named_twice_count_twice(queries, block):
    gen = _gen(queries + block)
    heads, keys, dtype = 2, 1000, torch.bfloat16
    q, k, v = (randn(gen, n, heads, D, dtype=dtype) for n in (queries, keys, keys))
    ids = torch.tensor([2, 5, 2, -1, 7, 5, 5], dtype=torch.int32, device="cuda")
    blocks = ids.expand(heads, -(-queries // 128), 7).contiguous()
    out, lse = h3b200.block_sparse_attention(q, k, v, blocks, block, return_lse=True)
    at = torch.cat([torch.arange(i * block, min(keys, (i + 1) * block), device="cuda") for i in ids.tolist()
                    if 0 <= i < -(-keys // block)])
    mask = torch.ones(queries, at.numel(), dtype=torch.bool, device="cuda")
    for h in range(heads):
        ref = attend64(q[:, h], k[at, h], v[at, h], mask, D ** -0.5)
        check_attention(out[:, h], lse[:, h], ref, dtype, float(v.abs().max()), f"head {h}")


def test_calls_at_once_on_two_streams():
    """Two streams, each with its own calls of every operator, some with workspaces and joins: the same bits as alone."""
    gen = _gen(51)
    dtype, kv, page = torch.bfloat16, 2, 32
    jobs = []
    for n, t in ((30000, 200), (5000, 1500)):
        pages = -(-n // page)
        kc, vc = (randn(gen, pages, kv, page, D) for _ in range(2))
        tab = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)[None]
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        q1, qs = randn(gen, 1, 8, D), randn(gen, t, 8, D)
        k, v = randn(gen, n, kv, D), randn(gen, n, kv, D)
        slots = torch.arange(t, device="cuda")
        f, kw = table(t, 64), randn(gen, D)

        def job(kc=kc, vc=vc, tab=tab, lens=lens, q1=q1, qs=qs, k=k, v=v, slots=slots, f=f, kw=kw, t=t):
            a = h3b200.paged_decode_attention(q1, kc, vc, tab, lens, return_lse=True)
            b = h3b200.sparse_attention(qs, k, v, 20, causal=True, return_lse=True, return_blocks=True)
            c = h3b200.sparse_attention(q1, k, v, 33)
            kn, vn = torch.zeros_like(kc), torch.zeros_like(vc)
            d = h3b200.append_paged_kv(k[:t], v[:t], kn, vn, slots, f, k_weight=kw, q=qs)
            return (*a, *b, c, kn, vn, d)

        jobs.append(job)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(20):
        got = []
        for s, job in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(job())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_one_page_of_more_than_a_million_keys():
    """A cache without paging is one long page per sequence."""
    gen = _gen(61)
    page, n, heads, dtype = (1 << 20) + 8, 5000, 4, torch.bfloat16
    kc, vc = (torch.zeros(2, 1, page, D, dtype=dtype, device="cuda") for _ in range(2))
    k, v = randn(gen, n, 1, D), randn(gen, n, 1, D)
    slots = page + (page - n) + torch.arange(n, device="cuda")     # the second page's last rows
    h3b200.append_paged_kv(k, v, kc, vc, slots)
    assert torch.equal(kc[1, 0, page - n:], k[:, 0]) and torch.equal(vc[1, 0, page - n:], v[:, 0])
    assert not bool(kc[0].any()) and not bool(kc[1, :, :page - n].any())
    q = randn(gen, 1, heads, D)
    tab = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([page], dtype=torch.int32, device="cuda")
    out, lse = h3b200.paged_decode_attention(q, kc, vc, tab, lens, return_lse=True)
    check_decode(q, [(kc[1].transpose(0, 1), vc[1].transpose(0, 1))], out, lse, D ** -0.5, dtype)
