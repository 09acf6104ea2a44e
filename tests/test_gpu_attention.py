"""Paged K/V append, paged decode attention and block-sparse attention on the GPU, against
plain 64-bit implementations of their definitions.

Tolerances. One rounding to the element type is off by at most h = eps / 2 of the value.
Append: one rounding, plus fp32 steps (norm, two products, one sum) of a few 2^-24 of the
terms. Attention: the scores of one row are 128-term fp32 sums, off by at most
e = 128 * 2^-24 * A with A the largest scale * sum |q_d k_d|, which moves a weight by a
factor 1 +- (2 e + 2^-20) (2^-20: exp2 and the sum's rounding); each weight is rounded once
(h), the n products are summed in fp32 (n 2^-24), the result is rounded once (h):
  |out - ref| <= sum p|v| * (h + 2 e + 2^-20 + 2 n 2^-24) + h |ref| + n t max|v|
with t half the smallest subnormal of the element type (weights that small), and
  |lse - ref| <= e + 2^-20 + n 2^-24 + 2^-23 |ref|.
"""

import math

import pytest
import torch

import h3b200

pytestmark = pytest.mark.gpu

D = 128
F64 = torch.float64
DTYPES = [torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(gen, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)


def table(rows, rot, dtype=torch.float32):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=F64, device="cuda") / rot)
    a = torch.arange(rows, dtype=F64, device="cuda")[:, None] * inv
    return torch.stack((a.cos(), -a.sin(), a.sin(), a.cos()), -1).reshape(rows, rot // 2, 2, 2).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def norm_rope64(x, w, coef, eps=1e-6):
    """(value, size of the terms) of the norm and the rotation, 64 bits."""
    x = x.to(F64)
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.to(F64)
    y, size = x.clone(), x.abs()
    if coef is not None:
        r = coef.shape[1]
        c = coef.to(F64)[:, None]
        a, b = x[..., :r], x[..., r:2 * r]
        for i, sl in ((0, slice(0, r)), (1, slice(r, 2 * r))):
            u, v = c[..., i, 0] * a, c[..., i, 1] * b
            y[..., sl], size[..., sl] = u + v, u.abs() + v.abs()
    return y, size


def check_rounded(got, ref, size, dtype, what):
    tol = half_step(dtype) * ref.abs() * 1.001 + 16 * 2.0 ** -24 * size + tiny(dtype)
    bad = (got.to(F64) - ref).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} values off"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv,rot,page,tab,norm,idx", [
    (1, 24, 24, 128, 64, torch.float32, True, torch.int64),
    (1, 1, 1, 16, 8, torch.bfloat16, False, torch.int32),
    (7, 5, 5, 96, 128, torch.bfloat16, True, torch.int64),
    (61, 32, 8, 64, 16, torch.float16, False, torch.int32),
    (130, 9, 3, 112, 24, torch.float32, True, torch.int64),
    (5000, 3, 1, 32, 8, torch.float32, True, torch.int32),
])
def test_append_matches_definition(dtype, tokens, heads, kv, rot, page, tab, norm, idx):
    gen = _gen(tokens + rot)
    pages = tokens // page + 3
    qkv = randn(gen, tokens, (heads + 2 * kv) * D, dtype=dtype)
    q, k, v = (x.reshape(tokens, -1, D) for x in qkv.split((heads * D, kv * D, kv * D), 1))
    kc = randn(gen, pages, kv, page, D, dtype=dtype)
    vc = randn(gen, pages, page, kv, D, dtype=dtype).transpose(1, 2)    # [pages, page, heads, D] storage
    kc0, vc0 = kc.clone(), vc.clone()
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].to(idx)
    if tokens > 3:
        slots[2], slots[tokens - 1] = -1, pages * page      # padding on either side of the pool
    f = table(tokens + 50, rot, tab)
    pos = torch.randint(0, tokens + 50, (tokens,), generator=gen, device="cuda").to(idx)
    kw, qw = (randn(gen, D, dtype=dtype), randn(gen, D, dtype=dtype)) if norm else (None, None)
    mark = randn(gen, tokens, heads, D, dtype=dtype)
    q_out = mark.clone()
    r = h3b200.append_paged_kv(k, v, kc, vc, slots, f, pos, k_weight=kw, q=q, q_weight=qw, q_out=q_out)
    assert r is q_out
    live = (slots >= 0) & (slots < pages * page)
    coef = f[pos.long()]
    kr, ks = norm_rope64(k, kw, coef)
    qr, qs = norm_rope64(q, qw, coef)
    check_rounded(q_out[live], qr[live], qs[live], dtype, "q")
    assert torch.equal(q_out[~live], mark[~live])
    at = slots[live].long()
    check_rounded(kc[at // page, :, at % page], kr[live], ks[live], dtype, "k")
    assert torch.equal(vc[at // page, :, at % page], v[live])
    kc[at // page, :, at % page] = kc0[at // page, :, at % page]
    vc[at // page, :, at % page] = vc0[at // page, :, at % page]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0), "rows that no slot names changed"


def test_append_forms():
    """No rotation, no norm: plain copies; rows by token; in place Q; 4-D and 6-D arguments."""
    gen = _gen(3)
    t, h, page = 21, 4, 8
    k, v, q = (randn(gen, 1, t, h, D) for _ in range(3))
    kc, vc = (torch.zeros(6, h, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.arange(3, 3 + t, device="cuda")
    assert h3b200.append_paged_kv(k, v, kc, vc, slots) is None
    flat = kc.transpose(1, 2).reshape(-1, h, D)
    assert torch.equal(flat[3:3 + t], k[0]) and not flat[:3].any() and not flat[3 + t:].any()
    f = table(t, 96)
    a = h3b200.append_paged_kv(k, v, kc, vc, slots, f.reshape(1, t, 1, 48, 2, 2), q=q)
    want = a.clone()
    b = h3b200.append_paged_kv(k, v, kc, vc, slots, f, torch.arange(t, device="cuda"), q=q, q_out=q)
    assert b is q and torch.equal(q, want)
    # a position outside the table shows as NaN in the rotated dims, and reads nothing
    pos = torch.arange(t, device="cuda")
    pos[4], pos[5] = -1, t
    h3b200.append_paged_kv(k, v, kc, vc, slots, f, pos)
    flat = kc.transpose(1, 2).reshape(-1, h, D)[3:3 + t]
    assert bool(flat[4:6, :, :96].isnan().all()) and torch.equal(flat[4:6, :, 96:], k[0, 4:6, :, 96:])
    assert not bool(flat[:4].isnan().any()) and not bool(flat[6:].isnan().any())
    h3b200.append_paged_kv(k[:, :0], v[:, :0], kc, vc, slots[:0], f)   # nothing to do


# ---------------------------------------------------------------------------
# attention references
# ---------------------------------------------------------------------------


def attend64(q, k, v, mask, scale):
    """(out, lse, sum p|v|, A, n) of q [m, D] over k, v [n, D] with mask [m, n]."""
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    k = torch.where(mask.any(0)[:, None], k, 0.0)
    v = torch.where(mask.any(0)[:, None], v, 0.0)
    x = (q @ k.T) * scale
    a = (q.abs() @ k.abs().T) * scale
    x = x.masked_fill(~mask, -math.inf)
    some = mask.any(1)
    lse = torch.logsumexp(x, 1)
    p = torch.where(some[:, None], torch.exp(x - torch.where(some, lse, 0.0)[:, None]), 0.0)
    big = torch.where(mask, a, 0.0).amax(1) if mask.shape[1] else torch.zeros_like(lse)
    return p @ v, lse, p @ v.abs(), big, mask.sum(1)


def check_attention(out, lse, ref, dtype, vmax, what=""):
    o, ls, pv, a, n = ref
    h = half_step(dtype)
    e = (128 * 2.0 ** -24 * a)[:, None]
    n = n.to(F64)[:, None]
    tol = pv * (h + 2 * e + 2.0 ** -20 + 2 * n * 2.0 ** -24) + h * o.abs() + n * tiny(dtype) * vmax
    bad = ~((out.to(F64) - o).abs() <= tol)
    assert not bool(bad.any()), f"{what} out: {int(bad.sum())} of {bad.numel()} off, worst {float((out.to(F64) - o).abs().max())}"
    if lse is not None:
        some = torch.isfinite(ls)
        assert torch.equal(torch.isneginf(lse), ~some), f"{what}: lse of empty rows"
        ltol = e[:, 0] + 2.0 ** -20 + n[:, 0] * 2.0 ** -24 + 2.0 ** -23 * ls.abs()
        off = (lse.to(F64) - ls).abs()
        assert bool((off[some] <= ltol[some]).all()), f"{what} lse: worst {float(off[some].max())}"


# ---------------------------------------------------------------------------
# paged decode
# ---------------------------------------------------------------------------


def paged_case(gen, lengths, kv, page, dtype, extra=3, width=None):
    b = len(lengths)
    width = max(1, max(-(-n // page) for n in lengths)) if width is None else width
    pages = b * width + extra
    kc = torch.full((pages, kv, page, D), float("nan"), dtype=dtype, device="cuda")
    vc = torch.full((pages, kv, page, D), float("inf"), dtype=dtype, device="cuda")
    tab = torch.randperm(pages, generator=gen, device="cuda")[:b * width].to(torch.int32).reshape(b, width)
    seqs = []
    for i, n in enumerate(lengths):
        k, v = randn(gen, n, kv, D, dtype=dtype), randn(gen, n, kv, D, dtype=dtype)
        at = torch.arange(n, device="cuda")
        pg = tab[i].long()[at // page] if n else at
        kc[pg, :, at % page], vc[pg, :, at % page] = k, v
        seqs.append((k, v))
    return kc, vc, tab, torch.tensor(lengths, dtype=torch.int32, device="cuda"), seqs


def check_decode(q, seqs, out, lse, scale, dtype):
    b, heads, _ = q.shape
    for i, (k, v) in enumerate(seqs):
        n, kv, _ = k.shape
        g = heads // kv
        vmax = float(v.abs().max()) if n else 0.0
        for h in range(kv):
            mask = torch.ones(g, n, dtype=torch.bool, device="cuda")
            ref = attend64(q[i, h * g:(h + 1) * g], k[:, h], v[:, h], mask, scale)
            check_attention(out[i, h * g:(h + 1) * g], None if lse is None else lse[i, h * g:(h + 1) * g], ref, dtype,
                            vmax, f"sequence {i} head {h}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,heads,kv,page", [
    ([1], 1, 1, 8),
    ([777], 24, 24, 64),
    ([0, 1, 7, 8, 9, 15, 16, 17, 63, 64, 65, 0], 8, 2, 8),
    ([1000, 3, 0, 511, 129], 32, 8, 16),
    ([300, 2], 48, 3, 24),           # 16 heads per key head
    ([65, 200], 40, 2, 128),         # 20 heads per key head: two row tiles
    ([40000], 4, 2, 256),
    ([100] * 70, 12, 4, 32),
])
def test_decode_matches_definition(dtype, lengths, heads, kv, page):
    gen = _gen(sum(lengths) + heads)
    kc, vc, tab, lens, seqs = paged_case(gen, lengths, kv, page, dtype)
    q = randn(gen, len(lengths), heads, D, dtype=dtype, std=1.5)
    out, lse = h3b200.paged_decode_attention(q, kc, vc, tab, lens, return_lse=True)
    check_decode(q, seqs, out, lse, D ** -0.5, dtype)
    again = h3b200.paged_decode_attention(q, kc, vc, tab, lens)
    assert torch.equal(out, again)


def test_decode_strides_scale_and_wide_tables():
    """A cache in [pages, page, heads, D] order, q and out as views, a far too wide table, lengths
    beyond the table, bad page ids (no keys), large scores."""
    gen = _gen(11)
    dtype, kv, page, heads = torch.bfloat16, 3, 16, 6
    kc, vc, tab, lens, seqs = paged_case(gen, [50, 0, 333], kv, page, dtype)
    kn = kc.transpose(1, 2).contiguous().transpose(1, 2)
    vn = vc.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((3, 4096), -7, dtype=torch.int32, device="cuda")
    wide[:, :tab.shape[1]] = tab
    q = randn(gen, 3, heads * 2, D, dtype=dtype, std=3.0)[:, ::2]
    out = torch.zeros(heads, 3, D, dtype=dtype, device="cuda").transpose(0, 1)
    got, lse = h3b200.paged_decode_attention(q, kn, vn, wide, lens, scale=0.7, out=out, return_lse=True)
    assert got is out
    check_decode(q, seqs, out, lse, 0.7, dtype)
    # lengths are clamped to what the table holds; ids outside the pool hold no keys
    k, v = seqs[2]
    short = wide[:, :21].contiguous()
    short[2, 1], short[2, 4] = -1, kc.shape[0]
    keep = torch.ones(333, dtype=torch.bool, device="cuda")
    keep[16:32] = keep[64:80] = False
    lens2 = torch.tensor([-5, 0, 1 << 30], dtype=torch.int32, device="cuda")
    out2, lse2 = h3b200.paged_decode_attention(q, kn, vn, short[:, :20], lens2, scale=0.7, return_lse=True)
    seqs2 = [(k[:0], v[:0]), (k[:0], v[:0]), (k[:320][keep[:320]], v[:320][keep[:320]])]
    check_decode(q, seqs2, out2, lse2, 0.7, dtype)


def test_decode_far_offsets():
    """Pages whose element offsets pass 2^31 and 2^32."""
    gen = _gen(12)
    kv, page, pages = 8, 64, 66000           # 66,000 * 8 * 64 * 128 = 4.3e9 elements
    kc = torch.empty(pages, kv, page, D, dtype=torch.float16, device="cuda")
    tab = torch.tensor([[pages - 1, 33000, 0, 50001]], dtype=torch.int32, device="cuda")
    data = randn(gen, 4, kv, page, D, dtype=torch.float16)
    kc[tab[0].long()] = data
    lens = torch.tensor([250], dtype=torch.int32, device="cuda")
    q = randn(gen, 1, 16, D, dtype=torch.float16)
    out, lse = h3b200.paged_decode_attention(q, kc, kc, tab, lens, return_lse=True)
    seq = data.transpose(1, 2).reshape(-1, kv, D)[:250]
    check_decode(q, [(seq, seq)], out, lse, D ** -0.5, torch.float16)
    slot = torch.tensor([(pages - 1) * page + 5], device="cuda")
    k = randn(gen, 1, kv, D, dtype=torch.float16)
    h3b200.append_paged_kv(k, k, kc, kc, slot)
    assert torch.equal(kc[pages - 1, :, 5], k[0])


def test_decode_extreme_scores():
    """Scores near the top of the range, equal scores, -inf scores: the maximum is taken out first."""
    gen = _gen(13)
    kc, vc, tab, lens, seqs = paged_case(gen, [200, 90], 1, 8, torch.float16)
    q = randn(gen, 2, 2, D, dtype=torch.float16, std=200.0)
    out, lse = h3b200.paged_decode_attention(q, kc, vc, tab, lens, return_lse=True)
    check_decode(q, seqs, out, lse, D ** -0.5, torch.float16)
    q = torch.zeros_like(q)
    out, lse = h3b200.paged_decode_attention(q, kc, vc, tab, lens, return_lse=True)
    check_decode(q, seqs, out, lse, D ** -0.5, torch.float16)


# ---------------------------------------------------------------------------
# block selection
# ---------------------------------------------------------------------------


def means64(x, block):
    t, h, _ = x.shape
    return torch.stack([x[i:i + block].to(F64).mean(0) for i in range(0, t, block)], 1) if t else x.new_zeros(h, 0, D)


def select64(qm, km, top_k, queries, keys, block, causal):
    kv, nk, _ = km.shape
    qb = qm.shape[1]
    s = torch.einsum("qd,kd->qk", qm.double().reshape(kv, -1, qb, D).sum(1).reshape(-1, D),
                     km.double().reshape(-1, D)).reshape(kv, qb, kv, nk)
    blocks = torch.full((kv, qb, top_k), -1, dtype=torch.int32)
    for h in range(kv):
        for i in range(qb):
            row = s[h, i, h].tolist()
            order = sorted(range(nk), key=lambda j: (-row[j], j))
            if causal:
                lo = i * 128 + keys - queries
                hi = min((i + 1) * 128, queries) - 1 + keys - queries
                order = [j for j in order if j * block <= hi]
                order.sort(key=lambda j: (j * block + block <= lo, -row[j] if j * block + block <= lo else 0, j))
            picked = sorted(order[:top_k])
            blocks[h, i, :len(picked)] = torch.tensor(picked, dtype=torch.int32)
    return blocks.cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,block", [(1, 1, 64), (63, 3, 64), (129, 2, 128), (1000, 5, 64), (700, 2, 300)])
def test_block_means(dtype, tokens, heads, block):
    gen = _gen(tokens)
    x = randn(gen, heads, tokens, D, dtype=dtype, std=3.0).transpose(0, 1)
    got = h3b200.attention_block_means(x, block)
    ref = means64(x, block)
    assert got.shape == ref.shape
    assert bool(((got.to(F64) - ref).abs() <= 2.0 ** -24 * 1.001 * ref.abs() + 1e-40).all())


@pytest.mark.parametrize("queries,keys,heads,kv,block,top_k,causal", [
    (1, 1, 1, 1, 64, 1, False),
    (1, 5000, 8, 2, 64, 7, False),
    (300, 300, 3, 3, 64, 2, False),
    (1000, 2500, 8, 4, 64, 40, False),      # more than there are
    (2000, 2000, 4, 2, 128, 5, True),
    (130, 1111, 2, 1, 64, 6, True),         # an offset that splits blocks
    (700, 300, 2, 2, 64, 3, True),          # rows before the first key
    (1100, 60000, 1, 1, 64, 16, False),
])
def test_selection(queries, keys, heads, kv, block, top_k, causal):
    gen = _gen(queries + keys)
    qm = h3b200.attention_block_means(randn(gen, queries, heads, D), 128)
    km = h3b200.attention_block_means(randn(gen, keys, kv, D), block)
    got = h3b200.select_key_blocks(qm, km, top_k, queries, keys, block, causal)
    assert torch.equal(got, select64(qm, km, top_k, queries, keys, block, causal))


@pytest.mark.parametrize("queries,keys,heads,kv,block,top_k,causal", [
    (1, 16385, 6, 2, 64, 33, False),        # a few key blocks for each of several CTAs
    (1, 32768, 24, 24, 64, 64, False),
    (100, 140000, 4, 1, 64, 500, True),     # more keys than a lane holds in registers
    (2048, 20000, 14, 2, 128, 1, False),
    (1024, 190000, 2, 1, 64, 100, False),   # as much shared memory as eight rows take, in a cluster
])
def test_selection_few_rows_many_blocks(queries, keys, heads, kv, block, top_k, causal):
    test_selection(queries, keys, heads, kv, block, top_k, causal)


def test_selection_refusals():
    """Counts that a 64-bit argument would wrap are refused like other bad ones."""
    m = torch.zeros(1, 1, D, device="cuda")
    for top_k, block in ((0, 64), (1 << 25, 64), ((1 << 64) + 1, 64), (1, 0), (1, (1 << 64) + 1)):
        with pytest.raises(ValueError):
            h3b200.select_key_blocks(m, m, top_k, 1, 64, block)
    x = torch.zeros(1, 1, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        h3b200.sparse_attention(x, x, x, (1 << 64) + 1)


def test_selection_ties_and_odd_scores():
    """Equal scores go to the lowest block, zero of either sign is one score, NaN ranks last."""
    km = torch.zeros(1, 100, D, device="cuda")
    qm = torch.zeros(1, 1, D, device="cuda")
    qm[0, 0, 0] = 1.0
    km[0, 40:60, 0] = 2.0
    km[0, 70, 0] = -0.0
    want = list(range(40, 60))
    got = h3b200.select_key_blocks(qm, km, 20, 1, 6400, 64)
    assert got[0, 0].tolist() == want
    got = h3b200.select_key_blocks(qm, km, 7, 1, 6400, 64)
    assert got[0, 0].tolist() == want[:7]
    got = h3b200.select_key_blocks(qm, km, 93, 1, 6400, 64)
    assert got[0, 0].tolist() == list(range(93))
    km[0, 3, 0], km[0, 5, 0], km[0, 9, 0] = float("nan"), float("inf"), float("-inf")
    got = h3b200.select_key_blocks(qm, km, 98, 1, 6400, 64)
    assert got[0, 0].tolist() == [j for j in range(100) if j not in (3, 9)]
    got = h3b200.select_key_blocks(qm, km, 100, 1, 6400, 64)
    assert got[0, 0].tolist() == list(range(100))


# ---------------------------------------------------------------------------
# block-sparse attention
# ---------------------------------------------------------------------------


def list_mask(blocks, h, queries, keys, block, causal):
    """[queries, keys] mask of key head h from a block list."""
    nk = -(-keys // block)
    held = torch.zeros(blocks.shape[1], nk + 1, dtype=torch.bool, device="cuda")
    ids = torch.where((blocks[h] >= 0) & (blocks[h] < nk), blocks[h], nk).long()
    held.scatter_(1, ids, True)
    rows, cols = torch.arange(queries, device="cuda"), torch.arange(keys, device="cuda")
    mask = held[rows // 128][:, cols // block]
    if causal:
        mask &= cols <= rows[:, None] + keys - queries
    return mask


def check_sparse(q, k, v, blocks, block, causal, out, lse, scale, dtype):
    t, heads, _ = q.shape
    s, kv, _ = k.shape
    vmax = float(v.abs().max())
    for h in range(heads):
        g = h // (heads // kv)
        ref = attend64(q[:, h], k[:, g], v[:, g], list_mask(blocks, g, t, s, block, causal), scale)
        check_attention(out[:, h], None if lse is None else lse[:, h], ref, dtype, vmax, f"head {h}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,keys,heads,kv,block,top_k,causal", [
    (1, 1, 1, 1, 64, 1, False),
    (1, 3000, 8, 2, 64, 9, False),
    (1, 500, 20, 1, 128, 2, True),
    (2, 100, 1, 1, 64, 1, False),
    (128, 128, 1, 1, 64, 2, False),
    (129, 65, 3, 3, 64, 2, False),
    (300, 700, 4, 2, 64, 3, False),          # an odd number of sub-blocks
    (257, 1000, 6, 3, 128, 4, False),
    (640, 640, 2, 2, 64, 4, True),
    (500, 1234, 4, 1, 128, 3, True),
    (200, 90, 2, 1, 64, 5, True),            # rows that see no key
    (3000, 3000, 24, 24, 64, 8, False),      # two query blocks per CTA, more CTAs than SMs
    (1400, 1600, 32, 8, 64, 5, False),       # grouped heads, more query blocks than streams
    (1300, 2000, 48, 8, 128, 4, True),
    (1500, 900, 64, 4, 64, 3, True),         # whole query blocks without a key among them
])
def test_sparse_matches_definition(dtype, queries, keys, heads, kv, block, top_k, causal):
    gen = _gen(queries * 7 + keys)
    q = randn(gen, queries, heads, D, dtype=dtype, std=1.5)
    k, v = randn(gen, keys, kv, D, dtype=dtype), randn(gen, keys, kv, D, dtype=dtype)
    out, lse, blocks = h3b200.sparse_attention(q, k, v, top_k, block, causal=causal, return_lse=True, return_blocks=True)
    qm = torch.stack([x for x in means64(q, 128)]).float()
    km = means64(k, block).float()
    assert torch.equal(blocks, select64(qm, km, top_k, queries, keys, block, causal))
    check_sparse(q, k, v, blocks, block, causal, out, lse, D ** -0.5, dtype)
    again = h3b200.sparse_attention(q, k, v, top_k, block, causal=causal,
                                    k_means=h3b200.attention_block_means(k, block))
    assert torch.equal(out, again)


def test_sparse_lists_views_and_growing_maxima():
    """A caller's own lists (gaps, ids outside, empty rows), HND-backed views, a scale, scores that
    grow from tile to tile by more than the rescale threshold."""
    gen = _gen(21)
    t, s, heads, block, dtype = 390, 1000, 4, 64, torch.bfloat16
    q = randn(gen, heads, t, D, dtype=dtype).transpose(0, 1)
    k = randn(gen, heads, s, D, dtype=dtype).transpose(0, 1)
    v = randn(gen, heads, s, D, dtype=dtype).transpose(0, 1)
    ramp = torch.linspace(0.05, 6.0, s, device="cuda")[:, None, None]
    k.copy_((k.float() * ramp).to(dtype))
    blocks = torch.full((heads, 4, 7), -1, dtype=torch.int32, device="cuda")
    blocks[0, 0] = torch.tensor([3, -1, 0, 99, 15, -2, 14], dtype=torch.int32)
    blocks[1, 1] = torch.tensor([-1, -1, -1, -1, -1, -1, 15], dtype=torch.int32)
    blocks[2, 2] = torch.tensor([0, 2, 4, 6, 8, 10, 12], dtype=torch.int32)
    blocks[3, 3] = torch.tensor([12, 10, 8, 6, 4, 2, 0], dtype=torch.int32)
    out = torch.full((heads, t, D), 7.0, dtype=dtype, device="cuda").transpose(0, 1)
    got, lse = h3b200.block_sparse_attention(q, k, v, blocks, block, scale=0.5, out=out, return_lse=True)
    assert got is out
    check_sparse(q, k, v, blocks, block, False, out, lse, 0.5, dtype)
    assert not bool(out[128:, 0].any()) and bool(torch.isneginf(lse[128:, 0]).all())
    out1, lse1 = h3b200.block_sparse_attention(q[:1], k, v, blocks[:, :1].contiguous(), block, return_lse=True)
    check_sparse(q[:1], k, v, blocks[:, :1], block, False, out1, lse1, D ** -0.5, dtype)


def test_sparse_keys_behind_the_last_are_not_read():
    """k and v as the head of larger buffers that hold NaN behind the last key."""
    gen = _gen(22)
    k, v = (torch.full((400, 2, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k[:333], v[:333] = randn(gen, 333, 2, D), randn(gen, 333, 2, D)
    for t in (1, 200):
        q = randn(gen, t, 2, D)
        out, lse, blocks = h3b200.sparse_attention(q, k[:333], v[:333], 6, return_lse=True, return_blocks=True)
        check_sparse(q, k[:333], v[:333], blocks, 64, False, out, lse, D ** -0.5, torch.bfloat16)


def test_sparse_hidden_values_count_nothing():
    """The weight of a key that a row may not see is zero, not just small: values near the largest
    finite one, hidden under `causal`, leave the rows before them as they are."""
    gen = _gen(24)
    t, seen = 256, 201
    q, k, v = randn(gen, t, 2, D), randn(gen, t, 1, D), randn(gen, t, 1, D)
    blocks = torch.arange(4, dtype=torch.int32, device="cuda").expand(1, 2, 4).contiguous()
    loud = v.clone()
    loud[seen:] = 3e38
    out, lse = h3b200.block_sparse_attention(q, k, loud, blocks, causal=True, return_lse=True)
    mask = list_mask(blocks, 0, t, t, 64, True)[:seen]
    for h in range(2):
        ref = attend64(q[:seen, h], k[:, 0], v[:, 0], mask, D ** -0.5)
        check_attention(out[:seen, h], lse[:seen, h], ref, torch.bfloat16, float(v.abs().max()), f"head {h}")
    # rows that see no key at all
    out, lse = h3b200.block_sparse_attention(q, k[:100], loud[-100:], blocks[..., :2].contiguous(), causal=True,
                                             return_lse=True)
    assert not bool(out[:t - 100].any()) and bool(torch.isneginf(lse[:t - 100]).all())


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def test_prompt_then_tokens():
    """A prompt enters the cache and runs block-sparse (here: every block), tokens follow one at a time;
    both read the same keys, and the tokens' results are those of causal attention over everything."""
    gen = _gen(31)
    heads, kv, page, prompt, steps = 8, 2, 64, 333, 5
    total = prompt + steps
    width = (heads + 2 * kv) * D
    x = randn(gen, total, width)
    kw, qw = randn(gen, D, std=0.1) + 1, randn(gen, D, std=0.1) + 1
    f = table(1024, 96)
    pages = 12
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    kc, vc = (torch.zeros(pages, kv, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pt = order[None, :6].contiguous()
    at = torch.arange(total, device="cuda")
    slots, pos = pt[0].long()[at // page] * page + at % page, at + 100

    def put(a, b):
        q, k, v = (y.reshape(b - a, -1, D) for y in x[a:b].split((heads * D, kv * D, kv * D), 1))
        return h3b200.append_paged_kv(k, v, kc, vc, slots[a:b], f, pos[a:b], k_weight=kw, q=q, q_weight=qw)

    def keys(n):
        return [c.transpose(1, 2).reshape(-1, kv, D)[slots[:n]] for c in (kc, vc)]

    q = put(0, prompt)
    k, v = keys(prompt)
    out, lse, blocks = h3b200.sparse_attention(q, k, v, 100, causal=True, return_lse=True, return_blocks=True)
    check_sparse(q, k, v, blocks, 64, True, out, lse, D ** -0.5, torch.bfloat16)
    for n in range(prompt, total):
        q = put(n, n + 1)
        lens = torch.tensor([n + 1], dtype=torch.int32, device="cuda")
        out = h3b200.paged_decode_attention(q, kc, vc, pt, lens)
        k, v = keys(n + 1)
        check_decode(q, [(k, v)], out, None, D ** -0.5, torch.bfloat16)
        # the same token over all key blocks of the gathered keys
        dense = h3b200.sparse_attention(q, k, v, 100)
        check_decode(q, [(k, v)], dense, None, D ** -0.5, torch.bfloat16)


def test_reads_what_the_qkv_build_writes():
    """qkv_qknorm_rope's HND-backed views go straight into the attention and the cache."""
    gen = _gen(33)
    m, heads, d = 200, 3, 256
    w, ws = h3b200.quantize_int8_convrot_weight(randn(gen, 3 * heads * D, d, std=0.05))
    xq, xs = h3b200.quantize_int8_rowwise_convrot(randn(gen, m, d), 256)
    nw = randn(gen, D, std=0.1) + 1
    q, k, v = h3b200.qkv_qknorm_rope(xq, xs, w, ws, None, heads, nw, nw, table(m, 96).reshape(1, m, 1, 48, 2, 2), 1e-6)
    out, lse, blocks = h3b200.sparse_attention(q, k, v, 2, return_lse=True, return_blocks=True)
    check_sparse(q, k, v, blocks, 64, False, out, lse, D ** -0.5, torch.bfloat16)
    kc, vc = (torch.zeros(8, heads, 32, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    h3b200.append_paged_kv(k, v, kc, vc, torch.arange(m, device="cuda"))
    lens = torch.tensor([m], dtype=torch.int32, device="cuda")
    pages = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    one = h3b200.paged_decode_attention(q[m - 1:m], kc, vc, pages, lens)
    check_decode(q[m - 1:m], [(k, v)], one, None, D ** -0.5, torch.bfloat16)


def test_graph_and_streams():
    """Captured steps replay after lengths, tables and inputs change in place; a side stream works."""
    gen = _gen(32)
    kc, vc, tab, lens, seqs = paged_case(gen, [100, 700], 2, 16, torch.bfloat16)
    kc, vc = torch.nan_to_num(kc), torch.nan_to_num(vc, posinf=0.0)
    q = randn(gen, 2, 8, D)
    k, v = randn(gen, 600, 2, D), randn(gen, 600, 2, D)
    qs = randn(gen, 300, 4, D)
    h3b200.paged_decode_attention(q, kc, vc, tab, lens)
    h3b200.sparse_attention(qs, k, v, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = h3b200.paged_decode_attention(q, kc, vc, tab, lens)
        b = h3b200.sparse_attention(qs, k, v, 3)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ga = h3b200.paged_decode_attention(q, kc, vc, tab, lens)
        gb = h3b200.sparse_attention(qs, k, v, 3)
    g.replay()
    assert torch.equal(ga, a) and torch.equal(gb, b)
    lens.copy_(torch.tensor([90, 13], dtype=torch.int32))
    q.copy_(randn(gen, 2, 8, D))
    qs.copy_(randn(gen, 300, 4, D))
    g.replay()
    assert torch.equal(ga, h3b200.paged_decode_attention(q, kc, vc, tab, lens))
    assert torch.equal(gb, h3b200.sparse_attention(qs, k, v, 3))


def test_refusals():
    k = torch.zeros(4, 2, D, dtype=torch.bfloat16, device="cuda")
    c = torch.zeros(3, 2, 16, D, dtype=torch.bfloat16, device="cuda")
    s = torch.zeros(4, dtype=torch.int64, device="cuda")
    f = table(4, 64)
    bad = [
        lambda: h3b200.append_paged_kv(k.cpu(), k, c, c, s),
        lambda: h3b200.append_paged_kv(k.float(), k, c, c, s),
        lambda: h3b200.append_paged_kv(k, k.half(), c, c, s),
        lambda: h3b200.append_paged_kv(k, k[:3], c, c, s),
        lambda: h3b200.append_paged_kv(k, k, c, c[:, :1], s),
        lambda: h3b200.append_paged_kv(k, k, c, c, s[:3]),
        lambda: h3b200.append_paged_kv(k, k, c, c, s.float()),
        lambda: h3b200.append_paged_kv(k, k, c, c, s, f[:3]),
        lambda: h3b200.append_paged_kv(k, k, c, c, s, table(4, 24)),
        lambda: h3b200.append_paged_kv(k, k, c, c, s, None, s),
        lambda: h3b200.append_paged_kv(k, k, c, c, s, q_weight=k[0, 0]),
        lambda: h3b200.append_paged_kv(k, k, c[:, :, :12], c[:, :, :12], s),
        lambda: h3b200.append_paged_kv(k, k, c, c, s, k_weight=k[0]),
    ]
    q = torch.zeros(2, 4, D, dtype=torch.bfloat16, device="cuda")
    pt = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    bad += [
        lambda: h3b200.paged_decode_attention(q[:, :3], c, c, pt, n),
        lambda: h3b200.paged_decode_attention(q.half(), c, c, pt, n),
        lambda: h3b200.paged_decode_attention(q, c[:, :, :12], c[:, :, :12], pt, n),
        lambda: h3b200.paged_decode_attention(q, c, c, pt.long(), n),
        lambda: h3b200.paged_decode_attention(q, c, c, pt[:1], n),
        lambda: h3b200.paged_decode_attention(q, c, c, pt, n.long()),
        lambda: h3b200.paged_decode_attention(q, c, c, pt, n, scale=0.0),
        lambda: h3b200.paged_decode_attention(q, c, c, pt, n, scale=float("nan")),
        lambda: h3b200.paged_decode_attention(q, c, c, pt, n, out=q.float()),
        lambda: h3b200.sparse_attention(q, k, k, 0),
        lambda: h3b200.sparse_attention(q[:, :3], k, k, 1),
        lambda: h3b200.sparse_attention(q, k[:0], k[:0], 1),
        lambda: h3b200.sparse_attention(q, k, k, 1, scale=-1.0),
        lambda: h3b200.sparse_attention(q, k, k, 1, k_means=torch.zeros(2, 2, D, device="cuda")),
        lambda: h3b200.block_sparse_attention(q, k, k, pt[None]),
        lambda: h3b200.attention_block_means(k, 0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    for call in (lambda: h3b200.sparse_attention(q, k, k, 1, block_size=96),
                 lambda: h3b200.sparse_attention(q, k[:1].expand(4, 2, D), k, 1)):
        with pytest.raises(NotImplementedError):
            call()
    empty = q[:0]
    assert h3b200.paged_decode_attention(empty, c, c, pt[:0], n[:0]).shape == empty.shape
    assert h3b200.sparse_attention(empty, k, k, 1).shape == empty.shape
    assert h3b200.device_status(0) == 0
