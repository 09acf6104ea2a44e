"""Attention around the Q/K/V build: what its operators are given and what they cost.

Three operators follow the projection and the QK-norm-RoPE of a transformer block:

* ``append_paged_kv``: new keys and values into a paged cache, K (and Q) normalised per head
  and rotated by their position on the way;
* ``paged_decode_attention``: attention of one new token per sequence over that cache;
* ``sparse_attention``: attention of 128-token query blocks over the key blocks that a cheap
  score (products of block means) selects, for whole prompts and for a single token.

Each case is one call. With ``own`` false, :func:`run` computes it with elementary torch
operations; with ``own`` true it calls the framework. :func:`exact` is the definition in 64 bits.
"""

import math
import os
import sys

import torch

own = False

D = 128           # head dim of every attention operator of the framework
Q_BLOCK = 128     # query tokens that share a selection
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TABLES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_LARGEST = 13_000_000_000_000   # flops a drawn sparse case may have, dense upper bound of the largest listed one


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200")
    if root not in sys.path:
        sys.path.insert(1, root)
    import h3b200

    return h3b200


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one sequence generates: one token of 24 heads enters the cache
        dict(name="append_one_token", op="append", tokens=1, heads=24, kv_heads=24, rot=128, page=64, pages=40,
             norm=True, dtype="bf16", table="fp32", padded=0),
        # a batch generates: one token per sequence, the last rows are padding, grouped heads, partial rotation
        dict(name="append_batch_gqa_fp16", op="append", tokens=61, heads=32, kv_heads=8, rot=64, page=16, pages=700,
             norm=False, dtype="fp16", table="fp32", padded=7),
        # one chunk of a long prompt through the 56-head attention with its 96 rotated dims and bf16 table
        dict(name="append_chunk_56_heads", op="append", tokens=4095, heads=56, kv_heads=56, rot=96, page=128, pages=80,
             norm=True, dtype="bf16", table="bf16", padded=0),
        # all tokens of a 21 x 39 x 40 grid at once
        dict(name="append_grid", op="append", tokens=32760, heads=24, kv_heads=24, rot=128, page=64, pages=560,
             norm=True, dtype="bf16", table="fp32", padded=0),
        # the first steps of one sequence: a call whose latency counts
        dict(name="decode_one_short", op="decode", batch=1, heads=24, kv_heads=24, longest=777, shortest=777, page=64,
             pages=40, dtype="bf16"),
        # a serving batch of very different lengths, empty sequences among them, small pages
        dict(name="decode_ragged_gqa_fp16", op="decode", batch=48, heads=32, kv_heads=8, longest=6000, shortest=0,
             page=16, pages=20000, dtype="fp16"),
        # a full batch of long sequences
        dict(name="decode_batch_long", op="decode", batch=64, heads=64, kv_heads=8, longest=9000, shortest=7000,
             page=64, pages=9100, dtype="bf16"),
        # one very long sequence in a pool whose offsets pass 32 bits: few rows, so the length has to be split
        dict(name="decode_one_very_long", op="decode", batch=1, heads=32, kv_heads=4, longest=250001, shortest=250001,
             page=128, pages=33000, dtype="bf16"),
        # one new token over the blocks that kept block means select from a long context
        dict(name="sparse_one_token", op="sparse", tokens=1, keys=32760, heads=24, kv_heads=24, block=64, top_k=32,
             causal=False, kept_means=True, dtype="bf16"),
        # one 39 x 40 frame of 56 heads
        dict(name="sparse_frame_56_heads", op="sparse", tokens=1560, keys=1560, heads=56, kv_heads=56, block=64,
             top_k=8, causal=False, kept_means=False, dtype="bf16"),
        # the rest of a causal prompt behind 2,048 tokens that are in the cache, grouped heads, wide blocks
        dict(name="sparse_causal_gqa_fp16", op="sparse", tokens=6145, keys=8193, heads=32, kv_heads=8, block=128,
             top_k=16, causal=True, kept_means=False, dtype="fp16"),
        # all tokens of a 21 x 39 x 40 grid, one key block of eight
        dict(name="sparse_grid", op="sparse", tokens=32760, keys=32760, heads=24, kv_heads=24, block=64, top_k=64,
             causal=False, kept_means=False, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _heads(rng):
    kv = rng.choice((1, 2, 3, 4, 8, 16, 24, 56))
    group = rng.choice((1, 1, 2, 3, 4, 8, 16)) if kv <= 8 else 1
    return kv * group, kv


def draw(rng):
    op = rng.choice(("append", "decode", "sparse"))
    heads, kv = _heads(rng)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "append":
        tokens = _spread(rng, 1, 32760 * 72 // (heads + 2 * kv) if heads + 2 * kv > 72 else 32760)
        page = rng.choice((8, 16, 32, 64, 128, 256))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, rot=rng.choice((16, 32, 64, 96, 112, 128)),
                    page=page, pages=tokens // page + rng.randint(2, 90), norm=rng.random() < 0.5, dtype=dtype,
                    table=rng.choice(("fp32", "bf16", "fp16")), padded=rng.choice((0, 0, min(3, tokens - 1))))
    if op == "decode":
        batch = _spread(rng, 1, 64)
        longest = _spread(rng, 1, min(250000, 4_000_000 // (batch * kv)))
        page = rng.choice((8, 16, 32, 64, 128, 256))
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv, longest=longest,
                    shortest=rng.choice((0, longest, longest // 2)), page=page,
                    pages=batch * (longest // page + 1) + rng.randint(1, 50), dtype=dtype)
    block = rng.choice((64, 64, 128))
    keys = _spread(rng, 1, 32760)
    causal = rng.random() < 0.4
    tokens = 1 if rng.random() < 0.2 else _spread(rng, 1, keys if causal else 32760)
    blocks = -(-keys // block)
    top_k = _spread(rng, 1, max(1, min(blocks, 4096 // block)))
    while 4 * D * heads * tokens * top_k * block > _LARGEST // 8:
        tokens = tokens // 2 + 1
    return dict(op=op, tokens=tokens, keys=keys, heads=heads, kv_heads=kv, block=block, top_k=top_k, causal=causal,
                kept_means=rng.random() < 0.5, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _randn(gen, *shape, dtype, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda").mul_(std).to(dtype)


def _angles(positions, rot):
    """[positions, rot / 2] rotation angles in 64 bits (far positions lose them in 32)."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    return positions.to(torch.float64)[:, None] * inv


def _table(count, rot, dtype):
    a = _angles(torch.arange(count, device="cuda"), rot)
    c, s = torch.cos(a), torch.sin(a)
    return torch.stack((c, -s, s, c), dim=-1).reshape(count, rot // 2, 2, 2).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    heads, kv = case["heads"], case["kv_heads"]
    if case["op"] == "append":
        t, page, pages = case["tokens"], case["page"], case["pages"]
        qkv = _randn(gen, t, (heads + 2 * kv) * D, dtype=dtype)     # one packed projection row per token
        q, k, v = (x.reshape(t, -1, D) for x in qkv.split((heads * D, kv * D, kv * D), dim=1))
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:t].contiguous()
        if t > 64:   # prompts fill whole pages in the order of their tokens, in pages from anywhere
            order = torch.randperm(pages, generator=gen, device="cuda")
            at = torch.arange(t, device="cuda")
            slots = order[at // page] * page + at % page
        if case["padded"]:
            slots[t - case["padded"]:] = -1
        rows = max(2 * t, 4096)
        first = int(torch.randint(0, rows - t + 1, (1,), generator=gen, device="cuda"))
        positions = torch.arange(first, first + t, device="cuda")
        if t <= 64:
            positions = torch.randint(0, rows, (t,), generator=gen, device="cuda")
        s = dict(case=case, q=q, k=k, v=v, slots=slots, positions=positions,
                 table=_table(rows, case["rot"], TABLES[case["table"]]),
                 k_cache=_randn(gen, pages, kv, page, D, dtype=dtype),
                 v_cache=_randn(gen, pages, kv, page, D, dtype=dtype),
                 q_out=torch.zeros(t, heads, D, dtype=dtype, device="cuda"), q_weight=None, k_weight=None)
        if case["norm"]:
            s["q_weight"] = (1 + _randn(gen, D, dtype=torch.float32, std=0.02)).to(dtype)
            s["k_weight"] = (1 + _randn(gen, D, dtype=torch.float32, std=0.02)).to(dtype)
        return s
    if case["op"] == "decode":
        b, page, pages = case["batch"], case["page"], case["pages"]
        lo, hi = case["shortest"], case["longest"]
        lengths = torch.randint(lo, hi + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        if lo == 0 and b > 2:
            lengths[b // 2], lengths[0], lengths[b - 1] = 0, hi, 1
        width = -(-hi // page)
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
        page_table = order[:b * width].reshape(b, width).contiguous()
        k_cache = torch.zeros(pages, kv, page, D, dtype=dtype, device="cuda")
        v_cache = torch.zeros(pages, kv, page, D, dtype=dtype, device="cuda")
        used, step = page_table.reshape(-1).long(), max(1, (1 << 27) // (kv * page * D))
        for at in range(0, used.numel(), step):
            ids = used[at:at + step]
            k_cache[ids] = _randn(gen, ids.numel(), kv, page, D, dtype=dtype)
            v_cache[ids] = _randn(gen, ids.numel(), kv, page, D, dtype=dtype)
        return dict(case=case, q=_randn(gen, b, heads, D, dtype=dtype, std=1.5), k_cache=k_cache, v_cache=v_cache,
                    page_table=page_table, lengths=lengths)
    t, n, block = case["tokens"], case["keys"], case["block"]
    # neighbouring tokens are alike: a part that changes every 48 tokens, beside each token's own
    def alike(tokens, hs, std):
        slow = torch.randn(tokens // 48 + 1, hs, D, generator=gen, device="cuda").mul_(std)
        x = torch.randn(tokens, hs, D, generator=gen, device="cuda")
        return x.add_(slow.repeat_interleave(48, dim=0)[:tokens]).to(dtype)
    s = dict(case=case, q=alike(t, heads, 0.7), k=alike(n, kv, 0.7), v=_randn(gen, n, kv, D, dtype=dtype),
             k_means=None)
    if case["kept_means"]:
        s["k_means"] = _means(s["k"], block)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _means(x, block):
    """fp32 [H, ceil(T / block), D] means of the blocks, summed in 64 bits: selections compare products of them."""
    t, h, d = x.shape
    n = -(-t // block)
    padded = torch.zeros(n * block, h, d, dtype=torch.float64, device=x.device)
    padded[:t] = x
    count = (t - torch.arange(n, device=x.device) * block).clamp(max=block).to(torch.float64)
    return (padded.reshape(n, block, h, d).sum(1) / count[:, None, None]).permute(1, 0, 2).to(torch.float32)


def _rotated(x, weight, table, dtype):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    half = table.shape[1]
    c = table.float()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    y0 = c[..., 0, 0] * a + c[..., 0, 1] * b
    y1 = c[..., 1, 0] * a + c[..., 1, 1] * b
    return torch.cat((y0, y1, x[..., 2 * half:]), dim=-1).to(dtype)


def _append(s):
    dtype = s["k"].dtype
    table = s["table"][s["positions"]]
    live = s["slots"] >= 0
    q = _rotated(s["q"], s["q_weight"], table, dtype)
    k = _rotated(s["k"], s["k_weight"], table, dtype)
    page = s["k_cache"].shape[2]
    slots = s["slots"][live]
    s["k_cache"][slots // page, :, slots % page] = k[live]
    s["v_cache"][slots // page, :, slots % page] = s["v"][live]
    s["q_out"].copy_(torch.where(live[:, None, None], q, s["q_out"]))
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": s["q_out"]}


def _decode(s):
    q, table, lengths = s["q"], s["page_table"].long(), s["lengths"]
    b, heads, _ = q.shape
    kv, page = s["k_cache"].shape[1:3]
    out, lse = [], []
    for i in range(b):   # one sequence at a time: the gathered keys of all of them are large
        n = table.shape[1] * page
        k = s["k_cache"][table[i]].transpose(0, 1).reshape(kv, n, D).float()
        v = s["v_cache"][table[i]].transpose(0, 1).reshape(kv, n, D).float()
        x = (q[i].float().reshape(kv, heads // kv, D) @ k.transpose(1, 2)) * D ** -0.5
        seen = torch.arange(n, device=q.device) < lengths[i]
        x = torch.where(seen, x, -math.inf)
        top = x.amax(-1, keepdim=True).clamp(min=-3e38)
        p = torch.exp(x - top)
        total = p.sum(-1, keepdim=True)
        out.append(torch.where(total > 0, (p @ v) / total.clamp(min=1e-30), 0.0).reshape(heads, D).to(q.dtype))
        lse.append((top + torch.log(total)).reshape(heads))
    return {"out": torch.stack(out), "lse": torch.stack(lse)}


def _selected(q_means, k_means, top_k, block, tokens, keys, causal):
    """int32 [kv heads, query blocks, top_k]: the key blocks of each query block, ascending, -1 behind them."""
    kv, n = k_means.shape[:2]
    scores = q_means.double().reshape(kv, -1, *q_means.shape[1:]).sum(1) @ k_means.double().transpose(1, 2)
    nq = scores.shape[1]
    if causal:
        first = torch.arange(nq, device=scores.device) * Q_BLOCK + keys - tokens
        last = torch.clamp(first + Q_BLOCK, max=keys) - 1
        start = torch.arange(n, device=scores.device) * block
        scores = torch.where(start[None] + block > first[:, None], math.inf, scores)   # the diagonal comes first
        scores = torch.where(start[None] > last[:, None], -math.inf, scores)           # the future never
    k = min(top_k, n)
    best, at = torch.sort(scores, dim=-1, descending=True, stable=True)
    best, at = best[..., :k], at[..., :k]
    at = torch.sort(torch.where(best > -math.inf, at, n), dim=-1).values
    blocks = torch.full((kv, nq, top_k), -1, dtype=torch.int32, device=scores.device)
    blocks[..., :k] = torch.where(at < n, at, -1)
    return blocks


def _sparse(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    t, heads, _ = q.shape
    n, kv, _ = k.shape
    block, top_k = c["block"], c["top_k"]
    group = heads // kv
    k_means = _means(k, block) if s["k_means"] is None else s["k_means"]
    blocks = _selected(_means(q, Q_BLOCK), k_means, top_k, block, t, n, c["causal"])
    nq = blocks.shape[1]
    rows = torch.arange(nq * Q_BLOCK, device=q.device).reshape(nq, Q_BLOCK) + (n - t)
    out = torch.empty_like(q)
    lse = torch.empty(t, heads, dtype=torch.float32, device=q.device)
    for h in range(kv):   # one key head at a time: its gathered keys are large
        at = (blocks[h].long()[..., None] * block + torch.arange(block, device=q.device)).reshape(nq, -1)
        seen = (at >= 0) & (at < n)
        at = at.clamp(0, n - 1)
        ks, vs = k[:, h][at].float(), v[:, h][at].float()
        mask = seen[:, None, :]
        if c["causal"]:
            mask = mask & (at[:, None, :] <= rows[:, :, None])
        for g in range(h * group, (h + 1) * group):
            qs = torch.zeros(nq * Q_BLOCK, D, device=q.device)
            qs[:t] = q[:, g]
            x = (qs.reshape(nq, Q_BLOCK, D) @ ks.transpose(1, 2)) * D ** -0.5
            x = torch.where(mask, x, -math.inf)
            top = x.amax(-1, keepdim=True).clamp(min=-3e38)
            p = torch.exp(x - top)
            total = p.sum(-1, keepdim=True)
            o = torch.where(total > 0, (p @ vs) / total.clamp(min=1e-30), 0.0)
            out[:, g] = o.reshape(-1, D)[:t].to(q.dtype)
            lse[:, g] = (top + torch.log(total)).reshape(-1)[:t]
    return {"out": out, "lse": lse, "blocks": blocks}


def run(state):
    c = state["case"]
    if own:
        h3 = _framework()
        if c["op"] == "append":
            q = h3.append_paged_kv(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slots"],
                                   state["table"], state["positions"], k_weight=state["k_weight"], q=state["q"],
                                   q_weight=state["q_weight"], q_out=state["q_out"])
            return {"k_cache": state["k_cache"], "v_cache": state["v_cache"], "q": q}
        if c["op"] == "decode":
            out, lse = h3.paged_decode_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"],
                                                 state["lengths"], return_lse=True)
            return {"out": out, "lse": lse}
        out, lse, blocks = h3.sparse_attention(state["q"], state["k"], state["v"], c["top_k"], c["block"],
                                               causal=c["causal"], k_means=state["k_means"], return_lse=True,
                                               return_blocks=True)
        return {"out": out, "lse": lse, "blocks": blocks}
    return {"append": _append, "decode": _decode, "sparse": _sparse}[c["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    heads, kv = case["heads"], case["kv_heads"]
    if case["op"] == "append":
        live = case["tokens"] - case["padded"]
        row = (heads + 2 * kv) * D * 2
        table = case["rot"] * 2 * torch.empty((), dtype=TABLES[case["table"]]).element_size()
        return {"bytes": live * (2 * row + table + 16), "flops": live * (heads + kv) * D * (7 if case["norm"] else 3)}
    if case["op"] == "decode":
        keys = case["batch"] * (case["longest"] + case["shortest"]) / 2
        return {"bytes": keys * kv * D * 4 + case["batch"] * heads * (4 * D + 4) + keys / case["page"] * 4,
                "flops": keys * heads * D * 4}
    t, n, block, top_k = case["tokens"], case["keys"], case["block"], case["top_k"]
    nq, nk = -(-t // Q_BLOCK), -(-n // block)
    pairs, most = 0, min(top_k * block, n)
    for i in range(nq):
        rows = min(Q_BLOCK, t - i * Q_BLOCK)
        seen = min(most, max(0, n - t + i * Q_BLOCK + rows // 2)) if case["causal"] else most
        pairs += rows * seen
    read = min(n, nq * most)
    means = nk * kv * D * 4 if case["kept_means"] else 0
    keys_read = read if case["kept_means"] else n
    return {"bytes": t * heads * (4 * D + 4) + (keys_read + read) * kv * D * 2 + means + nq * kv * top_k * 4,
            "flops": 4 * D * heads * pairs + 2 * D * kv * nq * nk}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_append(s):
    c, f = s["case"], torch.float64
    # the coefficients are the operator's inputs, in the table's own type
    coef = s["table"].to(f)[s["positions"]].reshape(c["tokens"], 1, c["rot"] // 2, 4)

    def turned(x, w):
        x = x.to(f)
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * w.to(f)
        y, r = x.clone(), c["rot"] // 2
        y[..., :r] = coef[..., 0] * x[..., :r] + coef[..., 1] * x[..., r:2 * r]
        y[..., r:2 * r] = coef[..., 2] * x[..., :r] + coef[..., 3] * x[..., r:2 * r]
        return y

    k, q = turned(s["k"], s["k_weight"]), turned(s["q"], s["q_weight"])
    k_cache, v_cache = s["k_cache"].to(f), s["v_cache"].to(f)
    n = c["tokens"] - c["padded"]
    flat_k = k_cache.transpose(1, 2).reshape(-1, c["kv_heads"], D)
    flat_v = v_cache.transpose(1, 2).reshape(-1, c["kv_heads"], D)
    flat_k[s["slots"][:n]] = k[:n]
    flat_v[s["slots"][:n]] = s["v"][:n].to(f)
    back = (c["pages"], c["page"], c["kv_heads"], D)
    q[n:] = 0
    return {"k_cache": flat_k.reshape(back).transpose(1, 2), "v_cache": flat_v.reshape(back).transpose(1, 2), "q": q}


def _exact_decode(s):
    c, f = s["case"], torch.float64
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(c["batch"], c["heads"], D, dtype=f, device="cuda")
    lse = torch.full((c["batch"], c["heads"]), -math.inf, dtype=f, device="cuda")
    for i, n in enumerate(s["lengths"].tolist()):
        if not n:
            continue
        at = torch.arange(n, device="cuda")
        page, row = s["page_table"][i].long()[at // c["page"]], at % c["page"]
        for h in range(c["kv_heads"]):
            k, v = s["k_cache"][page, h, row].to(f), s["v_cache"][page, h, row].to(f)
            own_q = slice(h * group, (h + 1) * group)
            x = torch.einsum("gd,nd->gn", s["q"][i, own_q].to(f), k) / math.sqrt(D)
            out[i, own_q] = torch.softmax(x, -1) @ v
            lse[i, own_q] = torch.logsumexp(x, -1)
    return {"out": out, "lse": lse}


def _exact_sparse(s):
    c, f = s["case"], torch.float64
    t, n, block, top_k = c["tokens"], c["keys"], c["block"], c["top_k"]
    group = c["heads"] // c["kv_heads"]
    nq, nk = -(-t // Q_BLOCK), -(-n // block)
    out = torch.zeros(t, c["heads"], D, dtype=f, device="cuda")
    lse = torch.full((t, c["heads"]), -math.inf, dtype=f, device="cuda")
    q_of, k_of = torch.arange(t, device="cuda") // Q_BLOCK, torch.arange(n, device="cuda") // block

    def mean(x, of, count):   # means are kept in 32 bits: the score is a product of those
        total = torch.zeros(count, D, dtype=f, device="cuda").index_add_(0, of, x.to(f))
        return (total / torch.bincount(of, minlength=count)[:, None]).float().to(f)

    for h in range(c["kv_heads"]):
        score = torch.zeros(nq, nk, dtype=f, device="cuda")
        km = mean(s["k"][:, h], k_of, nk)
        for g in range(group):
            score += torch.einsum("qd,kd->qk", mean(s["q"][:, h * group + g], q_of, nq), km)
        held = torch.zeros(nq, nk, dtype=torch.bool, device="cuda")
        for i in range(nq):
            row, last = score[i], nk
            if c["causal"]:
                lo, hi = i * Q_BLOCK + n - t, min((i + 1) * Q_BLOCK, t) + n - t - 1
                last = hi // block + 1
                row = row.clone()
                row[lo // block:last] = math.inf
            held[i, torch.sort(row[:last], descending=True, stable=True).indices[:top_k]] = True
        for at in range(0, t, 4096):
            of = q_of[at:at + 4096]
            mask = held[of][:, k_of]
            if c["causal"]:
                mask &= torch.arange(n, device="cuda") <= torch.arange(at, at + of.numel(), device="cuda")[:, None] + n - t
            for g in range(h * group, (h + 1) * group):
                x = torch.einsum("qd,kd->qk", s["q"][at:at + 4096, g].to(f), s["k"][:, h].to(f)) / math.sqrt(D)
                x.masked_fill_(~mask, -math.inf)
                lse[at:at + 4096, g] = torch.logsumexp(x, -1)
                out[at:at + 4096, g] = torch.softmax(x, -1) @ s["v"][:, h].to(f)
    return {"out": out, "lse": lse, "blocks": None}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "sparse": _exact_sparse}[case["op"]](s)
