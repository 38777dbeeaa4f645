"""Operators of tree-drafted decoding against plain 64-bit restatements:
step plan, tree attention over the paged cache, logits rules, tree commit."""
import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

# unit roundoff of the stored types
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _ops():
    from kvserve_b200 import ops
    return ops


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _indptr(new):
    return _i32(np.concatenate([[0], np.cumsum(new)]).tolist())


def _random_tree(rng, n):
    return [-1] + [rng.randrange(i) for i in range(1, n)]


def _paths(parents):
    """Node sets (the node and its ancestors) of one tree."""
    sets = []
    for i, p in enumerate(parents):
        sets.append((sets[p] if p >= 0 else set()) | {i})
    return sets


def _mask_tensor(sets_per_row, words):
    m = np.zeros((len(sets_per_row), words), np.uint32)
    for r, s in enumerate(sets_per_row):
        for j in s:
            m[r, j // 32] |= np.uint32(1 << (j % 32))
    return torch.from_numpy(m.view(np.int32)).cuda()


# ------------------------------------------------------------------ attention
def _attention_inputs(new, ctx, hq, hkv, D, bs, dtype, seed=0, layout="nhd", poison=True):
    """Inputs with shuffled blocks; whatever no row may read is NaN (cache
    slots past the context, blocks of nobody, rows of no request)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, B = sum(new), len(new)
    held = [-(-c // bs) for c in ctx]
    pool = sum(held) + 3
    perm = torch.randperm(pool, generator=g, device="cuda").tolist()
    width = max(held + [1]) + 2
    table = torch.full((B, width), pool + 1000, dtype=torch.int32)  # entries past the held blocks are no block ids
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = torch.tensor(perm[at:at + h], dtype=torch.int32)
        at += h

    def cache():
        if layout == "nhd":
            t = torch.empty(pool, bs, hkv, D, dtype=dtype, device="cuda")
        elif layout == "hnd":
            t = torch.empty(pool, hkv, bs, D, dtype=dtype, device="cuda").transpose(1, 2)
        else:  # one plane of an interleaved [blocks, 2, block_size, Hkv, D + 8] cache
            t = torch.empty(pool, 2, bs, hkv, D + 8, dtype=dtype, device="cuda")[:, 1, :, :, :D]
        t.copy_(torch.randn(pool, bs, hkv, D, generator=g, device="cuda").to(dtype))
        if poison:
            used = torch.zeros(pool, bs, dtype=torch.bool, device="cuda")
            for b, c in enumerate(ctx):
                for i in range(held[b]):
                    used[table[b, i].item(), : min(bs, c - i * bs)] = True
            t[~used] = math.nan
        return t

    def rows(heads):
        return torch.randn(R, heads, D, generator=g, device="cuda").to(dtype)
    return {"q": rows(hq), "kt": rows(hkv), "vt": rows(hkv), "kc": cache(), "vc": cache(), "table": table.cuda(),
            "ctx": _i32(ctx), "indptr": _indptr(new)}


def _attention_reference(x, new, ctx, sets, scale):
    """(result, bound) in 64 bits.  The bound: one rounding of the result, one
    of each probability to the K/V type before the second product (a relative
    error of at most U for each term of sum p |v|), and 2^-12 of the same sum
    for 32-bit scores (|score| below 32) and exponentials."""
    q = x["q"].double()
    u = U[x["q"].dtype]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    hkv, bs = x["kc"].shape[2], x["kc"].shape[1]
    group = q.shape[1] // hkv
    row = 0
    for b, n in enumerate(new):
        blocks = x["table"][b, : -(-ctx[b] // bs)].long()
        for h in range(hkv):
            kc = x["kc"][blocks][:, :, h].reshape(-1, q.shape[2])[: ctx[b]].double()
            vc = x["vc"][blocks][:, :, h].reshape(-1, q.shape[2])[: ctx[b]].double()
            for i in range(n):
                seen = [row + j for j in sorted(sets[row + i]) if j < n]
                k = torch.cat([kc, x["kt"][seen, h].double()])
                v = torch.cat([vc, x["vt"][seen, h].double()])
                if k.shape[0] == 0:
                    continue
                hs = slice(h * group, (h + 1) * group)
                p = torch.softmax(q[row + i, hs] @ k.T * scale, -1)
                out[row + i, hs] = p @ v
                bound[row + i, hs] = (u + 2.0 ** -12) * (p @ v.abs())
        row += n
    return out, bound + u * out.abs() + 1e-6


def _check_attention(x, new, ctx, sets, mask, scale=None):
    ops = _ops()
    got = ops.paged_tree_attention(x["q"], x["kt"], x["vt"], x["kc"], x["vc"], x["table"], x["ctx"], x["indptr"],
                                   tree_mask=mask, scale=scale)
    ops.check_device_status()
    ref, bound = _attention_reference(x, new, ctx, sets, scale or x["q"].shape[2] ** -0.5)
    bad = (got.double() - ref).abs() - bound
    assert torch.isfinite(got).all()
    assert (bad <= 0).all(), f"{bad.max().item():.3g} over the bound at {bad.argmax().item()}"
    return got


SHAPES = [
    # new, ctx, hq, hkv, D, bs, dtype, layout
    ([1], [0], 8, 2, 128, 16, torch.bfloat16, "nhd"),
    ([1], [1], 8, 2, 128, 16, torch.bfloat16, "nhd"),
    ([3], [63], 32, 8, 128, 16, torch.bfloat16, "nhd"),
    ([5, 1, 7], [64, 65, 129], 28, 4, 128, 16, torch.bfloat16, "nhd"),
    ([33, 0, 64], [128, 300, 17], 32, 8, 128, 16, torch.bfloat16, "nhd"),
    ([65, 2], [191, 256], 8, 1, 128, 32, torch.bfloat16, "nhd"),
    ([100, 31], [40, 77], 4, 4, 128, 64, torch.bfloat16, "nhd"),
    ([16, 9, 1, 1], [127, 0, 1000, 5], 16, 2, 64, 16, torch.bfloat16, "nhd"),
    ([7, 12], [513, 2], 28, 4, 128, 128, torch.float16, "nhd"),
    ([4, 4], [200, 90], 40, 8, 64, 8, torch.float16, "nhd"),
    ([9, 3], [77, 150], 8, 2, 128, 16, torch.bfloat16, "hnd"),
    ([9, 3], [77, 150], 8, 2, 128, 16, torch.bfloat16, "plane"),
    ([6, 3], [77, 150], 8, 2, 128, 5, torch.bfloat16, "nhd"),      # blocks that TMA boxes do not tile
    ([6, 3], [77, 31], 8, 2, 64, 1, torch.float16, "nhd"),
    ([6, 3], [177, 250], 8, 2, 128, 24, torch.bfloat16, "nhd"),
    ([6, 3], [177, 600], 8, 2, 128, 256, torch.bfloat16, "hnd"),
    ([40], [70], 32, 1, 128, 16, torch.bfloat16, "nhd"),            # 32 query heads on one KV head
    ([2], [5000], 16, 8, 128, 16, torch.bfloat16, "nhd"),
]


@pytest.mark.parametrize("new,ctx,hq,hkv,D,bs,dtype,layout", SHAPES)
def test_tree_attention_random_trees(new, ctx, hq, hkv, D, bs, dtype, layout):
    rng = random.Random(sum(ctx) + len(new))
    x = _attention_inputs(new, ctx, hq, hkv, D, bs, dtype, layout=layout)
    sets = [s for n in new if n for s in _paths(_random_tree(rng, n))]
    words = -(-max(new) // 32)
    _check_attention(x, new, ctx, sets, _mask_tensor(sets, words))


@pytest.mark.parametrize("group,D", [(17, 128), (20, 64), (24, 128), (64, 128), (128, 64)])
def test_tree_attention_large_groups(group, D):
    """More than 16 query heads a KV head, numbers among them that do not
    divide a row tile."""
    new, ctx = [9, 1, 15], [130, 0, 77]
    x = _attention_inputs(new, ctx, 2 * group, 2, D, 16, torch.bfloat16)
    sets = [s for n in new for s in _paths(_random_tree(random.Random(group), n))]
    _check_attention(x, new, ctx, sets, _mask_tensor(sets, 1))


@pytest.mark.parametrize("new,ctx", [([1, 1, 1], [0, 64, 200]), ([200], [100]), ([70, 3], [0, 33])])
def test_tree_attention_without_a_mask_is_causal(new, ctx):
    x = _attention_inputs(new, ctx, 8, 2, 128, 16, torch.bfloat16)
    sets = [set(range(i + 1)) for n in new for i in range(n)]
    _check_attention(x, new, ctx, sets, None)


def test_tree_attention_scale_and_sharp_scores():
    x = _attention_inputs([5, 5], [300, 90], 8, 2, 128, 16, torch.bfloat16)
    x["q"] *= 2
    sets = [s for _ in range(2) for s in _paths([-1, 0, 1, 1, 0])]
    _check_attention(x, [5, 5], [300, 90], sets, _mask_tensor(sets, 1), scale=0.11)


@pytest.mark.parametrize("drop", [9, 19.5, 25.2])
def test_tree_attention_fp16_tail_under_a_sink(drop):
    """Each request's fourth token takes nearly all of the weight and has a
    zero V; the result is what the many others (2^-drop of its weight each)
    leave.  Enough requests that a share holds many tiles with the sink's
    maximum: the others' probabilities must not lose bits to the smallest
    numbers that fp16 has."""
    new, ctx, D = [2] * 96, [1000 + b for b in range(96)], 128
    x = _attention_inputs(new, ctx, 8, 2, D, 16, torch.float16, poison=False)
    x["q"][:] = 1.0
    x["kc"] *= 2.0 ** -7                          # scores of the others: within a few hundredths of 0
    x["kt"] *= 2.0 ** -7
    x["vc"] = x["vc"].abs() + 0.5                 # nothing cancels
    x["vt"] = x["vt"].abs() + 0.5
    first = x["table"][:, 0].long()
    x["kc"][first, 3] = drop * math.log(2.0) / D ** 0.5  # a score of drop * ln 2
    x["vc"][first, 3] = 0.0
    sets = [s for n in new for s in _paths([-1] + [0] * (n - 1))]
    _check_attention(x, new, ctx, sets, _mask_tensor(sets, 1))


def test_tree_attention_rows_that_see_nothing_are_zero():
    new, ctx = [4, 3], [0, 50]
    x = _attention_inputs(new, ctx, 8, 2, 128, 16, torch.bfloat16)
    sets = [{0}, set(), {0, 1}, set(), {0}, set(), {1}]
    got = _check_attention(x, new, ctx, sets, _mask_tensor(sets, 1))
    assert (got[1] == 0).all() and (got[3] == 0).all() and (got[5] != 0).any()


def test_tree_attention_padding_rows_are_zero():
    x = _attention_inputs([6], [70], 8, 2, 128, 16, torch.bfloat16)
    x["indptr"] = _i32([0, 4])
    for name in ("q", "kt", "vt"):
        x[name][4:] = math.nan
    sets = _paths([-1, 0, 0, 2]) + [set(), set()]
    got = _check_attention(dict(x, q=x["q"]), [4], [70], sets, _mask_tensor(sets, 1))
    assert (got[4:] == 0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["kt", "vt"])
def test_tree_attention_masked_tokens_that_are_not_finite(value, where):
    """Node 2's own K or V is not finite; rows that do not see it are as if it
    were not there."""
    new, ctx = [40, 5], [90, 64]
    x = _attention_inputs(new, ctx, 8, 2, 128, 16, torch.bfloat16)
    rng = random.Random(3)
    trees = [_random_tree(rng, 40), [-1, 0, 0, 1, 0]]
    sets = [s for t in trees for s in _paths(t)]
    blind = [r for r, s in enumerate(sets) if 2 not in s]
    clean = _ops().paged_tree_attention(x["q"], x["kt"], x["vt"], x["kc"], x["vc"], x["table"], x["ctx"],
                                        x["indptr"], tree_mask=_mask_tensor(sets, 2))
    x[where][2, :, 5] = value
    x[where][42, 0] = value
    got = _ops().paged_tree_attention(x["q"], x["kt"], x["vt"], x["kc"], x["vc"], x["table"], x["ctx"], x["indptr"],
                                      tree_mask=_mask_tensor(sets, 2))
    assert len(blind) > 10 and torch.equal(got[blind], clean[blind])
    if where == "vt":  # rows that do see it carry it, in that column only
        row = next(r for r, s in enumerate(sets[:40]) if 2 in s)
        assert not torch.isfinite(got[row, :, 5]).any()
        assert torch.isfinite(got[row, :, :5]).all() and torch.isfinite(got[row, :, 6:]).all()


def test_tree_attention_reads_views_of_a_fused_projection():
    """q, K and V as views of one [R, (Hq + 2 Hkv) D] tensor, out as a view."""
    ops = _ops()
    hq, hkv, D, R = 8, 2, 128, 9
    x = _attention_inputs([9], [100], hq, hkv, D, 16, torch.bfloat16)
    qkv = torch.cat([x["q"].reshape(R, -1), x["kt"].reshape(R, -1), x["vt"].reshape(R, -1)], 1).contiguous()
    out = torch.full((R, hq + 3, D), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.paged_tree_attention(qkv[:, : hq * D].view(R, hq, D), qkv[:, hq * D:(hq + hkv) * D].view(R, hkv, D),
                             qkv[:, (hq + hkv) * D:].view(R, hkv, D), x["kc"], x["vc"], x["table"], x["ctx"],
                             x["indptr"], out=out[:, 1:hq + 1])
    want = ops.paged_tree_attention(x["q"], x["kt"], x["vt"], x["kc"], x["vc"], x["table"], x["ctx"], x["indptr"])
    assert torch.equal(out[:, 1:hq + 1], want) and (out[:, 0] == 7).all() and (out[:, hq + 1:] == 7).all()


def test_tree_attention_offsets_past_32_bits():
    """Blocks whose element offsets pass 2^31."""
    hq, hkv, D, bs = 8, 8, 128, 16
    pool = (1 << 31) // (bs * hkv * D) + 40
    ctx, new = [70], [3]
    x = _attention_inputs(new, ctx, hq, hkv, D, bs, torch.bfloat16, poison=False)
    far = torch.arange(pool - 5, pool, device="cuda")
    small = x["table"][0, :5].long()
    for name in ("kc", "vc"):
        big = torch.empty(pool, bs, hkv, D, dtype=torch.bfloat16, device="cuda")
        big[far] = x[name][small]
        x[name] = big
    x["table"][0, :5] = far.to(torch.int32)
    sets = _paths([-1, 0, 0])
    _check_attention(x, new, ctx, sets, _mask_tensor(sets, 1))


def test_tree_attention_many_requests_and_repeatability():
    rng = random.Random(9)
    new = [rng.randrange(0, 5) for _ in range(700)]
    ctx = [rng.choice([0, 1, rng.randrange(200)]) for _ in new]
    x = _attention_inputs(new, ctx, 8, 2, 64, 16, torch.bfloat16, poison=False)
    sets = [s for n in new if n for s in _paths(_random_tree(rng, n))]
    mask = _mask_tensor(sets, 1)
    first = _check_attention(x, new, ctx, sets, mask)
    for _ in range(3):
        again = _ops().paged_tree_attention(x["q"], x["kt"], x["vt"], x["kc"], x["vc"], x["table"], x["ctx"],
                                            x["indptr"], tree_mask=mask)
        assert torch.equal(first, again)


def test_tree_attention_long_context_splits():
    """One long context is shared out over the whole GPU; 512 query rows a KV head."""
    new, ctx = [64], [20011]
    x = _attention_inputs(new, ctx, 16, 2, 128, 16, torch.bfloat16, poison=False)
    sets = _paths(_random_tree(random.Random(5), 64))
    _check_attention(x, new, ctx, sets, _mask_tensor(sets, 2))


def test_tree_attention_single_tokens_match_paged_decode():
    """With one row a request the result is that of paged decode attention
    over a cache that already holds the token."""
    ops = _ops()
    ctx = [130, 15, 16, 64]
    x = _attention_inputs([1] * 4, ctx, 8, 2, 128, 16, torch.bfloat16, poison=False)
    got = ops.paged_tree_attention(x["q"], x["kt"], x["vt"], x["kc"], x["vc"], x["table"], x["ctx"], x["indptr"])
    kc, vc = torch.cat([x["kc"], x["kc"][:4]]), torch.cat([x["vc"], x["vc"][:4]])
    table = x["table"].clone()
    for b, c in enumerate(ctx):
        if c % 16 == 0:
            table[b, c // 16] = x["kc"].shape[0] + b
        blk = table[b, c // 16].item()
        kc[blk, c % 16], vc[blk, c % 16] = x["kt"][b], x["vt"][b]
    want = ops.paged_decode_attention(x["q"], kc, vc, table, x["ctx"] + 1, 131)
    # both round their result once and their probabilities at most once
    assert (got.float() - want.float()).abs().max() <= 4 * 2.0 ** -8 * want.float().abs().max()


def test_tree_attention_on_a_side_stream_and_in_a_graph():
    ops = _ops()
    x = _attention_inputs([5, 9], [300, 20], 8, 2, 128, 16, torch.bfloat16, poison=False)
    args = (x["q"], x["kt"], x["vt"], x["kc"], x["vc"], x["table"], x["ctx"], x["indptr"])
    want = ops.paged_tree_attention(*args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.paged_tree_attention(*args)
    s.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        ops.paged_tree_attention(*args, out=out)
    x["q"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.paged_tree_attention(*args)) and not torch.equal(out, want)


def test_tree_attention_refusals():
    ops = _ops()
    x = _attention_inputs([5], [40], 8, 2, 128, 16, torch.bfloat16, poison=False)

    def call(**kw):
        y = {**x, "mask": None, "out": None, **kw}
        return ops.paged_tree_attention(y["q"], y["kt"], y["vt"], y["kc"], y["vc"], y["table"], y["ctx"], y["indptr"],
                                        tree_mask=y["mask"], out=y["out"])
    call()
    bad = [
        dict(q=x["q"].float()), dict(q=x["q"].cpu()), dict(kt=x["kt"].half()), dict(q=x["q"][:, :7]),
        dict(q=x["q"][..., :96], kt=x["kt"][..., :96], vt=x["vt"][..., :96], kc=x["kc"][..., :96],
             vc=x["vc"][..., :96]),
        dict(kt=x["kt"][:4]), dict(table=x["table"].long()), dict(table=x["table"].repeat(2, 1)),
        dict(indptr=x["indptr"][:1]), dict(ctx=x["ctx"].long()), dict(mask=torch.zeros(4, 1, device="cuda", dtype=torch.int32)),
        dict(mask=torch.zeros(5, 1, device="cuda", dtype=torch.int64)), dict(out=torch.empty_like(x["q"][:4])),
        dict(q=torch.empty(5, 8, 129, device="cuda", dtype=torch.bfloat16)[..., 1:]), dict(vc=x["vc"][:-1]),
    ]
    for kw in bad:
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)
    empty = call(q=x["q"][:0], kt=x["kt"][:0], vt=x["vt"][:0], indptr=_i32([0, 0]))
    assert empty.shape == (0, 8, 128)


# ------------------------------------------------------------------------ plan
def _plan_reference(ctx, new, table, held, queue, head, tail, bs, R, parents, words):
    table, queue, held = [list(r) for r in table], list(queue), list(held)
    cap = len(queue)
    n = [max(v, 0) for v in new]
    need = [max(0, -(-(c + k) // bs) - h) if v >= 0 else 0 for c, k, h, v in zip(ctx, n, held, new)]
    dry = sum(need) > tail - head
    old = [list(r) for r in table]
    if not dry:
        for b, k in enumerate(need):
            for i in range(k):
                table[b][held[b] + i] = queue[head % cap]
                head += 1
    got = [h + (0 if dry else k) for h, k in zip(held, need)]
    for b, v in enumerate(new):
        if v < 0:
            for i in range(held[b]):
                queue[tail % cap] = old[b][i]
                tail += 1
            got[b] = 0
    indptr = np.concatenate([[0], np.cumsum(n)]).tolist()
    request, slots, pos, mask = [-1] * R, [-1] * R, [0] * R, [set() for _ in range(R)]
    for b in range(len(ctx)):
        par = parents[indptr[b]:indptr[b + 1]] if parents else None
        sets = _paths(par) if par else None
        for i in range(n[b]):
            r, p = indptr[b] + i, ctx[b] + i
            request[r], pos[r] = b, p
            if p // bs < got[b]:
                slots[r] = table[b][p // bs] * bs + p % bs
            if par:
                mask[r], pos[r] = sets[i], ctx[b] + len(sets[i]) - 1
    return indptr, request, pos, slots, mask, got, table, queue, head, tail


def _plan_state(rng, B, bs, n, spare, extra=0):
    ctx = [rng.choice([0, 1, rng.randrange(5 * bs + 2)]) for _ in range(B)]
    held = [-(-c // bs) + (rng.randrange(2) if extra else 0) for c in ctx]
    new = [rng.choice([-1, 0, 1, rng.randrange(n + 1)]) for _ in range(B)]
    width = max(max(held), max(-(-(c + max(v, 0)) // bs) for c, v in zip(ctx, new))) + 1
    pool = sum(held) + spare
    ids = list(range(pool))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    head = rng.randrange(3 * pool)
    queue = [-9] * pool
    for i in range(spare):
        queue[(head + i) % pool] = ids[at + i]
    return ctx, new, held, table, queue, head, head + spare


@pytest.mark.parametrize("B,bs,n,tree,spare,padding", [
    (1, 16, 1, False, 4, 0), (1, 16, 40, True, 8, 3), (7, 16, 30, True, 40, 0), (300, 16, 9, True, 900, 50),
    (700, 1, 5, False, 4000, 0), (2500, 7, 30, False, 14000, 100), (33, 100, 300, False, 200, 1),
    (6, 16, 20, True, 0, 0), (40, 16, 20, False, 3, 0), (5, 16, 100, True, 60, 0)])
def test_plan_step(B, bs, n, tree, spare, padding):
    ops = _ops()
    rng = random.Random(B * 131 + n)
    ctx, new, held, table, queue, head, tail = _plan_state(rng, B, bs, n, spare, extra=1)
    R = sum(max(v, 0) for v in new) + padding
    parents = None
    if tree:
        parents = [p for v in new if v > 0 for p in _random_tree(rng, v)] + [0] * padding
    words = -(-n // 32)
    want = _plan_reference(ctx, new, table, held, queue, head, tail, bs, R, parents, words)
    t_table, t_queue = _i32(table), _i32(queue)
    cursor = torch.tensor([head, tail], device="cuda")
    args = (_i32(ctx), _i32(new), t_table, _i32(held), t_queue, cursor, bs, R)
    p = ops.plan_step(*args, parents=_i32(parents) if tree else None, max_tree=n)
    dry = sum(want[5]) < sum(max(h, 0 if v < 0 else -(-(c + max(v, 0)) // bs))
                             for h, c, v in zip(held, ctx, new) if v >= 0)
    if dry:
        with pytest.raises(RuntimeError, match="no free KV blocks"):
            ops.check_device_status()
    else:
        ops.check_device_status()
    assert p.indptr.tolist() == want[0] and p.row_request.tolist() == want[1]
    assert p.positions.tolist() == want[2] and p.slot_mapping.tolist() == want[3]
    assert p.held.tolist() == want[5] and t_table.tolist() == want[6] and t_queue.tolist() == want[7]
    assert p.cursor.tolist() == [want[8], want[9]]
    if tree:
        assert torch.equal(p.tree_mask, _mask_tensor(want[4], words))


def test_plan_step_updates_its_state_in_place():
    """Steps that grow, end and restart requests, with the plan's own outputs
    as the state: blocks are never lost or handed out twice."""
    ops = _ops()
    rng = random.Random(4)
    B, bs, pool, W = 64, 16, 400, 40
    ctx = _i32([0] * B)
    table, queue = torch.zeros(B, W, dtype=torch.int32, device="cuda"), _i32(list(range(pool)))
    plan, R = None, B * 9
    held, cursor = _i32([0] * B), torch.tensor([0, pool], device="cuda")
    for _ in range(30):
        new = _i32([rng.choice([-1, 0, 3, 9]) for _ in range(B)])
        if plan is None:
            plan = ops.plan_step(ctx, new, table, held, queue, cursor, bs, R)
        else:
            plan = ops.plan_step(ctx, new, table, plan.held, queue, plan.cursor, bs, R, out=plan)
        ops.check_device_status()
        ctx = torch.where(new < 0, torch.zeros_like(ctx), ctx + new.clamp(min=0))
        h, (head, tail) = plan.held.tolist(), plan.cursor.tolist()
        owned = [v for b in range(B) for v in table[b, :h[b]].tolist()]
        free = [queue[i % pool].item() for i in range(head, tail)]
        assert sorted(owned + free) == list(range(pool))
        slots = plan.slot_mapping[: plan.indptr[-1]].tolist()
        assert len(set(slots)) == len(slots) and min(slots, default=0) >= 0


def test_plan_step_over_several_blocks_updates_its_state_in_place():
    """As above with more rows than one block of threads plans (the state is
    then written by a second launch), against separate outputs."""
    ops = _ops()
    rng = random.Random(8)
    B, bs, pool, W = 70, 16, 3000, 60
    R = B * 33
    ctx = _i32([0] * B)
    table, queue = torch.zeros(B, W, dtype=torch.int32, device="cuda"), _i32(list(range(pool)))
    held, cursor = _i32([0] * B), torch.tensor([0, pool], device="cuda")
    state = None
    for _ in range(25):
        new = _i32([rng.choice([-1, 0, 3, 33, 33]) for _ in range(B)])
        t2, q2 = table.clone(), queue.clone()
        want = ops.plan_step(ctx, new, t2, held, q2, cursor, bs, R)
        if state is None:
            state = want._replace(held=held.clone(), cursor=cursor.clone())
        got = ops.plan_step(ctx, new, table, state.held, queue, state.cursor, bs, R, out=state)
        ops.check_device_status()
        assert got is state and torch.equal(table, t2) and torch.equal(queue, q2)
        for a, b in zip(got, want):
            assert a is None and b is None or torch.equal(a, b)
        held, cursor = state.held.clone(), state.cursor.clone()
        ctx = torch.where(new < 0, torch.zeros_like(ctx), ctx + new.clamp(min=0))
        ctx = ctx.clamp(max=(W - 3) * bs)
        held_list, (head, tail) = held.tolist(), cursor.tolist()
        owned = [v for b in range(B) for v in table[b, :held_list[b]].tolist()]
        assert sorted(owned + [queue[i % pool].item() for i in range(head, tail)]) == list(range(pool))


def test_plan_step_reports_what_does_not_fit():
    ops = _ops()
    queue, cursor = _i32(list(range(8))), torch.tensor([0, 8], device="cuda")
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")

    def status(ctx, new, R, parents=None, max_tree=64, table=table):
        p = ops.plan_step(_i32(ctx), _i32(new), table.clone(), _i32([0, 0]), queue.clone(), cursor, 16, R,
                          parents=parents, max_tree=max_tree)
        code = ops.device_status()[0].item()
        ops.device_status().zero_()
        return code, p
    assert status([0, 0], [3, 4], 7)[0] == 0
    code, p = status([0, 0], [3, 4], 5)               # more rows than the row tensors hold
    assert code == 4 and p.indptr.tolist() == [0, 3, 5]
    code, p = status([0, 0], [3, 40], 43)             # table too narrow: 40 tokens need three blocks
    assert code == 4 and p.slot_mapping[3 + 32:].tolist() == [-1] * 8
    code, p = status([0, 0], [2, 3], 5, parents=_i32([-1, 0, -1, 5, 1]))   # a parent that comes later
    assert code == 3 and p.tree_mask[:, 0].tolist() == [1, 3, 1, 2, 6]
    assert status([0, 0], [1, 33], 34, parents=_i32([-1] + [-1] + list(range(32))), max_tree=32,
                  table=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))[0] == 4


def test_plan_step_refusals():
    ops = _ops()
    good = dict(ctx=_i32([1, 2]), new=_i32([1, 1]), table=torch.zeros(2, 3, dtype=torch.int32, device="cuda"),
                held=_i32([1, 1]), queue=_i32([3, 4]), cursor=torch.tensor([0, 2], device="cuda"), bs=16, R=2,
                parents=None)

    def call(**kw):
        y = dict(good, **kw)
        return ops.plan_step(y["ctx"], y["new"], y["table"], y["held"], y["queue"], y["cursor"], y["bs"], y["R"],
                             parents=y["parents"])
    call()
    for kw in [dict(ctx=good["ctx"].long()), dict(new=_i32([1])), dict(table=good["table"][:1]),
               dict(table=good["table"].t()), dict(held=good["held"].cpu()), dict(queue=_i32([])),
               dict(cursor=_i32([0, 2])), dict(bs=0), dict(bs=1 << 31), dict(parents=_i32([0])),
               dict(ctx=_i32([1, 2])[::1].repeat(9000), new=_i32([1, 1]).repeat(9000))]:
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)


# ---------------------------------------------------------------------- commit
def _commit_reference(drafts, targets, parents, indptr):
    paths = []
    for b in range(len(indptr) - 1):
        lo, n = indptr[b], indptr[b + 1] - indptr[b]
        path = [0] if n else []
        while path:
            kids = [i for i in range(path[-1] + 1, n) if parents[lo + i] == path[-1]
                    and drafts[lo + i] == targets[lo + path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        paths.append(path)
    return paths


@pytest.mark.parametrize("new,L,hkv,D,bs,dtype,chain", [
    ([1], 1, 2, 128, 16, torch.bfloat16, False), ([8], 3, 8, 128, 16, torch.bfloat16, False),
    ([0, 5, 1, 70], 2, 3, 64, 7, torch.float16, False), ([33, 200], 2, 1, 128, 32, torch.bfloat16, False),
    ([9, 4], 2, 2, 128, 16, torch.bfloat16, True), ([5] * 300, 1, 2, 8, 4, torch.float32, False)])
def test_commit_tree(new, L, hkv, D, bs, dtype, chain):
    ops = _ops()
    rng = random.Random(len(new) + sum(new))
    R, B = sum(new) + 3, len(new)
    indptr = np.concatenate([[0], np.cumsum(new)]).tolist()
    parents, drafts, targets = [], [], [rng.randrange(50) for _ in range(R)]
    for b, n in enumerate(new):
        tree = list(range(-1, n - 1)) if chain else _random_tree(rng, n) if n else []
        for i, p in enumerate(tree):
            parents.append(p)
            drafts.append(targets[indptr[b] + p] if p >= 0 and rng.random() < 0.7 else rng.randrange(50))
    parents, drafts = parents + [0] * 3, drafts + [0] * 3
    ctx = [rng.randrange(40) for _ in new]
    pool = sum(-(-(c + n) // bs) for c, n in zip(ctx, new)) + 2
    slots = rng.sample(range(pool * bs), R)
    g = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(L, 2, R, hkv, D, generator=g, device="cuda").to(dtype)
    cache = torch.randn(L, 2, pool, bs, hkv, D, generator=g, device="cuda").to(dtype)
    tokens = torch.full((B, 40 + max(new) + 1), -5, dtype=torch.int32, device="cuda")
    want_cache, want_tokens = cache.clone(), tokens.clone()
    paths = _commit_reference(drafts, targets, parents, indptr)
    want_path = [-1] * R
    for b, path in enumerate(paths):
        for k, node in enumerate(path):
            want_path[indptr[b] + k] = node
            s = slots[indptr[b] + k]
            want_cache[:, :, s // bs, s % bs] = kv[:, :, indptr[b] + node]
            want_tokens[b, ctx[b] + k] = drafts[indptr[b] + node]
    t_ctx = _i32(ctx)
    c = ops.commit_tree(_i32(drafts), _i32(targets), None if chain else _i32(parents), _i32(indptr), t_ctx,
                        _i32(slots), tree_kv=kv, kv_cache=cache, tokens=tokens)
    ops.check_device_status()
    assert c.accepted.tolist() == [len(p) for p in paths] and c.path.tolist() == want_path
    assert c.next_ids.tolist() == [targets[indptr[b] + p[-1]] if p else -1 for b, p in enumerate(paths)]
    assert c.ctx_lens.tolist() == [a + len(p) for a, p in zip(ctx, paths)]
    assert torch.equal(cache, want_cache) and torch.equal(tokens, want_tokens)
    assert max(len(p) for p in paths) > (1 if sum(new) > 4 else 0)


def test_commit_tree_updates_context_lengths_in_place():
    """Accepted chains longer than a block of threads, with ``ctx_lens`` as the
    output too: tokens and lengths are those of separate outputs."""
    ops = _ops()
    new = [300, 1, 700, 64, 1024, 33] * 4
    R, B = sum(new), len(new)
    indptr = np.concatenate([[0], np.cumsum(new)]).tolist()
    drafts = [1 + r for r in range(R)]
    targets = drafts[1:] + [0]  # every node carries what was chosen after the one before: all accepted
    ctx = _i32([(37 * b) % 50 for b in range(B)])
    width = 50 + max(new)

    def commit(out, ctx):
        tokens = torch.full((B, width), -5, dtype=torch.int32, device="cuda")
        c = ops.commit_tree(_i32(drafts), _i32(targets), None, _i32(indptr), ctx, _i32([0] * R), tokens=tokens, out=out)
        ops.check_device_status()
        return c, tokens
    want, want_tokens = commit(None, ctx)
    assert want.accepted.tolist() == new and want.ctx_lens.tolist() == (ctx + _i32(new)).tolist()
    for b, n in enumerate(new):
        c = ctx[b].item()
        assert want_tokens[b, c:c + n].tolist() == drafts[indptr[b]:indptr[b + 1]]
        assert (want_tokens[b, :c] == -5).all() and (want_tokens[b, c + n:] == -5).all()
    for _ in range(20):
        state = ctx.clone()
        out = ops.TreeCommit(torch.empty_like(ctx), torch.empty(R, dtype=torch.int32, device="cuda"),
                             torch.empty_like(ctx), state)
        got, tokens = commit(out, state)
        assert got.ctx_lens is state and torch.equal(tokens, want_tokens)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_commit_tree_lowest_child_wins_and_strided_rows():
    """Two children carry the accepted token; K/V rows and cache are views."""
    ops = _ops()
    parents, drafts = _i32([-1, 0, 0, 0, 2, 3]), _i32([4, 9, 7, 7, 5, 5])
    targets = _i32([7, 0, 5, 5, 8, 3])
    wide = torch.randn(2, 2, 6, 3, 200, device="cuda", dtype=torch.bfloat16)
    kv = wide[..., :2, 8:136]
    big = torch.zeros(2, 3, 2, 4, 16, 128, device="cuda", dtype=torch.bfloat16)  # [L, blocks, 2, Hkv, bs, D]
    cache = big.permute(0, 2, 1, 4, 3, 5)[..., :2, :]
    c = ops.commit_tree(drafts, targets, parents, _i32([0, 6]), _i32([3]), _i32([40, 41, 2, 3, 4, 5]), tree_kv=kv,
                        kv_cache=cache)
    assert c.path.tolist() == [0, 2, 4, -1, -1, -1] and c.next_ids.tolist() == [8]
    for k, (node, s) in enumerate([(0, 40), (2, 41), (4, 2)]):
        assert torch.equal(cache[:, :, s // 16, s % 16], kv[:, :, node])
    assert (big[:, :, :, 2:] == 0).all() and (big != 0).sum() == 3 * 2 * 2 * 2 * 128
    walk_only = ops.commit_tree(drafts, targets, parents, _i32([0, 6]), _i32([3]), _i32([0] * 6))
    assert walk_only.path.tolist() == c.path.tolist()


def test_commit_tree_without_a_slot_is_reported():
    ops = _ops()
    kv = torch.ones(1, 2, 2, 1, 64, device="cuda", dtype=torch.bfloat16)
    cache = torch.zeros(1, 2, 2, 16, 1, 64, device="cuda", dtype=torch.bfloat16)
    for slot in (-1, 32):
        ops.commit_tree(_i32([1, 2]), _i32([2, 3]), None, _i32([0, 2]), _i32([0]), _i32([5, slot]), tree_kv=kv,
                        kv_cache=cache)
        with pytest.raises(RuntimeError, match="bad size"):
            ops.check_device_status()
        assert cache.sum() == 2 * 64
    with pytest.raises(RuntimeError, match="bad size"):  # the token buffer is too short
        ops.commit_tree(_i32([1, 2]), _i32([2, 3]), None, _i32([0, 2]), _i32([0]), _i32([5, 6]),
                        tokens=torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
        ops.check_device_status()


def test_commit_tree_refusals():
    ops = _ops()
    kv = torch.ones(1, 2, 2, 1, 64, device="cuda", dtype=torch.bfloat16)
    cache = torch.zeros(1, 2, 2, 16, 1, 64, device="cuda", dtype=torch.bfloat16)
    good = dict(d=_i32([1, 2]), t=_i32([2, 3]), p=None, i=_i32([0, 2]), c=_i32([0]), s=_i32([5, 6]), kv=kv,
                cache=cache, tokens=None)

    def call(**kw):
        y = dict(good, **kw)
        return ops.commit_tree(y["d"], y["t"], y["p"], y["i"], y["c"], y["s"], tree_kv=y["kv"], kv_cache=y["cache"],
                               tokens=y["tokens"])
    call()
    for kw in [dict(d=good["d"].long()), dict(t=_i32([1])), dict(p=_i32([0])), dict(i=_i32([0])), dict(kv=None),
               dict(cache=cache.half()), dict(cache=cache[..., :32]), dict(kv=kv[:, :, :1]),
               dict(kv=torch.ones(1, 2, 2, 1, 65, device="cuda", dtype=torch.bfloat16)[..., 1:]),
               dict(tokens=torch.zeros(2, 4, dtype=torch.int32, device="cuda")), dict(s=good["s"].cpu())]:
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)


# ---------------------------------------------------------------------- logits
def _logits_inputs(B, new, V, M, dtype, seed=0, hist=None):
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    R = sum(new)
    lens = hist or [rng.choice([0, 1, rng.randrange(M + 1), M]) for _ in range(B)]
    prompt = [rng.randrange(n + 2) for n in lens]
    tokens = torch.randint(0, min(V, 60), (B, M), generator=g, device="cuda").to(torch.int32)
    trees = [_random_tree(rng, n) if n else [] for n in new]
    sets = [s for t in trees if t for s in _paths(t)]
    indptr = np.concatenate([[0], np.cumsum(new)]).tolist()
    request = [b for b, n in enumerate(new) for _ in range(n)]
    positions = [lens[request[r]] + len(sets[r]) - 1 for r in range(R)]
    return {"logits": (4 * torch.randn(R, V, generator=g, device="cuda")).to(dtype), "row_request": _i32(request),
            "tokens": tokens, "token_lens": _i32(lens), "prompt_lens": _i32(prompt),
            "repetition": torch.tensor([rng.choice([0.7, 1.0, 1.5]) for _ in range(B)], device="cuda"),
            "frequency": torch.tensor([rng.choice([0.0, 0.3, -0.2]) for _ in range(B)], device="cuda"),
            "presence": torch.tensor([rng.choice([0.0, 0.9, -0.4]) for _ in range(B)], device="cuda"),
            "draft_ids": torch.randint(0, min(V, 60), (R,), generator=g, device="cuda").to(torch.int32),
            "indptr": _i32(indptr), "positions": _i32(positions),
            "tree_mask": _mask_tensor(sets, -(-max(new) // 32))}, sets


def _logits_reference(x, sets, bias=None, allowed=None, index=None, vocab_begin=0):
    """(result, bound) in 64 bits: five 32-bit operations on terms no larger
    than the sum of magnitudes, one rounding to the stored type."""
    R, V = x["logits"].shape
    out, mag = x["logits"].double().clone(), x["logits"].double().abs()
    indptr = x["indptr"].tolist()
    for r in range(R):
        b = x["row_request"][r].item()
        if b >= 0:
            n, p0 = x["token_lens"][b].item(), x["prompt_lens"][b].item()
            text = [(t, i >= p0) for i, t in enumerate(x["tokens"][b, :n].tolist())]
            text += [(x["draft_ids"][indptr[b] + j].item(), x["positions"][indptr[b] + j].item() >= p0)
                     for j in sorted(sets[r])]
            counts = {}
            for t, made in text:
                counts[t] = counts.get(t, 0) + made
            rep, fr, pr = (x[k][b].double().item() for k in ("repetition", "frequency", "presence"))
            for t, c in counts.items():
                v = t - vocab_begin
                if not 0 <= v < V:
                    continue
                y = out[r, v].item()
                y = y / rep if y > 0 else y * rep
                out[r, v] = y - fr * c - (pr if c else 0)
                mag[r, v] = abs(y) + abs(fr) * c + abs(pr)
            for t, v in (bias or {}).get(b, []):
                if 0 <= t - vocab_begin < V:
                    out[r, t - vocab_begin] += v
                    mag[r, t - vocab_begin] += abs(v)
        if allowed is not None and (index is None or index[r] >= 0):
            row = allowed[r if index is None else index[r]]
            ok = torch.tensor([(int(row[v // 32]) >> (v % 32)) & 1 for v in range(V)], device="cuda")
            out[r, ok == 0] = -math.inf
    return out, 8 * 2.0 ** -24 * mag + U[x["logits"].dtype] * out.abs().nan_to_num(posinf=0.0)


def _check_logits(x, sets, bias=None, words=None, index=None, vocab_begin=0, **more):
    ops = _ops()
    R = x["logits"].shape[0]
    greedy, value = torch.empty(R, dtype=torch.int32, device="cuda"), torch.empty(R, device="cuda")
    kw = {k: v for k, v in x.items() if k != "logits"}
    got = ops.process_logits(x["logits"], vocab_begin=vocab_begin, greedy=greedy, greedy_val=value, **kw, **more)
    ref, bound = _logits_reference(x, sets, bias, words, index, vocab_begin)
    hidden = ref == -math.inf
    assert torch.equal(got == -math.inf, hidden)
    assert ((got.double() - ref).abs() <= bound)[~hidden].all()
    host = got.float().cpu().numpy()
    assert greedy.tolist() == (host.argmax(1) + vocab_begin).tolist()  # numpy: the first of equal values
    assert value.tolist() == host.max(1).tolist()
    return got


@pytest.mark.parametrize("B,new,V,M,dtype", [
    (1, [1], 128, 5, torch.float32), (1, [1], 1, 3, torch.float32), (3, [1, 1, 1], 1000, 40, torch.bfloat16),
    (2, [9, 40], 4099, 100, torch.bfloat16), (3, [3, 0, 2], 70001, 33, torch.float16),
    (2, [2, 1], 50257, 600, torch.float32), (40, [1] * 40, 333, 64, torch.float16)])
def test_process_logits_penalties(B, new, V, M, dtype):
    x, sets = _logits_inputs(B, new, V, M, dtype)
    _check_logits(x, sets)


def test_process_logits_long_history_and_counts():
    """One token a hundred thousand times."""
    x, sets = _logits_inputs(1, [1], 300, 100000, torch.float32, hist=[100000])
    x["tokens"][:] = 7
    x["frequency"][:] = 1.0 / 1024
    x["prompt_lens"][:] = 3
    _check_logits(x, sets)


def test_process_logits_bias_and_grammar():
    V, new = 5003, [3, 1, 2, 1]
    x, sets = _logits_inputs(4, new, V, 50, torch.bfloat16, seed=2)
    rng = random.Random(1)
    ids = [rng.sample(range(V), 39) + [-1] for _ in range(4)]
    ids[1][3], ids[1][4], ids[2] = ids[1][0], ids[1][0], [-1] * 40      # listed three times; none at all
    values = torch.randn(4, 40, device="cuda") * 5
    bias = {b: [(t, v) for t, v in zip(ids[b], values[b].double().tolist()) if t >= 0] for b in range(4)}
    words = np.random.RandomState(0).randint(-2**31, 2**31, (3, -(-V // 32)), dtype=np.int64)
    words[2] = 0                                                        # a grammar that allows nothing
    index = [0, -1, 2, 1, 0, 1, -1]
    got = _check_logits(x, sets, bias, words & 0xffffffff, index, bias_ids=_i32(ids), bias_values=values,
                        allowed=torch.from_numpy(words.astype(np.int32)).cuda(), allowed_index=_i32(index))
    assert (got[2] == -math.inf).all()


def test_process_logits_vocab_shard_and_rows_without_a_request():
    x, sets = _logits_inputs(2, [3, 2], 40, 30, torch.float32, seed=5)
    x["row_request"][1] = -1
    sets[1] = set()
    ids, values = _i32([[22, 21, 60], [1, 59, 20]]), torch.randn(2, 3, device="cuda")
    bias = {b: list(zip(ids[b].tolist(), values[b].double().tolist())) for b in range(2)}
    _check_logits(x, sets, bias, vocab_begin=20, bias_ids=ids, bias_values=values)


def test_process_logits_without_a_mask_counts_earlier_rows():
    x, _ = _logits_inputs(2, [5, 3], 100, 20, torch.float32, seed=6)
    x["positions"] = torch.cat([x["token_lens"][b] + torch.arange(n, device="cuda", dtype=torch.int32)
                                for b, n in enumerate([5, 3])])
    sets = [set(range(i + 1)) for n in (5, 3) for i in range(n)]
    del x["tree_mask"]
    _check_logits(x, sets)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_process_logits_values_that_are_not_finite(dtype):
    """The mask replaces whatever stands there; outside it infinities and NaN
    pass through; the greedy choice is the first NaN, else the first maximum."""
    ops = _ops()
    x = torch.zeros(5, 70, device="cuda", dtype=dtype)
    x[0, 3], x[0, 40] = math.nan, 2.0
    x[1, 5], x[1, 6] = math.inf, math.nan
    x[2] = -math.inf
    x[3, 0], x[3, 1] = -0.0, 0.0
    x[4] = torch.finfo(dtype).min
    x[4, 69] = -math.inf
    allowed = torch.full((5, 3), -1, dtype=torch.int32, device="cuda")
    allowed[0, 0] = ~8                      # hides the NaN
    greedy = torch.empty(5, dtype=torch.int32, device="cuda")
    got = ops.process_logits(x, allowed=allowed, greedy=greedy)
    assert got[0, 3] == -math.inf and greedy.tolist() == [40, 6, 0, 0, 0]
    want = x.clone()
    want[0, 3] = -math.inf
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_process_logits_in_place_strided_and_unaligned():
    ops = _ops()
    for V, off in ((1003, 1), (1003, 0), (1000, 3), (2048, 8)):
        x, sets = _logits_inputs(2, [3, 2], V, 30, torch.bfloat16, seed=7)
        want = _check_logits(x, sets)
        wide = torch.zeros(5, V + 13, device="cuda", dtype=torch.bfloat16)
        view = wide[:, off:off + V]
        view.copy_(x["logits"])
        kw = {k: v for k, v in x.items() if k != "logits"}
        got = ops.process_logits(view, out=view, **kw)
        assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
        assert (wide[:, :off] == 0).all() and (wide[:, off + V:] == 0).all()


def test_process_logits_refusals():
    ops = _ops()
    x, _ = _logits_inputs(2, [3, 2], 100, 30, torch.float32)
    logits = x.pop("logits")
    ops.process_logits(logits, **x)
    bad = [dict(logits=logits.double()), dict(logits=logits.cpu()), dict(logits=logits.t()), dict(token_lens=None),
           dict(indptr=None), dict(row_request=None), dict(frequency=x["frequency"].double()),
           dict(positions=x["positions"][:3]), dict(tokens=x["tokens"].long()),
           dict(bias_ids=_i32([[1], [2]])), dict(allowed=torch.zeros(5, 3, dtype=torch.int32, device="cuda")),
           dict(allowed=torch.zeros(4, 4, dtype=torch.int32, device="cuda")),
           dict(allowed_index=_i32([0] * 5)), dict(out=torch.empty(5, 99, device="cuda")),
           dict(greedy=torch.empty(5, dtype=torch.int64, device="cuda")), dict(greedy_val=torch.empty(5, device="cuda")),
           dict(vocab_begin=-1), dict(tree_mask=x["tree_mask"][:2])]
    for kw in bad:
        y = {**x, "logits": logits, **kw}
        with pytest.raises((ValueError, RuntimeError)):
            ops.process_logits(y.pop("logits"), **y)
    assert ops.process_logits(logits[:0]).shape == (0, 100)
