"""Workloads of the operators behind one step of tree-drafted decoding: the
step plan (block tables, slots, tree masks), attention of a tree of drafted
tokens over the paged cache, the rules on the logits (penalties, biases,
grammar masks) and the commit of the accepted path.

``own`` False computes each operator from elementary torch operations in 32
bits; ``own`` True calls ``kvserve_b200.ops``.  The layouts are those of the
public entry points: paged caches ``[num_blocks, block_size, Hkv, D]``, rows
of all requests packed in ``[R, ...]`` with ``indptr`` ``[B + 1]``.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BITS = 32


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one interactive request early in its answer: latency of a small verify step (8B heads)
        _attention("attn b1 n8 ctx700", B=1, n=8, ctx=700, hq=32, hkv=8, ragged=1),
        # a small batch of medium contexts with full 32-token trees: one 128-row tile per KV head
        _attention("attn b8 n32 ctx6k", B=8, n=32, ctx=6000, hq=32, hkv=8, ragged=2),
        # a loaded server: many requests, short trees, ragged contexts
        _attention("attn b64 n16 ctx3k", B=64, n=16, ctx=2900, hq=32, hkv=8, ragged=3),
        # single tokens (no drafts) of a big batch, seven query heads per KV head, fp16 cache
        _attention("attn b128 n1 ctx2k fp16", B=128, n=1, ctx=2047, hq=28, hkv=4, bs=32, dtype="fp16", ragged=4),
        # one very long context with a large tree: 512 query rows per KV head
        _attention("attn b1 n64 ctx128k", B=1, n=64, ctx=131000, hq=64, hkv=8, ragged=5),
        # one request, one row: the smallest call
        _logits("logits r1", B=1, n=1, V=128256, hist=1500, ragged=1),
        # verify rows of eight requests, every row under a grammar
        _logits("logits b8 n32 grammar", B=8, n=32, V=152064, hist=3000, grammar=1.0, bias=64, ragged=2),
        # a large fp32 batch with long histories, a few rows under a grammar
        _logits("logits b512 fp32", B=512, n=1, V=128256, hist=8000, grammar=0.1, bias=16, dtype="fp32", ragged=3),
        # plan of a small verify step
        _plan("plan b8 n16", B=8, n=16, ctx=3000, tree=True, ragged=1),
        # plan of a big mixed batch: chains of ragged length, some requests ended
        _plan("plan b2048 n40", B=2048, n=40, ctx=1500, tree=False, ragged=2),
        # commit of one request's tree, 32 layers
        _commit("commit b1 n8", B=1, n=8, layers=32, hkv=8, ragged=1),
        # commit of a full batch
        _commit("commit b128 n24", B=128, n=24, layers=28, hkv=4, ragged=2),
    ]


def _attention(name, B, n, ctx, hq, hkv, D=128, bs=16, dtype="bf16", ragged=0):
    return {"name": name, "op": "attention", "B": B, "n": n, "ctx": ctx, "hq": hq, "hkv": hkv, "D": D, "bs": bs,
            "dtype": dtype, "ragged": ragged}


def _logits(name, B, n, V, hist, grammar=0.0, bias=0, dtype="bf16", ragged=0):
    return {"name": name, "op": "logits", "B": B, "n": n, "V": V, "hist": hist, "grammar": grammar, "bias": bias,
            "dtype": dtype, "ragged": ragged}


def _plan(name, B, n, ctx, tree, bs=16, ragged=0):
    return {"name": name, "op": "plan", "B": B, "n": n, "ctx": ctx, "tree": tree, "bs": bs, "ragged": ragged}


def _commit(name, B, n, layers, hkv, D=128, bs=16, dtype="bf16", ragged=0):
    return {"name": name, "op": "commit", "B": B, "n": n, "layers": layers, "hkv": hkv, "D": D, "bs": bs,
            "dtype": dtype, "ragged": ragged}


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    ragged = 1000 + rng.randrange(1 << 20)
    op = rng.choice(["attention", "attention", "attention", "logits", "logits", "plan", "commit"])
    if op == "attention":
        hq, hkv = rng.choice([(32, 8), (28, 4), (64, 8), (40, 8), (8, 2), (16, 4)])
        D, n, B = rng.choice([64, 128, 128]), _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 128)
        # not more K/V than the longest listed context, scores of the plain form within a few GB
        most = min(131000, (1 << 27) // (B * hkv * D), (1 << 29) // (B * hq * n))
        c = _attention("", B, n, _log_uniform(rng, 1, max(1, most)), hq, hkv, D, rng.choice([8, 16, 32, 64, 128]),
                       rng.choice(["bf16", "bf16", "fp16"]), ragged)
    elif op == "logits":
        V = rng.choice([128256, 152064, 32000, 50257, _log_uniform(rng, 1000, 152064)])
        n, B = rng.choice([1, 1, _log_uniform(rng, 2, 64)]), _log_uniform(rng, 1, 400)
        n = max(1, min(n, 400 // B))
        c = _logits("", B, n, V, _log_uniform(rng, 1, 8000), rng.choice([0.0, 0.3, 1.0]), rng.choice([0, 1, 40, 300]),
                    rng.choice(["bf16", "fp16", "fp32"]), ragged)
    elif op == "plan":
        tree = rng.random() < 0.5
        B = _log_uniform(rng, 1, 512 if tree else 2048)
        c = _plan("", B, _log_uniform(rng, 1, 64 if tree else 40), _log_uniform(rng, 1, 1500), tree,
                  rng.choice([1, 8, 16, 32, 100]), ragged)
    else:
        hkv = rng.choice([2, 4, 8])
        layers = rng.choice([1, 4, 28, 32])
        c = _commit("", _log_uniform(rng, 1, 128), _log_uniform(rng, 1, 24), layers, hkv if layers < 28 else 4,
                    rng.choice([64, 128]), rng.choice([8, 16, 32]), rng.choice(["bf16", "fp16"]), ragged)
    del c["name"]
    return c


# ---------------------------------------------------- lengths and work of a case
def _lengths(case):
    """(new, ctx): drafted and committed tokens of every request.  One request
    has the case's own sizes; in a batch sizes spread over [1/2, 1] of them,
    one request in eight holds a short context."""
    r = random.Random(case["ragged"] * 1000003 + 17)
    B, n, ctx = case["B"], case["n"], case.get("ctx", 0)
    if B == 1:
        return [n], [ctx]
    new = [r.randint((n + 1) // 2, n) for _ in range(B)]
    ctxs = [r.randint(ctx // 8, ctx // 4) if r.randrange(8) == 0 else r.randint(ctx // 2, ctx) for _ in range(B)]
    new[0], ctxs[-1] = n, ctx
    if case["op"] == "plan":  # one request in sixteen ended, a few add nothing
        new = [(-1 if r.randrange(16) == 0 else v) if r.randrange(32) else 0 for v in new]
        new[0] = n
    return new, ctxs


def _blocks(case, tokens):
    return -(-tokens // case["bs"])


def work(case):
    new, ctx = _lengths(case)
    B, rows = case["B"], sum(max(v, 0) for v in new)
    if case["op"] == "attention":
        size = DTYPES[case["dtype"]].itemsize
        kv = 2 * case["hkv"] * case["D"] * size
        tables = 4 * sum(_blocks(case, c) for c in ctx)
        nbytes = kv * (sum(ctx) + rows) + 2 * rows * case["hq"] * case["D"] * size + tables + 8 * rows + 8 * B
        seen = sum(v * c for v, c in zip(new, ctx)) + 6 * rows
        return {"bytes": nbytes, "flops": 4 * case["D"] * case["hq"] * seen}
    if case["op"] == "logits":
        size = DTYPES[case["dtype"]].itemsize
        V = case["V"]
        nbytes = rows * (2 * V * size + 4) + int(rows * case["grammar"]) * (-(-V // BITS)) * 4
        nbytes += 4 * sum(_histories(case)) + 8 * B * case["bias"] + 24 * B + 16 * rows
        return {"bytes": nbytes, "flops": rows * V}
    if case["op"] == "plan":
        held = [_blocks(case, c) for c in ctx]
        got = sum(max(0, _blocks(case, c + max(v, 0)) - h) if v >= 0 else 2 * h for v, c, h in zip(new, ctx, held))
        per_row = 4 * (4 + (3 if case["tree"] else 0))
        return {"bytes": 20 * B + 8 * got + per_row * rows, "flops": rows}
    row = case["layers"] * 2 * case["hkv"] * case["D"] * DTYPES[case["dtype"]].itemsize
    kept = sum(len(_walk_on_host(case, b, v)) for b, v in enumerate(new))
    return {"bytes": 2 * kept * row + 20 * rows + 16 * B, "flops": rows}


def _histories(case):
    r = random.Random(case["ragged"] * 7919 + 3)
    h = case["hist"]
    return [h] + [r.randint(h // 4, h) for _ in range(case["B"] - 1)]


# ------------------------------------------------------------------ inputs
def _tree(case, b, n):
    """Parents and acceptance of a request's tree: node 0 is the certain root,
    later nodes hang off a recent earlier node; ``hit`` says that a node
    carries the token which the model will choose after its parent."""
    r = random.Random((case["ragged"] * 131071 + b) * 31 + n)
    parents = [-1] + [max(0, i - 1 - min(int(r.expovariate(0.5)), i - 1)) for i in range(1, n)]
    hit = [True] + [r.random() < 0.6 for _ in range(1, n)]
    return parents[:n], hit[:n]


def _walk_on_host(case, b, n):
    parents, hit = _tree(case, b, n)
    path = [0] if n else []
    for i in range(1, n):
        if hit[i] and parents[i] == path[-1]:
            path.append(i)
    return path


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _indptr(new):
    return _ints(np.concatenate([[0], np.cumsum([max(v, 0) for v in new])]).tolist())


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _mask_words(case, new):
    """Tree masks ``[R, W]`` (bit j of a row: tree token j is on its path) and
    depths, by walking each tree once on the host."""
    W = -(-max(max(new), 1) // BITS)
    words, depth = np.zeros((sum(new), W), np.uint32), np.zeros(sum(new), np.int32)
    at = 0
    for b, n in enumerate(new):
        for i, p in enumerate(_tree(case, b, n)[0]):
            if p >= 0:
                words[at + i] = words[at + p]
                depth[at + i] = depth[at + p] + 1
            words[at + i, i // BITS] |= np.uint32(1 << (i % BITS))
        at += n
    return torch.from_numpy(words.view(np.int32)).cuda(), torch.from_numpy(depth).cuda()


def _tables(case, ctx, width, pool, g):
    """Block tables over a shuffled pool, and the shuffled pool itself."""
    perm = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    held = [_blocks(case, c) for c in ctx]
    table = torch.zeros(case["B"], width, dtype=torch.int32, device="cuda")
    start = _ints(np.concatenate([[0], np.cumsum(held)[:-1]]).tolist())
    col = torch.arange(width, device="cuda")[None]
    inside = col < _ints(held)[:, None]
    table = torch.where(inside, perm[(start[:, None] + col).clamp(max=pool - 1).long()], table)
    return table, held, perm


def prepare(case, seed):
    g = _generator(seed)
    s = {"attention": _prepare_attention, "logits": _prepare_logits, "plan": _prepare_plan,
         "commit": _prepare_commit}[case["op"]](case, g)
    s["op"], s["case"] = case["op"], dict(case)
    return s


def _prepare_attention(case, g):
    new, ctx = _lengths(case)
    R, dt = sum(new), DTYPES[case["dtype"]]
    hq, hkv, D, bs = case["hq"], case["hkv"], case["D"], case["bs"]
    width = _blocks(case, max(ctx)) + 4
    pool = sum(_blocks(case, c) for c in ctx) + 8
    table, _, _ = _tables(case, ctx, width, pool, g)

    def normal(*shape):
        return torch.randn(shape, device="cuda", dtype=dt, generator=g)
    mask, _ = _mask_words(case, new)
    return {"q": normal(R, hq, D), "k_tree": normal(R, hkv, D), "v_tree": normal(R, hkv, D),
            "k_cache": normal(pool, bs, hkv, D), "v_cache": normal(pool, bs, hkv, D), "tables": table,
            "ctx": _ints(ctx), "indptr": _indptr(new), "mask": mask, "most_new": max(new), "most_ctx": max(ctx)}


def _prepare_logits(case, g):
    new, _ = _lengths(case)
    B, V, R, dt = case["B"], case["V"], sum(new), DTYPES[case["dtype"]]
    hist = _histories(case)
    prompt = [max(0, h - 1 - (h * 3) // 10) for h in hist]
    # frequent tokens repeat: squares of uniforms crowd the low ids
    u = torch.rand(B, max(hist), device="cuda", generator=g)
    tokens = (u * u * V).to(torch.int32).clamp(max=V - 1)
    drafts = (torch.rand(R, device="cuda", generator=g) ** 2 * V).to(torch.int32).clamp(max=V - 1)
    mask, depth = _mask_words(case, new)
    indptr = _indptr(new)
    request = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(new)).to(torch.int32)
    s = {"logits": (torch.randn(R, V, device="cuda", generator=g) * 3).to(dt), "request": request, "tokens": tokens,
         "lens": _ints(hist), "prompt": _ints(prompt), "drafts": drafts, "mask": mask, "indptr": indptr,
         "positions": _ints(hist)[request.long()] + depth, "most_new": max(new),
         "repetition": 1 + 0.3 * torch.rand(B, device="cuda", generator=g),
         "frequency": torch.rand(B, device="cuda", generator=g),
         "presence": torch.rand(B, device="cuda", generator=g) - 0.2,
         "bias_ids": None, "bias_values": None, "allowed": None, "allowed_index": None}
    if case["bias"]:
        # distinct ids: a random offset and an odd stride over the vocabulary
        first = torch.randint(0, V, (B, 1), device="cuda", generator=g)
        step = max(1, V // case["bias"] - 1)
        s["bias_ids"] = ((first + step * torch.arange(min(case["bias"], V), device="cuda")) % V).to(torch.int32)
        s["bias_values"] = torch.randn(s["bias_ids"].shape, device="cuda", generator=g) * 4
    if case["grammar"] > 0:
        index = torch.arange(R, device="cuda")
        index = torch.where(index % 100 < round(100 * case["grammar"]), index, -torch.ones_like(index))
        s["allowed_index"] = index.to(torch.int32)
        # half of the bits, in runs of words that are all set, all clear or mixed
        words = torch.randint(-2**31, 2**31, (R, -(-V // BITS)), device="cuda", generator=g)
        kind = torch.randint(0, 3, words.shape, device="cuda", generator=g)
        s["allowed"] = torch.where(kind == 0, words, torch.where(kind == 1, -torch.ones_like(words),
                                                                 torch.zeros_like(words))).to(torch.int32)
    return s


def _prepare_plan(case, g):
    new, ctx = _lengths(case)
    width = _blocks(case, max(ctx) + case["n"]) + 1
    held = [_blocks(case, c) for c in ctx]
    pool = sum(held) + sum(_blocks(case, max(v, 0)) + 1 for v in new) + 16
    table, held, perm = _tables(case, ctx, width, pool, g)
    used = sum(held)
    queue = torch.zeros(pool, dtype=torch.int32, device="cuda")
    head = pool - 5  # the ring wraps
    queue[(head + torch.arange(pool - used, device="cuda")) % pool] = perm[used:]
    parents = None
    if case["tree"]:
        parents = _ints([p for b, v in enumerate(new) for p in _tree(case, b, max(v, 0))[0]])
    return {"ctx": _ints(ctx), "new": _ints(new), "table": table, "held": _ints(held), "queue": queue,
            "cursor": _ints([head, head + pool - used], torch.int64), "rows": sum(max(v, 0) for v in new),
            "parents": parents, "most_new": case["n"]}


def _prepare_commit(case, g):
    new, ctx = _lengths(dict(case, ctx=40))
    R, B, dt = sum(new), case["B"], DTYPES[case["dtype"]]
    L, hkv, D, bs = case["layers"], case["hkv"], case["D"], case["bs"]
    whole = [c + n for c, n in zip(ctx, new)]
    pool = sum(_blocks(case, t) for t in whole) + 4
    table, _, _ = _tables(case, whole, _blocks(case, max(whole)), pool, g)
    indptr = _indptr(new)
    request = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(new))
    at = torch.arange(R, device="cuda") - indptr[request] + _ints(ctx)[request]
    slots = table[request, at // bs] * bs + (at % bs).to(torch.int32)
    trees = [_tree(case, b, n) for b, n in enumerate(new)]
    parents = _ints([p for t in trees for p in t[0]])
    hit = torch.tensor([h for t in trees for h in t[1]]).cuda()
    target = torch.randint(0, 100000, (R,), device="cuda", generator=g).to(torch.int32)
    other = torch.randint(100000, 128000, (R,), device="cuda", generator=g).to(torch.int32)
    above = (indptr[request] + parents.clamp(min=0)).long()
    drafts = torch.where(hit, target[above], other)
    return {"drafts": drafts, "targets": target, "parents": parents, "indptr": indptr, "ctx": _ints(ctx),
            "slots": slots.to(torch.int32), "request": request, "most_new": max(new),
            "tokens": torch.randint(0, 128000, (B, max(whole) + 3), device="cuda", generator=g).to(torch.int32),
            "tree_kv": torch.randn((L, 2, R, hkv, D), device="cuda", dtype=dt, generator=g),
            "cache": torch.randn((L, 2, pool, bs, hkv, D), device="cuda", dtype=dt, generator=g)}


# -------------------------------------------------------------------- runs
def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _pad_rows(indptr, most):
    """Index of row i of each request ``[B, most]`` and which of them exist."""
    i = torch.arange(most, device=indptr.device)[None]
    there = i < (indptr[1:] - indptr[:-1])[:, None]
    return torch.where(there, indptr[:-1, None] + i, torch.zeros_like(i)).long(), there


def _ancestors(parents, indptr, most):
    """``[B, n, n]``: entry (i, j) says that node j is i or one of its ancestors."""
    rows, there = _pad_rows(indptr, most)
    up = torch.where(there, parents[rows], torch.full_like(rows, -1).to(parents.dtype))
    step = (up[:, :, None] == torch.arange(most, device=up.device)) & there[:, :, None]
    step = step.float() + torch.eye(most, device=up.device)
    return (torch.matrix_power(step, 1 << (most - 1).bit_length()) > 0) & there[:, :, None]


def _unpack(words, count):
    """Bits ``[..., count]`` of int32 words ``[..., W]``."""
    at = torch.arange(count, device=words.device)
    return ((words[..., at // BITS] >> (at % BITS)) & 1).bool()


def _plain_attention(s):
    q, kc, vc, table = s["q"], s["k_cache"], s["v_cache"], s["tables"]
    bs, hkv = kc.shape[1], kc.shape[2]
    group = q.shape[1] // hkv
    rows, there = _pad_rows(s["indptr"], s["most_new"])
    B, N = rows.shape
    at = torch.arange(s["most_ctx"], device=q.device)
    where = (table[:, at // bs] * bs + (at % bs).to(torch.int32)).long()

    def keys(cache, tree):  # [B, Hkv, L + N, D]
        old = cache.reshape(-1, hkv, cache.shape[-1])[where]
        return torch.cat([old, tree[rows]], 1).float().transpose(1, 2)
    seen = torch.cat([(at[None, None] < s["ctx"][:, None, None]).expand(B, N, -1), _unpack(s["mask"], N)[rows]], -1)
    seen = (seen & there[:, :, None])[:, None]
    qf = q[rows].float().view(B, N, hkv, group, -1).permute(0, 2, 3, 1, 4).reshape(B, hkv, group * N, -1)
    x = qf @ keys(kc, s["k_tree"]).transpose(2, 3) / math.sqrt(q.shape[-1])
    x = x.view(B, hkv * group, N, -1).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = x.view(B, hkv, group * N, -1) @ keys(vc, s["v_tree"])
    o = o.view(B, hkv * group, N, -1) / torch.where(total > 0, total, torch.ones_like(total))
    row = torch.arange(q.shape[0], device=q.device, dtype=torch.int32)
    request = torch.searchsorted(s["indptr"][1:].contiguous(), row, right=True)
    return {"out": o[request, :, (row - s["indptr"][request]).long()].to(q.dtype)}


def _plain_logits(s):
    x = s["logits"].float()
    R, V = x.shape
    request = s["request"].long()
    B, H = s["tokens"].shape
    at = torch.arange(H, device=x.device)[None]
    ids = s["tokens"].long()
    known = (at < s["lens"][:, None])
    output = known & (at >= s["prompt"][:, None])
    zeros = torch.zeros(B, V, device=x.device, dtype=torch.int32)
    seen = zeros.scatter_add(1, ids, known.int())[request]
    count = zeros.scatter_add(1, ids, output.int())[request]
    rows, there = _pad_rows(s["indptr"], s["most_new"])
    path = _unpack(s["mask"], s["most_new"]) & there[request]
    drafts = s["drafts"].long()[rows][request]
    generated = path & (s["positions"][rows] >= s["prompt"][:, None])[request]
    seen.scatter_add_(1, drafts, path.int())
    count.scatter_add_(1, drafts, generated.int())
    rep = s["repetition"][request, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][request, None] * count
    x = torch.where(count > 0, x - s["presence"][request, None], x)
    if s["bias_ids"] is not None:
        x = x + torch.zeros(B, V, device=x.device).scatter_add(1, s["bias_ids"].long(), s["bias_values"])[request]
    if s["allowed"] is not None:
        index = s["allowed_index"].long()
        free = _unpack(s["allowed"][index.clamp(min=0)], V) | (index < 0)[:, None]
        x = torch.where(free, x, torch.full_like(x, -math.inf))
    out = x.to(s["logits"].dtype)
    best = torch.where(out == out.amax(1, keepdim=True), torch.arange(V, device=x.device), V).amin(1)
    return {"logits": out, "greedy": best.to(torch.int32)}


def _plain_plan(s):
    ctx, new, held, table, queue, bs = s["ctx"], s["new"], s["held"], s["table"], s["queue"], s["case"]["bs"]
    B, W = table.shape
    n, ended = new.clamp(min=0), new < 0
    zero = torch.zeros_like(held)
    need = torch.where(ended, zero, ((ctx + n + bs - 1) // bs - held).clamp(min=0))
    freed = torch.where(ended, held, zero)
    first = torch.cumsum(need, 0) - need
    back = torch.cumsum(freed, 0) - freed
    col = torch.arange(W, device=ctx.device)[None]
    head, tail = s["cursor"][0], s["cursor"][1]
    cap = queue.numel()
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    taken = queue[((head + first[:, None] + col - held[:, None]) % cap)]
    gone = col < freed[:, None]
    spot = torch.where(gone, (tail + back[:, None] + col) % cap, torch.full_like(col, cap))
    longer = torch.cat([queue, queue[:1]])
    longer[spot.reshape(-1)] = table.reshape(-1)
    table = torch.where(fresh, taken, table)
    queue.copy_(longer[:cap])
    s["table"].copy_(table)
    indptr = torch.nn.functional.pad(torch.cumsum(n, 0), (1, 0)).to(torch.int32)
    row = torch.arange(s["rows"], device=ctx.device, dtype=torch.int32)
    request = torch.searchsorted(indptr[1:].contiguous(), row, right=True)
    at = ctx[request] + row - indptr[request]
    slots = table[request, (at // bs).long()] * bs + at % bs
    out = {"indptr": indptr, "request": request.to(torch.int32), "slots": slots, "positions": at, "tables": table,
           "held": torch.where(ended, zero, held + need), "queue": queue,
           "cursor": torch.stack([head + need.sum(), tail + freed.sum()])}
    if s["parents"] is not None:
        most = s["most_new"]
        up = _ancestors(s["parents"], indptr, most)
        words = -(-most // BITS)
        padded = torch.nn.functional.pad(up, (0, words * BITS - most)).view(B, most, words, BITS).long()
        packed = (padded << torch.arange(BITS, device=ctx.device)).sum(-1)
        inside = (row - indptr[request]).long()
        out["mask"] = packed[request, inside].to(torch.int32)
        out["positions"] = ctx[request] + up.sum(-1)[request, inside].to(torch.int32) - 1
    return out


def _plain_commit(s):
    indptr, most, ctx = s["indptr"], s["most_new"], s["ctx"]
    rows, there = _pad_rows(indptr, most)
    up = _ancestors(s["parents"], indptr, most)
    parents = torch.where(there, s["parents"][rows], torch.full_like(s["parents"][rows], -2))
    drafts, targets = s["drafts"][rows], s["targets"][rows]
    i = torch.arange(most, device=ctx.device)
    # a node is good if it carries its parent's target and no earlier sibling carries the same token
    twin = (parents[:, :, None] == parents[:, None]) & (drafts[:, :, None] == drafts[:, None])
    first = ~(twin & (i[None, :] < i[:, None])).any(-1)
    good = (drafts == targets.gather(1, parents.clamp(min=0).long())) & first & (parents >= 0)
    good[:, 0] = there[:, 0]
    kept = there & ((up & ~good[:, None]).sum(-1) == 0)
    depth = up.sum(-1) - 1
    accepted = kept.sum(1)
    path = torch.full((rows.shape[0], most + 1), -1, dtype=torch.long, device=ctx.device)
    path.scatter_(1, torch.where(kept, depth, torch.full_like(depth, most)), i.expand_as(depth).contiguous())
    path = torch.where(i < accepted[:, None], path[:, :most], torch.full_like(path[:, :most], -1))
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    request, inside = s["request"], torch.arange(s["drafts"].numel(), device=ctx.device) - indptr[s["request"]]
    kept_row = path[request, inside]
    source = (indptr[request] + kept_row.clamp(min=0)).long()
    flat = s["cache"].view(*s["cache"].shape[:2], -1, *s["cache"].shape[4:])
    slots = s["slots"].long()
    flat[:, :, slots] = torch.where((kept_row >= 0)[:, None, None], s["tree_kv"][:, :, source], flat[:, :, slots])
    at = (ctx[request] + inside).long()
    s["tokens"][request, at] = torch.where(kept_row >= 0, s["drafts"][source], s["tokens"][request, at])
    return {"accepted": accepted.to(torch.int32), "path": kept_row.to(torch.int32),
            "next": targets.gather(1, last[:, None])[:, 0], "ctx": ctx + accepted.to(torch.int32),
            "tokens": s["tokens"], "cache": s["cache"]}


_plain = {"attention": _plain_attention, "logits": _plain_logits, "plan": _plain_plan, "commit": _plain_commit}


def _own_attention(s):
    from kvserve_b200 import ops
    return {"out": ops.paged_tree_attention(s["q"], s["k_tree"], s["v_tree"], s["k_cache"], s["v_cache"], s["tables"],
                                            s["ctx"], s["indptr"], tree_mask=s["mask"])}


def _own_logits(s):
    from kvserve_b200 import ops
    greedy = torch.empty(s["logits"].shape[0], dtype=torch.int32, device=s["logits"].device)
    out = ops.process_logits(s["logits"], row_request=s["request"], tokens=s["tokens"], token_lens=s["lens"],
                             prompt_lens=s["prompt"], repetition=s["repetition"], frequency=s["frequency"],
                             presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                             allowed=s["allowed"], allowed_index=s["allowed_index"], draft_ids=s["drafts"],
                             indptr=s["indptr"], tree_mask=s["mask"], positions=s["positions"], greedy=greedy)
    return {"logits": out, "greedy": greedy}


def _own_plan(s):
    from kvserve_b200 import ops
    p = ops.plan_step(s["ctx"], s["new"], s["table"], s["held"], s["queue"], s["cursor"], s["case"]["bs"], s["rows"],
                      parents=s["parents"], max_tree=s["most_new"])
    out = {"indptr": p.indptr, "request": p.row_request, "slots": p.slot_mapping, "positions": p.positions,
           "tables": s["table"], "held": p.held, "queue": s["queue"], "cursor": p.cursor}
    if s["parents"] is not None:
        out["mask"] = p.tree_mask
    return out


def _own_commit(s):
    from kvserve_b200 import ops
    c = ops.commit_tree(s["drafts"], s["targets"], s["parents"], s["indptr"], s["ctx"], s["slots"],
                        tree_kv=s["tree_kv"], kv_cache=s["cache"], tokens=s["tokens"])
    return {"accepted": c.accepted, "path": c.path, "next": c.next_ids, "ctx": c.ctx_lens, "tokens": s["tokens"],
            "cache": s["cache"]}


_own = {"attention": _own_attention, "logits": _own_logits, "plan": _own_plan, "commit": _own_commit}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return {"out": _exact_attention(s)}
    if case["op"] == "logits":
        return {"logits": _exact_logits(s), "greedy": None}
    return None  # indices and copied rows: nothing is computed


def _exact_attention(s):
    """Request by request and KV head by KV head from softmax(q k / sqrt(D)) v."""
    q = s["q"].double()
    out = torch.zeros_like(q)
    bounds, ctx = s["indptr"].tolist(), s["ctx"].tolist()
    bs, hkv = s["k_cache"].shape[1:3]
    group = q.shape[1] // hkv
    for b, c in enumerate(ctx):
        lo, hi = bounds[b], bounds[b + 1]
        if hi == lo:
            continue
        blocks = s["tables"][b, : -(-c // bs)].long()
        words = s["mask"][lo:hi].tolist()
        on_path = torch.tensor([[(w[j // BITS] >> (j % BITS)) & 1 for j in range(hi - lo)] for w in words],
                               dtype=torch.bool, device=q.device)
        for h in range(hkv):
            k = torch.cat([s["k_cache"][blocks, :, h].reshape(-1, q.shape[2])[:c], s["k_tree"][lo:hi, h]]).double()
            v = torch.cat([s["v_cache"][blocks, :, h].reshape(-1, q.shape[2])[:c], s["v_tree"][lo:hi, h]]).double()
            for g in range(group):
                score = torch.mm(q[lo:hi, h * group + g], k.T) * q.shape[2] ** -0.5
                score[:, c:][~on_path] = -math.inf
                out[lo:hi, h * group + g] = torch.mm(torch.softmax(score, -1), v)
    return out


def _exact_logits(s):
    """Row by row: histogram of the row's tokens, then the rules in order."""
    R, V = s["logits"].shape
    out = torch.empty(R, V, dtype=torch.float64, device="cuda")
    request, bounds = s["request"].tolist(), s["indptr"].tolist()
    lens, prompt, positions = s["lens"].tolist(), s["prompt"].tolist(), s["positions"].tolist()
    words = s["mask"].tolist()
    index = s["allowed_index"].tolist() if s["allowed"] is not None else [-1] * R
    for r in range(R):
        b = request[r]
        path = [bounds[b] + j for j in range(bounds[b + 1] - bounds[b]) if (words[r][j // BITS] >> (j % BITS)) & 1]
        made = [j for j in path if positions[j] >= prompt[b]]
        old = s["tokens"][b, :lens[b]]
        counted = torch.bincount(torch.cat([old[prompt[b]:], s["drafts"][made]]).long(), minlength=V).double()
        there = torch.bincount(torch.cat([old, s["drafts"][path]]).long(), minlength=V) > 0
        x = s["logits"][r].double()
        rep = s["repetition"][b].double()
        x = torch.where(there & (x > 0), x / rep, torch.where(there, x * rep, x))
        x -= s["frequency"][b].double() * counted + s["presence"][b].double() * (counted > 0)
        if s["bias_ids"] is not None:
            x[s["bias_ids"][b].long()] += s["bias_values"][b].double()
        if index[r] >= 0:
            row = s["allowed"][index[r]]
            bit = (row[:, None] >> torch.arange(BITS, device="cuda", dtype=torch.int32)) & 1
            x[bit.reshape(-1)[:V] == 0] = -math.inf
        out[r] = x
    return out
