"""Greedy decoding with drafted token trees on one GPU.

Every step verifies a small tree of drafted tokens per request in one pass of
the model: :func:`kvserve_b200.ops.plan_step` lays the rows out and hands out
KV blocks on the GPU, :meth:`LlamaShard.verify_step` runs the model with
:func:`~kvserve_b200.ops.paged_tree_attention`,
:func:`~kvserve_b200.ops.process_logits` applies penalties and biases and picks
the model's choice after every node, and
:func:`~kvserve_b200.ops.commit_tree` accepts a path and moves its K/V rows
into the paged cache.  A step yields one to ``max_tree`` tokens a request; the
result is that of one-token greedy decoding under the same rules (up to the
rounding of differently shaped products).  Steps are launched kernel by kernel,
not from a CUDA graph.  Grammar masks belong to rows, not to requests: whoever
needs them calls the operators one by one.

    dec = TreeDecoder(model, num_blocks=4096, max_len=4096)
    out = dec.generate(prompts, 128, rules={"repetition": torch.full((B,), 1.1, device="cuda")})

``propose(history, max_nodes) -> (tokens, parents)`` drafts for one request;
the default looks the last tokens up earlier in the request's own text.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Optional, Sequence

import torch

from .. import ops
from ..models.llama import LlamaShard
from .kv_cache import PagedKVCache

Drafts = tuple  # (tokens after the root, parents inside the tree; the root is node 0)


def lookup_drafts(history: Sequence[int], max_nodes: int, match: int = 2, width: int = 2) -> Drafts:
    """Continuations of the latest ``width`` earlier places where the last
    ``match`` tokens occur, as chains under the root (equal beginnings share
    their nodes)."""
    tokens: list = []
    parents: list = []
    children: dict = {}
    tail = list(history[-match:])
    found = 0
    for at in range(len(history) - match - 1, -1, -1):
        if found == width or len(history) < match + 1:
            break
        if list(history[at:at + match]) != tail:
            continue
        found += 1
        node = 0
        for tok in history[at + match:at + match + max_nodes]:
            key = (node, tok)
            if key not in children:
                if len(tokens) + 1 >= max_nodes:
                    break
                tokens.append(tok)
                parents.append(node)
                children[key] = len(tokens)
            node = children[key]
    return tokens, parents


@dataclass
class TreeResult:
    tokens: list          # generated token ids of the request
    steps: int            # verify steps that the request took part in


@dataclass
class _Requests:
    ctx: torch.Tensor     # int32 [B] committed tokens
    held: torch.Tensor    # int32 [B] blocks held
    tables: torch.Tensor  # int32 [B, W]


class TreeDecoder:
    def __init__(self, model: LlamaShard, num_blocks: int, max_len: int, block_size: int = 16, max_tree: int = 16,
                 propose: Callable[[Sequence[int], int], Drafts] = lookup_drafts):
        if model.tp_size != 1:
            raise ValueError("tree decoding runs on one GPU (TP size 1)")
        if not 1 <= max_tree <= 64:
            raise ValueError("max_tree must be 1 to 64")
        if max_len > model.cos_sin.shape[0]:
            raise ValueError(f"max_len {max_len} exceeds the model's rotary table "
                             f"(max_position {model.cos_sin.shape[0]})")
        self.model, self.max_len, self.max_tree, self.propose = model, max_len, max_tree, propose
        cfg, dev = model.cfg, model.device
        self.block_size = block_size
        self.kv = PagedKVCache(cfg.num_layers, num_blocks, block_size, model.hkv, model.D, dev).cache
        self.free_queue = torch.arange(num_blocks, dtype=torch.int32, device=dev)
        self.cursor = torch.tensor([0, num_blocks], dtype=torch.int64, device=dev)

    def _ints(self, values) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32).to(self.model.device, non_blocking=True)

    def free_blocks(self) -> int:
        head, tail = self.cursor.tolist()
        return tail - head

    def generate(self, prompts: Sequence[torch.Tensor], max_new_tokens: int, rules: Optional[dict] = None,
                 stop: Optional[int] = None) -> list:
        """Tokens of every prompt (int32 vectors); ``rules`` are keyword
        arguments of :func:`kvserve_b200.ops.process_logits` that belong to
        requests (``repetition``, ``frequency``, ``presence``, ``bias_ids``,
        ``bias_values``).  ``stop`` ends a request after that token."""
        m, dev = self.model, self.model.device
        B, bs = len(prompts), self.block_size
        history = [[int(t) for t in p.tolist()] for p in prompts]
        lens = [len(h) for h in history]
        if B == 0:
            return []
        if min(lens) < 1 or max(lens) + max_new_tokens > self.max_len:
            raise ValueError("prompt is empty, or prompt and new tokens exceed max_len")
        if max_new_tokens < 0:
            raise ValueError("max_new_tokens is negative")
        results = [TreeResult([], 0) for _ in range(B)]
        if max_new_tokens == 0:
            return results
        tables = torch.zeros(B, -(-self.max_len // bs), dtype=torch.int32, device=dev)
        tokens = torch.zeros(B, self.max_len, dtype=torch.int32, device=dev)
        for b, h in enumerate(history):
            tokens[b, :lens[b]] = self._ints(h)
        none = torch.zeros(B, dtype=torch.int32, device=dev)
        req = _Requests(none, none, tables)
        # the prompt without its last token, which is the root of the first tree
        new = self._ints(n - 1 for n in lens)
        try:
            plan = self._plan(req, new, sum(lens) - B)
            self._prefill(history, plan)
            req.ctx = new
            prompt_lens = self._ints(lens)
            live = list(range(B))
            while live:
                self._step(history, results, live, req, tokens, prompt_lens, rules or {}, max_new_tokens, stop)
                live = [b for b in live if len(results[b].tokens) < max_new_tokens
                        and not (results[b].tokens and results[b].tokens[-1] == stop)]
            ops.check_device_status(dev)  # the last step's; the others' were read after the next plan
            return results
        finally:  # all blocks go back
            self.cursor = ops.plan_step(req.ctx, torch.full_like(none, -1), tables, req.held, self.free_queue,
                                        self.cursor, bs, 0).cursor

    def _plan(self, req: _Requests, new: torch.Tensor, rows: int, parents=None) -> "ops.StepPlan":
        """Plan of a step.  The held blocks and the ring's cursor advance with
        it at once, so that whatever fails afterwards, what the plan took is
        known and goes back."""
        plan = ops.plan_step(req.ctx, new, req.tables, req.held, self.free_queue, self.cursor, self.block_size, rows,
                             parents=parents, max_tree=self.max_tree)
        req.held, self.cursor = plan.held, plan.cursor
        ops.check_device_status(self.model.device)  # blocks ran out, or a broken tree
        return plan

    def _prefill(self, history: list, plan: "ops.StepPlan") -> None:
        m, at = self.model, 0
        L, _, nb, bs, hkv, D = self.kv.shape
        for h in history:
            n = len(h) - 1
            if n == 0:
                continue
            k = torch.empty(L, n, hkv, D, dtype=self.kv.dtype, device=self.kv.device)
            v = torch.empty_like(k)
            m.prefill(self._ints(h[:n]), plan.positions[at:at + n], k, v)
            slots = plan.slot_mapping[at:at + n].long()
            self.kv[:, 0].view(L, nb * bs, hkv, D)[:, slots] = k
            self.kv[:, 1].view(L, nb * bs, hkv, D)[:, slots] = v
            at += n

    def _step(self, history, results, live, req: _Requests, tokens, prompt_lens, rules, max_new, stop):
        m = self.model
        B = len(history)
        new, drafts, parents = [0] * B, [], []
        for b in live:
            room = min(self.max_tree, max_new - len(results[b].tokens))
            toks, par = self.propose(history[b], room) if room > 1 else ([], [])
            toks, par = list(toks)[:room - 1], list(par)[:room - 1]
            new[b] = 1 + len(toks)
            drafts += [history[b][-1]] + toks
            parents += [-1] + par
        ids = self._ints(drafts)
        par = self._ints(parents)
        R = len(drafts)
        plan = self._plan(req, self._ints(new), R, parents=par)
        L, _, _, _, hkv, D = self.kv.shape
        tree_kv = torch.empty(L, 2, R, hkv, D, dtype=self.kv.dtype, device=self.kv.device)
        logits = m.verify_step(ids, plan, tree_kv, self.kv, req.tables, req.ctx)
        chosen = torch.empty(R, dtype=torch.int32, device=m.device)
        ops.process_logits(logits, row_request=plan.row_request, tokens=tokens, token_lens=req.ctx,
                           prompt_lens=prompt_lens, draft_ids=ids, indptr=plan.indptr, tree_mask=plan.tree_mask,
                           positions=plan.positions, out=logits, greedy=chosen, **rules)
        done = ops.commit_tree(ids, chosen, par, plan.indptr, req.ctx, plan.slot_mapping, tree_kv=tree_kv,
                               kv_cache=self.kv, tokens=tokens)
        req.ctx = done.ctx_lens
        # the drafts of the next step come from the host: one read back a step
        path, accepted, chosen = done.path.tolist(), done.accepted.tolist(), chosen.tolist()
        row = 0
        for b in live:
            got = [chosen[row + node] for node in path[row:row + accepted[b]]]
            if stop is not None and stop in got:
                got = got[:got.index(stop) + 1]
            history[b] += got
            results[b].tokens += got
            results[b].steps += 1
            row += new[b]
