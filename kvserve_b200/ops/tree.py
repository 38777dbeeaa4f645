"""Operators of one step of tree-drafted decoding.

A step verifies several drafted tokens of every request at once.  Its rows are
packed: request ``b`` owns rows ``indptr[b] .. indptr[b + 1]`` and row
``indptr[b] + i`` is node ``i`` of its tree.  Node 0 is the last chosen token
(certain, not yet in the cache); a node's parent has a lower index.

    plan = plan_step(ctx_lens, new_lens, ...)        # blocks, slots, masks
    paged_tree_attention(q, k_tree, v_tree, ...)     # every layer
    process_logits(logits, ..., greedy=targets)      # rules and model's choice
    commit_tree(drafts, targets, ...)                # accepted path -> cache

The K/V rows of drafted tokens stay in the step's own staging tensors until
:func:`commit_tree` moves the accepted ones into the paged cache, so the cache
never holds a rejected token.  Every call runs on the current stream, does
not synchronise, and can be captured in a CUDA graph; what only the device can
see (an exhausted free list, a broken tree) is reported through
:func:`kvserve_b200.ops.check_device_status`.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import count_launches, device_status
from ._ext import ext


class StepPlan(NamedTuple):
    """Row layout of a step.  Rows past ``indptr[B]`` are padding: request -1,
    slot -1, position 0, empty mask."""
    indptr: torch.Tensor                # int32 [B + 1]
    row_request: torch.Tensor           # int32 [R]
    positions: torch.Tensor             # int32 [R] ctx + depth in the tree (a chain: ctx + i)
    slot_mapping: torch.Tensor          # int32 [R] cache slot of position ctx + i
    tree_mask: Optional[torch.Tensor]   # int32 [R, W] bit j: node j is on the row's path (None: chains)
    held: torch.Tensor                  # int32 [B] blocks held after the plan
    cursor: torch.Tensor                # int64 [2] head and tail of the free ring after the plan


class TreeCommit(NamedTuple):
    accepted: torch.Tensor   # int32 [B] length of the accepted path (its root included)
    path: torch.Tensor       # int32 [R] node of the k-th accepted token at row indptr[b] + k, then -1
    next_ids: torch.Tensor   # int32 [B] the model's choice after the path (-1: no rows)
    ctx_lens: torch.Tensor   # int32 [B] committed tokens after the step


def plan_step(ctx_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, held: torch.Tensor,
              free_queue: torch.Tensor, cursor: torch.Tensor, block_size: int, num_rows: int,
              parents: Optional[torch.Tensor] = None, max_tree: int = 64,
              out: Optional[StepPlan] = None) -> StepPlan:
    """Row layout, KV blocks and tree masks of a step, from request lengths on
    the GPU.

    ``ctx_lens`` / ``new_lens`` int32 [B]: committed tokens and rows of the
    step (0: sits out; negative: ended, its blocks are returned).
    ``free_queue`` int32 [N] is a ring of free block ids between ``cursor`` =
    (head, tail), monotonic int64 counters.  Requests take the blocks they
    miss from its head in request order and ``block_tables`` [B, W] is
    extended in place; returned blocks join its tail.  If the ring holds too
    few blocks nobody gets one, rows without a block have slot -1, and the
    device status says so.  ``parents`` int32 [num_rows] (-1 for the root,
    index inside the tree otherwise) gives tree masks of ``max_tree`` bits and
    depths; without it the rows are chains.  At most 16384 requests.  ``held``
    and ``cursor`` may also be ``out.held`` and ``out.cursor`` (state updated
    in place).  Steps of more than 1024 rows or requests take 16 bytes of
    scratch memory.
    """
    # more than 1024 rows or requests: a second launch updates the state
    count_launches(1 if max(num_rows, ctx_lens.numel()) <= 1024 else 2)
    given = [] if out is None else [x for x in out if x is not None]
    got = ext().plan_step(ctx_lens, new_lens, block_tables, held, free_queue, cursor, block_size, num_rows, parents,
                          max_tree, given, device_status(ctx_lens.device))
    if out is not None:
        return out
    return StepPlan(*got) if parents is not None else StepPlan(*got[:4], None, *got[4:])


def paged_tree_attention(q: torch.Tensor, k_tree: torch.Tensor, v_tree: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                         indptr: torch.Tensor, tree_mask: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GQA attention of drafted tokens: row ``r`` of request ``b`` sees the
    ``ctx_lens[b]`` tokens of the paged cache (``[num_blocks, block_size, Hkv,
    D]``, any strides with contiguous head rows) and the tree rows of its
    request whose bit is set in ``tree_mask[r]`` (without a mask: the rows up
    to itself).  A row that sees nothing, and padding rows, give zeros.
    bf16 or fp16, head_dim 64 or 128, up to 128 query heads per KV head, a
    positive ``scale``; head rows start at 16-byte boundaries.  Block sizes
    that are no multiple of 8 tokens work, but many times slower.  ``k_tree`` /
    ``v_tree`` ``[R, Hkv, D]`` hold the step's own K and V.  Contexts end with
    the block table at the latest; block ids outside the cache read as zeros.
    Each call takes scratch memory from torch's allocator for the records of
    shared items: 4 x SMs x min(128, R x Hq / Hkv) x (4 D + 8) bytes, 39 MB at
    most on 148 SMs.  Probabilities are
    rounded to the K/V type before the product with V (fp16: with all bits
    down to 2^-21 of the row's largest one, none below 2^-32); sums are fp32."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    count_launches(2)
    ext().paged_tree_attention(q, k_tree, v_tree, k_cache, v_cache, block_tables, ctx_lens, indptr, tree_mask,
                               float(scale), out, device_status(q.device))
    return out


def process_logits(logits: torch.Tensor, *, row_request: Optional[torch.Tensor] = None,
                   tokens: Optional[torch.Tensor] = None, token_lens: Optional[torch.Tensor] = None,
                   prompt_lens: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                   bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
                   allowed: Optional[torch.Tensor] = None, allowed_index: Optional[torch.Tensor] = None,
                   draft_ids: Optional[torch.Tensor] = None, indptr: Optional[torch.Tensor] = None,
                   tree_mask: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                   vocab_begin: int = 0, out: Optional[torch.Tensor] = None, greedy: Optional[torch.Tensor] = None,
                   greedy_val: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties, biases and grammar masks on ``logits`` ``[R, V]`` (bf16, fp16
    or fp32; ``out`` may be ``logits``), and the greedy token of each result.

    In this order, in fp32, rounded once: a token that occurs in the row's
    text has its logit divided (positive) or multiplied (negative) by
    ``repetition``; then ``frequency`` times its count among generated tokens
    and, if that is not zero, ``presence`` are subtracted; then its bias is
    added; then a clear bit of the row's grammar mask gives ``-inf``, whatever
    was there.  All of these are fp32 ``[B]`` and optional.

    The text of row ``r`` is the committed tokens of its request
    (``tokens[b, :token_lens[b]]``, int32 [B, M]; those from ``prompt_lens[b]``
    on are generated) and the drafted tokens on its own tree path
    (``draft_ids`` [R] with ``indptr``, ``tree_mask`` and ``positions`` of the
    step plan; without ``tree_mask`` the rows up to itself), generated where
    their position is at least ``prompt_lens[b]``.  ``row_request`` [R] maps
    rows to requests (-1: no rules but the grammar; None: row r is request r).
    ``bias_ids`` / ``bias_values`` [B, K]: ids below 0 are padding, an id
    listed twice gets the sum; at most 2047 a request.  ``tokens`` may be up to
    2^19 wide (less the number of rows); at most 65535 rows.  ``allowed`` int32 [A, ceil(V / 32)] holds bit
    masks over the columns, ``allowed_index`` [R] names each row's mask (-1:
    none).  With ``vocab_begin`` the columns are a shard of the vocabulary;
    ids outside it are ignored.  ``greedy`` int32 [R] receives the index of
    the largest value of ``out`` (lowest index of equal ones, the first NaN if
    there is one) and ``greedy_val`` fp32 [R] the value; it takes 8 bytes of
    scratch memory for each row and slice (1024 to 16384 entries) of it."""
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    count_launches(1 if greedy is None else 2)
    ext().process_logits(logits, out, row_request, tokens, token_lens, prompt_lens, repetition, frequency, presence,
                         bias_ids, bias_values, allowed, allowed_index, draft_ids, indptr, tree_mask, positions,
                         int(vocab_begin), greedy, greedy_val)
    return out


def commit_tree(draft_ids: torch.Tensor, target_ids: torch.Tensor, parents: Optional[torch.Tensor],
                indptr: torch.Tensor, ctx_lens: torch.Tensor, slot_mapping: torch.Tensor,
                tree_kv: Optional[torch.Tensor] = None, kv_cache: Optional[torch.Tensor] = None,
                tokens: Optional[torch.Tensor] = None, out: Optional[TreeCommit] = None) -> TreeCommit:
    """Greedy verification and commit: from the root on, a child (the lowest
    one) is accepted if it carries the token in ``target_ids`` of its parent,
    the model's choice after it.  ``parents`` None: chains.  The accepted
    rows of ``tree_kv`` ``[L, 2, R, Hkv, D]`` are copied into ``kv_cache``
    ``[L, 2, blocks, block_size, Hkv, D]`` at ``slot_mapping[indptr[b] + k]``
    and their tokens written to ``tokens[b, ctx + k]`` (int32 [B, M]).  At
    most 1024 nodes a tree.  ``out.ctx_lens`` may be ``ctx_lens``."""
    count_launches(1)
    got = ext().commit_tree(draft_ids, target_ids, parents, indptr, ctx_lens, slot_mapping, tree_kv, kv_cache, tokens,
                            [] if out is None else list(out), device_status(draft_ids.device))
    return out if out is not None else TreeCommit(*got)
