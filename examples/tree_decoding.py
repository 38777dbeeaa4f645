"""Greedy decoding with drafted token trees: one request batch on one GPU.

    python examples/tree_decoding.py [--model tiny-gqa] [--new-tokens 64]

Random-init weights; the prompts repeat themselves, so that the default
drafter (looking the last tokens up earlier in the text) finds continuations.
Prints the tokens per verify step with and without drafts.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))  # run in a source tree

from kvserve_b200.engine.tree_decode import TreeDecoder  # noqa: E402
from kvserve_b200.models.config import get_config  # noqa: E402
from kvserve_b200.models.llama import LlamaShard  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--model", default="tiny-gqa")
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=120)
    ap.add_argument("--new-tokens", type=int, default=64)
    ap.add_argument("--repetition", type=float, default=1.0)
    args = ap.parse_args()
    cfg = get_config(args.model)
    max_len = args.prompt + args.new_tokens + 64
    model = LlamaShard(cfg, device="cuda:0", max_position=max_len)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, cfg.vocab, (args.prompt // 4 + 1,), generator=g).repeat(4)[:args.prompt].to(torch.int32)
               for _ in range(args.requests)]
    rules = {"repetition": torch.full((args.requests,), args.repetition, device="cuda:0")}
    blocks = args.requests * ((args.prompt + args.new_tokens) // 16 + 4)
    for name, nodes in (("one token a step", 1), ("trees of 16", 16)):
        dec = TreeDecoder(model, num_blocks=blocks, max_len=max_len, max_tree=nodes)
        dec.generate(prompts, 2, rules)  # warm-up
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = dec.generate(prompts, args.new_tokens, rules)
        torch.cuda.synchronize()
        steps, n = sum(r.steps for r in out), sum(len(r.tokens) for r in out)
        print(f"{name}: {n / steps:.2f} tokens a step, {(time.perf_counter() - t) * 1e3:.1f} ms, "
              f"first tokens {out[0].tokens[:8]}")


if __name__ == "__main__":
    main()
