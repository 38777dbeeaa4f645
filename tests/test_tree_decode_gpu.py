"""Tree-drafted greedy decoding through the model, and its host-side drafter."""
import pytest
import torch


def test_lookup_drafts_share_equal_beginnings():
    from kvserve_b200.engine.tree_decode import lookup_drafts
    #          0  1  2  3  4  5  6  7  8  9
    history = [1, 2, 3, 4, 1, 2, 3, 5, 1, 2]
    tokens, parents = lookup_drafts(history, 5, match=2, width=2)
    # latest first: 3 5 1 2 under the root, then 3 (shared) 4 if there is room
    assert tokens == [3, 5, 1, 2] and parents == [0, 1, 2, 3]
    tokens, parents = lookup_drafts(history, 6, match=2, width=2)
    assert tokens == [3, 5, 1, 2, 4] and parents == [0, 1, 2, 3, 1]
    assert lookup_drafts([1, 2], 4) == ([], []) and lookup_drafts([7, 8, 9, 6], 4) == ([], [])


def _model():
    from kvserve_b200.models.config import get_config
    from kvserve_b200.models.llama import LlamaShard
    return LlamaShard(get_config("tiny-gqa"), device="cuda:0", max_position=1024)


def _logits_of_text(model, text):
    """Logits after every token of ``text``: one step of a causal chain over an empty cache."""
    from kvserve_b200 import ops
    n, dev = len(text), model.device
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    table = torch.zeros(1, -(-n // 16), dtype=torch.int32, device=dev)
    plan = ops.plan_step(zero, zero + n, table, zero, torch.arange(table.numel(), dtype=torch.int32, device=dev),
                         torch.tensor([0, table.numel()], device=dev), 16, n)
    L = model.cfg.num_layers
    kv = torch.empty(L, 2, n, model.hkv, model.D, dtype=torch.bfloat16, device=dev)
    cache = torch.zeros(L, 2, table.numel(), 16, model.hkv, model.D, dtype=torch.bfloat16, device=dev)
    ids = torch.tensor(text, dtype=torch.int32, device=dev)
    return model.verify_step(ids, plan, kv, cache, table, zero).float()


@pytest.mark.gpu
@pytest.mark.parametrize("max_tree", [1, 8, 33])
def test_generated_tokens_are_greedy_choices(max_tree):
    """Every generated token is the model's choice after its own text (up to
    the rounding of logits that differently shaped products give)."""
    from kvserve_b200.engine.tree_decode import TreeDecoder
    model = _model()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 4096, (n,), generator=g).to(torch.int32) for n in (1, 40, 65)]
    prompts.append(torch.randint(0, 4096, (20,), generator=g).repeat(4).to(torch.int32))
    dec = TreeDecoder(model, num_blocks=64, max_len=256, max_tree=max_tree)
    out = dec.generate(prompts, 24)
    assert dec.free_blocks() == 64
    for p, r in zip(prompts, out):
        assert len(r.tokens) == 24 and 24 // max_tree <= r.steps <= 24
        text = p.tolist() + r.tokens
        logits = _logits_of_text(model, text)[len(p) - 1:-1]
        chosen = logits.gather(1, torch.tensor(r.tokens, device="cuda")[:, None])[:, 0]
        # 4 layers of bf16 activations: both passes are within a few roundings of each other
        slack = 16 * 2.0 ** -8 * logits.abs().amax(1)
        assert (chosen >= logits.amax(1) - slack).all()
    # the same blocks again
    again = dec.generate(prompts, 24)
    assert [r.tokens for r in again] == [r.tokens for r in out]


@pytest.mark.gpu
def test_good_drafts_are_accepted_and_bad_ones_are_not():
    from kvserve_b200.engine.tree_decode import TreeDecoder
    model = _model()
    prompt = torch.arange(100, 150, dtype=torch.int32)
    plain = TreeDecoder(model, num_blocks=32, max_len=256, max_tree=8, propose=lambda h, n: ([], []))
    want = plain.generate([prompt], 32)[0]
    assert want.steps == 32
    text = prompt.tolist() + want.tokens

    def right(history, nodes):  # the known continuation, beside a wrong child of the root
        rest = text[len(history):len(history) + nodes - 2]
        return [4095] + rest, [0, 0] + list(range(2, len(rest) + 1))[:max(0, len(rest) - 1)]

    good = TreeDecoder(model, num_blocks=32, max_len=256, max_tree=8, propose=right).generate([prompt], 32)[0]
    # Seven tokens a step (the root's choice and six drafts) for as long as the
    # texts agree.  They may part where two logits are within rounding of each
    # other; from there on the drafts are wrong: one token a step.
    same = next((i for i, (x, y) in enumerate(zip(want.tokens, good.tokens)) if x != y), 32)
    assert same >= 7 and good.steps <= -(-same // 7) + 32 - same
    if same < 32:
        logits = _logits_of_text(model, text)[len(prompt) - 1 + same]
        assert logits[good.tokens[same]] >= logits.max() - 16 * 2.0 ** -8 * logits.abs().max()
    wrong = TreeDecoder(model, num_blocks=32, max_len=256, max_tree=8,
                        propose=lambda h, n: ([h[-1]] * 3, [0, 0, 1])).generate([prompt], 32)[0]
    assert len(wrong.tokens) == 32 and wrong.steps >= 16


@pytest.mark.gpu
def test_rules_reach_the_choice():
    from kvserve_b200.engine.tree_decode import TreeDecoder
    model = _model()
    prompt = torch.arange(50, dtype=torch.int32)
    dec = TreeDecoder(model, num_blocks=32, max_len=256)
    ids = torch.tensor([[77]], dtype=torch.int32, device="cuda")
    big = torch.full((1, 1), 1e4, device="cuda")
    out = dec.generate([prompt], 6, rules={"bias_ids": ids, "bias_values": big})[0]
    assert out.tokens == [77] * 6
    # a presence penalty larger than the bias lets the token come once
    out = dec.generate([prompt], 6, rules={"bias_ids": ids, "bias_values": big,
                                           "presence": torch.full((1,), 3e4, device="cuda")})[0]
    assert out.tokens[0] == 77 and 77 not in out.tokens[1:] and len(set(out.tokens)) == 6
    stopped = dec.generate([prompt], 6, rules={"bias_ids": ids, "bias_values": big}, stop=77)[0]
    assert stopped.tokens == [77]


@pytest.mark.gpu
def test_running_out_of_blocks_is_an_error_and_gives_them_back():
    from kvserve_b200.engine.tree_decode import TreeDecoder
    model = _model()
    dec = TreeDecoder(model, num_blocks=4, max_len=512)
    with pytest.raises(RuntimeError, match="no free KV blocks"):
        dec.generate([torch.arange(40, dtype=torch.int32)], 64)
    assert dec.free_blocks() == 4
    assert len(dec.generate([torch.arange(40, dtype=torch.int32)], 8)[0].tokens) == 8


def test_refusals():
    from types import SimpleNamespace
    from kvserve_b200.engine.tree_decode import TreeDecoder
    with pytest.raises(ValueError, match="one GPU"):
        TreeDecoder(SimpleNamespace(tp_size=2), 4, 64)
    with pytest.raises(ValueError, match="max_tree"):
        TreeDecoder(SimpleNamespace(tp_size=1), 4, 64, max_tree=65)


def test_max_len_beyond_the_rotary_table_is_refused():
    """Refused on the host: the rotary kernels read the table by position."""
    from types import SimpleNamespace
    from kvserve_b200.engine.tree_decode import TreeDecoder
    cfg = SimpleNamespace(num_layers=1)
    model = SimpleNamespace(tp_size=1, cfg=cfg, device=torch.device("cpu"), hkv=1, D=64, cos_sin=torch.zeros(100, 64))
    with pytest.raises(ValueError, match="rotary table"):
        TreeDecoder(model, 4, 101)
    assert TreeDecoder(model, 4, 100).max_len == 100


def test_the_example_starts_from_the_source_tree(tmp_path):
    """Its documented command finds the package without an installation."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    run = subprocess.run([sys.executable, os.path.join(root, "examples", "tree_decoding.py"), "--help"], cwd=tmp_path,
                         env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "--new-tokens" in run.stdout, run.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("fault", ["rule", "parent"])
def test_a_step_that_fails_after_its_plan_gives_its_blocks_back(fault):
    """The step's plan takes a block (the prompt ends a block) before the rules
    are refused, or before the broken tree is reported."""
    from kvserve_b200.engine.tree_decode import TreeDecoder
    model = _model()
    prompt = torch.arange(33, dtype=torch.int32)  # 32 committed tokens: two whole blocks of 16

    def broken(history, nodes):  # a parent that comes later
        return [5, 6], [2, 0]
    dec = TreeDecoder(model, num_blocks=16, max_len=128, propose=broken if fault == "parent" else lambda h, n: ([], []))
    rules = {"repetition": torch.full((1,), 1.1)} if fault == "rule" else {}  # not on the GPU
    for _ in range(3):
        with pytest.raises((ValueError, RuntimeError)):
            dec.generate([prompt], 8, rules=rules)
        assert dec.free_blocks() == 16
    dec.propose = lambda h, n: ([], [])
    assert len(dec.generate([prompt], 8)[0].tokens) == 8 and dec.free_blocks() == 16


@pytest.mark.gpu
def test_no_new_tokens():
    from kvserve_b200.engine.tree_decode import TreeDecoder
    dec = TreeDecoder(_model(), num_blocks=16, max_len=128)
    out = dec.generate([torch.arange(n, dtype=torch.int32) for n in (1, 20)], 0)
    assert [(r.tokens, r.steps) for r in out] == [([], 0), ([], 0)] and dec.free_blocks() == 16
    with pytest.raises(ValueError, match="max_new_tokens"):
        dec.generate([torch.arange(20, dtype=torch.int32)], -1)


@pytest.mark.gpu
def test_text_may_fill_max_len():
    """Prompt and new tokens of exactly max_len give the tokens of a decoder
    with room to spare; one more is refused."""
    from kvserve_b200.engine.tree_decode import TreeDecoder
    model = _model()
    prompt = torch.arange(7, dtype=torch.int32).repeat(6)[:40]
    roomy = TreeDecoder(model, num_blocks=16, max_len=128).generate([prompt], 9)[0]
    dec = TreeDecoder(model, num_blocks=16, max_len=49)
    tight = dec.generate([prompt], 9)[0]
    assert tight.tokens == roomy.tokens and tight.steps == roomy.steps and len(tight.tokens) == 9
    with pytest.raises(ValueError, match="max_len"):
        dec.generate([prompt], 10)


@pytest.mark.gpu
def test_an_error_in_the_last_step_is_raised(monkeypatch):
    """What the kernels of the last step report does not wait for a later call."""
    from kvserve_b200 import ops
    from kvserve_b200.engine.tree_decode import TreeDecoder
    model = _model()
    dec = TreeDecoder(model, num_blocks=16, max_len=128)
    verify = model.verify_step

    def failing(*args):
        logits = verify(*args)
        ops.device_status(model.device)[0] = 1  # as a kernel whose wait ran out does
        return logits
    monkeypatch.setattr(model, "verify_step", failing)
    with pytest.raises(RuntimeError, match="timeout"):
        dec.generate([torch.arange(20, dtype=torch.int32)], 1)
    assert dec.free_blocks() == 16
    ops.check_device_status(model.device)
