"""Models whose cache is held in 4 bits: logits, generation, graphs, memory."""
import os

import numpy as np
import pytest
import torch

import helpers
import plain_q4
import plain_qwen2 as plain

pytestmark = pytest.mark.gpu


def _quantised_logits(folder, tokens, monkeypatch):
    """Plain logits in 64 bits where attention reads keys and values as 4 bits hold them."""
    config, weights = helpers.plain_model(folder)
    attend = plain.attention

    def held(x):
        return torch.from_numpy(plain_q4.stand_for(*plain_q4.quantise(x.numpy())))

    with monkeypatch.context() as patch:
        patch.setattr(plain, "attention", lambda q, k, v, **rest: attend(q, held(k), held(v), **rest))
        return plain.forward(config, weights, list(tokens), dtype=torch.float64).numpy()


def _replay(folder, dtype, steps, monkeypatch, page_size=16, graphs="1"):
    """The steps through the engine's runner; {(request, position): logits}."""
    from vipera_rs_b200.engine.replay import Replayer

    monkeypatch.setenv("VIPERA_POISON_CACHE", "1")
    monkeypatch.setenv("VIPERA_STEP_GRAPHS", graphs)
    replayer = Replayer(folder, dtype, max_tokens=512, page_size=page_size, max_live=4, kv_type="q4")
    replayer.runner.decode_graphs = graphs == "1"
    done, rows = {}, {}
    for entries, end in steps:
        logits = replayer.step([{"id": n, "tokens": t, "want": list(range(len(t)))} for n, t in entries], end)
        at = 0
        for name, tokens in entries:
            for _ in tokens:
                rows[name, done.get(name, 0)] = logits[at]
                done[name] = done.get(name, 0) + 1
                at += 1
    assert replayer.pools.audit() == ""
    return rows


def _steps(vocab):
    a, b, c = (helpers.random_tokens(vocab, n, seed) for n, seed in ((110, 1), (70, 2), (5, 3)))
    steps = [([("a", a[:50])], []), ([("a", a[50:51]), ("b", b[:33])], []), ([("a", a[51:52]), ("b", b[33:34])], []),
             ([("b", b[34:69]), ("c", c[:2]), ("a", a[52:100])], [])]
    steps += [([("a", a[100 + i:101 + i]), ("c", c[2 + i:3 + i])], ["c"] if i == 2 else []) for i in range(3)]
    steps += [([("a", a[103 + i:104 + i])], []) for i in range(7)] + [([("b", b[69:])], ["a", "b"])]
    return {"a": a, "b": b, "c": c}, steps


@pytest.mark.parametrize("name, page_size", [("A", 16), ("A", 24), ("B", 16)])
def test_logits_are_those_of_the_held_keys_and_values(name, page_size, monkeypatch):
    """32-bit steps against 64 bits over the same 4-bit cache.  A key that lies next to a border between two codes may fall to the
    other side there; few do, so a row is nearer to the plain logits over held keys than a tenth of what holding them changes."""
    folder = helpers.model_folder(name, "float32")
    sequences, steps = _steps(helpers.CONFIGS[name]["vocab_size"])
    rows = _replay(folder, "float32", steps, monkeypatch, page_size)
    for request, tokens in sequences.items():
        held = _quantised_logits(folder, tokens, monkeypatch)
        full = helpers.plain_logits(folder, tokens)
        got = np.stack([rows[request, i] for i in range(len(tokens))]).astype(np.float64)
        assert np.linalg.norm(got - held) < 0.1 * np.linalg.norm(held - full)


@pytest.mark.parametrize("name", ["A", "B"])
def test_bfloat16_steps_over_packed_pages(name, monkeypatch):
    """bfloat16 steps (single tokens over packed pages, portions through the expanded rows) are as far from the plain logits over held
    keys as bfloat16 is from 64 bits, and what holding the keys changes, at most."""
    folder = helpers.model_folder(name, "bfloat16")
    sequences, steps = _steps(helpers.CONFIGS[name]["vocab_size"])
    rows = _replay(folder, "bfloat16", steps, monkeypatch)
    for request, tokens in sequences.items():
        held = _quantised_logits(folder, tokens, monkeypatch)
        full, rounded = helpers.plain_logits(folder, tokens), helpers.plain_logits(folder, tokens, torch.bfloat16)
        got = np.stack([rows[request, i] for i in range(len(tokens))]).astype(np.float64)
        assert np.linalg.norm(got - held) < 2 * np.linalg.norm(rounded - full) + np.linalg.norm(held - full)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_captured_steps_give_the_bits_of_steps_launched_one_by_one(dtype, monkeypatch):
    """Rows of steps that fill their size class: the same kernels with the same cuts either way for tokens of portions; single tokens
    are cut for the block tables' width, which may differ, so theirs are compared within the type's rounding."""
    folder = helpers.model_folder("A", dtype)
    _, steps = _steps(helpers.CONFIGS["A"]["vocab_size"])
    captured = _replay(folder, dtype, steps, monkeypatch)
    eager = _replay(folder, dtype, steps, monkeypatch, graphs="0")
    scale = max(float(np.abs(row).max()) for row in eager.values())
    for key, row in captured.items():
        assert np.abs(row - eager[key]).max() <= scale * (2.0 ** -6 if dtype == "bfloat16" else 2.0 ** -10)


def _engine(name, dtype, **options):
    from vipera_rs_b200 import Engine

    return Engine(helpers.model_folder(name, dtype), dtype=dtype, kv_type="q4", **options)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_alone_together_ahead_and_again(dtype):
    """32-bit generation gives the same tokens alone and together; in either type the same run twice, and with steps launched ahead or
    not, gives the same tokens; pages come back."""
    from vipera_rs_b200 import SamplingParams

    vocab = helpers.CONFIGS["A"]["vocab_size"]
    prompts = [helpers.random_tokens(vocab, n, 900 + n) for n in (5, 33, 80)]
    params = SamplingParams(max_new_tokens=30)
    engine = _engine("A", dtype, page_size=16, ctx=256, max_num_seqs=3, max_tokens_per_step=48)
    together = [r.tokens for r in engine.generate(prompts, params)]
    assert all(len(t) == 30 for t in together)
    for lookahead in (True, False):
        other = _engine("A", dtype, page_size=16, ctx=256, max_num_seqs=3, max_tokens_per_step=48, lookahead=lookahead)
        assert [r.tokens for r in other.generate(prompts, params)] == together
        assert other.pools.audit() == ""
    if dtype == "float32":
        assert [engine.generate([p], params)[0].tokens for p in prompts] == together
    stats = engine.stats()
    assert stats["kv_used_pages"] == stats["kv_kept_pages"] and engine.pools.audit() == ""


def test_few_pages_preempt_and_windows_give_back():
    from vipera_rs_b200 import SamplingParams

    vocab = helpers.CONFIGS["B"]["vocab_size"]
    engine = _engine("B", "bfloat16", page_size=16, num_pages=18, max_num_seqs=3, max_tokens_per_step=64)
    prompts = [helpers.random_tokens(vocab, n, 50 + n) for n in (90, 100, 60)]
    results = engine.generate(prompts, SamplingParams(max_new_tokens=40))
    assert all(len(r.tokens) == 40 for r in results) and sum(r.preemptions for r in results) >= 1
    assert engine.pools.audit() == ""


def test_the_cache_is_as_large_as_planned():
    """The pools of a model of heads of 64 and 128: 4.5 bits a value, within the guards' and the scratch page's room."""
    from vipera_rs_b200.cache import CachePools
    from vipera_rs_b200.engine import planner
    from vipera_rs_b200.engine.loader import load_model

    for name in ("A", "B"):
        model = load_model(helpers.model_folder(name, "bfloat16"), "bfloat16")
        pools = CachePools(model.cache_requests, page_size=16, num_pages=64, num_state_slots=4, dtype=model.dtype, device=model.device, kv_type="q4")
        planned = 64 * 16 * planner.kv_bytes_per_token(model.spec, 2, "q4")
        per_page = planned // 64
        assert planned <= pools.bytes() <= planned + per_page + 4 * 256 * len(model.cache_requests)
        assert planned * 32 == 64 * 16 * planner.kv_bytes_per_token(model.spec, 2) * 9    # 4.5 bits for 16
        assert pools.audit() == ""
        pools.poison()
        assert pools.audit() == ""
