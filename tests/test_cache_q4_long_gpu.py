"""The 4-bit cache over long histories and in whole models, with bounds that a lost run of keys, or a cache that was never quantised, would not keep."""
import numpy as np
import pytest
import torch

import helpers
import plain_q4
import plain_qwen2
from test_cache_q4_engine_gpu import _quantised_logits, _replay, _steps
from test_cache_q4_gpu import DEVICE, Step, _int, _workspace, form, ops  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu
UNIT = 128     # keys: what a block of the single tokens' kernels, and a tile of the tensor cores', walks at a time


@pytest.fixture(params=[1, 2, 16, 0])
def shares(ops, request, monkeypatch):
    """Blocks that share a (request, KV head) pair's keys; 0: all pairs' keys in even runs."""
    monkeypatch.setattr(ops, "q4_shares", lambda *sizes: request.param)
    return request.param


def _walked(ops, shares, entries, pairs, units):
    """Units of keys that a block walks at most, and parts that are joined."""
    if shares:
        return -(-units // shares), shares
    runs = ops.Q4_BLOCKS_PER_SM * ops._sm_count_of(0)
    run = -(-entries * pairs * (units + 3) // runs)
    return min(run, units), -(-units // run) + 1


class Outlier:
    """Requests that share their pages but for one unit each, the unit of their number: there every value is `rise` times as large as elsewhere's
    scales and of one sign.  Queries of zeros weigh all keys alike, so an output is a mean of values, and a unit, or sixteen rows of it, that are left
    out or counted twice change its request's mean by more than all roundings."""

    def __init__(self, ops, keys, page_size, kv_heads, d, tokens):
        self.units = -(-keys // UNIT)
        held = -(-keys // page_size)
        each = UNIT // page_size
        raw = plain_q4.make_pages(held + each, page_size, kv_heads, d, 5, DEVICE)
        self.rise = 1024.0
        raw[2][held:] = 0                            # codes of -8
        raw[3][held:] = -self.rise
        self.pages = ops.Q4Pages(*raw)
        self.step = Step([tokens] * self.units, [keys - tokens] * self.units, page_size)
        self.step.tables = [[held + index - each * e if each * e <= index < each * (e + 1) else index for index in range(held)]
                            for e in range(self.units)]
        base = plain_q4.rows_of(raw[2][:held], raw[3][:held], False).swapaxes(1, 2).reshape(held * page_size, kv_heads, d)[:keys]
        steps = np.repeat(np.abs(raw[3][:held].double().cpu().numpy()), 32, -1).swapaxes(1, 2).reshape(held * page_size, kv_heads, d)[:keys]
        self.means, self.sizes, self.steps = [], [], []
        for e in range(self.units):
            at = slice(e * UNIT, min((e + 1) * UNIT, keys))
            v, s = base.copy(), steps.copy()
            v[at], s[at] = 8 * self.rise, self.rise
            for i in range(tokens):
                seen = keys - tokens + i + 1
                self.means.append(v[:seen].mean(0))
                self.sizes.append(np.abs(v[:seen]).mean(0))
                self.steps.append(s[:seen].mean(0))
        self.means, self.sizes, self.steps = (np.stack(x) for x in (self.means, self.sizes, self.steps))

    def run(self, ops, heads, kv_heads, d, dtype):
        tokens = len(self.step.positions)
        q = torch.zeros(tokens, heads * d, dtype=dtype, device=DEVICE)
        out = torch.zeros_like(q)
        ops.attention_q4(q, out, self.pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, scale=0.1, workspace=_workspace(),
                         **self.step.device())
        return out.double().cpu().numpy().reshape(tokens, kv_heads, heads // kv_heads, d)

    def check(self, got, keys, walk=None, parts=1, rounding=2.0 ** -8):
        # Weights of 1 are exact, times a scale too.  A sum of `keys` products is off by 2^-22 of its terms' sizes for each 16 of them and each
        # part; single tokens' codes are summed as 136 above, 144 steps at most, by 2^-20 for each product of 17 terms, of which
        # a warp has one for 16 keys, 2 for a unit, and four join it.
        limit = self.sizes * (keys / 16 + parts) * 2.0 ** -22 + np.abs(self.means) * rounding + 2.0 ** -30
        if walk is not None:
            limit = limit + self.steps * (2 * walk + 4 + parts) * 144 * 2.0 ** -20
        # sixteen rows of the outlying unit less, or twice, are seen (one row moves a mean by about twice what its bfloat16 rounding alone may)
        assert (limit * 2 < 16 * (8 * self.rise - np.abs(self.means)) / (keys + 16)).all()
        assert (np.abs(got - self.means[:, :, None]) <= limit[:, :, None]).all()


@pytest.mark.parametrize("heads, kv_heads, d, keys, page_size", [(2, 1, 64, 9000, 16), (6, 2, 128, 5000, 64), (12, 1, 128, 3000, 16)])
def test_no_key_of_a_long_history_is_lost_or_counted_twice(ops, shares, heads, kv_heads, d, keys, page_size):
    history = Outlier(ops, keys, page_size, kv_heads, d, 1)
    walk, parts = _walked(ops, shares, history.units, kv_heads, history.units)
    history.check(history.run(ops, heads, kv_heads, d, torch.bfloat16), keys, walk, parts)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, d, keys, tokens", [(2, 1, 64, 9000, 3), (6, 2, 128, 5000, 50)])
def test_no_key_of_a_long_history_is_lost_by_portions(ops, form, dtype, heads, kv_heads, d, keys, tokens):
    history = Outlier(ops, keys, 16, kv_heads, d, tokens)
    history.check(history.run(ops, heads, kv_heads, d, dtype), keys, parts=64, rounding=2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("counts, history", [([3, 1, 20], [5000, 5, 2500]), ([70], [4000])])
def test_long_histories_of_portions_within_their_own_roundings(ops, form, d, counts, history):
    """bfloat16 portions read codes as exact numbers: scores are off by 32-bit sums alone, a weight and the output by a rounding each."""
    step = Step(counts, history, 16, seed=d)
    heads, kv_heads = 2, 1
    raw = plain_q4.make_pages(step.num_pages, 16, kv_heads, d, 3, DEVICE)
    k_rows, v_rows = plain_q4.rows_of(raw[0], raw[1], True), plain_q4.rows_of(raw[2], raw[3], False)
    tokens, scale = sum(counts), d ** -0.5
    q = torch.randn(tokens, heads * d, device=DEVICE).to(torch.bfloat16)
    out = torch.zeros_like(q)
    ops.attention_q4(q, out, ops.Q4Pages(*raw), num_heads=heads, num_kv_heads=kv_heads, head_dim=d, scale=scale, workspace=_workspace(),
                     **dict(step.device(), any_single=False))         # every row a portion's
    expected, parts = plain_q4.attend(q.double().cpu().numpy(), k_rows, v_rows, counts=counts, history=history, tables=step.tables,
                                      page_size=16, num_heads=heads, num_kv_heads=kv_heads, d=d, scale=scale)
    # the terms of plain_q4.allowed that hold for these kernels: no offsets beside the codes
    unit, keys = 2.0 ** -22, max(c + h for c, h in zip(counts, history))
    relative = 2 * (d + 8) * parts["reach"] * unit + 2 * (keys + 16) * unit
    limit = parts["spread"] * (2.0 ** -8 + 2.0 ** -15 + relative[..., None]) + np.abs(expected) * 2.0 ** -8 + 2.0 ** -30
    assert (np.abs(out.double().cpu().numpy().reshape(expected.shape) - expected) <= limit).all()


@pytest.mark.parametrize("name", ["A", "B"])
def test_bfloat16_models_attend_over_held_keys(name, monkeypatch):
    """bfloat16 steps round as the plain model in bfloat16 over held keys does, and as often move a key over a border between two codes: over all
    rows they are as far from 64 bits, half as much again at most, which is less than what holding the keys changes."""
    folder = helpers.model_folder(name, "bfloat16")
    sequences, steps = _steps(helpers.CONFIGS[name]["vocab_size"])
    rows = _replay(folder, "bfloat16", steps, monkeypatch)
    config, weights = helpers.plain_model(folder)
    attend = plain_qwen2.attention
    held_of = lambda x: torch.from_numpy(plain_q4.stand_for(*plain_q4.quantise(x.numpy())))
    off = {"got": 0.0, "rounded": 0.0, "unheld": 0.0}
    for request, tokens in sequences.items():
        held = _quantised_logits(folder, tokens, monkeypatch)
        with monkeypatch.context() as patch:
            patch.setattr(plain_qwen2, "attention", lambda q, k, v, **rest: attend(q, held_of(k), held_of(v), **rest))
            rounded = plain_qwen2.forward(config, weights, list(tokens), dtype=torch.float64, round_to=torch.bfloat16).numpy()
        got = np.stack([rows[request, i] for i in range(len(tokens))]).astype(np.float64)
        for key, other in (("got", got), ("rounded", rounded), ("unheld", helpers.plain_logits(folder, tokens, torch.bfloat16))):
            off[key] += float(((other - held) ** 2).sum())
    got, rounded, unheld = (off[key] ** 0.5 for key in ("got", "rounded", "unheld"))
    assert 1.5 * rounded < unheld
    assert got < 1.5 * rounded


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_portion_that_fills_its_class_has_the_same_bits_captured(dtype, monkeypatch):
    """128 tokens, whose block table's width is the class's: captured or launched kernel by kernel, the keys are cut alike."""
    folder = helpers.model_folder("A", dtype)
    tokens = helpers.random_tokens(helpers.CONFIGS["A"]["vocab_size"], 128, 4)
    captured, eager = (_replay(folder, dtype, [([("a", tokens)], [])], monkeypatch, graphs=graphs) for graphs in ("1", "0"))
    assert all(np.array_equal(captured[key], eager[key]) for key in eager) and len(eager) == 128
