"""Attention over the 4-bit cache on the device, at its edges."""
import numpy as np
import pytest
import torch

import plain_q4 as plain
from test_cache_q4_gpu import DEVICE, Step, _int, _off, _workspace, deal, form, ops  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def _attend(ops, step, pages, q, heads, kv_heads, d, scale=0.1, workspace=None, **more):
    out = torch.zeros_like(q)
    ops.attention_q4(q, out, pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, scale=scale, workspace=workspace or _workspace(),
                     **dict(step.device(), **more))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_an_output_off_its_pieces_is_refused_by_steps_of_rows(ops, dtype, d):
    """32-bit steps, single tokens' too, and short bfloat16 portions: refused on the host, nothing is launched."""
    from vipera_rs_b200.errors import InternalError

    for counts in ([3, 2], [1, 1]):
        if dtype == torch.bfloat16 and counts == [1, 1]:
            continue
        step = Step(counts, [20, 3], 16)
        tokens = sum(counts)
        assert ops.attention_q4_takes_rows(dtype, d, 16, tokens * 2, 24, 2)
        pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, d, 3, DEVICE))
        q = torch.randn(tokens, 2 * d, device=DEVICE).to(dtype)
        before = ops.launches
        with pytest.raises(InternalError, match="bad argument"):
            ops.attention_q4(q, _off(q), pages, num_heads=2, num_kv_heads=1, head_dim=d, scale=0.1, workspace=_workspace(), **step.device())
        assert ops.launches == before
        # queries may begin anywhere: they are read value by value
        assert torch.equal(_attend(ops, step, pages, _off(q), 2, 1, d), _attend(ops, step, pages, q, 2, 1, d))


@pytest.mark.parametrize("captured", [False, True])
def test_layers_that_share_their_buffers_beside_portions(ops, deal, monkeypatch, captured):
    """Write, portions, single tokens, layer after layer as an engine runs them: queries, outputs and workspace are the same buffers in every
    layer, pages are the layer's own.  Each layer's outputs are those of the same launches with a pause behind each."""
    monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
    monkeypatch.setattr(ops, "q4_portion_plan", lambda *a: (128, 1 << 20, 1))
    heads, kv_heads, d, layers = 8, 2, 128, 12
    step = Step([1, 300, 1, 40, 1, 1], [900, 100, 700, 30, 1500, 3], 16)
    tokens = sum(step.counts)
    described, slots, room = step.device(), _int(step.slots), _workspace()
    qkv = torch.randn(layers, tokens, (heads + 2 * kv_heads) * d, device=DEVICE)
    start = [plain.make_pages(step.num_pages, 16, kv_heads, d, 3 + i, DEVICE) for i in range(layers)]
    q, out, kept = (torch.zeros(*n, tokens, heads * d, dtype=torch.bfloat16, device=DEVICE) for n in ((), (), (layers,)))

    def run(pages, pause):
        for i in range(layers):
            ops.rope_cache_q4(qkv[i], q, pages[i], num_heads=heads, num_kv_heads=kv_heads, head_dim=d, positions=described["positions"],
                              cos=None, sin=None, style=ops.ROPE_NONE, slots=slots)
            pause()
            ops.attention_q4(q, out, pages[i], num_heads=heads, num_kv_heads=kv_heads, head_dim=d, scale=0.09, workspace=room, settled=True,
                             **described)
            pause()
            kept[i].copy_(out)
            pause()

    fresh = lambda: [ops.Q4Pages(*[t.clone() for t in layer]) for layer in start]
    run(fresh(), torch.cuda.synchronize)
    expected = kept.clone()
    pages = fresh()
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(pages, lambda: None)
        again = graph.replay
    else:
        again = lambda: run(pages, lambda: None)
    for _ in range(5):
        kept.zero_()
        again()
        torch.cuda.synchronize()
        assert torch.equal(kept, expected)
    assert int(room.get("attention.q4_beside", (1,), torch.int32)) == 0        # taken back


@pytest.mark.parametrize("singles", [0, 1, 3])
@pytest.mark.parametrize("portions", [0, 2])
def test_steps_of_portions_alone_and_of_single_tokens_alone_said_to_hold_both(ops, deal, monkeypatch, singles, portions):
    """Either kernel may find nothing to do: the other's rows are right, and the word between them is taken back."""
    if not singles + portions:
        return
    monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
    monkeypatch.setattr(ops, "q4_portion_plan", lambda *a: (256, 1 << 20, 1))
    step = Step([1] * singles + [70, 150][:portions], [500, 2, 90][:singles] + [0, 900][:portions], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 2, 128, 3, DEVICE))
    q = torch.randn(sum(step.counts), 8 * 128, device=DEVICE).to(torch.bfloat16)
    room = _workspace()
    both = _attend(ops, step, pages, q, 8, 2, 128, workspace=room, all_single=False, any_single=True)
    assert int(room.get("attention.q4_beside", (1,), torch.int32)) == 0
    if portions:
        apart = _attend(ops, step, pages, q, 8, 2, 128, any_single=False)          # every row the portions' kernel's
        assert torch.equal(both[singles:], apart[singles:])
    if singles:
        alone = Step([1] * singles, [500, 2, 90][:singles], 16)
        alone.tables = step.tables[:singles]
        expected = _attend(ops, alone, pages, q[:singles].contiguous(), 8, 2, 128)
        assert torch.equal(both[:singles], expected)


@pytest.mark.parametrize("heads", [6, 22])
@pytest.mark.parametrize("d", [64, 128])
def test_a_group_that_is_not_finite_shows_in_its_own_channels_of_single_tokens(ops, deal, d, heads):
    """One group of one value, each in turn: the group's outputs of the heads that see it are NaN, all others those of the same step without,
    bit for bit."""
    kv_heads, key = 2, 141
    step = Step([1, 1, 1], [700, 60, 150], 16)
    raw = plain.make_pages(step.num_pages, 16, kv_heads, d, 3, DEVICE)
    pages = ops.Q4Pages(*raw)
    q = torch.randn(3, heads * d, device=DEVICE).to(torch.bfloat16)
    without = _attend(ops, step, pages, q, heads, kv_heads, d).view(3, heads, d)
    assert without.isfinite().all()
    for group in range(d // 32):
        usual = raw[3].clone()
        for entry in (0, 2):
            raw[3][step.tables[entry][key // 16], 1, key % 16, group] = float("nan")
        with_one = _attend(ops, step, pages, q, heads, kv_heads, d).view(3, heads, d)
        raw[3].copy_(usual)
        bad = torch.zeros(3, heads, d, dtype=torch.bool, device=DEVICE)
        bad[0::2, heads // 2:, 32 * group:32 * group + 32] = True
        assert with_one[bad].isnan().all()
        assert torch.equal(with_one[~bad], without[~bad])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page_size", [16, 24])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales_that_are_not_positive(ops, form, dtype, page_size, scale):
    """A scale below 0 turns the order of the scores, one of 0 weighs all keys alike; hidden keys stay hidden."""
    heads, kv_heads, d = 6, 2, 64
    step = Step([50, 1, 70], [40, 300, 0], page_size)
    raw = plain.make_pages(step.num_pages, page_size, kv_heads, d, 3, DEVICE)
    k_rows, v_rows = plain.rows_of(raw[0], raw[1], True), plain.rows_of(raw[2], raw[3], False)
    q = torch.randn(121, heads * d, device=DEVICE).to(dtype)
    got = _attend(ops, step, ops.Q4Pages(*raw), q, heads, kv_heads, d, scale=scale).double().cpu().numpy().reshape(121, heads, d)
    expected, parts = plain.attend(q.double().cpu().numpy(), k_rows, v_rows, counts=step.counts, history=step.history, tables=step.tables,
                                   page_size=page_size, num_heads=heads, num_kv_heads=kv_heads, d=d, scale=scale,
                                   k_steps=raw[1].double().cpu().numpy(), v_steps=raw[3].double().cpu().numpy())
    for name in ("reach", "full"):      # sizes of scores' terms
        parts[name] = np.abs(parts[name])
    limit = plain.allowed(expected, parts, 301, d, dtype)
    assert (np.abs(got - expected) <= limit).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("queries, keys", [(126, -100), (124, -100), (100, -20), (-100, 60), (0, 117), (0, -90)])
def test_single_tokens_with_numbers_near_the_ends_of_the_type(ops, deal, d, queries, keys):
    """Queries and keys times powers of two, the scale divided by them: nothing on the way to a score leaves its type, so the outputs are the
    same bits."""
    step = Step([1, 1], [190, 17], 16)
    raw = plain.make_pages(step.num_pages, 16, 1, d, 3, DEVICE)
    q = torch.randn(2, 4 * d, device=DEVICE).clamp(-1.9, 1.9).to(torch.bfloat16)
    usual = _attend(ops, step, ops.Q4Pages(*raw), q, 4, 1, d)
    far = q.double() * 2.0 ** queries
    assert torch.equal(far.to(torch.bfloat16).double(), far)
    raw[1].mul_(2.0 ** keys)
    assert torch.equal(_attend(ops, step, ops.Q4Pages(*raw), far.to(torch.bfloat16), 4, 1, d, scale=0.1 * 2.0 ** -(queries + keys)), usual)


def test_a_first_mixed_step_leaves_captured_steps_valid(ops, monkeypatch):
    """A workspace that has seen a step of portions alone holds all that a mixed one asks for: nothing captured before goes stale."""
    monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
    monkeypatch.setattr(ops, "q4_portion_plan", lambda *a: (256, 1 << 20, 1))
    room, seen = _workspace(), []
    for counts in ([70, 150], [70, 150, 1]):
        step = Step(counts, [0, 900, 30][:len(counts)], 16)
        pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 2, 128, 3, DEVICE))
        q = torch.randn(sum(counts), 8 * 128, device=DEVICE).to(torch.bfloat16)
        _attend(ops, step, pages, q, 8, 2, 128, workspace=room)
        seen.append(room.generation)
    assert seen[0] == seen[1]


@pytest.mark.parametrize("page_size", [16, 24])
@pytest.mark.parametrize("per_head", [False, True])
def test_a_sink_of_score_0_beside_a_gate(ops, form, page_size, per_head):
    """No flash kernel has both endings: over expanded rows such a step is the general kernel's, and is not refused."""
    from test_cache_q4_gpu import _attend as attend_and_compare

    heads, d = 4, 64
    gate = np.random.default_rng(9).standard_normal((60, heads * (1 if per_head else d))).astype(np.float32)
    attend_and_compare(ops, Step([19, 1, 40], [33, 64, 0], page_size), torch.bfloat16, heads, 2, d, sink=True, gate=gate, gate_per_head=per_head)
