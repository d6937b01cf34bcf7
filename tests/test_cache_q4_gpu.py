"""Operators of the 4-bit cache on the device against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

import plain_q4 as plain

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.kernels import ops

    return ops


def _workspace():
    from vipera_rs_b200.parts.base import Workspace

    return Workspace(DEVICE)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


class Step:
    """A step's description: lengths, pages in random order, block tables, and the maps of its tokens."""

    def __init__(self, counts, history, page_size, seed=0, spare=3, width=None):
        rng = np.random.default_rng(seed)
        self.counts, self.history, self.page_size = counts, history, page_size
        self.held = [-(-(c + h) // page_size) for c, h in zip(counts, history)]
        self.num_pages = sum(self.held) + spare
        order = rng.permutation(self.num_pages)
        self.tables, at = [], 0
        width = width or max(self.held + [1])
        self.pages = order[:sum(self.held)]
        for n in self.held:
            self.tables.append([int(x) for x in order[at:at + n]] + [-1] * (width - n))
            at += n
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(int)
        self.positions = [h + i for c, h in zip(counts, history) for i in range(c)]
        self.entry = [e for e, c in enumerate(counts) for _ in range(c)]
        self.slots = [self.tables[e][p // page_size] * page_size + p % page_size for e, p in zip(self.entry, self.positions)]

    def device(self):
        return dict(entry_starts=_int(self.starts), entry_pos0=_int(self.history), positions=_int(self.positions),
                    token_entry=_int(self.entry), block_table=_int(self.tables),
                    max_keys=max(c + h for c, h in zip(self.counts, self.history)), all_single=all(c == 1 for c in self.counts),
                    any_single=any(c == 1 for c in self.counts))


@pytest.mark.parametrize("page_size", [1, 7, 16, 64])
@pytest.mark.parametrize("counts, history", [
    ([1], [0]), ([1, 1, 1], [5, 0, 100]), ([3, 1, 200], [0, 63, 17]), ([0, 2, 0, 1, 0], [0, 3, 9, 0, 0]), ([700], [1]),
    ([1] * 70, list(range(70)))])
def test_maps_are_those_of_the_lengths(ops, page_size, counts, history):
    step = Step(counts, history, page_size, width=60 if page_size >= 16 else None)
    tokens = len(step.positions)
    table = torch.full((len(counts), len(step.tables[0])), 77, dtype=torch.int32, device=DEVICE)
    out = {name: torch.full((tokens + 3,), 77, dtype=torch.int32, device=DEVICE) for name in ("positions", "token_entry", "slots")}
    page_starts = _int(np.concatenate([[0], np.cumsum(step.held)]))
    ops.step_maps(_int(step.starts), _int(history), page_size=page_size, page_starts=page_starts, pages=_int(step.pages),
                  block_table=table, **out)
    assert table.tolist() == step.tables
    for name, expected in (("positions", step.positions), ("token_entry", step.entry), ("slots", step.slots)):
        assert out[name].tolist() == expected + [77] * 3       # what lies behind the last token stays
    again = torch.full_like(out["slots"], 77)
    ops.step_maps(_int(step.starts), _int(history), page_size=page_size, block_table=table, slots=again)   # from the tables alone
    assert again.tolist() == step.slots + [77] * 3
    assert table.tolist() == step.tables


def test_maps_where_pages_are_missing_or_tables_are_short(ops):
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEVICE)
    slots = torch.zeros(6, dtype=torch.int32, device=DEVICE)
    # the first holds one page of the two that its tokens need, the second three where the table has room for two
    ops.step_maps(_int([0, 3, 6]), _int([2, 7]), page_size=4, page_starts=_int([0, 1, 4]), pages=_int([5, 1, 2, 9]), block_table=table,
                  slots=slots)
    assert table.tolist() == [[5, -1], [1, 2]]
    assert slots.tolist() == [22, 23, -1, 11, 36, 37]
    ops.step_maps(_int([0, 3, 6]), _int([2, 7]), page_size=4, block_table=table, slots=slots)
    assert slots.tolist() == [22, 23, -1, 11, -1, -1]
    ops.step_maps(_int([0]), _int([]), page_size=4, block_table=table[:0], slots=slots[:0])   # a step of nothing


def _turn(x, cos, sin, rot, interleaved):
    """The rotation in 32 bits, every product and sum rounded by itself (numpy does not fuse)."""
    x = x.astype(np.float32).copy()
    half = rot // 2
    first = 2 * np.arange(half) if interleaved else np.arange(half)
    second = first + 1 if interleaved else first + half
    a, b = x[..., first].copy(), x[..., second].copy()
    c, s = cos[:, None, :], sin[:, None, :]
    x[..., first], x[..., second] = a * c - b * s, a * s + b * c
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, d, rot, style, extra", [
    (4, 2, 64, 64, "neox", 0), (12, 2, 128, 128, "neox", 0), (5, 1, 128, 64, "neox", 4), (3, 3, 96, 96, "interleaved", 0),
    (2, 1, 32, 6, "interleaved", 3), (2, 1, 32, 20, "neox", 0), (2, 2, 256, 256, "neox", 1), (7, 1, 64, 0, "neox", 0),
    (4, 4, 64, 64, "none", 0)])
def test_keys_and_values_are_the_nearest_codes(ops, dtype, heads, kv_heads, d, rot, style, extra):
    step = Step([1, 37, 2], [40, 0, 15], 16, seed=d + rot)
    tokens = len(step.positions)
    rng = np.random.default_rng(d)
    x = (rng.standard_normal((tokens, heads + 2 * kv_heads, d)) * np.exp(rng.standard_normal(d))).astype(np.float32)
    x[3, heads, :32] = 0.0                       # a group of zeros
    x[4, heads + kv_heads, 5] = np.nan           # groups that are not finite show as a whole
    x[5, heads + kv_heads, 7] = -np.inf
    x[6, heads + kv_heads, :32] *= np.float32(1e-42) / 3    # a group whose scale has no bits left
    x[7, heads + kv_heads, :32] *= np.float32(2.0 ** 100)
    x[8, heads + kv_heads, :32] = 3.0            # all alike
    x[9, heads + kv_heads, :4] = [2.0, -2.0, 1.875, -1.875]
    angles = np.arange(64)[:, None] * 10000.0 ** (-np.arange(max(rot // 2, 1)) / max(rot // 2, 1))
    cos, sin = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    turned = x.copy()
    if style != "none" and rot:
        turned[:, :heads + kv_heads] = _turn(x[:, :heads + kv_heads], cos[step.positions], sin[step.positions], rot, style == "interleaved")
    qkv = torch.full((tokens, x[0].size + extra), 9e9, dtype=torch.float32, device=DEVICE)
    qkv[:, :x[0].size] = torch.from_numpy(x.reshape(tokens, -1)).to(DEVICE)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, kv_heads, d, 1, DEVICE))
    before = [t.clone() for t in pages]
    q_out = torch.zeros(tokens, heads * d, dtype=dtype, device=DEVICE)
    slots = _int(step.slots)
    slots[2] = -1                                # not written
    slots[10] = step.num_pages * 16              # nor is a slot outside the pool
    tables = [torch.from_numpy(t[:, :rot // 2].copy()).to(DEVICE) if rot else None for t in (cos, sin)]
    ops.rope_cache_q4(qkv, q_out, pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, rot_dims=rot, positions=_int(step.positions),
                      cos=tables[0], sin=tables[1], slots=slots,
                      style={"neox": ops.ROPE_NEOX, "interleaved": ops.ROPE_INTERLEAVED, "none": ops.ROPE_NONE}[style])
    expected_q = torch.from_numpy(turned[:, :heads].reshape(tokens, -1)).to(dtype)
    assert torch.equal(q_out.cpu(), expected_q)
    written = [t for t in range(tokens) if t not in (2, 10)]
    for which, keys in ((0, True), (1, False)):
        codes, scales = plain.quantise(turned[written, heads + which * kv_heads:heads + (which + 1) * kv_heads])
        tiny = np.abs(scales) < 2.0 ** -126       # 19 bits go there too, of a number that has fewer
        expected_codes, expected_scales = before[2 * which].cpu().numpy().copy(), before[2 * which + 1].float().cpu().numpy().copy()
        got_codes, got_scales = pages[2 * which].cpu().numpy(), pages[2 * which + 1].float().cpu().numpy()
        at = np.asarray([step.slots[t] for t in written])
        page, place = at // 16, at % 16
        if tiny.any():
            assert np.abs(got_scales[page, :, place][tiny]).max() < 2.0 ** -126
            scales = np.where(tiny, got_scales[page, :, place], scales)
            codes = np.where(tiny[..., None], plain.unpack(got_codes[page, :, place], keys), codes)
        expected_codes[page, :, place] = plain.pack(codes, keys)
        expected_scales[page, :, place] = scales
        assert np.array_equal(got_codes, expected_codes)
        assert np.array_equal(got_scales, expected_scales, equal_nan=True)


def test_queries_alone_leave_the_pages(ops):
    step = Step([3], [0], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, 64, 1, DEVICE))
    before = [t.clone() for t in pages]
    qkv = torch.randn(3, 4 * 64, device=DEVICE)
    q = torch.zeros(3, 2 * 64, device=DEVICE)
    ops.rope_cache_q4(qkv, q, pages, num_heads=2, num_kv_heads=1, head_dim=64, positions=_int([0, 1, 2]), cos=None, sin=None,
                      style=ops.ROPE_NONE, slots=None)
    assert torch.equal(q, qkv[:, :128]) and all(torch.equal(a, b) for a, b in zip(pages, before))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page_size, kv_heads, d, window, keep_first, skip", [
    (16, 2, 128, 0, 0, False), (16, 1, 64, 20, 3, False), (5, 3, 96, 33, 40, True), (32, 2, 32, 1, 0, False), (16, 2, 256, 50, 17, True)])
def test_rows_are_read_back_where_the_step_sees_them(ops, dtype, page_size, kv_heads, d, window, keep_first, skip):
    counts, history = [1, 30, 0, 5, 1], [90, 61, 10, 0, 0]
    step = Step(counts, history, page_size, seed=3)
    raw = plain.make_pages(step.num_pages, page_size, kv_heads, d, 2, DEVICE)
    raw[1][0, 0, 0, 0] = float("nan")
    pages = ops.Q4Pages(*raw)
    rooms = [torch.full((step.num_pages, page_size, kv_heads, d), 5.5, dtype=dtype, device=DEVICE) for _ in range(2)]
    described = step.device()
    ops.expand_q4(pages, *rooms, window=window, keep_first=keep_first, skip_single=skip,
                  **{name: described[name] for name in ("entry_starts", "entry_pos0", "block_table")})
    seen = np.zeros((step.num_pages, page_size), dtype=bool)
    for e, (count, held) in enumerate(zip(counts, history)):
        if count == 0 or (skip and count == 1):
            continue
        first = max(0, held - window + 1) if window else 0
        for j in range(held + count):
            if j >= first or (window and j < keep_first):
                seen[step.tables[e][j // page_size], j % page_size] = True
    for room, (codes, scales), keys in ((rooms[0], pages[:2], True), (rooms[1], pages[2:], False)):
        rows = np.swapaxes(plain.rows_of(codes, scales, keys), 1, 2)
        expected = np.where(seen[:, :, None, None], rows, 5.5)
        assert np.array_equal(room.double().cpu().numpy(), expected, equal_nan=True)


def _hide(step, pages, window=0, keep_first=0):
    """NaN in every row that no token of the step sees, and tables that name no page where a window has left one behind."""
    seen = np.zeros((step.num_pages, step.page_size), dtype=bool)
    for e, (count, held) in enumerate(zip(step.counts, step.history)):
        for j in range(held + count):
            if not window or j > held - window or j < keep_first:
                seen[step.tables[e][j // step.page_size], j % step.page_size] = True
        for index, page in enumerate(step.tables[e]):
            if page >= 0 and window and not any(index * step.page_size <= j < (index + 1) * step.page_size
                                                for j in range(held + count) if j > held - window or j < keep_first):
                step.tables[e][index] = -1
    hidden = torch.from_numpy(~seen).to(DEVICE)[:, None, :, None]
    for scales in (pages.k_scales, pages.v_scales):
        scales.masked_fill_(hidden, float("nan"))


def _attend(ops, step, dtype, heads, kv_heads, d, seed=0, window=0, keep_first=0, sink=False, sink_values=None, gate=None,
            gate_per_head=False, workspace=None):
    raw = plain.make_pages(step.num_pages, step.page_size, kv_heads, d, seed + 10, DEVICE)
    k_rows, v_rows = plain.rows_of(raw[0], raw[1], True), plain.rows_of(raw[2], raw[3], False)
    k_steps, v_steps = raw[1].double().cpu().numpy(), raw[3].double().cpu().numpy()
    pages = ops.Q4Pages(*raw)
    tables = [list(row) for row in step.tables]
    _hide(step, pages, window, keep_first)
    tokens = len(step.positions)
    generator = torch.Generator().manual_seed(seed)
    q = (torch.randn(tokens, heads * d, generator=generator) * 1.5).to(dtype)
    out = torch.full((tokens + 2, heads * d), 7.0, dtype=dtype, device=DEVICE)
    scale = d ** -0.5
    gates = None if gate is None else torch.from_numpy(np.concatenate([np.full((tokens, 4), 9.0, dtype=np.float32), gate], 1)).to(DEVICE)
    ops.attention_q4(q.to(DEVICE), out[:tokens], pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, scale=scale,
                     workspace=workspace or _workspace(), window=window, keep_first=keep_first, sink=sink,
                     sink_values=None if sink_values is None else torch.from_numpy(sink_values).to(DEVICE),
                     gate=gates, gate_offset=4, gate_per_head=gate_per_head, **step.device())
    expected, parts = plain.attend(q.double().numpy(), k_rows, v_rows, counts=step.counts, history=step.history, tables=tables,
                                   page_size=step.page_size, num_heads=heads, num_kv_heads=kv_heads, d=d, scale=scale, window=window,
                                   keep_first=keep_first, sink=sink, sink_values=sink_values, gate=gate, k_steps=k_steps, v_steps=v_steps)
    got = out[:tokens].double().cpu().numpy().reshape(expected.shape)
    keys = max(c + h for c, h in zip(step.counts, step.history))
    limit = plain.allowed(expected, parts, keys, d, dtype)
    assert np.isfinite(got).all()
    worst = (np.abs(got - expected) / limit).max()
    assert worst <= 1.0, worst
    assert (out[tokens:] == 7.0).all()          # rows behind the step's last token


@pytest.fixture(params=["cluster", "runs"])
def deal(ops, request, monkeypatch):
    """How single tokens' keys are shared: by the blocks of a cluster, or dealt out in even runs as where requests are many."""
    ops.q4_shares.cache_clear()
    monkeypatch.setattr(ops, "Q4_RUNS_UNITS", 0 if request.param == "runs" else 1e9)
    monkeypatch.setattr(ops, "Q4_RUNS_PAIRS", 0)
    yield request.param
    ops.q4_shares.cache_clear()


@pytest.mark.parametrize("heads, kv_heads, d", [(12, 2, 128), (14, 2, 64), (4, 4, 128), (20, 1, 128), (5, 1, 64), (16, 1, 64), (40, 2, 64)])
@pytest.mark.parametrize("history", [[0], [15, 16, 17, 0, 31], [300, 127, 128, 1, 129], [5] * 40 + [1500]])
def test_single_tokens_over_packed_pages(ops, deal, heads, kv_heads, d, history):
    _attend(ops, Step([1] * len(history), history, 16, seed=heads), torch.bfloat16, heads, kv_heads, d)


@pytest.mark.parametrize("page_size", [32, 48, 64])
def test_single_tokens_over_pages_of_other_sizes(ops, deal, page_size):
    _attend(ops, Step([1, 1], [200, 47], page_size), torch.bfloat16, 6, 2, 128)


@pytest.mark.parametrize("window, keep_first", [(1, 0), (16, 0), (100, 4), (40, 37), (1000, 5), (33, 64)])
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_windows_kept_keys_and_sinks(ops, deal, window, keep_first, sink, d):
    _attend(ops, Step([1, 1, 1], [300, 39, 0], 16, seed=window), torch.bfloat16, 8, 2, d, window=window, keep_first=keep_first, sink=sink)


@pytest.fixture(params=["packed", "tensor", "cut", "expanded"])
def form(ops, request, monkeypatch):
    """Which way bfloat16 portions take: the kernel of any number of rows, the tensor cores' with its keys in one piece or in several, or rows
    that are expanded first."""
    if request.param != "packed":
        monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
        assert not ops.attention_q4_takes_rows(torch.bfloat16, 64, 16, 2, 2, 1)
        if request.param == "expanded":
            monkeypatch.setattr(ops, "attention_q4_takes_portions", lambda *sizes: False)
        else:
            assert ops.attention_q4_takes_portions(torch.bfloat16, 64, 16)
            rows, keys = (128, 128) if request.param == "cut" else (256, 1 << 20)
            monkeypatch.setattr(ops, "q4_portion_plan", lambda tokens, heads, kv_heads, d, seen, *rest: (rows, keys, -(-seen // keys)))
    else:
        monkeypatch.setattr(ops, "Q4_ROWS_WORK", 1e12)
        monkeypatch.setattr(ops, "Q4_ROWS_PORTIONS", 1 << 20)
    return request.param


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts, history", [([1, 1], [70, 3]), ([20, 1, 40], [33, 64, 0])])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("keep_first", [0, 4])
def test_learned_sinks_and_gates(ops, form, dtype, counts, history, per_head, keep_first):
    heads, d = 4, 64
    rng = np.random.default_rng(8)
    gate = rng.standard_normal((sum(counts), heads * (1 if per_head else d))).astype(np.float32)
    sinks = rng.standard_normal(heads).astype(np.float32)
    _attend(ops, Step(counts, history, 16), dtype, heads, 2, d, sink=True, sink_values=sinks, gate=gate, gate_per_head=per_head,
            window=50 if keep_first else 0, keep_first=keep_first)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, d, page_size", [(6, 2, 128, 16), (7, 1, 64, 32), (4, 2, 96, 16), (3, 3, 32, 5), (2, 1, 256, 16), (6, 2, 64, 24)])
@pytest.mark.parametrize("counts, history, window", [([50], [0], 0), ([1, 33, 1, 2], [40, 70, 0, 15], 0), ([20, 1], [100, 64], 30)])
def test_portions_and_mixed_steps(ops, form, dtype, heads, kv_heads, d, page_size, counts, history, window):
    _attend(ops, Step(counts, history, page_size, seed=d), dtype, heads, kv_heads, d, window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window, keep_first", [(1, 3), (8, 0), (33, 64), (20, 5), (500, 4), (40, 30)])
@pytest.mark.parametrize("heads, kv_heads, d", [(3, 1, 64), (8, 2, 128)])
def test_portions_with_windows_and_kept_keys(ops, form, dtype, window, keep_first, heads, kv_heads, d):
    """Rows of one block see different keys: the window leaves keys behind in the middle of a portion."""
    _attend(ops, Step([20, 1, 41], [33, 64, 0], 16), dtype, heads, kv_heads, d, window=window, keep_first=keep_first, sink=keep_first == 5)


def test_single_tokens_beside_portions_in_either_deal(ops, deal, monkeypatch):
    """The entries of one token of a mixed step, the others skipped: none of them first, some last, several in a row."""
    monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
    _attend(ops, Step([5, 1, 1, 40, 1, 3, 1], [9, 300, 0, 0, 77, 20, 500], 16), torch.bfloat16, 6, 2, 64)
    _attend(ops, Step([1, 20, 2], [130, 10, 0], 16), torch.bfloat16, 4, 2, 128, window=50, keep_first=7)


def test_many_requests_take_the_even_runs(ops):
    ops.q4_shares.cache_clear()
    assert ops.q4_shares(180, 3000, ops._sm_count_of(0)) == 0
    rng = np.random.default_rng(12)
    _attend(ops, Step([1] * 90, [int(x) for x in rng.integers(0, 300, 89)] + [2999], 16), torch.bfloat16, 4, 2, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_entries_without_tokens_take_no_part(ops, form, dtype):
    _attend(ops, Step([0, 3, 0, 1, 0, 20, 0], [5, 40, 0, 33, 100, 0, 1], 16), dtype, 4, 2, 64)


@pytest.mark.parametrize("counts", [[1, 1], [3, 2]])
def test_a_query_that_is_not_finite_shows_in_its_own_head(ops, deal, counts):
    """NaN and infinities in one head of one token: that head's outputs are NaN, all others those of the same step without."""
    step = Step(counts, [70, 20], 16)
    tokens, heads, d = sum(counts), 6, 64
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 2, d, 3, DEVICE))
    q = torch.randn(tokens, heads * d, device=DEVICE).to(torch.bfloat16)
    outs = []
    for bad in (None, float("nan"), float("inf")):
        x, out = q.clone(), torch.zeros_like(q)
        if bad is not None:
            x[1, 2 * d + 5] = bad
        ops.attention_q4(x, out, pages, num_heads=heads, num_kv_heads=2, head_dim=d, scale=0.125, workspace=_workspace(), **step.device())
        outs.append(out.view(tokens, heads, d))
    for out in outs[1:]:
        assert out[1, 2].isnan().all()
        keep = torch.ones(tokens, heads, dtype=torch.bool, device=DEVICE)
        keep[1, 2] = False
        assert torch.equal(out[keep], outs[0][keep])


def test_queries_of_any_size_keep_their_bits(ops, deal):
    """Queries times a power of two and the scale divided by it: the same outputs, from numbers near the smallest to near the largest."""
    step = Step([1, 1], [90, 17], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, 128, 3, DEVICE))
    q = torch.randn(2, 4 * 128, device=DEVICE).to(torch.bfloat16)
    outs = []
    for up in (0, -80, 80, 20):
        out = torch.zeros_like(q)
        ops.attention_q4(q * 2.0 ** up, out, pages, num_heads=4, num_kv_heads=1, head_dim=128, scale=128 ** -0.5 * 2.0 ** -up,
                         workspace=_workspace(), **step.device())
        outs.append(out)
    assert all(torch.equal(out, outs[0]) for out in outs[1:])


def _off(tensor):
    """The same numbers a place further on: contiguous, and not where rows of 16 bytes begin."""
    room = torch.zeros(tensor.numel() + 1, dtype=tensor.dtype, device=DEVICE)
    room[1:] = tensor.reshape(-1)
    return room[1:].view(tensor.shape)


def test_tensors_that_do_not_begin_on_16_bytes_are_refused(ops):
    """Before a launch: the kernels move pieces of 16 bytes."""
    from vipera_rs_b200.errors import InternalError

    step = Step([1, 1], [20, 3], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, 64, 3, DEVICE))
    q, qkv = torch.zeros(2, 2 * 64, dtype=torch.bfloat16, device=DEVICE), torch.zeros(2, 4 * 64, device=DEVICE)
    rooms = [torch.zeros(step.num_pages, 16, 1, 64, dtype=torch.bfloat16, device=DEVICE) for _ in range(2)]
    described = step.device()
    lengths = {name: described[name] for name in ("entry_starts", "entry_pos0", "block_table")}
    stores = dict(num_heads=2, num_kv_heads=1, head_dim=64, positions=described["positions"], cos=None, sin=None, style=ops.ROPE_NONE,
                  slots=_int(step.slots))
    attends = dict(num_heads=2, num_kv_heads=1, head_dim=64, scale=0.125, workspace=_workspace(), **described)
    off_codes = pages._replace(k_codes=_off(pages.k_codes))
    calls = [lambda: ops.rope_cache_q4(qkv, _off(q), pages, **stores), lambda: ops.rope_cache_q4(qkv, q, off_codes, **stores),
             lambda: ops.expand_q4(pages, _off(rooms[0]), rooms[1], **lengths), lambda: ops.expand_q4(off_codes, *rooms, **lengths),
             lambda: ops.attention_q4(_off(q), q.clone(), pages, **attends), lambda: ops.attention_q4(q, _off(q), pages, **attends),
             lambda: ops.attention_q4(q, q.clone(), off_codes, **attends),
             lambda: ops.attention_q4(q, q.clone(), pages._replace(v_scales=_off(pages.v_scales)), **attends),
             lambda: ops.attention_q4(q.float(), q.float(), off_codes, **attends)]
    for call in calls:
        with pytest.raises(InternalError, match="bad argument"):
            call()
    # a row that begins anywhere is read value by value
    out, far = torch.zeros_like(q), torch.zeros_like(q)
    qkv.normal_()
    ops.rope_cache_q4(qkv, out, pages, **stores)
    ops.rope_cache_q4(_off(qkv), far, pages, **stores)
    assert torch.equal(out, far)


def test_a_long_history_in_many_splits(ops, deal):
    """Thousands of keys, the longest beside a short one, of single tokens and of portions."""
    _attend(ops, Step([1, 1], [9000, 5], 16), torch.bfloat16, 2, 1, 64)
    for dtype in (torch.bfloat16, torch.float32):
        _attend(ops, Step([3, 1], [5000, 5], 16), dtype, 2, 1, 64)


def test_values_that_are_not_finite_show_where_they_are_seen(ops, deal):
    """A NaN key or value makes the outputs of the tokens that see it NaN, and of no others."""
    for which in ("k_scales", "v_scales"):
        step = Step([1, 1, 1], [200, 40, 40], 16)
        pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, 64, 3, DEVICE))
        getattr(pages, which)[step.tables[1][40 // 16], 0, 40 % 16] = float("nan")     # the second's own token
        q = torch.randn(3, 4 * 64, device=DEVICE).to(torch.bfloat16)
        out = torch.zeros_like(q)
        ops.attention_q4(q, out, pages, num_heads=4, num_kv_heads=1, head_dim=64, scale=0.125, workspace=_workspace(), **step.device())
        assert out[1].isnan().all() and out[[0, 2]].isfinite().all()
    # in a portion the tokens in front of a NaN key or value do not see it
    for dtype in (torch.bfloat16, torch.float32):
        for which in ("k_scales", "v_scales"):
            step = Step([6, 3], [40, 8], 16)
            pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, 64, 3, DEVICE))
            getattr(pages, which)[step.tables[0][43 // 16], 0, 43 % 16] = float("nan")     # its fourth token
            q = torch.randn(9, 4 * 64, device=DEVICE).to(dtype)
            out = torch.zeros_like(q)
            ops.attention_q4(q, out, pages, num_heads=4, num_kv_heads=1, head_dim=64, scale=0.125, workspace=_workspace(), **step.device())
            assert out[3:6].isnan().all() and out[[0, 1, 2, 6, 7, 8]].isfinite().all()
    # every key of a whole split is NaN
    step = Step([1], [700], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, 64, 3, DEVICE))
    for index in range(8):
        pages.k_scales[step.tables[0][index]] = float("nan")
    q = torch.randn(1, 4 * 64, device=DEVICE).to(torch.bfloat16)
    out = torch.zeros_like(q)
    ops.attention_q4(q, out, pages, num_heads=4, num_kv_heads=1, head_dim=64, scale=0.125, workspace=_workspace(), **step.device())
    assert out.isnan().all()


def test_scores_of_zero_and_equal_keys_give_the_mean(ops, deal):
    """A query of zeros weighs its keys alike: scores whose maximum is exactly 0."""
    step = Step([1], [99], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 1, 64, 4, DEVICE))
    q = torch.zeros(1, 2 * 64, dtype=torch.bfloat16, device=DEVICE)
    out = torch.zeros_like(q)
    ops.attention_q4(q, out, pages, num_heads=2, num_kv_heads=1, head_dim=64, scale=0.125, workspace=_workspace(), **step.device())
    v = plain.rows_of(pages.v_codes, pages.v_scales, False)[:, 0]
    seen = np.stack([v[step.tables[0][j // 16], j % 16] for j in range(100)])
    got = out.double().cpu().numpy().reshape(2, 64)
    # weights of 1 are exact, times a scale too: the sums in 32 bits (of codes + 136, see plain.allowed) and the output's rounding are left
    steps = np.stack([pages.v_scales.double().cpu().numpy()[step.tables[0][j // 16], 0, j % 16] for j in range(100)])
    limit = (np.abs(seen).mean(0) * 2.0 ** -14 + np.abs(seen.mean(0)) * 2.0 ** -8
             + np.repeat(np.abs(steps).mean(0), 32) * (100 / 64 + 4) * 144 * 2.0 ** -20)
    assert (np.abs(got - seen.mean(0)) <= limit).all()


def test_a_step_as_it_is_used_eager_captured_and_on_a_stream_of_its_own(ops):
    """Maps, write and attention in a row, step after step: captured and replayed they give the eager run's bits, and the cache's
    rows those of the keys and values that went in."""
    heads, kv_heads, d, page = 6, 2, 128, 16
    counts, history = [40, 1, 9], [0, 0, 0]
    rng = np.random.default_rng(6)

    def steps():
        held = [0, 0, 0]
        for number in range(4):
            now = counts if number == 0 else [1, 1, 1]
            yield now, list(held)
            held = [h + c for h, c in zip(held, now)]

    table_pages = rng.permutation(30)
    inputs = [rng.standard_normal((sum(c), (heads + 2 * kv_heads) * d)).astype(np.float32) for c, _ in steps()]
    cos = torch.from_numpy(np.cos(np.arange(64)[:, None] * 0.1 ** np.arange(64)).astype(np.float32)).to(DEVICE)
    sin = torch.from_numpy(np.sin(np.arange(64)[:, None] * 0.1 ** np.arange(64)).astype(np.float32)).to(DEVICE)

    def play(captured):
        pages = ops.Q4Pages(*[t.clone().zero_() for t in plain.make_pages(30, page, kv_heads, d, 0, DEVICE)])
        workspace = _workspace()
        outs = []
        for (now, held), x in zip(steps(), inputs):
            tokens = sum(now)
            need = [-(-(h + c) // page) for h, c in zip(held, now)]
            lists = [table_pages[e * 10:e * 10 + n] for e, n in enumerate(need)]
            starts, pos0 = _int(np.concatenate([[0], np.cumsum(now)])), _int(held)
            page_starts, page_list = _int(np.concatenate([[0], np.cumsum(need)])), _int(np.concatenate(lists))
            table = torch.empty(3, 4, dtype=torch.int32, device=DEVICE)
            maps = {n: torch.empty(tokens, dtype=torch.int32, device=DEVICE) for n in ("positions", "token_entry", "slots")}
            qkv = torch.from_numpy(x).to(DEVICE)
            q, out = (torch.zeros(tokens, heads * d, dtype=torch.bfloat16, device=DEVICE) for _ in range(2))

            def one():
                ops.step_maps(starts, pos0, page_size=page, page_starts=page_starts, pages=page_list, block_table=table, **maps)
                ops.rope_cache_q4(qkv, q, pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, positions=maps["positions"],
                                  cos=cos, sin=sin, style=ops.ROPE_NEOX, slots=maps["slots"])
                ops.attention_q4(q, out, pages, entry_starts=starts, entry_pos0=pos0, positions=maps["positions"],
                                 token_entry=maps["token_entry"], block_table=table, num_heads=heads, num_kv_heads=kv_heads, head_dim=d,
                                 scale=d ** -0.5, max_keys=64, all_single=tokens == 3, any_single=True, workspace=workspace)

            if captured:
                one()
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    one()
                out.zero_()
                graph.replay()
            else:
                one()
            torch.cuda.synchronize()
            outs.append(out.clone())
        return pages, outs

    pages, outs = play(False)
    again, replayed = play(True)
    with torch.cuda.stream(torch.cuda.Stream()):
        elsewhere, streamed = play(False)
    for other in (replayed, streamed):
        assert all(torch.equal(a, b) for a, b in zip(outs, other))
    for other in (again, elsewhere):
        assert all(torch.equal(a, b) for a, b in zip(pages, other))
    # the last step's outputs are attention over what the pages hold
    k_rows, v_rows = plain.rows_of(pages.k_codes, pages.k_scales, True), plain.rows_of(pages.v_codes, pages.v_scales, False)
    held = [42, 3, 11]
    q = _turn(inputs[3].reshape(3, -1, d)[:, :heads], cos.cpu().numpy()[held], sin.cpu().numpy()[held], d, False)
    q = torch.from_numpy(q.reshape(3, -1)).to(torch.bfloat16).double().numpy()
    tables = [list(table_pages[e * 10:e * 10 + 4]) for e in range(3)]
    expected, parts = plain.attend(q, k_rows, v_rows, counts=[1, 1, 1], history=held, tables=tables, page_size=page, num_heads=heads,
                                   num_kv_heads=kv_heads, d=d, scale=d ** -0.5, k_steps=pages.k_scales.double().cpu().numpy(),
                                   v_steps=pages.v_scales.double().cpu().numpy())
    limit = plain.allowed(expected, parts, 64, d, torch.bfloat16)
    assert (np.abs(outs[3].double().cpu().numpy().reshape(expected.shape) - expected) <= limit).all()


def _portions(step, pages, q, ops, heads, kv_heads, d, scale=0.1, **more):
    out = torch.zeros_like(q)
    ops.attention_q4(q, out, pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, scale=scale, workspace=_workspace(), **step.device(), **more)
    return out


@pytest.mark.parametrize("heads, kv_heads, d", [(7, 1, 128), (14, 2, 64), (3, 3, 128), (40, 1, 64)])
@pytest.mark.parametrize("counts, history, window", [([300], [0], 0), ([130, 2, 37], [0, 700, 251], 0), ([200, 64], [120, 1000], 150)])
def test_long_portions_on_the_tensor_cores(ops, form, heads, kv_heads, d, counts, history, window):
    """Several tiles of rows and of keys, tiles that begin inside a token's heads, buffers used again and again."""
    if form == "packed":
        pytest.skip("the kernel of few rows")
    _attend(ops, Step(counts, history, 16, seed=d), torch.bfloat16, heads, kv_heads, d, window=window)


@pytest.mark.parametrize("keep_first", [0, 5])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_not_finite_show_in_the_rows_that_see_them(ops, form, keep_first, d):
    """One group of one value: the group's outputs of the rows whose keys it is among are NaN, all others those of the same step without."""
    heads, kv_heads, key = 6, 2, 141
    step = Step([90, 3], [100, 60], 16)
    window = 30 if keep_first else 0
    raw = plain.make_pages(step.num_pages, 16, kv_heads, d, 3, DEVICE)
    pages = ops.Q4Pages(*raw)
    q = torch.randn(93, heads * d, device=DEVICE).to(torch.bfloat16)
    more = dict(window=window, keep_first=keep_first)
    without = _portions(step, pages, q, ops, heads, kv_heads, d, **more).view(93, heads, d)
    raw[3][step.tables[0][key // 16], 1, key % 16, 1] = float("nan")
    with_one = _portions(step, pages, q, ops, heads, kv_heads, d, **more).view(93, heads, d)
    sees = [i < 90 and key <= 100 + i and (not window or key > 100 + i - window) for i in range(93)]
    assert 0 < sum(sees) < 93
    if form == "expanded":      # rows of one tile of the flash kernel share what they do not see
        assert with_one[sees, 3:, 32:64].isnan().all()
        return
    bad = torch.zeros(93, heads, d, dtype=torch.bool, device=DEVICE)
    bad[sees, 3:, 32:64] = True
    assert with_one[bad].isnan().all()
    assert torch.equal(with_one[~bad], without[~bad])


@pytest.mark.parametrize("d", [64, 128])
def test_steps_near_the_largest_number(ops, form, d):
    """Scales whose multiples leave the type: only their codes' own are asked for."""
    step = Step([40], [30], 16)
    raw = plain.make_pages(step.num_pages, 16, 1, d, 3, DEVICE)
    pages = ops.Q4Pages(*raw)
    q = torch.randn(40, 2 * d, device=DEVICE).to(torch.bfloat16)
    usual = _portions(step, pages, q, ops, 2, 1, d)
    raw[3].mul_(2.0 ** 117)
    huge = _portions(step, pages, q, ops, 2, 1, d)
    assert huge.isfinite().all() and raw[3].abs().max() > 2.0 ** 117
    assert torch.equal(huge.float() * 2.0 ** -117, usual.float())
    raw[3].mul_(2.0 ** -117)
    raw[1].mul_(2.0 ** 117)
    assert raw[1].abs().max() > 2.0 ** 117
    assert torch.equal(_portions(step, pages, q, ops, 2, 1, d, scale=0.1 * 2.0 ** -117), usual)


def test_the_tensor_cores_kernel_in_a_captured_step_on_another_stream(ops, monkeypatch):
    monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
    step = Step([200, 1, 60], [30, 500, 900], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 2, 128, 3, DEVICE))
    q = torch.randn(261, 8 * 128, device=DEVICE).to(torch.bfloat16)
    described, room, out = step.device(), _workspace(), torch.zeros_like(q)
    run = lambda: ops.attention_q4(q, out, pages, num_heads=8, num_kv_heads=2, head_dim=128, scale=0.09, workspace=room, **described)
    run()
    first = out.clone()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        run()
    for scale in (1.0, 0.5):
        q.mul_(scale)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        if scale == 1.0:
            assert torch.equal(out, first)
    run()
    last = out.clone()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, last) and not torch.equal(out, first)
    assert int(ops.kernel_status_word(q.device)[0]) == 0


def test_keys_that_are_not_finite_show_in_the_rows_that_see_them(ops, form):
    heads, d, key = 4, 64, 77
    step = Step([60], [40], 16)
    raw = plain.make_pages(step.num_pages, 16, 2, d, 3, DEVICE)
    pages = ops.Q4Pages(*raw)
    q = torch.randn(60, heads * d, device=DEVICE).to(torch.bfloat16)
    without = _portions(step, pages, q, ops, heads, 2, d).view(60, heads, d)
    raw[1][step.tables[0][key // 16], 1, key % 16, 0] = float("nan")
    with_one = _portions(step, pages, q, ops, heads, 2, d).view(60, heads, d)
    sees = torch.arange(60, device=DEVICE) + 40 >= key
    assert with_one[sees, 2:].isnan().all()
    assert torch.equal(with_one[~sees], without[~sees]) and torch.equal(with_one[:, :2], without[:, :2])


@pytest.mark.parametrize("settled", [False, True])
def test_a_step_that_was_said_to_hold_single_tokens_and_does_not(ops, monkeypatch, settled):
    """The single tokens' kernel finds nothing to do; what follows must still see the portions' outputs."""
    monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
    step = Step([150, 70], [900, 0], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 2, 128, 3, DEVICE))
    q = torch.randn(220, 8 * 128, device=DEVICE).to(torch.bfloat16)
    described = dict(step.device(), any_single=True)
    outs = []
    for said in (False, True):
        out = torch.zeros_like(q)
        ops.attention_q4(q, out, pages, num_heads=8, num_kv_heads=2, head_dim=128, scale=0.09, workspace=_workspace(), settled=settled,
                         **dict(described, any_single=said))
        outs.append(out.clone())
    assert torch.equal(outs[0], outs[1]) and outs[0].abs().amax() > 0


def test_mixed_steps_behind_their_writes_in_a_graph(ops, monkeypatch):
    """Write, portions, single tokens, again and again without a pause: the single tokens' kernel starts while the portions' one runs, and
    finds the step's own rows and queries."""
    monkeypatch.setattr(ops, "Q4_ROWS_WORK", 0)
    heads, kv_heads, d, steps = 8, 2, 128, 6
    step = Step([300, 1, 1, 40, 1], [100, 700, 0, 30, 1500], 16)
    tokens = sum(step.counts)
    monkeypatch.setattr(ops, "q4_portion_plan", lambda *a: (128, 1 << 20, 1))
    described, slots, room = step.device(), _int(step.slots), _workspace()
    qkv = torch.randn(steps, tokens, (heads + 2 * kv_heads) * d, device=DEVICE)
    start = plain.make_pages(step.num_pages, 16, kv_heads, d, 3, DEVICE)

    def run(pause):
        pages = ops.Q4Pages(*[t.clone() for t in start])
        q, outs = (torch.zeros(steps, tokens, heads * d, dtype=torch.bfloat16, device=DEVICE) for _ in range(2))

        def all_steps():
            for i in range(steps):
                ops.rope_cache_q4(qkv[i], q[i], pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, positions=described["positions"],
                                  cos=None, sin=None, style=ops.ROPE_NONE, slots=slots)
                pause()
                ops.attention_q4(q[i], outs[i], pages, num_heads=heads, num_kv_heads=kv_heads, head_dim=d, scale=0.09, workspace=room, **described)
                pause()
        return all_steps, outs

    slow, expected = run(torch.cuda.synchronize)
    slow()
    fast, outs = run(lambda: None)
    fast()
    torch.cuda.synchronize()
    assert torch.equal(outs, expected)
    again, outs = run(lambda: None)
    again()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again()
    for _ in range(3):
        outs.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs, expected)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_behind_the_last_request_stay_as_they_are(ops, form, dtype):
    """A padded step: more rows of q and out than the requests bring."""
    heads, d = 4, 64
    step = Step([30, 2], [200, 0], 16)
    pages = ops.Q4Pages(*plain.make_pages(step.num_pages, 16, 2, d, 3, DEVICE))
    q = torch.randn(40, heads * d, device=DEVICE).to(dtype)
    out = torch.full_like(q, 7.0)
    described = step.device()
    for name in ("positions", "token_entry"):
        described[name] = torch.cat([described[name], torch.zeros(8, dtype=torch.int32, device=DEVICE)])
    run = lambda q, out: ops.attention_q4(q, out, pages, num_heads=heads, num_kv_heads=2, head_dim=d, scale=0.125, workspace=_workspace(), **described)
    run(q, out)
    alone = torch.zeros_like(q[:32])
    run(q[:32].contiguous(), alone)
    assert torch.equal(out[:32], alone)
    assert (out[32:] == 7.0).all()


def test_a_key_that_is_not_finite_and_alone_in_its_cut(ops, form):
    """A window whose first key is the last one of a cut of the keys: its row is NaN, and no other."""
    heads, d, key = 2, 64, 127
    step = Step([40], [110], 16)
    raw = plain.make_pages(step.num_pages, 16, 1, d, 3, DEVICE)
    pages = ops.Q4Pages(*raw)
    q = torch.randn(40, heads * d, device=DEVICE).to(torch.bfloat16)
    without = _portions(step, pages, q, ops, heads, 1, d, window=10)
    raw[1][step.tables[0][key // 16], 0, key % 16, 0] = float("nan")
    with_one = _portions(step, pages, q, ops, heads, 1, d, window=10)
    sees = [key <= 110 + i < key + 10 for i in range(40)]
    assert sees[26] and not sees[27]
    assert with_one[sees].isnan().all()
    assert torch.equal(with_one[[not s for s in sees]], without[[not s for s in sees]])
