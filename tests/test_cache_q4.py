"""A cache in 4 bits, without a device: the format, what its entry points refuse, what the memory plan counts."""
import numpy as np
import pytest
import torch

import plain_q4 as plain


def test_a_group_keeps_its_largest_value_to_a_64th_and_the_others_to_half_a_step():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((50, 128)) * np.exp(rng.standard_normal((50, 1)) * 3)).astype(np.float32)
    codes, scales = plain.quantise(x)
    back = plain.stand_for(codes, scales).reshape(50, 4, 32)
    groups = x.reshape(50, 4, 32).astype(np.float64)
    largest = np.abs(groups).max(-1, keepdims=True)
    step = np.abs(scales)[..., None]
    # the largest value lies on code -8 but for the scale's rounding, half of 1/16 of it at most; what passes +7 steps is cut there
    assert (np.abs(back - groups) <= np.where(np.abs(groups) == largest, largest / 32, np.maximum(step / 2, np.abs(groups) - 7 * step) + 1e-12)).all()
    assert codes.min() == -8 and codes.max() <= 7


def test_what_a_row_stands_for_is_a_bfloat16_exactly():
    rng = np.random.default_rng(4)
    values = plain.stand_for(*plain.quantise((rng.standard_normal((200, 256)) * 7).astype(np.float32)))
    assert np.array_equal(torch.from_numpy(values).to(torch.bfloat16).double().numpy(), values)


@pytest.mark.parametrize("keys", [True, False])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_packing_and_unpacking_agree_and_use_every_nibble_once(keys, d):
    codes = np.random.default_rng(5).integers(-8, 8, size=(3, 7, d // 32, 32))
    packed = plain.pack(codes, keys)
    assert packed.shape == (3, 7, d // 2)
    assert np.array_equal(plain.unpack(packed, keys), codes)


def _pages(ops, pages=3, page_size=16, kv_heads=2, d=64):
    u8 = dict(dtype=torch.uint8)
    return ops.Q4Pages(torch.zeros(pages, kv_heads, page_size, d // 2, **u8),
                       torch.zeros(pages, kv_heads, page_size, d // 32, dtype=torch.bfloat16),
                       torch.zeros(pages, kv_heads, page_size, d // 2, **u8),
                       torch.zeros(pages, kv_heads, page_size, d // 32, dtype=torch.bfloat16))


@pytest.fixture
def entry_points(monkeypatch):
    """The wrappers with the kernels' libraries out of reach: what they refuse, they refuse before a launch."""
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.kernels import ops

    def no_launch(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(ops, "_function", lambda *_: no_launch)
    monkeypatch.setattr(ops, "_check_struct", lambda *_: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return ops


def _int(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_step_maps_refuses_lengths_that_do_not_agree(entry_points):
    from vipera_rs_b200.errors import InvalidArgumentError

    ops = entry_points
    table = torch.zeros(2, 4, dtype=torch.int32)
    good = dict(page_size=16, block_table=table, page_starts=_int(0, 1, 2), pages=_int(0, 1), slots=torch.zeros(5, dtype=torch.int32))
    starts, pos0 = _int(0, 2, 5), _int(0, 9)
    for change in (dict(page_size=0), dict(block_table=table[:1]), dict(page_starts=None), dict(pages=None),
                   dict(page_starts=_int(0, 1)), dict(positions=torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(InvalidArgumentError):
            ops.step_maps(starts, pos0, **{**good, **change})
    with pytest.raises(InvalidArgumentError):
        ops.step_maps(_int(0, 2), pos0, **good)


def test_rope_cache_q4_refuses_shapes_and_sizes_it_does_not_take(entry_points):
    from vipera_rs_b200.errors import InvalidArgumentError, UnsupportedError

    ops = entry_points
    good = dict(num_heads=4, num_kv_heads=2, head_dim=64, positions=_int(0, 1, 2), cos=torch.zeros(8, 32), sin=torch.zeros(8, 32),
                style=ops.ROPE_NEOX, slots=_int(0, 1, 2))
    qkv, q = torch.zeros(3, 8 * 64), torch.zeros(3, 4 * 64)
    for change in (dict(positions=_int(0)), dict(slots=_int(0)), dict(rot_dims=33), dict(rot_dims=66), dict(cos=None),
                   dict(cos=torch.zeros(8, 16)), dict(num_kv_heads=3), dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32))):
        with pytest.raises(InvalidArgumentError):
            ops.rope_cache_q4(qkv, q, _pages(ops), **{**good, **change})
    for bad_qkv, bad_q in ((qkv[:, :-1], q), (qkv.t(), q), (qkv, q[:2]), (qkv.double(), q), (qkv, q)):   # the last: on another device
        with pytest.raises(InvalidArgumentError):
            ops.rope_cache_q4(bad_qkv, bad_q, _pages(ops), **good)
    with pytest.raises(UnsupportedError):
        ops.rope_cache_q4(torch.zeros(3, 8 * 48), torch.zeros(3, 4 * 48), _pages(ops), **{**good, "head_dim": 48})
    huge = ops.Q4Pages(*[t[:1].expand(2 ** 27, *t.shape[1:]) for t in _pages(ops)])      # 2^31 slots
    with pytest.raises(UnsupportedError):
        ops.rope_cache_q4(qkv, q, huge, **good)
    bad = _pages(ops)._replace(v_scales=torch.zeros(3, 2, 16, 4, dtype=torch.bfloat16))
    with pytest.raises(InvalidArgumentError):
        ops.rope_cache_q4(qkv, q, bad, **good)


def test_tensors_elsewhere_of_another_type_or_in_pieces_are_refused(entry_points):
    from vipera_rs_b200.errors import InternalError, InvalidArgumentError

    ops = entry_points
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(InternalError):            # on the host
        ops.step_maps(_int(0, 1), _int(0), page_size=16, block_table=table)
    with pytest.raises(InvalidArgumentError):     # 64-bit lengths
        ops.step_maps(_int(0, 1).long(), _int(0), page_size=16, block_table=table)
    with pytest.raises(InvalidArgumentError):     # every second number of a tensor
        ops.step_maps(torch.zeros(4, dtype=torch.int32)[::2], _int(0), page_size=16, block_table=table)


def test_expand_q4_refuses_rooms_of_another_cache(entry_points):
    from vipera_rs_b200.errors import InvalidArgumentError

    ops = entry_points
    room = torch.zeros(3, 16, 2, 64)
    good = dict(entry_starts=_int(0, 1), entry_pos0=_int(4), block_table=torch.zeros(1, 2, dtype=torch.int32))
    for k, v in ((room, room[:2]), (room, room.double()), (room[:2], room[:2]), (room[:, :8], room[:, :8])):
        with pytest.raises(InvalidArgumentError):
            ops.expand_q4(_pages(ops), k, v, **good)
    with pytest.raises(InvalidArgumentError):
        ops.expand_q4(_pages(ops), room, room, **{**good, "entry_starts": _int(0)})


def test_attention_q4_refuses_steps_that_do_not_agree(entry_points):
    from vipera_rs_b200.errors import InvalidArgumentError

    ops = entry_points
    q = torch.zeros(3, 4 * 64, dtype=torch.bfloat16)
    good = dict(entry_starts=_int(0, 1, 3), entry_pos0=_int(5, 0), positions=_int(5, 0, 1), token_entry=_int(0, 1, 1),
                block_table=torch.zeros(2, 2, dtype=torch.int32), num_heads=4, num_kv_heads=2, head_dim=64, scale=0.125, max_keys=6,
                all_single=False, any_single=True, workspace=None)
    for change in (dict(num_heads=3), dict(entry_starts=_int(0, 3)), dict(all_single=True), dict(positions=_int(5)),
                   dict(max_keys=0), dict(max_keys=33), dict(window=-1), dict(sink_values=torch.zeros(3)), dict(keep_first=-2),
                   dict(block_table=torch.zeros(1, 2, dtype=torch.int32))):
        with pytest.raises(InvalidArgumentError):
            ops.attention_q4(q, torch.zeros_like(q), _pages(ops), **{**good, **change})
    with pytest.raises(InvalidArgumentError):
        ops.attention_q4(q, torch.zeros(3, 4 * 64), _pages(ops), **good)


def _spec(raw):
    from vipera_rs_b200.config import architecture_of

    arch = architecture_of(raw)
    return arch.model_spec(arch.config_from_dict(raw))


def test_the_memory_plan_counts_packed_pages_and_one_slots_room():
    import helpers
    from vipera_rs_b200.engine import planner

    for name in ("A", "B"):
        spec = _spec(helpers.CONFIGS[name])
        run = planner.plan_memory(spec, 256, 3, "bfloat16", device_bytes=10**9)
        packed = planner.plan_memory(spec, 256, 3, "bfloat16", device_bytes=10**9, kv_type="q4")
        assert packed["kv_bytes"] * 32 == run["kv_bytes"] * 9 and packed["kv_bytes_per_token"] * 32 == run["kv_bytes_per_token"] * 9
        room = packed["workspace_bytes"] - run["workspace_bytes"]
        assert room == planner.room_bytes(spec, 256, 3, 2) > 0
    # (outputs, maximum, sum) of every token and head of a step; A's heads of 64 are read packed
    spec, parts = _spec(helpers.CONFIGS["A"]), planner.PLANNED_STEP_TOKENS * 4 * (64 + 2) * 4
    assert planner.room_bytes(spec, 256, 3, 2) == planner.room_bytes(spec, 256, 3, 4) == parts
    # in pages that the kernels do not read, one layer's of the two alike, and one page more
    assert planner.room_bytes(spec, 256, 3, 2, page_size=8) == planner.cache_bytes(spec, 256, 3, 2) // 2 + 8 * 2 * 2 * 64 * 2 + parts


def test_models_whose_mixers_need_the_runs_type_refuse_4_bits():
    import helpers
    from nobupel_cases import MIXED
    from vipera_rs_b200.engine import planner
    from vipera_rs_b200.errors import InvalidArgumentError, UnsupportedError

    for raw in (helpers.CONFIGS["C"], MIXED):    # heads of 48; values of another size than keys
        with pytest.raises(UnsupportedError):
            planner.plan_memory(_spec(raw), 64, 1, "bfloat16", device_bytes=10**9, kv_type="q4")
    with pytest.raises(InvalidArgumentError):
        planner.plan_memory(_spec(helpers.CONFIGS["A"]), 64, 1, "bfloat16", device_bytes=10**9, kv_type="q5")


@pytest.mark.parametrize("option", [dict(chunk=16), dict(values_from_keys=True), dict(row_norm=True, norm_eps=1e-6), dict(talking_heads=True),
                                    dict(out_scale=0.5), dict(value_mix="source"), dict(head_norm=True, norm_eps=1e-6), dict(value_dim=32),
                                    dict(head_dim=48)])
def test_attention_says_which_options_packed_pages_serve(option):
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.parts.attention import GQAttention

    plain_params = dict(hidden_size=256, num_heads=4, num_kv_heads=2, head_dim=64, window=None)
    assert GQAttention.cache_request_for(plain_params).four_bit
    assert GQAttention.cache_request_for(dict(plain_params, window=40, keep_first=3, sink="learned", output_gate=True)).four_bit
    assert not GQAttention.cache_request_for(dict(plain_params, **option)).four_bit


def test_keys_are_shared_by_a_clusters_blocks_and_cut_into_whole_walks():
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.kernels import ops

    for tiles in (1, 3, 8, 64, 300, 12000):
        for keys in (1, 128, 129, 2049, 40000, 10**6):
            shares = ops.q4_shares(tiles, keys, 148)
            assert (shares == 0) == (tiles >= 16 and tiles * -(-keys // 128) >= 8 * 444)      # in even runs where there is much to read
            assert shares in (0, 1, 2, 4, 8, 16) and (shares < 2 or keys > 64 * shares)    # no more than there are walks for, but for one
            chunk, splits = ops.q4_rows_splits(tiles, keys, 148)
            assert chunk % 64 == 0 and 0 < splits <= 64 and chunk * (splits - 1) < keys <= chunk * splits


def test_page_lists_are_the_requests_pages_one_behind_the_other():
    from vipera_rs_b200.build import runtime_module

    manager = runtime_module().CacheManager([(16, 20, 0, 0), (16, 20, 32, 0)], 4, False)
    for request, length in ((0, 40), (1, 5), (2, 80)):
        manager.open(request)
        manager.reserve(request, length)
    manager.commit(2, 80)                    # the window's group gives pages back
    for group in (0, 1):
        starts, pages = manager.page_lists([2, 0, 1], group)
        table = manager.tables([2, 0, 1], group, 8)
        assert starts.tolist()[0] == 0 and starts.tolist()[-1] == len(pages)
        for row, (first, last) in enumerate(zip(starts[:-1], starts[1:])):
            assert table[row].tolist() == pages[first:last].tolist() + [-1] * (8 - (last - first))


def test_the_command_line_plans_packed_pages(tmp_path, capsys):
    import json

    import helpers
    from nobupel_cases import MIXED
    from vipera_rs_b200 import cli

    for raw, code in ((helpers.CONFIGS["A"], 0), (MIXED, 2)):
        (tmp_path / "config.json").write_text(json.dumps(raw))
        plans = []
        for flags in ([], ["--kv-type", "q4"]):
            assert cli.main(["plan", str(tmp_path), "--ctx", "64", "--batch", "2", "--json", *flags]) == (code if flags else 0)
            plans.append(capsys.readouterr())
        if code:
            assert plans[1].err.startswith("vipera: unsupported:")
        else:
            run, packed = (json.loads(p.out) for p in plans)
            assert packed["kv_bytes"] * 32 == run["kv_bytes"] * 9


def test_how_the_tensor_cores_kernel_is_cut(entry_points):
    """Whole cuts of 128 keys that cover what is seen, few enough for their places, one where a window leaves little of a history."""
    ops = entry_points
    rng = np.random.default_rng(3)
    for _ in range(300):
        d, kv_heads, group = int(rng.choice([64, 128])), int(rng.integers(1, 9)), int(rng.integers(1, 17))
        tokens = int(2 ** rng.uniform(0, 13))
        seen = tokens + int(2 ** rng.uniform(0, 17))
        window = int(rng.choice([0, 0, 500]))
        rows, keys, cuts = ops.q4_portion_plan(tokens, kv_heads * group, kv_heads, d, seen, window, 148)
        assert rows in (128, 256) and keys % 128 == 0 and 1 <= cuts <= 127 and (cuts - 1) * keys < seen <= cuts * keys
        assert cuts == 1 or keys >= 256
        if window and 2 * (window + tokens) < seen:
            assert cuts == 1
    # blocks enough for the device: two tiles of rows each, in one piece; few rows behind a long history: in many
    assert ops.q4_portion_plan(2048, 28, 4, 128, 2048, 0, 148) == (256, 2048, 1)
    assert ops.q4_portion_plan(8, 28, 4, 128, 20008, 0, 148)[2] >= 8
    assert not ops.attention_q4_takes_portions(torch.float32, 128, 16) and not ops.attention_q4_takes_portions(torch.bfloat16, 96, 16)
    assert not ops.attention_q4_takes_portions(torch.bfloat16, 128, 24)
    assert ops.attention_q4_takes_rows(torch.float32, 128, 16, 10 ** 6, 10 ** 6, 50) and not ops.attention_q4_takes_rows(torch.float32, 96, 16, 1, 1, 1)
    assert ops.attention_q4_takes_rows(torch.bfloat16, 128, 16, 60, 500, 1) and not ops.attention_q4_takes_rows(torch.bfloat16, 128, 16, 60, 500, 3)
