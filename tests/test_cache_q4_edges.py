"""A cache in 4 bits at its edges, without a device: what launchers refuse before a launch, what plans and flags say."""
import pytest


@pytest.mark.parametrize("dtype, d, off", [("float32", 128, 4), ("float32", 128, 8), ("float32", 64, 4), ("bfloat16", 128, 2), ("bfloat16", 128, 4),
                                           ("bfloat16", 64, 2)])
def test_rows_are_not_stored_to_places_that_do_not_fit_their_pieces(dtype, d, off):
    """The launcher of the kernel of any number of rows looks at `out` before it launches anything (every address here is made up)."""
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.kernels import ops

    fn = ops._function("attention_q4", "vipera_attention_q4_rows", ops._ROWS_Q4_ARGS)
    at = 1 << 20
    block = ops._pack_rows_q4(at, at, at, at, at, at, at, at, 0, 0, 2, 16, 4, 1, 3, 4, 2, 0.125, 0, 0, 64, 1)
    code = ops.F32 if dtype == "float32" else ops.BF16
    call = lambda out, scratch: fn(block, out, code, d, at, 0, None, None, 0, 0, scratch, 1 << 20, None)
    assert call(at + off, at) == -3
    assert call(at, at + 4) == -3        # as a scratch that does not fit
    assert fn(block, at, 7, d, at, 0, None, None, 0, 0, at, 1 << 20, None) == -1      # no such type


@pytest.mark.parametrize("kernel", ["tensor", "mma"])
def test_the_flash_kernels_behind_an_expansion_refuse_rows_off_their_pieces(kernel):
    """Pages that no kernel reads packed are expanded for the flash kernels, which move a row's 16 bytes at once."""
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.kernels import ops

    kinds = [ops._c_void] * 7 + [ops._c_int] * 7 + [ops._c_float, ops._c_int]
    at = 1 << 20

    def call(q, out):
        places, sizes = (q, out, at, at, at, at, at), (2, 24, 1, 3, 4, 2, 64, 0.125, 0)
        if kernel == "tensor":
            fn = ops._function("attention_tc", "vipera_attention_prefill_tc", kinds + [ops._c_int, ops._c_int, ops._c_void, ops._c_void])
            return fn(*places, *sizes, 4, 0, at, None)
        return ops._function("attention_mma", "vipera_attention_prefill", kinds + [ops._c_int, ops._c_void])(*places, *sizes, 0, None)

    assert call(at + 2, at) == -3 and call(at + 8, at) == -3 and call(at, at + 2) == -3
    if kernel == "tensor":
        assert call(at, at + 8) == -3


def test_single_tokens_beside_portions_are_refused_without_their_word():
    """A launch that may begin while the portions run needs the word that says what is complete."""
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.kernels import ops

    fn = ops._function("attention_q4", "vipera_attention_q4_decode", ops._DECODE_Q4_ARGS)
    at = 1 << 20
    for settled, beside in ((2, 0), (3, at), (-1, at)):
        block = ops._pack_decode_q4(at, at, at, at, at, at, at, at, at, 0, 0, 0, 0, 2, 16, 0, 4, 1, 4, 2, 64, 0.125, 0, 0, 0, 1, settled, beside, 0)
        assert fn(block, None, 0, 0, None) == -3


def test_the_command_line_plans_no_other_cache_than_the_one_it_was_asked_for(tmp_path, capsys):
    import json

    import helpers
    from vipera_rs_b200 import cli

    (tmp_path / "config.json").write_text(json.dumps(helpers.CONFIGS["A"]))
    command = ["plan", str(tmp_path), "--ctx", "64", "--json"]
    assert cli.main(command) == 0
    usual = capsys.readouterr().out
    for name in ("bf16", "bfloat16", "f32", "float32"):       # names of the run's type, as for generate
        assert cli.main([*command, "--kv-type", name]) == 0
        assert capsys.readouterr().out == usual
    for name in ("q5", "Q4", "q8_0", ""):
        assert cli.main([*command, "--kv-type", name]) == 2
        told = capsys.readouterr()
        assert told.out == "" and "--kv-type" in told.err


@pytest.mark.parametrize("heads, kv_heads, head_dim, window, keep_first", [(8, 8, 128, 0, 0), (12, 2, 128, 0, 0), (28, 4, 128, 0, 0), (14, 2, 64, 0, 0),
                                                                         (28, 4, 128, 5000, 4)])
@pytest.mark.parametrize("ctx", [256, 8192, 32000])
def test_the_plan_counts_the_parts_that_a_step_asks_for(heads, kv_heads, head_dim, window, keep_first, ctx):
    """Buffers of parts as the launches size them, for steps of any length up to the planned one, stay within the plan."""
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.engine import planner
    from vipera_rs_b200.kernels import ops

    kept = 1 if keep_first else 0
    for batch in (1, 64):
        planned = planner.part_bytes(heads, kv_heads, head_dim, window, keep_first, ctx, batch, 2, 16)
        asked = [0]
        for tokens in (64, 128, 512, 1024, 1536, 2048):
            for keys in {ctx, ctx * 3 // 4, 2048}:
                if tokens <= keys <= ctx:
                    cuts = ops.q4_portion_plan(tokens, heads, kv_heads, head_dim, keys, window, 148)[2] + kept
                    asked.append(ops.attention_decode_scratch_floats(tokens, heads, head_dim, cuts) if cuts > 1 else 0)
                    splits = ops.q4_rows_splits(kv_heads * -(-tokens * (heads // kv_heads) // 16), keys, 148)[1] + kept
                    asked.append(ops.attention_decode_scratch_floats(tokens, heads, head_dim, splits))
        assert 4 * max(asked) <= planned + 16
    if ctx == 8192 and not window:
        assert planner.part_bytes(8, 8, 128, 0, 0, ctx, 1, 2, 16) >= 3 * 2048 * 8 * 130 * 4


def test_the_plan_of_a_model_holds_its_layers_parts():
    import helpers
    from vipera_rs_b200.config import architecture_of
    from vipera_rs_b200.engine import planner

    raw = dict(helpers.CONFIGS["A"], hidden_size=1536, num_attention_heads=12, num_key_value_heads=2, max_position_embeddings=32768)
    arch = architecture_of(raw)
    spec = arch.model_spec(arch.config_from_dict(raw))
    assert planner.room_bytes(spec, 8192, 1, 2) == planner.part_bytes(12, 2, 128, 0, 0, 8192, 1, 2, 16) >= 2 * 2048 * 12 * 130 * 4


def test_what_a_step_builds_on_the_device_shares_no_line_with_what_it_builds_it_from():
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200.engine.runner import step_offsets

    for copied in ([3, 2, 1, 1, 1, 0, 2, 5], [32], [31, 1], [100, 4, 29]):
        offsets, places = step_offsets(copied, [3, 3, 8, 0])
        assert offsets == [sum(copied[:i]) for i in range(len(copied) + 1)]
        assert places[0] % 32 == 0 and offsets[-1] <= places[0] < offsets[-1] + 32
        assert [b - a for a, b in zip(places, places[1:])] == [3, 3, 8, 0]


def test_a_steps_pieces_are_written_one_behind_the_other_for_the_device():
    import numpy as np

    from vipera_rs_b200.build import runtime_module
    from vipera_rs_b200.errors import InvalidArgumentError

    manager = runtime_module().CacheManager([(16, 20, 0, 0), (8, 40, 32, 0)], 4, False)
    for request, length in ((0, 40), (1, 5), (2, 80)):
        manager.open(request)
        manager.reserve(request, length)
    manager.commit(2, 72)                    # the window's group gives pages back
    requests, counts, pos0, fresh = [2, 0, 1], [8, 1, 5], [72, 39, 0], [0, 0, 1]
    tokens, rows = np.arange(100, 114, dtype=np.int32), np.asarray([7, 13], dtype=np.int32)
    lists = [manager.page_lists(requests, g) for g in (0, 1)]
    expected = [tokens, [0, 8, 9, 14], pos0, [manager.state_slot(r) for r in requests], fresh, rows] + [p for pair in lists for p in pair]
    buffer = np.full(300, 77, dtype=np.int32)
    sizes, longest = manager.fill_step(requests, tokens, counts, pos0, fresh, rows, buffer.ctypes.data, buffer.size)
    assert sizes == [len(piece) for piece in expected] and longest == [5, 10]
    assert buffer[:sum(sizes)].tolist() == [int(x) for piece in expected for x in piece]
    assert (buffer[sum(sizes):] == 77).all()
    # a buffer that is too small stays as it was, and the sizes are told all the same
    small = np.full(sum(sizes) - 1, 77, dtype=np.int32)
    assert manager.fill_step(requests, tokens, counts, pos0, fresh, rows, small.ctypes.data, small.size) == (sizes, longest)
    assert (small == 77).all()
    for change in (dict(pos0=[72, 60, 0]), dict(pos0=[0, 39, 0], counts=[8, 1, 20])):      # no page for a last position
        given = dict(dict(counts=counts, pos0=pos0), **change)
        with pytest.raises(InvalidArgumentError):
            manager.fill_step(requests, tokens, given["counts"], given["pos0"], fresh, rows, buffer.ctypes.data, buffer.size)
    with pytest.raises(InvalidArgumentError):
        manager.fill_step(requests, tokens, counts[:2], pos0, fresh, rows, buffer.ctypes.data, buffer.size)


def test_a_mixer_finds_the_view_of_packed_pages_beside_the_other_one():
    import vipera_rs_b200  # noqa: F401
    from vipera_rs_b200 import parts

    for name in ("PagedKV", "PagedKVView", "PagedQ4View"):
        assert name in parts.__all__ and hasattr(parts, name)
