"""What the operators of the 4-bit cache are measured on.

A case is a dict of plain values whose ``kind`` says which operator runs:

``maps``    block tables, positions, entries and cache slots of a step from its requests' lengths and pages (``ops.step_maps``)
``store``   rotation of q and k and the write of k and v into 4-bit pages (``ops.rope_cache_q4``), then the rows that the
            step's tokens see, read back as the numbers that they stand for (``ops.expand_q4``)
``attend``  attention of a step's tokens over 4-bit pages (``ops.attention_q4``)

``counts`` lists the tokens that each request of the step brings and ``history`` how many it has in the cache, as "700,13"
or "64x1" (sixty-four requests of one token).

A row of the cache (one token, one KV head) holds d channels in groups of 32.  A group's scale s is -m / 8 rounded to five
significant bits, m being its value of the largest magnitude (the positive one of two), a code the nearest whole number to
x / s (ties to even) within -8 and 7, and the cache stands for code * s; a group with a value that is not finite has the scale
NaN.  Keys are packed eight channels to a 32-bit word (channel 32 g + 8 t + 2 j + e of the row at bit 4 j + 16 e of word
[t][g]), values four to a 16-bit one (channel 32 g + 4 r + j at bit 4 j of half word [r][g]), a code c as c + 8.
"""
import math

import torch

own = False

DEVICE = "cuda"
PAGE = 16        # the engine's default page size
THETA = 10000.0
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------
def listed():
    shape_1_5b = dict(dtype="bfloat16", heads=12, kv_heads=2, dim=128, page=PAGE)
    shape_7b = dict(dtype="bfloat16", heads=28, kv_heads=4, dim=128, page=PAGE)
    shape_32b = dict(dtype="bfloat16", heads=40, kv_heads=8, dim=128, page=PAGE)
    shape_0_5b = dict(dtype="bfloat16", heads=14, kv_heads=2, dim=64, page=PAGE)
    plain = dict(kind="attend", window=0, keep_first=0, sink=False)
    store = dict(kind="store", rot=128, interleaved=False)
    return [
        # the maps of a full serving batch's decode step
        dict(kind="maps", name="maps_decode_64", page=PAGE, counts="64x1", history="48x2048,15x777,3000"),
        # the maps of a step under the engine's token budget, portions of prompts beside decoding requests of long histories
        dict(kind="maps", name="maps_mixed_8192", page=PAGE, counts="4096,1999,1,2000,97x1", history="0,6,32000,17,97x30000"),
        # a decode step's write, 7B shape
        dict(shape_7b, **store, name="store_decode_64", counts="64x1", history="32x37,31x50,3"),
        # a prompt's write, 7B shape
        dict(shape_7b, **store, name="store_2048", counts="2048", history="0"),
        # portions of odd lengths, heads of 64 of which half turn in neighbouring pairs, queries in 32 bits
        dict(shape_0_5b, kind="store", rot=32, interleaved=True, dtype="float32", name="store_portions_fp32",
             counts="700,1,323", history="0,900,41"),
        # one user's chat: the smallest call, 1.5B shape
        dict(shape_1_5b, **plain, name="attend_decode_1", counts="1", history="2048"),
        # a full serving batch of the 7B shape, histories of every length
        dict(shape_7b, **plain, name="attend_decode_64", counts="64x1", history="32x2048,16x1999,8x4095,7x333,0"),
        # the 32B shape at the benchmark's longest batch: the largest read of the cache
        dict(shape_32b, **plain, name="attend_decode_48_8k", counts="48x1", history="48x8192"),
        # a window with kept first keys and a sink over heads of 64
        dict(shape_0_5b, kind="attend", name="attend_window_32", window=1024, keep_first=4, sink=True, counts="32x1",
             history="16x8000,8x1023,7x5000,2"),
        # a prompt of the benchmark's length
        dict(shape_7b, **plain, name="attend_2048", counts="2048", history="0"),
        # a mixed step: portions behind histories beside requests that decode
        dict(shape_7b, **plain, name="attend_mixed", counts="512,200,16x1,37", history="1000,0,16x2048,2500"),
        # the 32-bit run: requests that decode and a portion
        dict(shape_1_5b, **plain, name="attend_fp32", dtype="float32", counts="8x1,64", history="8x1000,500"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _step(rng, most_tokens, most_history, most_entries):
    """Counts and histories of a step: single tokens, portions, or a few of both."""
    kind = rng.choice(["single", "single", "portions", "mixed"])
    if kind == "mixed":
        most_tokens, most_entries = min(most_tokens, 400), min(most_entries, 8)
    counts, history, left = [], [], most_tokens
    if kind != "single":
        for _ in range(rng.choice([1, 1, 2, 3])):
            count = min(left, _log_int(rng, 2, most_tokens))
            if count < 2:
                break
            counts.append(count)
            history.append(_log_int(rng, 1, most_history) if rng.random() < 0.5 else 0)
            left -= count
    if kind != "portions":
        longest = _log_int(rng, 8, most_history)
        for _ in range(_log_int(rng, 1, most_entries)):
            counts.append(1)
            history.append(longest if rng.random() < 0.5 else rng.randint(0, longest))
    return ",".join(map(str, counts)), ",".join(map(str, history))


def draw(rng):
    kind = rng.choice(["maps", "store", "attend", "attend", "attend"])
    page = rng.choice([16, 16, 16, 32, 64])
    if kind == "maps":
        counts, history = _step(rng, 4000, 30000, 90)
        return dict(kind="maps", page=rng.choice([page, 24]), counts=counts, history=history)
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (16, 4, 64), (8, 8, 128), (40, 8, 128), (20, 1, 128)])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    case = dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    if kind == "store":
        counts, history = _step(rng, 2000, 500, 64)
        return dict(case, rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.25, counts=counts, history=history)
    window = rng.choice([0, 0, 0, 512, 1000])
    case.update(window=window, keep_first=rng.choice([0, 4, 37]) if window else 0, sink=rng.random() < 0.25)
    if dtype == "float32":
        counts, history = _step(rng, 150, 2000, 8)
    else:
        counts, history = _step(rng, 1000, rng.choice([2000, 6000]), 40)
    return dict(case, counts=counts, history=history)


def _list(text):
    out = []
    for item in text.split(","):
        times, _, value = item.rpartition("x")
        out.extend([int(value)] * (int(times) if times else 1))
    return out


def _sizes(case):
    counts, history = _list(case["counts"]), _list(case["history"])
    held = [-(-(c + h) // case["page"]) for c, h in zip(counts, history)]
    return counts, history, held


# ---------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------
def _generator(seed, salt):
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(int(seed) * 1000003 + salt)
    return generator


def _rows(shape, generator):
    """Keys or values as layers project them: channels of different spread, some of them far out."""
    dim = shape[-1]
    spread = torch.randn(dim, generator=generator, device=DEVICE).mul_(0.6).exp_()
    spread[::37] *= 4.0
    return torch.randn(shape, generator=generator, device=DEVICE) * spread


def _step_inputs(case, seed):
    """What the host knows of a step, and the pages that its requests hold: pages of the pool in any order."""
    counts, history, held = _sizes(case)
    int32 = dict(dtype=torch.int32, device=DEVICE)
    pages_in_pool = sum(held) + 5
    order = torch.randperm(pages_in_pool, generator=_generator(seed, 1), device=DEVICE).to(torch.int32)
    starts = torch.tensor([0] + counts, **int32).cumsum(0).to(torch.int32)
    page_starts = torch.tensor([0] + held, **int32).cumsum(0).to(torch.int32)
    return dict(case=case, entry_starts=starts, entry_pos0=torch.tensor(history, **int32), page_starts=page_starts,
                pages=order[: sum(held)].contiguous(), pages_in_pool=pages_in_pool, num_tokens=sum(counts), width=max(held),
                max_keys=max(c + h for c, h in zip(counts, history)), max_count=max(counts))


def _maps(state):
    """The maps of a step in plain torch: (block table, positions, token_entry, slots)."""
    starts, pos0, page_starts = (state[k].long() for k in ("entry_starts", "entry_pos0", "page_starts"))
    page = state["case"]["page"]
    tokens = torch.arange(state["num_tokens"], device=DEVICE)
    entry = torch.searchsorted(starts[1:].contiguous(), tokens, right=True)
    positions = pos0[entry] + tokens - starts[entry]
    places = page_starts[:-1, None] + torch.arange(state["width"], device=DEVICE)
    inside = places < page_starts[1:, None]
    table = torch.where(inside, state["pages"].long()[places.clamp(max=state["pages"].numel() - 1)], -1)
    slots = table[entry, positions // page] * page + positions % page
    return tuple(t.to(torch.int32) for t in (table, positions, entry, slots))


def _round5(x):
    """32-bit numbers to five significant bits, ties to even."""
    bits = x.view(torch.int32)
    return ((bits + 0x3FFFF + ((bits >> 19) & 1)) & -0x80000).view(torch.float32)


def _quantise(x):
    """Codes -8 .. 7 (32-bit numbers [..., groups, 32]) and scales [..., groups] of rows x [..., d]."""
    groups = x.unflatten(-1, (-1, 32))
    high, low = groups.amax(-1), groups.amin(-1)
    scale = _round5(torch.where(high >= -low, high, low) / -8.0)
    scale = torch.where(torch.isfinite(groups).all(-1), scale, torch.nan)
    codes = torch.round(groups / scale.unsqueeze(-1)).clamp(-8, 7)
    return torch.where((scale == 0).logical_or(scale.isnan()).unsqueeze(-1), 0.0, codes), scale


def _pack_keys(codes):
    digits = (codes + 8).to(torch.int64).unflatten(-1, (4, 4, 2))                      # [..., g, t, j, e]
    shifts = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], device=DEVICE)
    words = (digits << shifts).sum((-1, -2)).transpose(-1, -2).flatten(-2)             # [..., t * groups + g]
    return words.to(torch.int32).contiguous().view(torch.uint8)


def _pack_values(codes):
    digits = (codes + 8).to(torch.int32).unflatten(-1, (8, 4))                         # [..., g, r, j]
    units = (digits << torch.tensor([0, 4, 8, 12], device=DEVICE, dtype=torch.int32)).sum(-1).transpose(-1, -2).flatten(-2)
    return units.to(torch.int16).contiguous().view(torch.uint8)


def _unpack_keys(data, groups):
    words = data.contiguous().view(torch.int32).unflatten(-1, (4, groups)).transpose(-1, -2)     # [..., g, t]
    shifts = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], device=DEVICE, dtype=torch.int32)
    return ((words[..., None, None] >> shifts) & 15).flatten(-3).float() - 8


def _unpack_values(data, groups):
    units = data.contiguous().view(torch.int16).to(torch.int32).unflatten(-1, (8, groups)).transpose(-1, -2)   # [..., g, r]
    shifts = torch.tensor([0, 4, 8, 12], device=DEVICE, dtype=torch.int32)
    return ((units[..., None] >> shifts) & 15).flatten(-2).float() - 8


def _stand_for(codes, scales):
    """Rows [..., d] that codes [..., groups, 32] and scales [..., groups] stand for, in 32 bits."""
    return (codes * scales.float().unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    state = _step_inputs(case, seed)
    if case["kind"] == "maps":
        int32 = dict(dtype=torch.int32, device=DEVICE)
        state.update(block_table=torch.empty(state["entry_pos0"].numel(), state["width"], **int32),
                     positions=torch.empty(state["num_tokens"], **int32), token_entry=torch.empty(state["num_tokens"], **int32),
                     slots=torch.empty(state["num_tokens"], **int32))
        return state
    state["block_table"], state["positions"], state["token_entry"], state["slots"] = _maps(state)
    heads, kv_heads, dim, page, tokens = case["heads"], case["kv_heads"], case["dim"], case["page"], state["num_tokens"]
    shape, dtype = (state["pages_in_pool"], kv_heads, page), DTYPES[case["dtype"]]
    for name, pack, salt in (("k", _pack_keys, 2), ("v", _pack_values, 3)):
        generator = _generator(seed, salt)
        codes = torch.empty(*shape, dim // 2, dtype=torch.uint8, device=DEVICE)
        scales = torch.empty(*shape, dim // 32, dtype=torch.bfloat16, device=DEVICE)
        for first in range(0, shape[0], 2048):
            some = slice(first, min(first + 2048, shape[0]))
            digits, scale = _quantise(_rows((some.stop - first, kv_heads, page, dim), generator))
            codes[some], scales[some] = pack(digits), scale.to(torch.bfloat16)
        state[name + "_codes"], state[name + "_scales"] = codes, scales
    generator = _generator(seed, 4)
    if case["kind"] == "store":
        parts = [torch.randn(tokens, heads, dim, generator=generator, device=DEVICE)]
        parts += [_rows((tokens, kv_heads, dim), generator) for _ in range(2)]
        half = case["rot"] // 2
        angles = torch.arange(state["max_keys"], device=DEVICE).double()[:, None] * \
            THETA ** (-torch.arange(half, device=DEVICE).double() / half)
        state.update(qkv=torch.cat([p.flatten(1) for p in parts], 1), cos=angles.cos().float(), sin=angles.sin().float(),
                     q_out=torch.zeros(tokens, heads * dim, dtype=dtype, device=DEVICE))
        for name in ("k_room", "v_room"):
            state[name] = torch.zeros(shape[0], page, kv_heads, dim, dtype=dtype, device=DEVICE)
        return state
    state.update(q=torch.randn(tokens, heads * dim, generator=generator, device=DEVICE).to(dtype),
                 out=torch.zeros(tokens, heads * dim, dtype=dtype, device=DEVICE),
                 sink_values=torch.randn(heads, generator=generator, device=DEVICE) if case["sink"] and not case["keep_first"] else None)
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own_maps(state) if kind == "maps" else _own_store(state) if kind == "store" else _own_attend(state)
    return _maps(state) if kind == "maps" else _store(state) if kind == "store" else _attend(state)


def _own_maps(state):
    from vipera_rs_b200.kernels import ops
    ops.step_maps(state["entry_starts"], state["entry_pos0"], page_size=state["case"]["page"], page_starts=state["page_starts"],
                  pages=state["pages"], block_table=state["block_table"], positions=state["positions"],
                  token_entry=state["token_entry"], slots=state["slots"])
    return state["block_table"], state["positions"], state["token_entry"], state["slots"]


def _own_store(state):
    from vipera_rs_b200.kernels import ops
    case = state["case"]
    pages = ops.Q4Pages(state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"])
    ops.rope_cache_q4(state["qkv"], state["q_out"], pages, num_heads=case["heads"], num_kv_heads=case["kv_heads"],
                      head_dim=case["dim"], rot_dims=case["rot"], positions=state["positions"], cos=state["cos"],
                      sin=state["sin"], style=ops.ROPE_INTERLEAVED if case["interleaved"] else ops.ROPE_NEOX, slots=state["slots"])
    ops.expand_q4(pages, state["k_room"], state["v_room"], entry_starts=state["entry_starts"], entry_pos0=state["entry_pos0"],
                  block_table=state["block_table"])
    return state["q_out"], state["k_room"], state["v_room"]


def _own_attend(state):
    from vipera_rs_b200.kernels import ops
    case = state["case"]
    if "workspace" not in state:
        from vipera_rs_b200.parts.base import Workspace
        state["workspace"] = Workspace(DEVICE)
    pages = ops.Q4Pages(state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"])
    ops.attention_q4(state["q"], state["out"], pages, entry_starts=state["entry_starts"], entry_pos0=state["entry_pos0"],
                     positions=state["positions"], token_entry=state["token_entry"], block_table=state["block_table"],
                     num_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["dim"], scale=case["dim"] ** -0.5,
                     max_keys=state["max_keys"], all_single=state["max_count"] == 1, any_single="1" in _items(case["counts"]),
                     workspace=state["workspace"], window=case["window"], keep_first=case["keep_first"], sink=case["sink"],
                     sink_values=state["sink_values"])
    return state["out"]


def _items(counts):
    return [item.rpartition("x")[2] for item in counts.split(",")]


def _store(state):
    case = state["case"]
    heads, kv_heads, dim, page, rot = case["heads"], case["kv_heads"], case["dim"], case["page"], case["rot"]
    rows = state["qkv"].unflatten(1, (-1, dim))
    turning = rows[:, : heads + kv_heads, :rot]
    if case["interleaved"]:
        a, b = turning[..., 0::2], turning[..., 1::2]
    else:
        a, b = turning[..., : rot // 2], turning[..., rot // 2:]
    positions = state["positions"].long()
    cos, sin = state["cos"][positions, None, :], state["sin"][positions, None, :]
    # every product and every sum is rounded by itself: a key next to a border between two codes falls the same way everywhere
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(turned, -1).flatten(-2) if case["interleaved"] else torch.cat(turned, -1)
    turned = torch.cat([turned, rows[:, : heads + kv_heads, rot:]], -1)
    k, v = turned[:, heads:], rows[:, heads + kv_heads:]
    slots = state["slots"].long()
    at = (slots // page, slice(None), slots % page)
    for name, x, pack in (("k", k, _pack_keys), ("v", v, _pack_values)):
        codes, scale = _quantise(x)
        state[name + "_codes"][at] = pack(codes)
        state[name + "_scales"][at] = scale.to(torch.bfloat16)
    # the rows that the step's tokens see
    place = torch.arange(state["width"] * page, device=DEVICE)
    last = state["entry_pos0"].long() + state["entry_starts"].long().diff()
    held = state["block_table"].long().repeat_interleave(page, 1) * page + place % page
    seen = held[place < last[:, None]]
    at = (seen // page, slice(None), seen % page)
    groups = dim // 32
    for name, unpack in (("k", _unpack_keys), ("v", _unpack_values)):
        values = _stand_for(unpack(state[name + "_codes"][at], groups), state[name + "_scales"][at])
        state[name + "_room"][seen // page, seen % page] = values.to(state[name + "_room"].dtype)
    q = turned[:, :heads].flatten(1)
    state["q_out"].copy_(q)
    return state["q_out"], state["k_room"], state["v_room"]


def _attend(state):
    case = state["case"]
    heads, kv_heads, dim, page, groups = case["heads"], case["kv_heads"], case["dim"], case["page"], case["dim"] // 32
    entries, count, keys = state["entry_pos0"].numel(), state["max_count"], state["width"] * page
    table = state["block_table"].long().clamp(min=0)
    rows = []
    rows.append(_stand_for(_unpack_keys(state["k_codes"][table], groups), state["k_scales"][table]))
    rows.append(_stand_for(_unpack_values(state["v_codes"][table], groups), state["v_scales"][table]))
    k, v = (r.transpose(1, 2).reshape(entries, kv_heads, keys, dim) for r in rows)          # [entry, kv head, key, d]
    starts, pos0 = state["entry_starts"].long(), state["entry_pos0"].long()
    token = starts[:-1, None] + torch.arange(count, device=DEVICE)                          # [entry, place]
    real = token < starts[1:, None]
    position = pos0[:, None] + torch.arange(count, device=DEVICE)
    q = state["q"].float()[torch.where(real, token, 0)].view(entries, count, kv_heads, -1, dim).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(entries, kv_heads, -1, dim) @ k.transpose(-1, -2)).view(entries, kv_heads, -1, count, keys)
    key = torch.arange(keys, device=DEVICE)
    seen = (key <= position[..., None]) & real[..., None]
    if case["window"]:
        seen &= (key > position[..., None] - case["window"]) | (key < case["keep_first"])
    seen = seen[:, None, None]
    scores = torch.where(seen, scores * case["dim"] ** -0.5, -torch.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -torch.inf, 0.0, most)
    weights = (scores - most).exp()
    total = weights.sum(-1, keepdim=True)
    if case["sink"]:
        sinks = torch.zeros(heads, device=DEVICE) if state["sink_values"] is None else state["sink_values"]
        total = total + (sinks.view(1, kv_heads, -1, 1, 1) - most).exp()
    mixed = (weights.reshape(entries, kv_heads, -1, keys) @ v).view(entries, kv_heads, -1, count, dim) / total
    mixed = mixed.permute(0, 3, 1, 2, 4).reshape(entries, count, heads * dim)
    state["out"].copy_(mixed[real])
    return state["out"]


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def _visible(case, position):
    """How many keys the query at `position` sees."""
    window, kept = case.get("window", 0), case.get("keep_first", 0)
    if not window:
        return position + 1
    first = max(0, position + 1 - window)
    return position + 1 - first + min(kept, first)


def work(case):
    counts, history, held = _sizes(case)
    tokens, entries = sum(counts), len(counts)
    if case["kind"] == "maps":
        return {"bytes": 4.0 * (3 * entries + 2 + sum(held) + entries * max(held) + 3 * tokens), "flops": 0.0}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["dtype"] == "float32" else 2
    row = dim / 2 + dim / 16                       # bytes of a key's or a value's codes and scales
    if case["kind"] == "store":
        seen = sum(c + h for c, h in zip(counts, history))
        wrote = tokens * ((heads + 2 * kv_heads) * dim * 4 + case["rot"] * 4 + 8 + heads * dim * size + 2 * kv_heads * row)
        return {"bytes": wrote + seen * 2 * kv_heads * (row + dim * size), "flops": 0.0}
    pairs = sum(_visible(case, h + i) for c, h in zip(counts, history) for i in range(c))
    window, kept = case["window"], case["keep_first"]
    keys = 0
    for c, h in zip(counts, history):
        first = max(0, h + 1 - window) if window else 0
        keys += h + c - first + min(kept, first)
    return {"bytes": keys * 2 * kv_heads * row + 2.0 * tokens * heads * dim * size, "flops": 4.0 * heads * dim * pairs}


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------
def _row_numbers(codes, scales, keys):
    """The numbers in 64 bits of rows of codes [n, d/2] with scales [n, d/32], nibble by nibble."""
    dim = codes.shape[1] * 2
    channel = torch.arange(dim, device=DEVICE)
    group, inside = channel // 32, channel % 32
    if keys:    # word [t][g], bit 4 j + 16 e
        bit = 32 * (inside // 8 * (dim // 32) + group) + 4 * (inside % 8 // 2) + 16 * (inside % 2)
    else:       # half word [r][g], bit 4 j
        bit = 16 * (inside // 4 * (dim // 32) + group) + 4 * (inside % 4)
    digits = (codes[:, bit // 8].long() >> (bit % 8)) & 15
    return (digits.double() - 8) * scales.double()[:, group]


def _exact_codes(x):
    """What rows x [n, d] in 64 bits are held as: the numbers that their codes stand for."""
    groups = x.view(x.shape[0], -1, 32)
    high, low = groups.max(-1).values, groups.min(-1).values
    peak = torch.where(high >= -low, high, low)
    fraction, exponent = torch.frexp(-peak / 8)
    scale = torch.ldexp(torch.round(fraction * 32), exponent - 5).unsqueeze(-1)
    codes = torch.where(scale == 0, 0.0, torch.round(groups / scale)).clamp(-8, 7)
    return (codes * scale).view(x.shape)


def exact(case, seed):
    if case["kind"] == "maps":
        return None
    state = prepare(case, seed)
    counts, history, _ = _sizes(case)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    tables = state["block_table"].tolist()
    if case["kind"] == "store":
        x = state["qkv"].double().view(state["num_tokens"], -1, dim)
        half = case["rot"] // 2
        first = 2 * torch.arange(half, device=DEVICE) if case["interleaved"] else torch.arange(half, device=DEVICE)
        second = first + 1 if case["interleaved"] else first + half
        angle = torch.complex(state["cos"].double(), state["sin"].double())[state["positions"].long()]
        turned = torch.complex(x[:, : heads + kv_heads, first], x[:, : heads + kv_heads, second]) * angle[:, None]
        x[:, : heads + kv_heads, first], x[:, : heads + kv_heads, second] = turned.real, turned.imag
        rooms = []
        for which, name in ((0, "k"), (1, "v")):
            room = torch.zeros_like(state[name + "_room"], dtype=torch.float64)
            new = x[:, heads + which * kv_heads: heads + (which + 1) * kv_heads]
            new = _exact_codes(new.reshape(-1, dim)).view(-1, kv_heads, dim)
            token = 0
            for entry, (count, held) in enumerate(zip(counts, history)):
                for index in range(-(-(held + count) // page)):
                    number = tables[entry][index]
                    old = min(max(held - index * page, 0), page)             # rows of the page from earlier steps
                    end = min(held + count - index * page, page)
                    if old:
                        rows = _row_numbers(state[name + "_codes"][number, :, :old].flatten(0, 1),
                                            state[name + "_scales"][number, :, :old].flatten(0, 1), which == 0)
                        room[number, :old] = rows.view(kv_heads, old, dim).transpose(0, 1)
                    if end > old:
                        at = token + index * page + old - held
                        room[number, old:end] = new[at: at + end - old]
                token += count
            rooms.append(room)
        return x[:, :heads].reshape(state["num_tokens"], heads * dim), rooms[0], rooms[1]
    group = heads // kv_heads
    out = torch.empty(state["num_tokens"], heads, dim, dtype=torch.float64, device=DEVICE)
    token = 0
    for entry, (count, held) in enumerate(zip(counts, history)):
        length = count + held
        numbers = torch.tensor(tables[entry][: -(-length // page)], device=DEVICE)
        position = torch.arange(held, length, device=DEVICE)[:, None]
        key = torch.arange(length, device=DEVICE)[None, :]
        hidden = key > position
        if case["window"]:
            hidden |= (key <= position - case["window"]) & (key >= case["keep_first"])
        for head in range(kv_heads):
            k, v = (_row_numbers(state[n + "_codes"][numbers, head].reshape(-1, dim // 2)[:length],
                                 state[n + "_scales"][numbers, head].reshape(-1, dim // 32)[:length], n == "k") for n in ("k", "v"))
            for h in range(head * group, (head + 1) * group):
                q = state["q"][token: token + count, h * dim: (h + 1) * dim].double()
                s = (q @ k.T / math.sqrt(dim)).masked_fill_(hidden, -math.inf)
                if case["sink"]:
                    sink = 0.0 if state["sink_values"] is None else state["sink_values"][h].double()
                    s = torch.cat([s, torch.zeros(count, 1, dtype=torch.float64, device=DEVICE) + sink], 1)
                out[token: token + count, h] = torch.softmax(s, -1)[:, :length] @ v
        token += count
    return out.view(state["num_tokens"], heads * dim)
