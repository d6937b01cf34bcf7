"""Memory plan of a model from its description: weights, cache, workspace against the device.

The reference plans before it loads (crates/vipera-core/src/planner.rs:224-263 for the sums,
:276-430 for ``feasible`` and ``violations``; bins/vipera/src/main.rs:186-251 prints the plan
and exits with 3 when it is infeasible).  Here the sums are asked of the architecture-neutral
description and of the parts' classes, so that a plan for another architecture needs no change:
weights from the tensor schema, cache bytes from what every scheduled layer says it keeps
between steps, workspace from what every part says it asks for in a step.
"""
from __future__ import annotations

from typing import Dict, Optional

from ..cache.pools import check_kv_type, plan_groups
from ..config.registry import BLOCKS
from ..config.spec import ModelSpec
from ..parts.model import model_schema
from ..weights.loader import FREE_EXTENT

DEVICE_RESERVE_BYTES = 16 << 20  # kept free on the device (crates/vipera-core/src/planner.rs:23)
PLANNED_STEP_TOKENS = 2048       # the step the workspace is sized for
PLANNED_MULTIPROCESSORS = 148    # of the device it runs on
PRODUCT_SCRATCH_BYTES = 32 << 20  # partial sums of split products (the buffer starts at this size)
PRODUCT_PARTS_BYTES = 96 << 20    # the parts of a 32-bit product's left operand, at most (gemm_split.cuh: kMostParts)


def _element_bytes(dtype: str) -> int:
    return 4 if str(dtype).replace("torch.", "") in ("float32", "fp32", "f32") else 2


def spec_cache_requests(spec: ModelSpec) -> Dict[int, object]:
    """What every cache slot of the schedule has to hold, from the description alone."""
    requests = {}
    for entry in spec.schedule:
        if entry.writes_cache:
            layer = spec.layers[entry.layer]
            requests[entry.cache] = BLOCKS.find(layer.block).cache_request_for(layer)
    return requests


def weight_bytes(spec: ModelSpec, element_bytes: int) -> int:
    """Bytes of all tensors of the schema as the engine keeps them: tensors that follow the
    run's type in `element_bytes`, 32-bit tensors and integer tables in 4."""
    total = 0
    for tensor in model_schema(spec).values():
        count = 1
        for extent in tensor.shape:
            count *= FREE_EXTENT if extent is None else int(extent)
        total += count * (element_bytes if tensor.store == "model" else 4)
    return total


def parameter_count(spec: ModelSpec) -> int:
    total = 0
    for tensor in model_schema(spec).values():
        count = 1
        for extent in tensor.shape:
            count *= FREE_EXTENT if extent is None else int(extent)
        total += count
    return total


def _group_tokens(group, ctx: int, page_size: int) -> int:
    """Tokens that a request of `ctx` tokens holds pages for in a group, whole pages of them."""
    tokens = ctx if not group.window else min(ctx, group.window + page_size)
    return -(-tokens // page_size) * page_size


def cache_bytes(spec: ModelSpec, ctx: int, batch: int, element_bytes: int, page_size: int = 16, kv_type: Optional[str] = None) -> int:
    """Pages for `batch` requests of `ctx` tokens in every group of layers (a windowed group
    holds a window and a page's slack per request), and the fixed-size states."""
    groups, states = plan_groups(spec_cache_requests(spec))
    total = 0
    for group in groups:
        total += batch * _group_tokens(group, ctx, page_size) * group.bytes_per_token(element_bytes, kv_type)
    for state in states.values():
        count = 1
        for extent in state.shape:
            count *= int(extent)
        total += batch * count * state.dtype.itemsize
    return total


def kv_bytes_per_token(spec: ModelSpec, element_bytes: int, kv_type: Optional[str] = None) -> int:
    groups, _ = plan_groups(spec_cache_requests(spec))
    return sum(group.bytes_per_token(element_bytes, kv_type) for group in groups)


def part_bytes(heads: int, kv_heads: int, head_dim: int, window: int, keep_first: int, ctx: int, batch: int, element_bytes: int,
               page_size: int) -> int:
    """The parts of a layer's outputs where attention over pages of 4 bits cuts its keys: outputs, maximum and sum of every token and head of a
    planned step, once, or as often as a bfloat16 step of any size up to that is cut (`ops.q4_portion_plan`), and once more for kept first keys; or
    those of the even runs of a batch's single tokens.  (The kernel of any number of rows has 9,472 rows of parts at most, of four blocks of 16 rows
    a multiprocessor, unless a row has one part: no more than the planned step's from five heads on.)"""
    from ..kernels import ops

    kept = 1 if window and keep_first else 0
    places = PLANNED_STEP_TOKENS * (1 + kept)
    most = 0
    if element_bytes == 2 and head_dim in ops.TC_ATTENTION_HEAD_DIMS and page_size % 16 == 0:
        lengths = [ctx] + [2 ** i for i in range(8, 31) if 2 ** i < ctx]
        for tokens in range(64, PLANNED_STEP_TOKENS + 1, 64):
            for keys in lengths:
                cuts = ops.q4_portion_plan(tokens, heads, kv_heads, head_dim, keys, window, PLANNED_MULTIPROCESSORS)[2]
                places = max(places, tokens * (cuts + kept))
        wide = heads // kv_heads > 8
        pairs = batch * kv_heads * -(-(heads // kv_heads) // (16 if wide else 8))
        if not ops.q4_shares(pairs, min(ctx, window + keep_first) if window else ctx, PLANNED_MULTIPROCESSORS, batch <= ops.Q4_RUNS_ENTRIES):
            runs = (2 if wide else ops.Q4_BLOCKS_PER_SM) * PLANNED_MULTIPROCESSORS
            most = runs * 2 * (16 if wide else 8) * (head_dim + 4) * 4
    return max(most, places * heads * (head_dim + 2) * 4)


def room_bytes(spec: ModelSpec, ctx: int, batch: int, element_bytes: int, page_size: int = 16) -> int:
    """What attention over pages of 4 bits needs beside them: the parts of a step's outputs, and, where it does not read them packed (heads
    other than 64 and 128, pages not of a multiple of 16 tokens), a room to expand a layer's rows to: one cache slot's pages in the run's
    type, of the group where they are the largest (layers share the room)."""
    groups, _ = plan_groups(spec_cache_requests(spec))
    room = max([(batch * _group_tokens(group, ctx, page_size) + page_size) * group.bytes_per_token(element_bytes) // len(group.slots)
                for group in groups if group.head_dim not in (64, 128) or page_size % 16] or [0])
    params = [part.params for layer in spec.layers for part in layer.parts.values()]
    attends = {tuple(int(p.get(key) or 0) for key in ("num_heads", "num_kv_heads", "head_dim", "window", "keep_first"))
               for p in params if p.get("num_heads") and p.get("num_kv_heads") and p.get("head_dim")}
    return room + max([part_bytes(*sizes, ctx, batch, element_bytes, page_size) for sizes in attends] or [0])


def workspace_bytes(spec: ModelSpec, batch: int, element_bytes: int, tokens: int = PLANNED_STEP_TOKENS) -> int:
    """The 32-bit residual stream (twice where the embedding's rows are kept beside it), the normalised input, the most any layer asks for (layers
    share their buffers), the products' scratch for partial sums (and, in 32-bit runs, for the parts of
    their left operands), and the 32-bit logits rows of a batch."""
    layers = max(BLOCKS.find(layer.block).workspace_bytes(layer, tokens, element_bytes) for layer in spec.layers)
    stream = 8 if any(entry.adds_embedding for entry in spec.schedule) else 4
    products = PRODUCT_SCRATCH_BYTES + (PRODUCT_PARTS_BYTES if element_bytes == 4 else 0)
    return tokens * spec.hidden_size * (stream + element_bytes) + layers + products + batch * spec.vocab_size * 4


def plan_memory(spec: ModelSpec, ctx: int, batch: int, dtype: str, device_bytes: Optional[int] = None,
                page_size: int = 16, kv_type: Optional[str] = None) -> dict:
    """Weights + cache + workspace against the device's memory; what does not fit is listed in
    ``violations``, and ``feasible`` says whether the list is empty.  ``kv_type`` as the engine's."""
    element = _element_bytes(dtype)
    kv_type = check_kv_type(kv_type, spec_cache_requests(spec))
    weights = weight_bytes(spec, element)
    kv = cache_bytes(spec, ctx, batch, element, page_size, kv_type)
    workspace = workspace_bytes(spec, batch, element)
    if kv_type:
        workspace += room_bytes(spec, ctx, batch, element, page_size)
    if device_bytes is None:
        try:
            import torch

            device_bytes = torch.cuda.get_device_properties(0).total_memory if torch.cuda.is_available() else None
        except Exception:
            device_bytes = None
    if device_bytes is None:
        device_bytes = 180 * 10**9  # one B200
    required = weights + kv + workspace + DEVICE_RESERVE_BYTES
    violations = []
    if ctx > spec.max_position_embeddings:
        violations.append({"constraint": "context_limit", "required": ctx,
                           "available": spec.max_position_embeddings,
                           "message": f"ctx {ctx} exceeds the model's limit of {spec.max_position_embeddings}"})
    if required > device_bytes:
        violations.append({"constraint": "device_memory", "required_bytes": required,
                           "available_bytes": device_bytes,
                           "message": f"{required} bytes needed, {device_bytes} on the device"})
    return {"architecture": spec.architecture, "ctx": ctx, "batch_size": batch, "dtype": dtype,
            "weight_bytes": weights, "kv_bytes": kv, "kv_bytes_per_token": kv_bytes_per_token(spec, element, kv_type),
            "workspace_bytes": workspace, "reserve_bytes": DEVICE_RESERVE_BYTES,
            "predicted_device_bytes": required, "device_bytes": int(device_bytes),
            "feasible": not violations, "violations": violations}
