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
