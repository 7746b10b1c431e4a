"""Calls of rotary positions and of paged caches at the edges of what they take: operands without heads, gradients that nobody
asked for, frequencies that leave while they are read, batches whose first rows go backwards, broadcast queries, pools that moved.
Tolerances are those of test_rotary_gpu.py and test_paged_gpu.py."""

import pytest
import torch

from attn_engine import RotaryEmbedding
from core.native import lib

pytestmark = pytest.mark.gpu


def draw(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---------------------------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_without_heads_leave_the_keys_their_rotation(packed, dtype):
    """q [.., 0, D] beside k with heads: k turns as it does alone, forward, in place and backward."""
    rope, lead = RotaryEmbedding(64), (7,) if packed else (2, 7)
    q = torch.empty(*lead, 0, 64, dtype=dtype, device="cuda")
    k, g = draw((*lead, 3, 64), dtype, 1).cuda(), draw((*lead, 3, 64), dtype, 2).cuda()
    pos = torch.arange(7, device="cuda") + 500
    want = rope(k, positions=pos)
    a, b = rope(q, k, positions=pos)
    assert a.shape == q.shape and torch.equal(b, want)
    own = k.clone()
    with torch.no_grad():
        a, b = rope(q, own, positions=pos, inplace=True)
    assert b.data_ptr() == own.data_ptr() and torch.equal(own, want)
    leaf, empty = k.clone().requires_grad_(), q.clone().requires_grad_()
    (alone,) = torch.autograd.grad(rope(leaf, positions=pos), leaf, g)
    a, b = rope(empty, leaf, positions=pos)
    dq, dk = torch.autograd.grad((a, b), (empty, leaf), (torch.empty_like(a), g))
    assert dq.shape == q.shape and torch.equal(dk, alone)
    assert lib.last_device_status() == 0
