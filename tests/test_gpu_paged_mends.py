"""The paged KV cache on the GPU, where calls are joined, captured or laid out in ways of their own; tolerances as in
test_gpu_paged.py unless a test derives its own."""
import math

import pytest
import torch

import test_gpu_paged as P

pytestmark = pytest.mark.gpu


# ---- weights -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", P.TYPES)
@pytest.mark.parametrize("slots", [200, 900, 4000])  # one piece; joined by the last workgroup; by a second launch
@pytest.mark.parametrize("bad", ["", "query", "key"])
def test_weights_of_holes(hip, dtype, slots, bad):
    """A hole's weights keep every bit: -0 stays -0, and a head whose query or key is NaN leaves its NaN at the slots it attends to."""
    cache, table, n = P.make([slots, slots - 7], 2, 64, 64, dtype)
    q = P.queries([0] * 2, 8, 64)
    if bad == "query":
        q[0, 0, 1, 3] = math.nan
    if bad == "key":
        cache[0, table[0, 0].long(), 0, 5, 9] = math.nan
    table[0, 1], table[1, 2] = -1, cache.shape[1]
    start = torch.full((2, 2, table.shape[1] * 64 + 4), -0.0)
    start[0, 0, 100] = 7.0
    w = start.cuda()
    hip.paged_attention(q.cuda(), cache.cuda(), table.cuda(), n.cuda(), weights=w)
    w = w.cpu()
    t = torch.arange(start.shape[2])
    for b in range(2):
        there = (t < n[b]) & (t // 64 != 1 + b)
        assert torch.equal(w[b, :, ~there].view(torch.int32), start[b, :, ~there].view(torch.int32)), b
        for h in range(2):
            nan = bad and b == 0 and h == 0
            assert w[b, h, there].isnan().all() if nan else (w[b, h, there] > 0).all()
