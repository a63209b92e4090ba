"""The fine-tuning operators on the GPU where ordinary random inputs do not lead: every place of a 16-byte piece, numbers at the ends of
float32's range, recordings that differ between the forward and the backward pass."""
import math

import pytest
import torch

from tests.test_finetune_cpu import U32

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def dev():
    return torch.device('cuda:0')


# ------------------------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('n', [8, 9, 15, 16, 257, 2048, 16384, 16391, 205539])
def test_grad_norm_counts_every_element(dtype, n):
    """one element that is not zero, at every place of the first and last pieces and around the ends of a block's part: its square's root is
    exact; then random values, whose squares are summed in 64 bits (below 1e-10 off) and whose root is rounded once"""
    from mit_semseg import ops
    places = sorted({i for a in (0, n - 16, 8 * 256, 16384) for i in range(a - 8, a + 24) if 0 <= i < n})
    g = torch.zeros(n, device=dev(), dtype=dtype)
    for i in places:
        g[i] = 3.0
        assert float(ops.grad_norm([g])[0]) == 3.0, i
        g[i] = 0.0
    gen = torch.Generator().manual_seed(n)
    g = (1e-3 * torch.randn(n, generator=gen)).to(dev(), dtype)
    for t in (g, torch.cat([g[:1], g])[1:]):                         # aligned, and from an odd address
        want = math.sqrt(float(t.cpu().double().square().sum()))
        assert abs(float(ops.grad_norm([t])[0]) - want) <= (U32 + 1e-10) * want
    more = [g, g[:1], g[: n // 2], g[n // 3:]]
    want = math.sqrt(sum(float(t.cpu().double().square().sum()) for t in more))
    assert abs(float(ops.grad_norm(more)[0]) - want) <= (U32 + 1e-10) * want
