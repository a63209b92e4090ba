"""The fine-tuning operators on the GPU where ordinary random inputs do not lead: every place of a 16-byte piece, numbers at the ends of
float32's range, recordings that differ between the forward and the backward pass."""
import math

import pytest
import torch

from tests.test_finetune_cpu import U32, check_codes, decoded, mix, reference_step

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


# ----------------------------------------------------------------------------------------------------- AdamW, states in 8 bits
def placed(t, odd):
    """on the GPU; `odd`: one element behind an aligned address"""
    t = t.to(dev())
    return torch.cat([t[:1], t])[1:] if odd else t


def state_of(n, odd):
    from mit_semseg import ops
    return ops.AdamW8State(*(placed(torch.zeros(k, dtype=d), odd and d == torch.uint8) for k, d in
                             ((n, torch.uint8), (-(-n // 256), torch.float32)) * 2))


@pytest.mark.parametrize('odd', [False, True])
@pytest.mark.parametrize('eps', [0.0, 1e-30, 1e-20])
def test_adamw8_small_second_moments(eps, odd):
    """gradients whose squares are denormal numbers (below 1.2e-38, down to 1e-42 here), three steps each from the states the one before
    left: parameters and root against float64.  Beside the roundings that check_step8 counts, the three products and the sum of v are
    each rounded to a multiple of 2^-149: dv <= 4 * 2^-150, so r and what is divided by it are dv / (2 v) of themselves off"""
    from mit_semseg import ops
    n, lr, wd, betas = 900, 1e-2, 0.01, (0.9, 0.999)
    gen = torch.Generator().manual_seed(31)
    size = 10 ** (torch.arange(-(-n // 256)).repeat_interleave(256)[:n] * 0.7 - 19.4 + 0.3 * torch.rand(n, generator=gen))
    g = torch.where(torch.rand(n, generator=gen) < 0.5, -size, size)
    p, state, step = placed(torch.randn(n, generator=gen), odd), state_of(n, odd), torch.zeros(1, dtype=torch.int32, device=dev())
    G, lr_t = placed(g, odd), torch.tensor([lr], device=dev())
    for t in range(1, 4):
        m0, r0 = decoded([x.cpu() for x in state])
        p0 = p.cpu()
        ops.adamw8_step([p], [G], [state], [step], [wd], lr_t, betas, eps, seed=9)
        rp, rm, rv, move = reference_step(p0, g, m0, r0 * r0, t, float(lr_t), wd, betas, eps)
        off = 4 * 2.0 ** -150 / (2 * rv)
        assert float(off.max()) < 0.01 and float(rv.min()) < 1e-40
        terms = betas[0] * m0.abs() + (1 - betas[0]) * g.double().abs()
        spread = terms / (1 - betas[0] ** t) * lr / ((rv / (1 - betas[1] ** t)).sqrt() + eps)
        bound = U32 * rp.abs() + (20 * U32 + 1.02 * off) * (spread + lr * wd * p0.double().abs())
        assert torch.all((p.cpu().double() - rp).abs() <= bound), float(((p.cpu().double() - rp).abs() / bound).max())
        bits = mix((torch.arange(n) + mix(9 ^ mix(t ^ mix(0)))) & 0xFFFFFFFF)
        r = rv.sqrt()
        check_codes(r, (7 * U32 + 1.02 * off) * r, state[2].cpu(), state[3].cpu(), bits >> 16, True)
        check_codes(rm, 6 * U32 * terms, state[0].cpu(), state[1].cpu(), bits & 0xFFFF, False)
