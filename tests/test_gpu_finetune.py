"""The fine-tuning operators on the GPU against float64: label log probability, clipped policy loss, gradient norm, AdamW with states in
32 and in 8 bits.  Tolerances count roundings: U32 is half a step of float32, half(t) of another type."""
import math

import pytest
import torch

from tests.test_finetune_cpu import U32, check_step, check_step8, decoded

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def dev():
    return torch.device('cuda:0')


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """half of the smallest spacing of a type"""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


# -------------------------------------------------------------------------------------------------------- logits and labels
def make_logits(shape, dtype, layout, gen, scale=3.0):
    """[N, C, H, W] in one of the layouts a caller may hand in; [P, C] for layouts that begin with 'rows'"""
    n, c, h, w = shape
    if layout.startswith('rows'):
        z = torch.randn(n * h * w, c, generator=gen) * scale
        if layout == 'rows':
            return z.to(dev(), dtype)
        if layout == 'rows_slice':                                  # columns of a wider matrix, starting at an odd one
            return torch.zeros(n * h * w, c + 5, device=dev(), dtype=dtype)[:, 3:3 + c].copy_(z)
        return z.t().contiguous().to(dev(), dtype).t()               # rows_t: classes outside
    z = (torch.randn(shape, generator=gen) * scale).to(dev(), dtype)
    if layout == 'nchw':
        return z.contiguous()
    if layout == 'apart':                                            # pixels of a much wider buffer
        buf = torch.zeros(n, h, w, 3 * c, device=dev(), dtype=dtype)
        return buf[..., 1:1 + c].permute(0, 3, 1, 2).copy_(z)
    if layout == 'nhwc':
        return z.contiguous(memory_format=torch.channels_last) if c > 1 else z
    pad = {'slice': 7, 'slice8': 8}[layout]
    buf = torch.zeros(n, h, w, c + pad, device=dev(), dtype=dtype)
    return buf[..., pad // 2:pad // 2 + c].permute(0, 3, 1, 2).copy_(z)


def as_rows(z):
    return z if z.dim() == 2 else z.permute(0, 2, 3, 1).reshape(-1, z.shape[1])


def reference_logp(z, label, ignore=-1):
    """float64 on the CPU: (lp, valid, log softmax, largest logit) per row"""
    x = as_rows(z).detach().cpu().double()
    a = label.reshape(-1).cpu()
    valid = (a != ignore) & (a >= 0) & (a < x.shape[1])
    logp = torch.log_softmax(x, dim=1)
    lp = logp.gather(1, torch.where(valid, a, torch.zeros_like(a)).unsqueeze(1)).squeeze(1)
    return torch.where(valid, lp, torch.zeros_like(lp)), valid, logp, x.max(dim=1)[0], x


def log_sum_roundings(c):
    """roundings of the logarithm of the sum: at most max(64, C / 256) serial additions of a lane and 8 of the lanes, 8 of an exponential
    and of the rescaling, ln C + 1 times 2 for the exponents' products (weighted by their terms), 2 of the logarithm"""
    return max(64, c / 256) + 8 + 8 + 2 * (math.log(c) + 1) + 2


def logp_bound(lp, za, top, c):
    logs = (lp - (za - top)).abs()
    return U32 * ((za - top).abs() + lp.abs() + 2 * logs + log_sum_roundings(c))


def check_gradient(dz, g, logp, x, top, label, valid, dtype):
    """dz against g (1[c = a] - p): p's error is its exponent's (two differences and the logarithm of the sum) and 4 of the exponential"""
    rows, c = logp.shape
    p = logp.exp()
    hit = torch.zeros_like(p)
    hit[valid, label.reshape(-1).cpu()[valid]] = 1.0
    want = torch.where(valid.unsqueeze(1), g.unsqueeze(1) * (hit - p), torch.zeros_like(p))
    d = (x - top.unsqueeze(1)).abs()
    logs = (logp - (x - top.unsqueeze(1))).abs()
    err_p = p * U32 * (3 * d + 3 * logs + log_sum_roundings(c) + 6)
    bound = g.abs().unsqueeze(1) * (err_p + 3 * U32) + want.abs() * (half(dtype) + 4 * U32) + tiny(dtype) + 1e-37 * g.abs().unsqueeze(1)
    got = as_rows(dz).cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    bad &= valid.unsqueeze(1) | (got != 0)
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / bound)[bad].max()))


def make_labels(shape, c, gen, kind='some'):
    label = torch.randint(0, c, shape, generator=gen)
    if kind == 'some':
        u = torch.rand(shape, generator=gen)
        label[u < 0.2] = -1
        label[(u >= 0.2) & (u < 0.25)] = c                            # outside: takes no part
        label[(u >= 0.25) & (u < 0.3)] = -100
    elif kind == 'none':
        label.fill_(-1)
    return label.to(dev())


ROW_CASES = [((1, 1, 1, 1), 'nhwc'), ((1, 2, 1, 1), 'nhwc'), ((2, 3, 5, 7), 'nhwc'), ((3, 19, 33, 17), 'nhwc'), ((2, 150, 9, 13), 'nhwc'),
             ((2, 150, 9, 13), 'nchw'), ((2, 150, 9, 13), 'slice'), ((2, 152, 9, 13), 'slice8'), ((1, 128, 16, 16), 'nhwc'),
             ((1, 129, 16, 16), 'slice'), ((2, 513, 3, 5), 'nhwc'), ((1, 1000, 5, 5), 'slice8'), ((1, 8, 40, 50), 'nhwc'),
             ((1, 9, 40, 50), 'nhwc'), ((1, 33, 1, 700), 'rows'), ((1, 150, 3, 70), 'rows_slice'), ((1, 150, 3, 70), 'rows_t'),
             ((1, 2049, 1, 67), 'rows'), ((1, 4096, 1, 5), 'rows'), ((1, 50001, 1, 3), 'rows'), ((1, 131072, 1, 1), 'rows_slice'),
             ((1, 1, 3, 50), 'rows_slice'), ((4, 21, 130, 131), 'nhwc'),
             # rows far apart (16 lanes a row), the lengths around which the number of lanes and of loads changes, few long rows
             ((1, 2, 5, 70), 'slice8'), ((1, 31, 9, 41), 'slice8'), ((1, 250, 3, 37), 'apart'), ((1, 300, 3, 37), 'apart'), ((1, 320, 7, 11), 'rows'),
             ((1, 321, 7, 11), 'rows'), ((1, 641, 7, 11), 'rows_slice'), ((1, 1024, 7, 11), 'rows'), ((1, 1027, 7, 11), 'rows_slice'),
             ((1, 2047, 5, 7), 'rows_slice'), ((1, 4097, 5, 7), 'rows_slice'), ((1, 8191, 1, 2), 'rows'), ((1, 32003, 1, 511), 'rows')]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('shape,layout', ROW_CASES, ids=str)
def test_label_log_prob(shape, layout, dtype):
    from mit_semseg import ops
    n, c, h, w = shape
    gen = torch.Generator().manual_seed(n * 1000 + c + h)
    z = make_logits(shape, dtype, layout, gen).requires_grad_(True)
    rows = (n * h * w,) if z.dim() == 2 else (n, h, w)
    label = make_labels(rows, c, gen)
    g = torch.randn(rows, generator=gen)
    lp = ops.label_log_prob(z, label)
    assert lp.shape == label.shape and lp.dtype == torch.float32
    want, valid, logp, top, x = reference_logp(z, label)
    za = x.gather(1, torch.where(valid, label.reshape(-1).cpu(), 0).unsqueeze(1)).squeeze(1)
    got = lp.detach().reshape(-1).cpu().double()
    assert torch.all(got[~valid] == 0)
    assert torch.all(((got - want).abs() <= logp_bound(want, za, top, c))[valid])
    dz = torch.autograd.grad(lp, z, g.to(dev()))[0]
    assert dz.shape == z.shape and dz.dtype == dtype
    check_gradient(dz, g.reshape(-1).double(), logp, x, top, label, valid, dtype)
    with torch.no_grad():
        assert torch.equal(ops.label_log_prob(z, label), lp)              # the same bits without the parts kept for the gradient


def test_label_log_prob_extreme_logits():
    """rows far from zero, masked classes (-infinity, the type's lowest value), rows that take no part whatever they hold"""
    from mit_semseg import ops
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        base = torch.tensor([0.5, -1.0, 2.0, 0.25, -3.0])
        rows = torch.stack([base, base + 1000, base - 1000, base, base, torch.full((5,), low), torch.full((5,), -math.inf), base, base])
        rows[3, 1:3] = -math.inf
        rows[4, 0:4] = low
        rows[7] = math.nan
        rows[8, 2] = math.inf
        z = rows.to(dev(), dtype).requires_grad_(True)
        label = torch.tensor([2, 2, 2, 0, 4, 1, -1, -1, -1], device=dev())
        lp = ops.label_log_prob(z, label)
        want, valid, logp, top, x = reference_logp(z, label)
        got = lp.detach().cpu().double()
        za = x.gather(1, label.cpu().clamp(min=0).unsqueeze(1)).squeeze(1)
        assert torch.all(got[6:] == 0)
        assert torch.all((got - want).abs()[:6] <= logp_bound(want, za, top, 5)[:6])
        dz = torch.autograd.grad(lp, z, torch.ones(9, device=dev()))[0]
        assert torch.isfinite(dz).all() and torch.all(dz[6:] == 0)
        check_gradient(dz[:6], torch.ones(6, dtype=torch.float64), logp[:6].clamp(min=-1e4), x[:6].clamp(min=-1e4), top[:6].clamp(min=-1e4),
                       label[:6], valid[:6], dtype)
        # a chosen class of probability zero, a valid row of nothing but -infinity, NaN and +infinity in a valid row
        z2 = torch.stack([rows[3], rows[6], rows[7], rows[8]]).to(dev(), dtype)
        lp2 = ops.label_log_prob(z2, torch.tensor([1, 0, 0, 0], device=dev())).cpu()
        assert lp2[0] == -math.inf and torch.isnan(lp2[1:3]).all() and not lp2[3] > -math.inf


def test_empty_inputs():
    from mit_semseg import ops
    z = torch.zeros(0, 5, device=dev(), requires_grad=True)
    lp = ops.label_log_prob(z, torch.zeros(0, dtype=torch.long, device=dev()))
    assert lp.shape == (0,) and torch.autograd.grad(lp.sum(), z)[0].shape == z.shape
    z = torch.zeros(0, 5, 3, 3, device=dev(), requires_grad=True)
    e = torch.zeros(0, 3, 3, device=dev())
    loss, kl, clipped = ops.policy_loss(z, e.long(), torch.zeros(0, device=dev()), e)
    assert float(loss.detach()) == 0 and torch.autograd.grad(loss, z)[0].shape == z.shape


def policy_inputs(shape, dtype, layout, gen, per_row=False, kind='some'):
    n, c, h, w = shape
    z = make_logits(shape, dtype, layout, gen).requires_grad_(True)
    rows = (n * h * w,) if z.dim() == 2 else (n, h, w)
    label = make_labels(rows, c, gen, kind)
    want = reference_logp(z, label)[0].reshape(rows)
    d = 0.3 * torch.randn(rows, generator=gen, dtype=torch.float64)
    for border in (math.log(0.8), math.log(1.2), math.log(0.9), math.log(1.3)):       # away from the clip's borders: the answer jumps there
        d[(d - border).abs() < 2e-3] = 0.0
    old = (want - d).float().to(dev())
    ref = (want + 0.3 * torch.randn(rows, generator=gen, dtype=torch.float64)).float().to(dev())
    adv = torch.randn(rows if per_row or z.dim() == 2 else (n,), generator=gen).to(dev())
    return z, label, adv, old, ref


def reference_policy(z, label, adv, old, ref, lo, hi, w):
    """float64: (loss, kl, clipped, d loss / d lp per row, rows' error in lp)"""
    lp, valid, logp, top, x = reference_logp(z, label)
    rows, c = logp.shape
    a = adv.detach().cpu().double()
    a = a.reshape(-1) if a.numel() == rows else a.repeat_interleave(rows // a.numel())
    count = max(1, int(valid.sum()))
    ratio = (lp - old.cpu().double().reshape(-1)).exp()
    cut = ratio.clamp(1 - lo, 1 + hi) * a
    clip = (cut < ratio * a) & valid
    row = -torch.minimum(ratio * a, cut)
    g = torch.where(clip, torch.zeros_like(a), -ratio * a)
    k = torch.zeros_like(a)
    if ref is not None:
        d = ref.cpu().double().reshape(-1) - lp
        k = d.exp() - d - 1
        row, g = row + w * k, g + w * (1 - d.exp())
    zero = torch.zeros_like(a)
    za = x.gather(1, torch.where(valid, label.reshape(-1).cpu(), 0).unsqueeze(1)).squeeze(1)
    elp = logp_bound(lp, za, top, c) + 2 * U32
    erow = (ratio * a).abs() * (elp + 6 * U32) + 3 * U32 * row.abs()
    eg = (ratio * a).abs() * (elp + 6 * U32)
    if ref is not None:
        erow = erow + w * ((d.exp() - 1).abs() * (elp + U32 * d.abs()) + 5 * U32 * (d.abs() + k))
        eg = eg + w * (d.exp() * (elp + U32 * d.abs()) + 5 * U32 * (d.exp() - 1).abs() + U32 * g.abs())
    ek = (torch.where(valid, ((d.exp() - 1).abs() * (elp + U32 * d.abs()) + 5 * U32 * (d.abs() + k)), zero).sum() / count) if ref is not None else 0.0
    pick = lambda t: torch.where(valid, t, zero)                                 # noqa: E731
    out = pick(row).sum() / count, pick(k).sum() / count, float(clip.sum()) / count
    return out, (pick(erow).sum() / count, ek), pick(g) / count, pick(eg) / count, (logp, x, top, valid)


# more logits whose gradient the forward pass writes (float32, dense, 8 to 320 classes): every number of lanes a row, whole and partial last
# tiles, odd and even rows, and neighbours of the rule
ONE_PASS = [((2, 150, 100, 80), 'nhwc'), ((1, 151, 121, 117), 'nhwc'), ((1, 2, 1000, 1100), 'nhwc'), ((1, 19, 333, 335), 'nhwc'),
            ((2, 40, 180, 150), 'nhwc'), ((1, 77, 1, 27301), 'rows'), ((1, 300, 70, 101), 'nhwc'), ((1, 319, 80, 83), 'nhwc'),
            ((1, 1, 1500, 1401), 'nhwc'), ((2, 64, 128, 130), 'nchw')]


@pytest.mark.parametrize('shape,layout,dtype', [(*c, t) for c in ROW_CASES if c[0][1] < 60000 for t in TYPES] +
                         [(*c, torch.float32) for c in ONE_PASS], ids=str)
def test_policy_loss(shape, layout, dtype):
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(sum(shape))
    with_ref, per_row = shape[1] % 2 == 0, shape[3] % 2 == 1
    z, label, adv, old, ref = policy_inputs(shape, dtype, layout, gen, per_row)
    ref, w = (ref, 0.07) if with_ref else (None, 0.0)
    lo, hi = (0.2, 0.2) if shape[2] % 2 else (0.1, 0.3)
    loss, kl, clipped = ops.policy_loss(z, label, adv, old, ref, lo, hi, w)
    assert loss.shape == kl.shape == clipped.shape == () and not kl.requires_grad and not clipped.requires_grad
    want, err, g, eg, (logp, x, top, valid) = reference_policy(z, label, adv, old, ref, lo, hi, w)
    for got, value, e in ((loss.detach(), want[0], err[0]), (kl, want[1], err[1]), (clipped, torch.tensor(want[2]), 0.0)):
        assert abs(float(got) - float(value)) <= float(e) + 2 * U32 * abs(float(value)), (float(got), float(value), float(e))
    up = 0.4
    dz = torch.autograd.grad(loss * up, z)[0]
    assert dz.shape == z.shape and dz.dtype == dtype
    # the row's own factor is off by eg: shift it into the bound through the rows' 1-norm
    p = logp.exp()
    got = as_rows(dz).cpu().double()
    hit = torch.zeros_like(p)
    hit[valid, label.reshape(-1).cpu()[valid]] = 1.0
    wantz = up * g.unsqueeze(1) * (hit - p)
    d, logs = (x - top.unsqueeze(1)).abs(), (logp - (x - top.unsqueeze(1))).abs()
    err_p = p * U32 * (3 * d + 3 * logs + log_sum_roundings(shape[1]) + 6)
    bound = up * ((eg + 4 * U32 * g.abs()).unsqueeze(1) * (hit - p).abs() + (g.abs() + eg).unsqueeze(1) * (err_p + 3 * U32)) + \
        wantz.abs() * (half(dtype) + 4 * U32) + tiny(dtype) + 1e-37
    assert torch.all((got - wantz).abs() <= bound), float(((got - wantz).abs() / bound).max())
    assert torch.all(got[~valid] == 0)
    loss, _, _ = ops.policy_loss(z, label, adv, old, ref, lo, hi, w)
    one = as_rows(torch.autograd.grad(loss, z)[0]).cpu().double()         # upstream 1
    assert torch.all((up * one - wantz).abs() <= bound + up * tiny(dtype))


def test_policy_gradient_against_differences():
    """the gradient along random directions against central differences of the float64 loss: their error is h^2 times the third
    derivative (below 10 here) and 1e-16 / h of rounding"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(5)
    z, label, adv, old, ref = policy_inputs((2, 11, 5, 6), torch.float32, 'nhwc', gen)
    loss, _, _ = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.3)
    dz = torch.autograd.grad(loss, z)[0].cpu().double()
    h = 1e-4
    for _ in range(5):
        v = torch.randn(z.shape, generator=gen, dtype=torch.float64)
        f = [float(reference_policy(z.detach().cpu().double() + s * h * v, label, adv, old, ref, 0.2, 0.2, 0.3)[0][0]) for s in (1, -1)]
        diff = (f[0] - f[1]) / (2 * h)
        assert abs(float((dz * v).sum()) - diff) <= 10 * h * h + 1e-15 / h + 1e-5 * float((dz * v).abs().sum())


@pytest.mark.parametrize('what', ['none valid', 'one valid', 'not finite in rows that take no part', 'huge ratio'])
def test_policy_loss_edges(what):
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(8)
    z, label, adv, old, ref = policy_inputs((2, 7, 4, 5), torch.float32, 'nhwc', gen, kind='all')
    if what == 'none valid':
        label.fill_(-1)
        with torch.no_grad():
            z.fill_(math.nan)
        loss, kl, clipped = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1)
        assert float(loss.detach()) == float(kl) == float(clipped) == 0
        assert torch.all(torch.autograd.grad(loss, z)[0] == 0)
        return
    if what == 'one valid':
        keep = label[1, 2, 3].clone()
        label.fill_(255)
        label[1, 2, 3] = keep
        loss, kl, clipped = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1, ignore_index=255)
        label = torch.where(label == 255, -1, label)
    elif what == 'huge ratio':
        old = old - 200.0                                             # the ratio overflows: a positive advantage is cut, a negative one is not
        adv = torch.tensor([1.0, 2.0], device=dev())
        loss, kl, clipped = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1)
        assert float(clipped) == 1.0 and math.isfinite(float(loss))
        adv = torch.tensor([-1.0, 2.0], device=dev())
        assert float(ops.policy_loss(z, label, adv, old, ref)[0]) == math.inf
        return
    else:
        label[0] = -1
        with torch.no_grad():
            z[0] = math.nan
        old[0], ref[0], adv[0] = math.nan, math.inf, math.nan
        loss, kl, clipped = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1)
    dz = torch.autograd.grad(loss, z)[0]
    if what.startswith('not'):
        assert torch.all(dz[0] == 0) and torch.isfinite(dz).all()
        loss1, kl1, clipped1 = ops.policy_loss(z.detach()[1:], label[1:], adv[1:], old[1:], ref[1:], kl_weight=0.1)
        assert torch.equal(kl, kl1) and torch.equal(clipped, clipped1) and abs(float(loss - loss1)) <= 2 * U32 * abs(float(loss))
        return
    want, err, g, eg, _ = reference_policy(z, label, adv, old, ref, 0.2, 0.2, 0.1)
    assert abs(float(loss) - float(want[0])) <= float(err[0]) + 2 * U32 * abs(float(want[0]))
    assert int((as_rows(dz) != 0).any(dim=1).sum()) == 1


def test_backward_twice_and_shared_logits():
    """retain_graph gives the same gradient again; logits used by two operators get the sum"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(9)
    big = policy_inputs((2, 150, 96, 97), torch.float32, 'nhwc', gen)            # its gradient is written by the forward pass
    z, label, adv, old, ref = policy_inputs((2, 150, 6, 7), torch.float32, 'nhwc', gen)
    for zz, *rest in (big, (z, label, adv, old, ref)):
        loss, _, _ = ops.policy_loss(zz, *rest, kl_weight=0.1)
        a, b, c = [torch.autograd.grad(loss, zz, grad_outputs=torch.tensor(u, device=dev()), retain_graph=True)[0] for u in (1.0, 1.0, 3.0)]
        # a second backward computes p from the kept parts instead of from the row's sum: within p's roundings
        close = 2 * U32 * (3 * 24.0 + 3 * math.log(150) + log_sum_roundings(150) + 6)
        scale = a.abs().amax(dim=1, keepdim=True)
        assert torch.all((a - b).abs() <= close * scale) and torch.all((c - 3 * b).abs() <= 4 * U32 * (3 * b).abs() + 1e-37)
        assert a.data_ptr() != b.data_ptr()
        loss, _, _ = ops.policy_loss(zz, *rest, kl_weight=0.1)
        d = torch.autograd.grad(2.0 * loss, zz)[0]
        assert torch.all((d - 2 * b).abs() <= close * 2 * scale)
        loss, _, _ = ops.policy_loss(zz, *rest, kl_weight=0.1)
        with torch.no_grad():
            zz.add_(0.0)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(loss, zz)
    lp = ops.label_log_prob(z, label)
    loss, _, _ = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1)
    both = torch.autograd.grad(loss + lp.sum(), z)[0]
    lp = ops.label_log_prob(z, label)
    c = torch.autograd.grad(lp.sum(), z)[0]
    assert torch.all((both - (a + c)).abs() <= U32 * (a + c).abs())
    # an expanded input: its gradient is the sum over the copies
    one = torch.randn(1, 150, 1, 1, generator=gen).to(dev()).requires_grad_(True)
    lp = ops.label_log_prob(one.expand(2, 150, 6, 7), label)
    got = torch.autograd.grad(lp.sum(), one)[0].reshape(-1).cpu().double()
    p = torch.softmax(one.detach().cpu().double().reshape(-1), 0)
    lab = label.cpu().reshape(-1)
    ok = (lab >= 0) & (lab < 150)
    want = torch.bincount(lab[ok], minlength=150).double() - int(ok.sum()) * p
    n = int(ok.sum())
    assert torch.all((got - want).abs() <= U32 * n * (p * (log_sum_roundings(150) + 60) + 2) + 84 * U32 * n)


def test_second_derivatives_are_refused_and_nodes_are_freed():
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(10)
    z, label, adv, old, ref = policy_inputs((2, 150, 6, 7), torch.float32, 'nhwc', gen)
    for out in (ops.policy_loss(z, label, adv, old)[0], ops.label_log_prob(z, label).sum()):
        dz = torch.autograd.grad(out, z, create_graph=True)[0]
        with pytest.raises(RuntimeError, match='differentiated'):
            torch.autograd.grad(dz.sum(), z)
    out = ops.label_log_prob(z, label).sum()
    torch.autograd.grad(out, z)
    with pytest.raises(RuntimeError, match='second time'):
        torch.autograd.grad(out, z)
    del out, dz
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for backward in (True, False) * 5:
        loss, _, _ = ops.policy_loss(z, label, adv, old)
        lp = ops.label_log_prob(z, label)
        if backward:
            torch.autograd.grad(loss + lp.sum(), z)
        del loss, lp, _
    assert torch.cuda.memory_allocated() == before
    # a leaf's .grad, accumulated
    leaf = z.detach().clone(memory_format=torch.channels_last).requires_grad_(True)
    for i in range(2):
        ops.label_log_prob(leaf, label).sum().backward()
    want = torch.autograd.grad(ops.label_log_prob(z, label).sum(), z)[0]
    assert torch.equal(leaf.grad, want + want)


# ------------------------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize('sizes', [[1], [3, 5], [16384], [16385, 7], [100001, 64, 1, 4096], [5] * 300], ids=lambda s: str(s[:4]))
def test_grad_norm(sizes):
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(len(sizes))
    gs = [torch.randn(s, generator=gen).to(dev(), TYPES[i % 3]) for i, s in enumerate(sizes)]
    gs[0] = torch.cat([gs[0][:1], gs[0]])[1:]                        # starts at an odd address
    gs.append(torch.zeros(0, device=dev()))
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs)) * 0.5
    for max_norm in (None, 0.0, 0.1 * want, 10 * want):
        norm, factor = ops.grad_norm(gs, max_norm, grad_scale=0.5).tolist()
        f = 1.0 if max_norm is None else min(1.0, max_norm / (want + 1e-6))
        assert abs(norm - want) <= 2 * U32 * want and abs(factor - f) <= 2 * U32 * f
    assert torch.equal(ops.grad_norm(gs, 1.0), ops.grad_norm(gs, 1.0))


def test_grad_norm_extremes():
    from mit_semseg import ops
    for value, want in ((1e30, 1e30 * math.sqrt(1000)), (1e-30, 1e-30 * math.sqrt(1000)), (0.0, 0.0)):
        norm, factor = ops.grad_norm([torch.full((1000,), value, device=dev())], 1.0).tolist()
        assert abs(norm - want) <= 4 * U32 * want and 0 <= factor <= 1
    for bad in (math.inf, math.nan, -math.inf):
        g = torch.ones(70000, device=dev())
        g[-1] = bad
        norm, factor = ops.grad_norm([torch.ones(5, device=dev()), g], 1.0).tolist()
        assert not math.isfinite(norm) and factor == 0.0
    assert ops.grad_norm([torch.zeros(0, device=dev())], 1.0).tolist() == [0.0, 1.0]


# ------------------------------------------------------------------------------------------------------------------ AdamW
def adam_tensors(kind, gen, grad):
    """(params, grads, exp_avgs, exp_avg_sqs, copies) on the CPU; place() puts them on the GPU in the layout that `kind` names"""
    shapes = {'small': [(1,), (3,), (255,), (256,), (257,)], 'net': [(64, 32, 3, 3), (77,), (5, 3, 1, 1), (64,), (128, 64, 1, 1), (9000,)],
              'many': [(1 + (i * 7) % 40,) for i in range(500)], 'large': [(4096 * 5 + 1,), (4096 * 3,), (1000003,)],
              'odd address': [(5000,), (4096,), (777,)]}[kind]
    ps = [torch.randn(s, generator=gen) for s in shapes]
    gs = [(0.1 * torch.randn(s, generator=gen)).to(grad) for s in shapes]
    ms = [0.1 * torch.randn(s, generator=gen) for s in shapes]
    vs = [0.01 * torch.rand(s, generator=gen) for s in shapes]
    return ps, gs, ms, vs


def place(t, kind):
    if kind == 'odd address':
        return torch.cat([torch.zeros(1, dtype=t.dtype), t]).to(dev())[1:]
    t = t.to(dev())
    return t.contiguous(memory_format=torch.channels_last) if t.dim() == 4 else t


KINDS = ['small', 'net', 'many', 'large', 'odd address']


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('grad', TYPES, ids=str)
@pytest.mark.parametrize('copy', [None, torch.bfloat16, torch.float16], ids=str)
def test_adamw_step(kind, grad, copy):
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(len(kind))
    ps, gs, ms, vs = adam_tensors(kind, gen, grad)
    n = len(ps)
    P, G, M, V = ([place(t, kind) for t in l] for l in (ps, gs, ms, vs))
    copies = None if copy is None else [torch.empty_like(p, dtype=copy) if i % 3 else None for i, p in enumerate(P)]
    steps = torch.arange(n, dtype=torch.int32, device=dev()) * 13
    wds = [0.01 if i % 2 else 0.0 for i in range(n)]
    lr = torch.tensor([2e-3], device=dev())
    clip = torch.tensor([7.0, 0.25], device=dev())
    ops.adamw_step(P, G, M, V, list(steps.unbind()), wds, lr, (0.9, 0.98), 1e-7, grad_scale=2.0, clip=clip, copies=copies)
    assert steps.tolist() == [13 * i + 1 for i in range(n)]
    for i in range(n):
        check_step(ps[i], gs[i], ms[i], vs[i], P[i].cpu(), M[i].cpu(), V[i].cpu(), 13 * i + 1, float(lr), wds[i], (0.9, 0.98), 1e-7, 0.5)
        if copies is not None and copies[i] is not None:
            assert torch.equal(copies[i], P[i].to(copy))


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('grad', TYPES, ids=str)
@pytest.mark.parametrize('copy', [None, torch.bfloat16, torch.float16], ids=str)
def test_adamw8_step(kind, grad, copy):
    """three steps, each from the states that the one before left, against float64"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(len(kind) + 50)
    ps, gs, _, _ = adam_tensors(kind, gen, grad)
    n = len(ps)
    P = [place(t, kind) for t in ps]
    S = [ops.adamw8_state(p) for p in P]
    if kind == 'odd address':
        S = [ops.AdamW8State(*(place(x.view(torch.uint8).cpu(), kind) if x.element_size() == 1 else x for x in s)) for s in S]
    steps = torch.arange(n, dtype=torch.int32, device=dev()) * 5
    wds = [0.01 if i % 2 else 0.0 for i in range(n)]
    copies = None if copy is None else [torch.empty_like(p, dtype=copy) if i % 3 else None for i, p in enumerate(P)]
    lr = torch.tensor([2e-3], device=dev())
    for it in range(3):
        G = [place((x.float() * (1 + it)).to(grad), kind) for x in gs]
        before = [(p.cpu(), [x.cpu() for x in s]) for p, s in zip(P, S)]
        ops.adamw8_step(P, G, S, list(steps.unbind()), wds, lr, (0.9, 0.98), 1e-7, grad_scale=0.5, copies=copies, seed=it)
        for i in range(n):
            m0, r0 = decoded(before[i][1])
            check_step8(before[i][0], G[i].cpu(), m0, r0, P[i].cpu(), [x.cpu() for x in S[i]], 5 * i + it + 1, float(lr), wds[i], (0.9, 0.98),
                        1e-7, it, i, 0.5)
            if copies is not None and copies[i] is not None:
                assert torch.equal(copies[i], P[i].to(copy))
    assert steps.tolist() == [5 * i + 3 for i in range(n)]


def test_adamw8_is_repeatable():
    """the same call gives the same bits, another seed other codes"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(6)
    p0, g = torch.randn(100000, generator=gen).to(dev()), torch.randn(100000, generator=gen).to(dev())

    def run(seed):
        p, s, step = p0.clone(), ops.adamw8_state(p0), torch.zeros((), dtype=torch.int32, device=dev())
        for _ in range(3):
            ops.adamw8_step([p], [g], [s], [step], [0.1], torch.tensor([1e-3], device=dev()), seed=seed)
        return [p, s.m.view(torch.uint8), s.m_scale, s.r.view(torch.uint8), s.r_scale]
    a, b, c = run(1), run(1), run(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert 0.1 < float((a[1] != c[1]).float().mean()) < 0.9


@pytest.mark.parametrize('bits', [32, 8])
def test_adamw_more_tensors_than_a_launch_holds(bits):
    """2500 tensors (a launch holds 1024, the small kernel before it about 50): every one as if it were alone"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(2)
    sizes = [1 + (i * 37) % 700 for i in range(2500)]
    sizes[1030] = 9000
    at = [0]
    for n in sizes:
        at.append(at[-1] + -(-n // 256) * 256)
    flat = torch.randn(at[-1], generator=gen).to(dev())
    p0, g = flat.clone(), torch.randn(at[-1], generator=gen).to(dev())
    cut = lambda t: [t[a:a + n] for a, n in zip(at, sizes)]             # noqa: E731
    steps, lr = torch.zeros(2500, dtype=torch.int32, device=dev()), torch.tensor([1e-2], device=dev())
    if bits == 32:
        m, v = torch.zeros_like(flat), torch.zeros_like(flat)
        ops.adamw_step(cut(flat), cut(g), cut(m), cut(v), list(steps.unbind()), [0.1] * 2500, lr)
    else:
        m, v = (torch.zeros(at[-1], dtype=torch.uint8, device=dev()) for _ in range(2))
        ms, vs = (torch.zeros(at[-1] // 256, device=dev()) for _ in range(2))
        blocks = [slice(a // 256, a // 256 + -(-n // 256)) for a, n in zip(at, sizes)]
        ops.adamw8_step(cut(flat), cut(g), [(a, ms[b], c, vs[b]) for a, b, c in zip(cut(m), blocks, cut(v))], list(steps.unbind()),
                        [0.1] * 2500, lr)
    assert torch.all(steps == 1)
    # the first step from zero states moves by lr (sign(g) up to eps) + lr wd p
    live = torch.zeros(at[-1], dtype=torch.bool)
    for a, n in zip(at, sizes):
        live[a:a + n] = True
    want = p0.cpu().double() * (1 - 1e-2 * 0.1) - 1e-2 * g.cpu().double() / (g.cpu().double().abs() + 1e-8)
    got = flat.cpu().double()
    assert torch.all((got - want).abs()[live] <= U32 * got.abs()[live] + 20 * U32 * 1e-2 + U32 * 1e-3)
    assert torch.equal(got[~live], p0.cpu().double()[~live])


@pytest.mark.parametrize('bits', [32, 8])
def test_adamw_writes_nothing_else(bits):
    """guard elements around every tensor of a call stay as they were"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(1)
    made = []

    def guarded(n, dtype, fill=None):
        buf = torch.full((n + 64,), 7, device=dev(), dtype=torch.float32).to(dtype) if dtype != torch.uint8 else \
            torch.full((n + 64,), 0x38, device=dev(), dtype=dtype)
        made.append((buf, n, buf.clone()))
        t = buf[32:32 + n]
        t.copy_(torch.zeros(n, dtype=dtype) if fill is None else fill)
        return t
    ns = [1, 255, 257, 4095, 4097, 9001]
    P = [guarded(n, torch.float32, torch.randn(n, generator=gen)) for n in ns]
    G = [guarded(n, torch.float32, torch.randn(n, generator=gen)) for n in ns]
    C = [guarded(n, torch.bfloat16) for n in ns]
    steps = torch.zeros(len(ns), dtype=torch.int32, device=dev())
    lr = torch.tensor([1e-3], device=dev())
    if bits == 32:
        M, V = ([guarded(n, torch.float32) for n in ns] for _ in range(2))
        ops.adamw_step(P, G, M, V, list(steps.unbind()), [0.1] * len(ns), lr, copies=C)
    else:
        S = [ops.AdamW8State(guarded(n, torch.uint8), guarded(-(-n // 256), torch.float32), guarded(n, torch.uint8),
                             guarded(-(-n // 256), torch.float32)) for n in ns]
        ops.adamw8_step(P, G, S, list(steps.unbind()), [0.1] * len(ns), lr, copies=C)
    for buf, n, before in made:
        assert torch.equal(buf[:32], before[:32]) and torch.equal(buf[32 + n:], before[32 + n:])


def test_clip_that_is_not_finite_changes_nothing():
    from mit_semseg import ops
    p, g = torch.randn(5000, device=dev()), torch.randn(5000, device=dev())
    g[77] = math.inf
    m, v, s8 = torch.rand(5000, device=dev()), torch.rand(5000, device=dev()), ops.adamw8_state(p)
    steps, lr = torch.full((2,), 4, dtype=torch.int32, device=dev()), torch.tensor([0.1], device=dev())
    clip = ops.grad_norm([g], 1.0)
    before = [x.clone() for x in (p, m, v)]
    ops.adamw_step([p], [g], [m], [v], [steps[:1]], [0.1], lr, clip=clip)
    ops.adamw8_step([p], [g], [s8], [steps[1:]], [0.1], lr, clip=clip)
    assert all(torch.equal(a, b) for a, b in zip(before, (p, m, v))) and steps.tolist() == [4, 4]
    assert torch.all(s8.m.float() == 0) and torch.all(s8.m_scale == 0)


# --------------------------------------------------------------------------------------------------- streams, graphs, runs
def test_two_streams_at_once():
    """the same operators on two streams, without waiting in between, give what they give one after the other"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(3)
    sets = [policy_inputs(shape, torch.float32, 'nhwc', gen) for shape in ((2, 150, 64, 64), (2, 150, 96, 90))]

    def work(z, label, adv, old, ref):
        loss, kl, clipped = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1)
        dz = torch.autograd.grad(loss, z)[0]
        return [loss.detach(), kl, clipped, dz, ops.grad_norm([dz, dz], 1e-3)]
    want = [work(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = work(*sets[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('bits', [32, 8])
def test_captured_step_replays(bits):
    """loss, gradient, norm and AdamW step in one graph: every replay equals an eager step on the same data, with eager work of the
    program between the replays"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(4)
    feats = torch.randn(512, 24, generator=gen).to(dev())
    label = torch.randint(-1, 33, (512,), generator=gen).to(dev())
    adv, old = torch.randn(512, generator=gen).to(dev()), torch.full((512,), -3.5, device=dev())
    w0 = (0.3 * torch.randn(33, 24, generator=gen)).to(dev())

    def make():
        w = w0.clone()
        return dict(w=w, m=torch.zeros_like(w), v=torch.zeros_like(w), s=ops.adamw8_state(w), step=torch.zeros(1, dtype=torch.int32, device=dev()),
                    lr=torch.tensor([0.05], device=dev()))

    def step(o):
        z = (feats @ o['w'].t()).requires_grad_(True)
        loss, kl, clipped = ops.policy_loss(z, label, adv, old)
        dz = torch.autograd.grad(loss, z)[0]
        g = dz.t().contiguous() @ feats
        clip = ops.grad_norm([g], 0.05)
        if bits == 32:
            ops.adamw_step([o['w']], [g], [o['m']], [o['v']], [o['step']], [0.01], o['lr'], clip=clip)
        else:
            ops.adamw8_step([o['w']], [g], [o['s']], [o['step']], [0.01], o['lr'], clip=clip, seed=5)
        return loss.detach(), clip
    eager, cap = make(), make()
    step(make())                                                       # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cap)
    for it in range(5):
        for o in (eager, cap):
            o['lr'].fill_(0.05 / (1 + it))
        want = step(eager)
        graph.replay()
        assert torch.equal(eager['w'], cap['w']) and torch.equal(eager['step'], cap['step'])
        assert all(torch.equal(a, b) for a, b in zip(want, out))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(eager['s'], cap['s']))
        torch.cuda.synchronize()
    assert int(cap['step']) == 5


def test_capture_beside_a_living_graph_of_the_same_leaf_is_refused():
    """a leaf's earlier graph on another stream: the capture is refused with an error, and works once that graph is gone"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(12)
    z, label, adv, old, ref = policy_inputs((2, 150, 6, 7), torch.float32, 'nhwc', gen)
    z = z.detach().requires_grad_(True)
    loss = ops.policy_loss(z, label, adv, old)[0]
    want = torch.autograd.grad(loss, z, retain_graph=True)[0]
    lp = ops.label_log_prob(z, label)
    for call in (lambda: ops.policy_loss(z, label, adv, old), lambda: ops.label_log_prob(z, label)):
        with pytest.raises(RuntimeError, match='another stream'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        torch.cuda.synchronize()
    ops.policy_loss(z, label, adv, old)                               # eager calls go on
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                                  # no gradient, nothing to refuse
            value = ops.label_log_prob(z, label)
        graph.replay()
        assert torch.equal(value, lp)
    del loss, lp
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.policy_loss(z, label, adv, old)[0]
        dz = torch.autograd.grad(out, z)[0]
    for _ in range(3):
        dz.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dz, want)


# ------------------------------------------------------------------------------------- offsets that do not fit 32 bits
@pytest.mark.parametrize('rows,c', [(14400000, 150), (33000, 65601)])
def test_more_than_2_31_logits(rows, c):
    """the last rows of maps of more than 2^31 elements"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(20)
    assert rows * c > 2 ** 31
    z = torch.zeros(rows, c, device=dev(), dtype=torch.bfloat16)
    n = 70
    z[-n:] = (3 * torch.randn(n, c, generator=gen)).to(dev(), torch.bfloat16)
    z.requires_grad_(True)
    label = torch.full((rows,), -1, device=dev())
    label[-n:] = torch.randint(0, c, (n,), generator=gen).to(dev())
    g = torch.randn(n, generator=gen)
    up = torch.zeros(rows, device=dev())
    up[-n:] = g.to(dev())
    lp = ops.label_log_prob(z, label)
    want, valid, logp, top, x = reference_logp(z.detach()[-n:], label[-n:])
    za = x.gather(1, label[-n:].cpu().unsqueeze(1)).squeeze(1)
    assert torch.all((lp.detach()[-n:].cpu().double() - want).abs() <= logp_bound(want, za, top, c))
    assert float(lp.detach()[:-n].abs().max()) == 0
    dz = torch.autograd.grad(lp, z, up)[0]
    check_gradient(dz[-n:], g.double(), logp, x, top, label[-n:], valid, torch.bfloat16)
    assert int(torch.count_nonzero(dz[:-n])) == 0
    old = (want + 0.05).float()
    olds = torch.zeros(rows, device=dev())
    olds[-n:] = old.to(dev())
    adv = torch.ones(rows, device=dev())
    loss, _, clipped = ops.policy_loss(z.detach(), label, adv, olds)
    value, err = reference_policy(z.detach()[-n:], label[-n:], adv[-n:], olds[-n:], None, 0.2, 0.2, 0.0)[:2]
    assert abs(float(loss) - float(value[0])) <= float(err[0]) + 2 * U32 * abs(float(value[0])) and float(clipped) == 0.0
    del z, dz
    torch.cuda.empty_cache()


@pytest.mark.parametrize('bits', [32, 8])
def test_more_than_2_31_parameters(bits):
    """the ends and the middle of a tensor of more than 2^31 elements (more than 2^32 in 8 bits: the counter of the random bits goes round)"""
    from mit_semseg import ops
    n = 2 ** 31 + 5003 if bits == 32 else 2 ** 32 + 5003
    p = torch.full((n,), 0.5, device=dev())
    g = torch.full((n,), 0.25, device=dev(), dtype=torch.bfloat16)
    gen = torch.Generator().manual_seed(21)
    spots = [slice(0, 512), slice(2 ** 31 - 256, 2 ** 31 + 256), slice(n - 5003 - 256, n)] + ([slice(2 ** 32 - 256, 2 ** 32 + 256)] if bits == 8 else [])
    for s in spots:
        k = len(range(*s.indices(n)))
        p[s], g[s] = torch.randn(k, generator=gen).to(dev()), torch.randn(k, generator=gen).to(dev(), torch.bfloat16)
    before = [(p[s].cpu(), g[s].cpu()) for s in spots]
    step, lr = torch.zeros(1, dtype=torch.int32, device=dev()), torch.tensor([1e-2], device=dev())
    norm = float(ops.grad_norm([g])[0])
    apart = [before[0], before[2]] if bits == 32 else before[:3]       # the others lie inside the last one
    want = sum(float(x[1].double().square().sum()) for x in apart) + (n - sum(x[1].numel() for x in apart)) * 0.0625
    assert abs(norm - math.sqrt(want)) <= 2 * U32 * norm
    if bits == 32:
        m, v = torch.zeros(n, device=dev()), torch.zeros(n, device=dev())
        ops.adamw_step([p], [g], [m], [v], [step], [0.1], lr)
    else:
        state = ops.adamw8_state(p)
        ops.adamw8_step([p], [g], [state], [step], [0.1], lr, seed=3)
    for s, (p0, g0) in zip(spots, before):
        zero = torch.zeros_like(p0)
        if bits == 32:
            check_step(p0, g0, zero, zero, p[s].cpu(), m[s].cpu(), v[s].cpu(), 1, float(lr), 0.1, (0.9, 0.999), 1e-8)
        else:
            a, b, c = s.indices(n)
            q = slice(a // 256, -(-b // 256))
            got = [state.m[s].cpu(), state.m_scale[q].cpu(), state.r[s].cpu(), state.r_scale[q].cpu()]
            check_step8(p0, g0, zero.double(), zero.double(), p[s].cpu(), got, 1, float(lr), 0.1, (0.9, 0.999), 1e-8, 3, 0, start=a)
    middle = p[1 << 20:1 << 30]
    assert float(middle.min()) == float(middle.max()) != 0.5
    del p, g, middle
    torch.cuda.empty_cache()


def test_two_graphs_replayed_at_once():
    """two captured steps on two streams share no scratch: every replay equals the eager result"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(14)
    sets = [policy_inputs(shape, t, 'nhwc', gen) for shape, t in (((2, 150, 48, 64), torch.float32), ((1, 9000, 5, 7), torch.bfloat16))]
    sets = [(z.detach(), *rest) for z, *rest in sets]

    def work(z, label, adv, old, ref):
        z = z.clone(memory_format=torch.preserve_format).requires_grad_(True)
        loss, kl, clipped = ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1)
        dz = torch.autograd.grad(loss, z)[0]
        return [loss.detach(), kl, clipped, dz, ops.grad_norm([dz], 1e-3)]
    want = [work(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in sets]
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work(*s))
    for _ in range(4):
        for out in outs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('shape,layout', [((2, 150, 6, 7), 'slice'), ((2, 400, 6, 7), 'apart'), ((1, 33, 1, 50), 'rows_slice'), ((2, 19, 5, 6), 'nchw')], ids=str)
def test_saved_tensor_hooks(shape, layout):
    """what is kept for the backward pass may come back from a hook in another layout"""
    from mit_semseg import ops
    for dtype in TYPES:
        gen = torch.Generator().manual_seed(16)
        z, label, adv, old, ref = policy_inputs(shape, dtype, layout, gen)
        calls = (lambda: ops.label_log_prob(z, label).sum(), lambda: ops.policy_loss(z, label, adv, old, ref, kl_weight=0.1)[0])
        for call in calls:
            out = call()
            torch.autograd.grad(out, z, retain_graph=True)            # (what the forward pass has written is handed out)
            want = torch.autograd.grad(out, z)[0]
            with torch.autograd.graph.save_on_cpu():
                out = call()
            torch.autograd.grad(out, z, retain_graph=True)
            assert torch.equal(torch.autograd.grad(out, z)[0], want)
