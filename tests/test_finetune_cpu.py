"""The AdamW steps, the gradient norm, the label log probability and the policy loss without a GPU: refusals of the entry points (the
native call must not be reached), and the AdamW arithmetic (csrc/adamw_math.h compiled for the host behind the same C ABI,
tests/native/adamw_emulate.cpp) against float64."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U32 = 2.0 ** -24                    # half a step of float32


def build_emulator(folder):
    out = os.path.join(str(folder), 'libadamw_emulate.so')
    subprocess.run(['g++', '-O2', '-std=c++17', '-ffp-contract=off', '-shared', '-fPIC', '-I' + os.path.join(ROOT, 'include'),
                    '-I' + os.path.join(ROOT, 'semantic-segmentation-pytorch_amd', 'csrc'),
                    os.path.join(ROOT, 'tests', 'native', 'adamw_emulate.cpp'), '-o', out], check=True)
    from mit_semseg import _native
    lib = ctypes.CDLL(out)
    for name in ('semseg_adamw_workspace_bytes', 'semseg_adamw_step', 'semseg_adamw8_step', 'semseg_grad_norm_workspace_bytes',
                 'semseg_grad_norm'):
        getattr(lib, name).restype, getattr(lib, name).argtypes = _native.SIGNATURES[name]
    return lib


class Unreachable:
    def __getattr__(self, name):
        raise AssertionError('%s was reached' % name)


@pytest.fixture
def host(monkeypatch):
    """the entry points on CPU tensors; native calls fail the test"""
    from mit_semseg import _native, ops
    monkeypatch.setattr(ops, '_require_cuda', lambda *a: None)
    monkeypatch.setattr(ops, '_st', lambda: ops.vp(0))
    monkeypatch.setattr(_native, 'lib', lambda: Unreachable())
    return ops


@pytest.fixture(scope='module')
def emulator(tmp_path_factory):
    return build_emulator(tmp_path_factory.mktemp('adamw'))


@pytest.fixture
def emulated(host, emulator, monkeypatch):
    from mit_semseg import _native
    monkeypatch.setattr(_native, 'lib', lambda: emulator)
    return host


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_no_cpu_fallback():
    from mit_semseg import ops
    z, label = torch.randn(2, 5, 3, 3), torch.zeros(2, 3, 3, dtype=torch.long)
    with pytest.raises(RuntimeError, match='HIP device'):
        ops.label_log_prob(z, label)
    with pytest.raises(RuntimeError, match='HIP device'):
        ops.policy_loss(z, label, torch.zeros(2), torch.zeros(2, 3, 3))
    with pytest.raises(RuntimeError, match='HIP device'):
        ops.grad_norm([torch.zeros(3)])
    with pytest.raises(RuntimeError, match='HIP device'):
        ops.adamw_step([torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], [torch.zeros((), dtype=torch.int32)], [0.0],
                       torch.zeros(1))


def test_label_log_prob_refusals(host):
    z, label = torch.randn(2, 5, 3, 4), torch.zeros(2, 3, 4, dtype=torch.long)
    for bad, err in ((z.double(), TypeError), (z[0], ValueError), (z.int(), TypeError), (z[:, :0], ValueError)):
        with pytest.raises(err):
            host.label_log_prob(bad, label if bad.dim() == 4 else label[0])
    for bad, err in ((label.float(), TypeError), (label.bool(), TypeError), (label[:1], ValueError), (label.transpose(1, 2), ValueError),
                     (label.unsqueeze(1), ValueError)):
        with pytest.raises(err):
            host.label_log_prob(z, bad)


def test_policy_loss_refusals(host):
    z, label = torch.randn(2, 5, 3, 4), torch.zeros(2, 3, 4, dtype=torch.long)
    adv, old, ref = torch.zeros(2), torch.zeros(2, 3, 4), torch.zeros(2, 3, 4)
    ok = dict(z=z, label=label, advantage=adv, old_logp=old, ref_logp=ref, clip_low=0.2, clip_high=0.2, kl_weight=0.1)

    def call(**k):
        a = {**ok, **k}
        return host.policy_loss(a['z'], a['label'], a['advantage'], a['old_logp'], a['ref_logp'], a['clip_low'], a['clip_high'],
                                a['kl_weight'])
    for bad in (torch.zeros(3), torch.zeros(2, dtype=torch.float64), torch.zeros(4)[::2], torch.zeros(2, requires_grad=True)):
        with pytest.raises(ValueError, match='scalars'):
            host.policy_loss(z, label, adv, old, scalars=bad)
    for k, err in ((dict(advantage=torch.zeros(3)), ValueError), (dict(advantage=torch.zeros(2, dtype=torch.long)), TypeError),
                   (dict(advantage=torch.zeros(2, requires_grad=True)), ValueError), (dict(old_logp=torch.zeros(2, 12)), ValueError),
                   (dict(old_logp=torch.zeros(2, 3, 4, requires_grad=True)), ValueError), (dict(ref_logp=None), ValueError),
                   (dict(ref_logp=torch.zeros(1, 3, 4)), ValueError), (dict(clip_low=1.5), ValueError), (dict(clip_low=-0.1), ValueError),
                   (dict(clip_high=-0.1), ValueError), (dict(clip_high=float('inf')), ValueError), (dict(clip_low=float('nan')), ValueError),
                   (dict(kl_weight=-1.0), ValueError), (dict(kl_weight=float('nan')), ValueError), (dict(label=label.float()), TypeError),
                   (dict(z=z.double()), TypeError)):
        with pytest.raises(err):
            call(**k)


def test_grad_norm_refusals(host):
    g = torch.zeros(4, 6)
    for bad, err in (([], ValueError), ([g.double()], TypeError), ([g[:, ::2]], RuntimeError), ([g, g[:1].expand(4, 6)], RuntimeError)):
        with pytest.raises(err):
            host.grad_norm(bad)
    with pytest.raises(ValueError):
        host.grad_norm([g], max_norm=-1.0)
    with pytest.raises(ValueError):
        host.grad_norm([g], max_norm=float('nan'))
    for bad in (torch.zeros(3), torch.zeros(2, dtype=torch.float64), torch.zeros(4)[::2]):
        with pytest.raises(ValueError, match='out'):
            host.grad_norm([g], out=bad)


@pytest.mark.parametrize('bits', [32, 8])
def test_adamw_refusals(host, bits):
    def call(**k):
        p = k.get('p', torch.zeros(6, 300))
        a = dict(p=[p], g=[torch.zeros(6, 300)], m=[torch.zeros(6, 300)], v=[torch.zeros(6, 300)], state=[host.adamw8_state(p)],
                 steps=[torch.zeros((), dtype=torch.int32)], wd=[0.0], lr=torch.zeros(1), betas=(0.9, 0.999), eps=1e-8, clip=None, copies=None)
        a.update({n: v for n, v in k.items() if n != 'p'})
        if bits == 32:
            return host.adamw_step(a['p'], a['g'], a['m'], a['v'], a['steps'], a['wd'], a['lr'], a['betas'], a['eps'], clip=a['clip'],
                                   copies=a['copies'])
        return host.adamw8_step(a['p'], a['g'], a['state'], a['steps'], a['wd'], a['lr'], a['betas'], a['eps'], clip=a['clip'],
                                copies=a['copies'])
    t = torch.zeros
    bad = [(dict(p=t(6, 300).double()), TypeError), (dict(p=t(6, 300).bfloat16()), TypeError), (dict(g=[t(6, 300).double()]), TypeError),
           (dict(g=[]), ValueError), (dict(wd=[0.0, 0.0]), ValueError), (dict(steps=[t(())]), TypeError),
           (dict(steps=[t(2, dtype=torch.int32)]), TypeError), (dict(g=[t(300, 6).t()]), RuntimeError), (dict(g=[t(6, 299)]), RuntimeError),
           (dict(p=t(6, 600)[:, ::2], g=[t(6, 600)[:, ::2]]), RuntimeError), (dict(lr=t(2)), ValueError), (dict(lr=t(1).double()), ValueError),
           (dict(clip=t(1)), ValueError), (dict(betas=(1.0, 0.9)), ValueError), (dict(betas=(0.9, -0.1)), ValueError),
           (dict(betas=(float('nan'), 0.9)), ValueError), (dict(eps=-1.0), ValueError), (dict(eps=float('inf')), ValueError),
           (dict(copies=[t(6, 300)]), RuntimeError), (dict(copies=[t(300, 6).bfloat16().t()]), RuntimeError),
           (dict(copies=[None, None]), ValueError)]
    if bits == 32:
        bad += [(dict(m=[t(6, 300).half()]), RuntimeError), (dict(v=[t(300, 6).t()]), RuntimeError), (dict(m=[]), ValueError)]
    else:
        s = host.adamw8_state(t(6, 300))
        bad += [(dict(state=[s._replace(m=s.m[:-1])]), RuntimeError), (dict(state=[s._replace(m_scale=s.m_scale[:-1])]), RuntimeError),
                (dict(state=[s._replace(r=t(1800))]), RuntimeError), (dict(state=[s._replace(r_scale=s.r_scale.double())]), RuntimeError),
                (dict(state=[]), ValueError)]
    for k, err in bad:
        with pytest.raises(err):
            call(**k)
    # the same tensor twice
    p, s = t(6), t((), dtype=torch.int32)
    twice = [p, p]
    for steps in ([s, s.clone()],):
        with pytest.raises(ValueError, match='twice'):
            if bits == 32:
                host.adamw_step(twice, [t(6), t(6)], [t(6), t(6)], [t(6), t(6)], steps, [0.0, 0.0], t(1))
            else:
                host.adamw8_step(twice, [t(6), t(6)], [host.adamw8_state(p) for _ in range(2)], steps, [0.0, 0.0], t(1))
    with pytest.raises(ValueError, match='twice'):
        if bits == 32:
            host.adamw_step([t(6), t(6)], [t(6), t(6)], [t(6), t(6)], [t(6), t(6)], [s, s], [0.0, 0.0], t(1))
        else:
            host.adamw8_step([t(6), t(6)], [t(6), t(6)], [host.adamw8_state(p) for _ in range(2)], [s, s], [0.0, 0.0], t(1))
    # the same state, a state that is another's parameter, a copy that overlaps another
    a, b, w = t(600), t(600), t(1000, dtype=torch.bfloat16)
    two = dict(steps=list(t(2, dtype=torch.int32).unbind()), weight_decays=[0.0, 0.0], lr_tensor=t(1))
    with pytest.raises(ValueError, match='twice'):
        if bits == 32:
            host.adamw_step([a, b], [t(600), t(600)], [t(600), t(600)], [s2 := t(600), s2], **two)
        else:
            st = host.adamw8_state(a)
            host.adamw8_step([a, b], [t(600), t(600)], [st, host.adamw8_state(b)._replace(r=st.r)], **two)
    with pytest.raises(ValueError, match='twice'):
        if bits == 32:
            host.adamw_step([a, b], [t(600), t(600)], [b, t(600)], [t(600), t(600)], **two)
        else:
            host.adamw8_step([a, b], [t(600), t(600)], [host.adamw8_state(a)._replace(m_scale=b[:3]), host.adamw8_state(b)], **two)
    with pytest.raises(ValueError, match='twice'):
        if bits == 32:
            host.adamw_step([a, b], [t(600), t(600)], [t(600), t(600)], [t(600), t(600)], **two, copies=[w[:600], w[400:]])
        else:
            host.adamw8_step([a, b], [t(600), t(600)], [host.adamw8_state(a), host.adamw8_state(b)], **two, copies=[w[:600], w[400:]])
    # nothing to do is not an error
    if bits == 32:
        host.adamw_step([], [], [], [], [], [], t(1))
        host.adamw_step([t(0)], [t(0)], [t(0)], [t(0)], [s], [0.0], t(1))
    else:
        host.adamw8_step([], [], [], [], [], t(1))
        host.adamw8_step([t(0)], [t(0)], [host.adamw8_state(t(0))], [s], [0.0], t(1))


# -------------------------------------------------------------------------------------------------------------- arithmetic
def reference_step(p, g, m, v, t, lr, wd, betas, eps, factor=1.0):
    """(p, m, v, what p's rounding errors are relative to) in float64, from the definition"""
    g = g.double() * factor
    m = betas[0] * m.double() + (1 - betas[0]) * g
    v = betas[1] * v.double() + (1 - betas[1]) * g * g
    move = lr * (m / (1 - betas[0] ** t)) / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p.double() * (1 - lr * wd) - move, m, v, move


def check_step(p0, g, m0, v0, p, m, v, t, lr, wd, betas, eps, factor=1.0):
    """the three results against float64.  Bounds: m is two products and a sum, with (1 - b1), b1 and the factor rounded once each:
    at most 5 roundings of the two terms; v the same with one product more: 6; the step divides m by a root of v (half of v's error, a
    root, a product, a sum), with 1 / sqrt(1 - b2^t) and lr / (1 - b1^t) rounded once each: 5 + 3 + 5 roundings of the step, whose m
    may be the difference of two larger terms, and half a unit of p."""
    rp, rm, rv, move = reference_step(p0, g, m0, v0, t, lr, wd, betas, eps, factor)
    terms = betas[0] * m0.double().abs() + (1 - betas[0]) * (g.double() * factor).abs()
    tiny = 2.0 ** -148                      # the last bit of subnormal products
    assert torch.all((m.double() - rm).abs() <= 5 * U32 * terms + tiny)
    assert torch.all((v.double() - rv).abs() <= 7 * U32 * rv + tiny)
    spread = terms / (1 - betas[0] ** t) * lr / ((rv / (1 - betas[1] ** t)).sqrt() + eps)
    assert torch.all((p.double() - rp).abs() <= U32 * rp.abs() + 14 * U32 * (spread + lr * wd * p0.double().abs()) + tiny)


@pytest.mark.parametrize('t0', [0, 1, 999, 2000000])
@pytest.mark.parametrize('grad', [torch.float32, torch.bfloat16, torch.float16])
def test_adamw_arithmetic(emulated, t0, grad):
    ops = emulated
    gen = torch.Generator().manual_seed(t0 + 1)
    shapes, wds = [(7, 5, 3, 3), (1,), (300,), (2, 0)], [1e-2, 0.0, 1e-4, 0.0]
    ps = [torch.randn(s, generator=gen) for s in shapes]
    ps[0] = ps[0].contiguous(memory_format=torch.channels_last)
    gs = [torch.empty_like(p, dtype=grad).copy_(torch.randn(p.shape, generator=gen) * 0.1) for p in ps]
    ms = [torch.empty_like(p).copy_(0.1 * torch.randn(p.shape, generator=gen)) for p in ps]
    vs = [torch.empty_like(p).copy_(0.01 * torch.rand(p.shape, generator=gen)) for p in ps]
    old = [[x.clone() for x in l] for l in (ps, ms, vs)]
    steps = torch.full((4,), t0, dtype=torch.int32)
    copies = [torch.empty_like(ps[0], dtype=torch.bfloat16), None, torch.empty_like(ps[2], dtype=torch.float16), None]
    lr = torch.tensor([3e-3])
    ops.adamw_step(ps, gs, ms, vs, list(steps.unbind()), wds, lr, (0.9, 0.999), 1e-8, grad_scale=0.5, copies=copies)
    assert steps.tolist() == [t0 + 1] * 3 + [t0]                    # an empty tensor takes no part
    for i in range(3):
        check_step(old[0][i], gs[i], old[1][i], old[2][i], ps[i], ms[i], vs[i], t0 + 1, float(lr), wds[i], (0.9, 0.999), 1e-8, 0.5)
    assert torch.equal(copies[0], ps[0].bfloat16()) and torch.equal(copies[2], ps[2].half())


def test_adamw_matches_torch(emulated):
    ops = emulated
    gen = torch.Generator().manual_seed(3)
    ref = torch.nn.Parameter(torch.randn(50, generator=gen))
    p, m, v = ref.detach().clone(), torch.zeros(50), torch.zeros(50)
    opt = torch.optim.AdamW([ref], lr=1e-2, weight_decay=0.1)
    step, lr = torch.zeros(1, dtype=torch.int32), torch.tensor([1e-2])
    for _ in range(20):
        g = torch.randn(50, generator=gen)
        ref.grad = g.clone()
        opt.step()
        ops.adamw_step([p], [g], [m], [v], [step], [0.1], lr)
    # 20 steps of at most 20 roundings each, of values of order 1 and steps of order lr
    torch.testing.assert_close(p, ref.detach(), rtol=400 * U32, atol=400 * U32 * 1e-1)


@pytest.mark.parametrize('case', ['zero gradient', 'beta 0', 'eps 0', 'not finite', 'clip', 'clip not finite'])
def test_adamw_edges(emulated, case):
    ops = emulated
    p, g = torch.tensor([1.0, -2.0, 3.0]), torch.tensor([0.5, -0.25, 2.0])
    m, v, step, lr = torch.zeros(3), torch.zeros(3), torch.zeros((), dtype=torch.int32), torch.tensor([0.1])
    betas, eps, clip = (0.9, 0.999), 1e-8, None
    if case == 'zero gradient':
        g = torch.zeros(3)
    elif case == 'beta 0':
        betas = (0.0, 0.0)
    elif case == 'eps 0':
        eps = 0.0
    elif case == 'not finite':
        g[1] = float('nan')
    elif case == 'clip':
        clip = torch.tensor([4.0, 0.25])
    else:
        clip = torch.tensor([float('inf'), 0.0])
    before = [x.clone() for x in (p, m, v)]
    ops.adamw_step([p], [g], [m], [v], [step], [0.1], lr, betas, eps, clip=clip)
    if case == 'clip not finite':
        assert int(step) == 0 and all(torch.equal(a, b) for a, b in zip(before, (p, m, v)))
        return
    assert int(step) == 1
    if case == 'not finite':
        assert torch.isnan(p).tolist() == [False, True, False] and torch.isnan(v).tolist() == [False, True, False]
        keep = torch.tensor([0, 2])
        check_step(before[0][keep], g[keep], before[1][keep], before[2][keep], p[keep], m[keep], v[keep], 1, 0.1, 0.1, betas, eps)
        return
    if case == 'zero gradient':
        torch.testing.assert_close(p, before[0] * (1 - 0.1 * 0.1), rtol=4 * U32, atol=0)
        return
    check_step(before[0], g, before[1], before[2], p, m, v, 1, float(lr), 0.1, betas, eps, 0.25 if case == 'clip' else 1.0)


def spacing(a):
    """distance between neighbouring e4m3 values at |a| (float64)"""
    return torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def check_codes(x, err, codes, scales, random16, positive):
    """codes and scales against the definition applied to the exact states `x` (float64), of which the float32 ones are off by `err`: a
    scale is its largest value's error and 2 roundings off, a code equals the stochastic rounding unless the value is within its error
    (its own, and 8 roundings of scale, reciprocal and product) of a border"""
    n = x.numel()
    pad = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    top = pad.abs().amax(1)
    want = torch.where(top < 2.0 ** -100, torch.zeros_like(top), top / 448)
    off = torch.nn.functional.pad(err, (0, -n % 256)).view(-1, 256).amax(1) / 448 + 2 * U32 * want
    assert torch.all((scales.double() - want).abs() <= off)
    s = want.repeat_interleave(256)[:n]
    live = s > 0
    safe = torch.where(live, s, torch.ones_like(s))
    a = torch.where(live, x.abs() / safe, torch.zeros_like(s)).clamp(max=448)
    if positive:
        a = torch.where((x > 0) & live, a.clamp(min=2.0 ** -9), a)
    q = spacing(a)
    exact = a / q + random16.double() / 65536
    low = torch.floor(exact) * q
    got = codes.view(torch.float8_e4m3fn).double()
    differ = (got.abs() != low) & live
    border = (err / safe + a * (8 * U32 + off.repeat_interleave(256)[:n] / safe)) / q + 2.0 ** -20
    near = (exact - exact.round()).abs() <= border
    assert not torch.any(differ & ~near)
    assert torch.all((got.abs() - low).abs()[differ] <= q[differ] * 1.001)
    nonzero = (got != 0) & live
    assert torch.equal(torch.sign(got)[nonzero], torch.sign(x)[nonzero])


def check_step8(p0, g, m0, r0, p, state, t, lr, wd, betas, eps, seed, ordinal, factor=1.0, start=0):
    """one 8-bit step from the decoded states m0, r0 (float64).  m, r^2: as check_step, each with one rounding more (the decoding), a
    product of codes and scales; root and reciprocal are up to one unit (2 roundings) off."""
    n = p.numel()
    flat = [x.reshape(-1) if x.is_contiguous() else x.as_strided((n,), (1,)) for x in (p0, g, p)]
    p0, g, p = flat
    rp, rm, rv, move = reference_step(p0, g, m0, r0 * r0, t, lr, wd, betas, eps, factor)
    terms = betas[0] * m0.abs() + (1 - betas[0]) * (g.double() * factor).abs()
    spread = terms / (1 - betas[0] ** t) * lr / ((rv / (1 - betas[1] ** t)).sqrt() + eps)
    assert torch.all((p.double() - rp).abs() <= U32 * rp.abs() + 20 * U32 * (spread + lr * wd * p0.double().abs()) + 2.0 ** -148)
    bits = mix((torch.arange(start, start + n) + mix(seed ^ mix(t ^ mix(ordinal)))) & 0xFFFFFFFF)
    check_codes(rm, 6 * U32 * terms, state[0], state[1], bits & 0xFFFF, False)
    r = rv.sqrt()
    check_codes(r, 7 * U32 * r + 1.1e-19, state[2], state[3], bits >> 16, True)


def decoded(state):
    """(m, r) of a state in float64"""
    n = state[0].numel()
    return [c.view(torch.float8_e4m3fn).double() * s.double().repeat_interleave(256)[:n] for c, s in ((state[0], state[1]), (state[2], state[3]))]


@pytest.mark.parametrize('n', [1, 3, 255, 256, 257, 1000, 4099])
@pytest.mark.parametrize('grad', [torch.float32, torch.bfloat16, torch.float16])
def test_adamw8_arithmetic(emulated, n, grad):
    ops = emulated
    gen = torch.Generator().manual_seed(n)
    p = torch.randn(n, generator=gen)
    state = ops.adamw8_state(p)
    step, lr, betas, eps, wd, seed = torch.zeros(1, dtype=torch.int32), torch.tensor([1e-2]), (0.9, 0.999), 1e-8, 0.01, 77
    for t in range(1, 5):
        g = (torch.randn(n, generator=gen) * 10 ** (torch.rand(n, generator=gen) * 3 - 3)).to(grad)
        m0, r0 = decoded(state)
        p0 = p.clone()
        copy = torch.empty(n, dtype=torch.bfloat16)
        ops.adamw8_step([p], [g], [state], [step], [wd], lr, betas, eps, copies=[copy], seed=seed)
        assert int(step) == t
        assert torch.equal(copy, p.bfloat16())
        check_step8(p0, g, m0, r0, p, state, t, float(lr), wd, betas, eps, seed, 0)
        m1, v1 = ops.adamw8_values(state, p)
        m, r = decoded(state)
        assert torch.all((m1.double() - m).abs() <= 2 * U32 * m.abs()) and torch.all((v1.double() - r * r).abs() <= 6 * U32 * r * r)
        assert torch.all(v1 >= 0) and torch.all(v1[g != 0] > 0)


def test_adamw8_rounding_is_right_on_average(emulated):
    """r that should follow its gradient does so, although one step is far below half a spacing: over 64 runs with different seeds the
    mean of the decoded r^2 is within 5 standard errors of the exact second moment after 100 steps"""
    ops = emulated
    g = torch.linspace(0.1, 1.0, 256)
    lr, vs = torch.zeros(1), []
    for seed in range(64):
        p, step = torch.zeros(256), torch.zeros(1, dtype=torch.int32)
        state = ops.adamw8_state(p)
        for _ in range(100):
            ops.adamw8_step([p], [g], [state], [step], [0.0], lr, seed=seed)
        vs.append(ops.adamw8_values(state, p)[1].double().sqrt())
    r = torch.stack(vs)
    want = (g.double() ** 2 * (1 - 0.999 ** 100)).sqrt()
    err, dev = (r.mean(0) - want), r.std(0) / 8
    # squaring and taking the root again at every step bends the mean down by half the relative variance of one rounding (below 1 %)
    assert torch.all(err.abs() <= 5 * dev + 0.01 * want)


def test_adamw8_blocks_that_are_not_finite_or_empty(emulated):
    ops = emulated
    p, g = torch.ones(700), torch.ones(700)
    g[300] = float('inf')
    g[600:] = 0
    state, step = ops.adamw8_state(p), torch.zeros(1, dtype=torch.int32)
    ops.adamw8_step([p], [g], [state], [step], [0.0], torch.tensor([0.1]))
    m, v = ops.adamw8_values(state, p)
    assert torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all()
    assert torch.isfinite(m[:256]).all() and torch.isfinite(m[512:]).all() and torch.isfinite(p[:256]).all()
    assert torch.all(m[600:] == 0) and torch.all(v[600:] == 0) and torch.all(p[600:] == 1)
    g = torch.full((700,), 1e-38)
    p, state, step = torch.ones(700), ops.adamw8_state(p), torch.zeros(1, dtype=torch.int32)
    ops.adamw8_step([p], [g], [state], [step], [0.0], torch.tensor([0.1]))
    assert torch.all(state.m_scale == 0) and torch.all(state.r_scale == 0) and torch.all(state.m.float() == 0)


def test_adamw8_state_layout(host):
    p = torch.zeros(5, 4, 3, 3).contiguous(memory_format=torch.channels_last)
    s = host.adamw8_state(p)
    assert s.m.dtype == torch.float8_e4m3fn and s.m.numel() == 180 and s.m_scale.numel() == 1 and s.r_scale.numel() == 1
    s.m.view(torch.uint8)[7] = 0x38                       # 1.0 at place 7 of the parameter's memory
    s.m_scale.fill_(2.0)
    m, v = host.adamw8_values(s, p)
    assert m.stride() == p.stride() and float(m.as_strided((180,), (1,))[7]) == 2.0 and float(m.sum()) == 2.0
    assert math.isclose(float(v.sum()), 0.0)


def _train_ranks(rank, world, folder, port, bits):
    """three steps of a small network on its own data, gradients in buckets, AdamW with clipping; the replicas go to a file"""
    import ctypes as C
    import torch.distributed as dist
    from mit_semseg import _native, ops
    from mit_semseg.engine import FusedAdamW
    from mit_semseg.parallel import GradientBuckets
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group('gloo', rank=rank, world_size=world)
    lib = C.CDLL(os.path.join(folder, 'libadamw_emulate.so'))
    for name in ('semseg_adamw_workspace_bytes', 'semseg_adamw_step', 'semseg_adamw8_step', 'semseg_grad_norm_workspace_bytes',
                 'semseg_grad_norm'):
        getattr(lib, name).restype, getattr(lib, name).argtypes = _native.SIGNATURES[name]
    _native.lib, ops._require_cuda, ops._st = (lambda: lib), (lambda *a: None), (lambda: ops.vp(0))
    net, data = _network()
    opt = FusedAdamW([dict(params=list(net.parameters()), lr=1e-2, weight_decay=0.1)], bits=bits, max_norm=0.5)
    buckets = GradientBuckets(list(net.parameters()), 1 << 14) if world > 1 else None
    for it in range(3):
        opt.zero_grad()
        if buckets is not None:
            buckets.prepare()
        x = data[it]
        loss = net(x[rank::world]).square().mean()
        loss.backward()
        if buckets is not None:
            buckets.finish()
        opt.step(grad_scale=1.0 / world)
    torch.save(dict(net=net.state_dict(), clip=opt.clip, counts=[int(opt.state[p][0]) for p in net.parameters()]),
               os.path.join(folder, 'rank%d_of_%d_%d.pt' % (rank, world, bits)))
    dist.barrier()
    dist.destroy_process_group()


def _network():
    torch.manual_seed(4)
    net = torch.nn.Sequential(torch.nn.Linear(40, 120), torch.nn.ReLU(), torch.nn.Linear(120, 37))
    return net, torch.randn(3, 16, 40, generator=torch.Generator().manual_seed(5))


@pytest.mark.parametrize('bits', [32, 8])
def test_adamw_on_two_ranks(bits, emulator, tmp_path):
    """two ranks with half of the batch each end with the same replicas, and with those of one rank that sees the whole batch"""
    import socket
    import torch.multiprocessing as mp
    build_emulator(tmp_path)
    for world in (1, 2):
        with socket.socket() as s:
            s.bind(('127.0.0.1', 0))
            port = s.getsockname()[1]
        mp.spawn(_train_ranks, args=(world, str(tmp_path), port, bits), nprocs=world, join=True)
    one, a, b = (torch.load(str(tmp_path / ('rank%d_of_%d_%d.pt' % (r, w, bits))), weights_only=True) for r, w in ((0, 1), (0, 2), (1, 2)))
    assert a['counts'] == b['counts'] == one['counts'] == [3] * 4
    assert torch.equal(a['clip'], b['clip']) and abs(float(a['clip'][0] - one['clip'][0])) <= 1e-5 * float(one['clip'][0])
    for k in one['net']:
        assert torch.equal(a['net'][k], b['net'][k])
        if bits == 32:
            # the halves' gradients and the whole one differ by the roundings of sums of 16 products.  A step is lr m / sqrt(v): it feels
            # them as much as the gradient does, fully (up to 2 lr) where the sum cancels to nothing, which few elements' do
            off = (a['net'][k] - one['net'][k]).abs() > 1e-2 * 1e-2
            assert float(off.float().mean()) <= 0.02
