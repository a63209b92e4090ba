"""The fine-tuning operators on the GPU where ordinary random inputs do not lead: every place of a 16-byte piece, numbers at the ends of
float32's range, recordings that differ between the forward and the backward pass."""
import math

import pytest
import torch

from tests.test_finetune_cpu import U32, check_codes, check_step8, decoded, mix, reference_step

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


EDGES = ['zero gradient', 'beta 0', 'eps 0', 'inf in a block', 'nan in a block', 'below the smallest scale', 'large']


@pytest.mark.parametrize('odd', [False, True])
@pytest.mark.parametrize('n', [256, 1024, 4096, 5000, 700, 3])
@pytest.mark.parametrize('case', EDGES)
def test_adamw8_edges(case, n, odd):
    """three steps of the kernel itself (its root, reciprocal, conversion and maxima differ from the host's form of the arithmetic)"""
    from mit_semseg import ops
    gen = torch.Generator().manual_seed(n)
    p, g = torch.randn(n, generator=gen), torch.randn(n, generator=gen)
    betas, eps, wd, hit = (0.9, 0.999), 1e-8, 0.01, n - 2
    if case == 'zero gradient':
        g.zero_()
    elif case == 'beta 0':
        betas = (0.0, 0.0)
    elif case == 'eps 0':
        eps = 0.0
    elif case.endswith('block'):
        g[hit] = math.inf if case.startswith('inf') else math.nan
    elif case.startswith('below'):
        g = torch.full((n,), 1e-38)
    else:
        g *= 1e18
    P, G, S, step = placed(p, odd), placed(g, odd), state_of(n, odd), torch.zeros(1, dtype=torch.int32, device=dev())
    lr = torch.tensor([1e-2], device=dev())
    for t in range(1, 4):
        m0, r0 = decoded([x.cpu() for x in S])
        p0 = P.cpu()
        ops.adamw8_step([P], [G], [S], [step], [wd], lr, betas, eps, seed=4)
        assert int(step) == t
        got = [x.cpu() for x in S]
        if case == 'zero gradient':
            assert all(torch.all(x.float() == 0) for x in got)
            assert torch.all((P.cpu().double() - p0.double() * (1 - float(lr) * wd)).abs() <= 2 * U32 * p0.double().abs())
            continue
        if case.startswith('below'):
            assert all(torch.all(x.float() == 0) for x in (got[0] & 0x7f, got[1], got[3])) and torch.isfinite(P).all()
            continue
        if not case.endswith('block'):
            check_step8(p0, g, m0, r0, P.cpu(), got, t, float(lr), wd, betas, eps, 4, 0)
            continue
        # the block with the number that is not finite decodes to NaN, the others are right
        b = hit // 256
        m, r = decoded(got)
        bad = torch.zeros(n, dtype=torch.bool)
        bad[b * 256:b * 256 + 256] = True
        assert torch.isnan(m[bad]).all() and torch.isnan(r[bad]).all() and torch.isnan(got[1][b]) and torch.isnan(got[3][b])
        assert torch.isfinite(m[~bad]).all() and torch.isfinite(r[~bad]).all() and torch.isfinite(P.cpu()[~bad]).all()
        if t == 1:                                                    # the step itself still takes the block's other elements
            keep = torch.arange(n) != hit
            assert torch.isfinite(P.cpu()[keep]).all()
        if b:
            check_step8(p0[:b * 256], g[:b * 256], m0[:b * 256], r0[:b * 256], P.cpu()[:b * 256],
                        [x[:b * 256] if x.numel() == n else x[:b] for x in got], t, float(lr), wd, betas, eps, 4, 0)


def test_adamw8_codes_are_the_definition_s():
    """4 M values of each sign convention: with both betas 0 the states are the gradient and its size, and every code equals the rounding
    of value / scale as bit operations define it (16 random bits added below the last of 3 mantissa bits), to the bit"""
    from mit_semseg import ops
    n = 1 << 22
    gen = torch.Generator(device=dev()).manual_seed(3)
    g = torch.randn(n, generator=gen, device=dev()) * 10 ** (4 * torch.rand(n, generator=gen, device=dev()) - 4)
    p, step, S = torch.zeros(n, device=dev()), torch.zeros(1, dtype=torch.int32, device=dev()), state_of(n, False)
    ops.adamw8_step([p], [g], [S], [step], [0.0], torch.zeros(1, device=dev()), (0.0, 0.0), 1e-8, seed=12)
    bits = mix((torch.arange(n, device=dev()) + mix(12 ^ mix(1 ^ mix(0)))) & 0xFFFFFFFF)
    r = (g * g).sqrt()
    for x, u, codes, scale, low in ((g, bits & 0xFFFF, S[0], S[1], 0.0), (r, bits >> 16, S[2], S[3], 2.0 ** -9)):
        top = x.abs().view(-1, 256).amax(1)
        want = top * torch.tensor(1.0 / 448.0, device=dev())
        assert torch.equal(scale, want)
        a = (x * (1.0 / want).repeat_interleave(256)).clamp(-448.0, 448.0)
        if low:
            a = torch.where(x > 0, a.clamp(min=low), a)
        add = torch.where(a.abs() < 2.0 ** -6, torch.full_like(a, 2.0 ** -6), torch.zeros_like(a))
        size = ((((a.abs() + add).view(torch.int32).long() + (u << 4)) & ~0xFFFFF).int().view(torch.float32)) - add
        got = codes.view(torch.float8_e4m3fn).float()
        assert torch.equal(got, torch.copysign(size, a))


# ----------------------------------------------------------------------------------- forward and backward pass recorded apart
def loss_inputs(seed, shape=(2, 150, 24, 30)):
    n, c, h, w = shape
    g = torch.Generator().manual_seed(seed)
    z = (2 * torch.randn(n, h, w, c, generator=g)).to(dev()).permute(0, 3, 1, 2).requires_grad_(True)       # its gradient is written by the forward pass
    label = torch.randint(-1, c, (n, h, w), generator=g).to(dev())
    return z, label, torch.randn(n, generator=g).to(dev()), (-5 + 0.3 * torch.randn(n, h, w, generator=g)).to(dev())


def close(a, b):
    """the same gradient, p from its row's sum in one and from the kept parts in the other: within the roundings of p that the tests of
    the gradient count (its exponent's, up to 3 (d + log) + 2 log C + 90, with d below 20 here), per row of the largest factor"""
    scale = b.abs().amax(dim=1, keepdim=True)
    return bool(torch.all((a - b).abs() <= 2 * U32 * (3 * 20.0 + 3 * math.log(150) + 2 * math.log(150) + 90) * scale))


def test_recorded_backward_of_an_eager_loss_is_refused():
    """every replay would scale the gradient that the forward pass has written once more; the eager backward pass goes on"""
    from mit_semseg import ops
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):                          # a leaf that has been used on the recording's stream alone
        z, label, adv, old = loss_inputs(40)
        x = z.detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
        want = torch.autograd.grad(ops.policy_loss(x, label, adv, old)[0], x)[0]
        loss, lp = ops.policy_loss(z, label, adv, old)[0], ops.label_log_prob(z, label)
        up, ups = torch.ones((), device=dev()), torch.ones_like(lp)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        for out, g in ((loss, up), (lp, ups)):
            with pytest.raises(RuntimeError, match='recorded apart'):
                torch.autograd.grad(out, z, grad_outputs=g, retain_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = torch.autograd.grad(loss, z)[0]
    torch.cuda.synchronize()
    assert close(got, want)


def test_eager_backward_of_a_recorded_loss():
    """gradients that were handed out stay what they are when the recorded loss is replayed on other logits"""
    from mit_semseg import ops
    z, label, adv, old = loss_inputs(41)
    values = [loss_inputs(s)[0].detach() for s in (42, 43, 44)]
    ops.policy_loss(z, label, adv, old)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        loss = ops.policy_loss(z, label, adv, old)[0]
    got = []
    for v in values:
        z.data.copy_(v)
        graph.replay()
        got.append(torch.autograd.grad(loss, z, retain_graph=True)[0])
        torch.cuda.synchronize()
    for v, dz in zip(values, got):
        x = v.clone(memory_format=torch.preserve_format).requires_grad_(True)
        assert close(dz, torch.autograd.grad(ops.policy_loss(x, label, adv, old)[0], x)[0])


def test_one_recording_still_hands_out_what_the_forward_pass_wrote():
    """forward and backward pass in one recording: the bits of the eager pass"""
    from mit_semseg import ops
    z, label, adv, old = loss_inputs(45)
    values = [loss_inputs(s)[0].detach() for s in (46, 47, 48)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        dz = torch.autograd.grad(0.25 * ops.policy_loss(z, label, adv, old)[0], z)[0]
    for v in values:
        z.data.copy_(v)
        graph.replay()
        x = v.clone(memory_format=torch.preserve_format).requires_grad_(True)
        assert torch.equal(dz, torch.autograd.grad(0.25 * ops.policy_loss(x, label, adv, old)[0], x)[0])
        torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------------------ tuning a network
@pytest.mark.parametrize('graph', [False, True])
def test_a_fresh_draw_starts_from_ratio_one_whatever_the_decoder_drops(graph):
    """ppm_deepsup drops channels in training: the first step after taking the log probabilities still has the policy that was asked.  Two
    forward passes of one network differ by less than 5e-4 in a log probability (each is within 2.3e-4 of the reference's), so the KL
    term against them is below 0.5 d^2 = 1.25e-7 and no ratio is near a border; and asking moves no running statistics"""
    import torch.nn as nn
    from mit_semseg.engine import TrainStep
    from mit_semseg.models import ModelBuilder, PolicyLoss, SegmentationModule, resnet
    from mit_semseg.models.models import ResnetDilated
    torch.manual_seed(7)
    enc = ResnetDilated(resnet.resnet18(pretrained=False), 8)
    dec = ModelBuilder.build_decoder('ppm_deepsup', fc_dim=512, num_class=150)
    sm = SegmentationModule(enc, dec, nn.NLLLoss(ignore_index=-1), 0.4).to(dev()).train()
    sm.crit = PolicyLoss(kl_weight=0.1).to(dev())
    ts = TrainStep(sm, lr_encoder=1e-5, lr_decoder=1e-4, max_iters=100, optim='AdamW', graph=graph)
    g = torch.Generator().manual_seed(8)
    for it in range(5):
        feed = {'img_data': torch.randn(2, 3, 64, 96, generator=g).to(dev()), 'seg_label': torch.randint(-1, 150, (2, 8, 12), generator=g).to(dev()),
                'advantage': torch.ones(2, device=dev())}
        before = {k: t.clone() for k, t in sm.state_dict().items()}
        with torch.no_grad():
            lp = sm.label_log_prob(feed)
        for k, t in sm.state_dict().items():
            assert torch.equal(t, before[k]), k
        loss, _ = ts.step(dict(feed, old_logp=lp, ref_logp=lp))
        assert float(sm.crit.clipped) == 0.0 and 0.0 <= float(sm.crit.kl) <= 1.25e-7 and abs(float(loss) + 1.0) <= 5e-4
        assert not torch.equal(sm.state_dict()['encoder.bn1.running_mean'], before['encoder.bn1.running_mean'])
    assert not graph or ts.stats['replayed'] >= 3


def test_numbers_changed_between_replays():
    """KL weight, clip range and gradient bound that a program changes between steps act on the next step, recorded or not"""
    import torch.nn as nn
    from mit_semseg.engine import TrainStep
    from mit_semseg.models import ModelBuilder, PolicyLoss, SegmentationModule, resnet
    from mit_semseg.models.models import ResnetDilated
    rows = []
    for graph in (False, True):
        torch.manual_seed(9)
        enc = ResnetDilated(resnet.resnet18(pretrained=False), 8)
        sm = SegmentationModule(enc, ModelBuilder.build_decoder('c1', fc_dim=512, num_class=150), PolicyLoss(kl_weight=0.05)).to(dev()).train()
        ts = TrainStep(sm, lr_encoder=1e-5, lr_decoder=1e-4, max_iters=100, optim='AdamW', clip_grad_norm=0.5, graph=graph)
        g = torch.Generator().manual_seed(10)
        feed = {'img_data': torch.randn(2, 3, 64, 96, generator=g).to(dev()), 'seg_label': torch.randint(-1, 150, (2, 8, 12), generator=g).to(dev()),
                'advantage': torch.randn(2, generator=g).to(dev()), 'old_logp': (-5 + 0.5 * torch.randn(2, 8, 12, generator=g)).to(dev()),
                'ref_logp': (-5 + 0.5 * torch.randn(2, 8, 12, generator=g)).to(dev())}
        seen = []
        for it in range(9):
            if it == 4:
                sm.crit.kl_weight = 5.0
            elif it == 6:
                sm.crit.clip_low, ts.opt.max_norm = 0.9, 0.01
            elif it == 8:
                sm.crit.kl_weight, sm.crit.clip_low, ts.opt.max_norm = 0.05, 0.2, 0.5
            loss, _ = ts.step(feed)
            seen.append(torch.stack([loss, sm.crit.kl, sm.crit.clipped, *ts.opt.clip]).clone())
        rows.append(torch.stack(seen))
    assert ts.stats['captured'] == 3 and ts.stats['replayed'] == 7, ts.stats
    assert torch.equal(rows[0], rows[1])


# ------------------------------------------------------------------------------------------------------ a KL term that is only watched
@pytest.mark.parametrize('shape', [(2, 150, 9, 13), (2, 2, 9, 13), (1, 700, 9, 13), (1, 40000, 1, 3)], ids=str)
def test_a_kl_term_of_weight_0_does_not_reach_the_loss(shape):
    """rows whose reference is e^100 times as likely (exp overflows) or has probability 0, and a chosen class that is masked: with weight 0
    loss and gradient are, to the bit, those without a reference"""
    from mit_semseg import ops
    z, label, adv, old = loss_inputs(50, shape)
    label.clamp_(min=0)
    with torch.no_grad():
        z[0, int(label[0, 0, 0]), 0, 0] = -math.inf
    ref = old.clone()
    ref.view(-1)[1], ref.view(-1)[2] = 100.0, -math.inf
    want, _, clipped = ops.policy_loss(z, label, adv, old)
    dz = torch.autograd.grad(want, z)[0]
    loss, kl, share = ops.policy_loss(z, label, adv, old, ref)
    assert torch.isfinite(want) and torch.equal(loss, want) and torch.equal(share, clipped) and float(kl) == math.inf
    got = torch.autograd.grad(loss, z)[0]
    assert torch.isfinite(got).all() and torch.equal(got, dz)


@pytest.mark.parametrize('up', [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize('shape,dtype', [((2, 150, 9, 13), torch.float32), ((1, 9, 5, 7), torch.float32), ((2, 150, 9, 13), torch.bfloat16),
                                         ((1, 700, 9, 13), torch.float32)], ids=str)
def test_rows_that_do_not_count_have_no_gradient_under_an_overflowed_scale(shape, dtype, up):
    """an upstream gradient that is not finite (a loss scale that overflowed): zero for rows that do not count, not finite for the others,
    whichever pass writes the gradient"""
    from mit_semseg import ops
    z, label, adv, old = loss_inputs(51, shape)
    label[0, 0, :3] = -1
    z = z.detach().to(dtype).requires_grad_(True)
    loss = ops.policy_loss(z, label, adv, old)[0]
    for _ in range(2):                                                # what the forward pass wrote, and a pass of its own
        dz = torch.autograd.grad(loss, z, grad_outputs=torch.tensor(up, device=dev()), retain_graph=True)[0].permute(0, 2, 3, 1)
        out = label < 0
        assert torch.all(dz[out] == 0)
        assert not torch.isfinite(dz[~out]).all(dim=-1).all()


def test_policy_step_in_segments_equals_eager():
    """a step recorded as a chain of graphs (collectives between them, forced on one rank) has its loss and its backward pass in recordings
    of their own: losses and weights are the eager ones to the bit, at every replay"""
    from mit_semseg import ops
    from mit_semseg.engine import TrainStep
    from mit_semseg.models import ModelBuilder, PolicyLoss, SegmentationModule, resnet
    from mit_semseg.models.models import ResnetDilated
    prev, out = ops._SYNC_GROUP['force'], []
    ops._SYNC_GROUP['force'] = True
    try:
        for graph in (False, True):
            torch.manual_seed(11)
            enc = ResnetDilated(resnet.resnet18(pretrained=False), 8)
            sm = SegmentationModule(enc, ModelBuilder.build_decoder('c1', fc_dim=512, num_class=150), PolicyLoss(kl_weight=0.05)).to(dev()).train()
            ts = TrainStep(sm, lr_encoder=1e-5, lr_decoder=1e-4, max_iters=100, optim='AdamW', clip_grad_norm=0.5, graph=graph)
            g = torch.Generator().manual_seed(12)
            feed = {'img_data': torch.randn(2, 3, 64, 96, generator=g).to(dev()), 'seg_label': torch.randint(-1, 150, (2, 8, 12), generator=g).to(dev()),
                    'advantage': torch.randn(2, generator=g).to(dev()), 'old_logp': (-5 + 0.5 * torch.randn(2, 8, 12, generator=g)).to(dev()),
                    'ref_logp': (-5 + 0.5 * torch.randn(2, 8, 12, generator=g)).to(dev())}
            losses = []
            for _ in range(6):
                loss, _ = ts.step(feed)
                losses.append(loss.clone())
                torch.cuda.synchronize()
            out.append(losses + [p.detach().clone() for p in sm.parameters()])
    finally:
        ops._SYNC_GROUP['force'] = prev
    assert ts.stats['replayed'] >= 3 and ts.launch_mode() != 'eager'
    assert ts._graph.counts().get('allreduce', 0) > 0                 # really a chain
    assert all(torch.equal(a, b) for a, b in zip(*out))
