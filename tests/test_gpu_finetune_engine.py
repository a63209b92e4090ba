"""The AdamW optimisers and the policy criterion inside TrainStep on the GPU: one step against float64 on the gradients that the step
itself produced, captured steps against eager ones, and a tuning run as a program makes it -- sample, log probabilities, loss, backward,
norm, step."""
import os
import sys

import pytest
import torch
import torch.nn as nn

from tests.test_finetune_cpu import U32, check_step, check_step8, decoded
from tests.test_gpu_drivers import PKG, _dataset, _run
from tests.test_gpu_finetune import log_sum_roundings, reference_policy

pytestmark = pytest.mark.gpu


def dev():
    return torch.device('cuda:0')


def make(crit, seed=3, arch='c1', dss=None):
    from mit_semseg.models import ModelBuilder, SegmentationModule, resnet
    from mit_semseg.models.models import ResnetDilated
    torch.manual_seed(seed)
    enc = ResnetDilated(resnet.resnet18(pretrained=False), 8)
    dec = ModelBuilder.build_decoder(arch, fc_dim=512, num_class=150)
    return SegmentationModule(enc, dec, crit, dss).to(dev()).train()


def images(seed):
    g = torch.Generator().manual_seed(seed)
    return {'img_data': torch.randn(2, 3, 64, 96, generator=g).to(dev()),
            'seg_label': torch.randint(-1, 150, (2, 8, 12), generator=g).to(dev())}


def flat(t):
    """a dense tensor's elements in the order of its memory"""
    return t.detach().as_strided((t.numel(),), (1,)).cpu()


@pytest.mark.parametrize('optim', ['AdamW', 'AdamW8bit'])
@pytest.mark.parametrize('clip', [None, 0.05])
def test_train_step_against_float64(optim, clip):
    from mit_semseg import ops
    from mit_semseg.engine import TrainStep
    sm = make(nn.NLLLoss(ignore_index=-1))
    ts = TrainStep(sm, lr_encoder=1e-3, lr_decoder=2e-3, weight_decay=0.05, max_iters=100, optim=optim, clip_grad_norm=clip)
    for it in range(2):
        before = {}
        for g in ts.opt.groups:
            for p in g['params']:
                s = ts.opt.state[p][1]
                before[p] = (flat(p), [x.clone().cpu() for x in s] if isinstance(s, ops.AdamW8State) else [flat(x) for x in s])
        ts.step(images(it))
        factor = 1.0
        if clip is not None:
            norm = sum(float(p.grad.double().square().sum()) for p in before) ** 0.5
            got = ts.opt.clip.tolist()
            assert abs(got[0] - norm) <= 2 * U32 * norm and got[1] < 1.0
            factor = got[1]                                     # the float32 that the step multiplies with
        for gi, g in enumerate(ts.opt.groups):
            coded = [p for p in g['params'] if isinstance(ts.opt.state[p][1], ops.AdamW8State)]
            assert (len(coded) > 0) == (optim == 'AdamW8bit' and any(p.numel() >= 4096 for p in g['params']))
            for p in g['params']:
                count, s = ts.opt.state[p]
                p0, s0 = before[p]
                assert int(count) == it + 1
                if isinstance(s, ops.AdamW8State):
                    m0, r0 = decoded(s0)
                    check_step8(p0, flat(p.grad), m0, r0, flat(p), [x.cpu() for x in s], it + 1, float(g['lr_t']), g['weight_decay'],
                                (0.9, 0.999), 1e-8, gi, [id(x) for x in coded].index(id(p)), factor)
                else:
                    check_step(p0, flat(p.grad), s0[0], s0[1], flat(p), flat(s[0]), flat(s[1]), it + 1, float(g['lr_t']),
                               g['weight_decay'], (0.9, 0.999), 1e-8, factor)


def run_steps(graph, optim, steps, clip):
    from mit_semseg.engine import TrainStep
    sm = make(nn.NLLLoss(ignore_index=-1))
    ts = TrainStep(sm, lr_encoder=1e-3, lr_decoder=2e-3, max_iters=100, optim=optim, clip_grad_norm=clip, graph=graph)
    losses = []
    for it in range(steps):
        loss, _ = ts.step(images(it))
        losses.append(loss.clone())
        torch.randn(1000, device=dev()).sum()                   # the program's own work between the steps
        if it % 2:
            torch.cuda.synchronize()
    return ts, sm, losses


@pytest.mark.parametrize('optim,clip', [('AdamW', None), ('AdamW8bit', 0.05), ('AdamW8bit', float('inf'))])
def test_captured_steps_equal_eager(optim, clip):
    a, sa, la = run_steps(False, optim, 6, clip)
    b, sb, lb = run_steps(True, optim, 6, clip)
    assert b.stats['replayed'] >= 3, b.stats
    assert all(torch.equal(x, y) for x, y in zip(la, lb))
    for (n, x), (_, y) in zip(sa.state_dict().items(), sb.state_dict().items()):
        assert torch.equal(x, y), n
    for ga, gb in zip(a.opt.groups, b.opt.groups):
        for p, q in zip(ga['params'], gb['params']):
            (ca, xs), (cb, ys) = a.opt.state[p], b.opt.state[q]
            assert int(ca) == int(cb) == 6
            for x, y in zip(xs, ys):
                assert torch.equal(x.view(torch.uint8) if x.element_size() == 1 else x, y.view(torch.uint8) if y.element_size() == 1 else y)


def test_gradients_that_are_not_finite_are_skipped():
    from mit_semseg.engine import TrainStep
    sm = make(nn.NLLLoss(ignore_index=-1))
    ts = TrainStep(sm, lr_encoder=1e-3, lr_decoder=1e-3, max_iters=100, optim='AdamW8bit', clip_grad_norm=1.0)
    ts.step(images(0))
    before = [p.detach().clone() for p in sm.parameters()]
    bad = images(1)
    bad['img_data'][0, 0, 0, 0] = float('inf')
    ts.step(bad)
    assert not torch.isfinite(ts.opt.clip[0]) and float(ts.opt.clip[1]) == 0.0
    assert all(torch.equal(a, b) for a, b in zip(before, sm.parameters()))
    assert all(int(ts.opt.state[p][0]) == 1 for p in sm.parameters())


def tuning_run(graph):
    """three rounds of: draw a label map per image, reward it, take two steps on it"""
    from mit_semseg.engine import TrainStep
    from mit_semseg.models import PolicyLoss
    sm = make(PolicyLoss(kl_weight=0.05), arch='c1_deepsup')
    start = make(PolicyLoss(), arch='c1_deepsup')
    ts = TrainStep(sm, lr_encoder=1e-5, lr_decoder=1e-4, max_iters=100, optim='AdamW8bit', clip_grad_norm=1.0, graph=graph)
    g = torch.Generator().manual_seed(11)
    out = []
    for it in range(3):
        img = images(it)['img_data']
        noise = -torch.log(-torch.log(torch.rand(2, 150, 8, 12, generator=g).clamp(1e-6, 1 - 1e-6))).to(dev())
        with torch.no_grad():
            scores = sm._main_scores(sm.encoder(img, return_feature_maps=True))
            label = (scores + noise).argmax(dim=1)
            label[:, 0, 0] = -1
            f = {'img_data': img, 'seg_label': label, 'advantage': torch.randn(2, generator=g).to(dev())}
            f['old_logp'], f['ref_logp'] = sm.label_log_prob(f), start.label_log_prob(f)
        for _ in range(2):
            loss, acc = ts.step(f)
            out.append([loss.clone(), acc.clone(), sm.crit.kl.clone(), sm.crit.clipped.clone()])
    return sm, ts, out, f, scores


def test_policy_tuning_run():
    sa, ta, oa, f, scores = tuning_run(False)
    sb, tb, ob, _, _ = tuning_run(True)
    assert tb.stats['replayed'] >= 3, tb.stats
    for x, y in zip(oa, ob):
        assert all(torch.equal(a, b) for a, b in zip(x, y)) and all(torch.isfinite(a) for a in x)
    for (n, x), (_, y) in zip(sa.state_dict().items(), sb.state_dict().items()):
        assert torch.equal(x, y), n
    # the first step on a fresh draw starts from the policy that drew it: every ratio is 1, nothing is clipped
    assert all(float(oa[i][3]) == 0.0 for i in (0, 2, 4))


def test_scalars_of_replayed_steps_of_two_shapes():
    """the KL term, the clipped share and the gradient norm are those of the step that ran last, whichever recording it replayed"""
    from mit_semseg.engine import TrainStep
    from mit_semseg.models import PolicyLoss
    out = []
    for graph in (False, True):
        sm = make(PolicyLoss(kl_weight=0.05))
        ts = TrainStep(sm, lr_encoder=1e-5, lr_decoder=1e-4, max_iters=100, optim='AdamW', clip_grad_norm=1.0, graph=graph)
        g = torch.Generator().manual_seed(13)
        feeds = []
        for w in (12, 8):
            feeds.append({'img_data': torch.randn(2, 3, 64, 8 * w, generator=g).to(dev()), 'seg_label': torch.randint(-1, 150, (2, 8, w), generator=g).to(dev()),
                          'advantage': torch.randn(2, generator=g).to(dev()), 'old_logp': (-5 + 0.5 * torch.randn(2, 8, w, generator=g)).to(dev()),
                          'ref_logp': (-5 + 0.5 * torch.randn(2, 8, w, generator=g)).to(dev())})
        seen = []
        for i in range(8):
            loss, _ = ts.step(feeds[i % 2])
            seen.append(torch.stack([loss, sm.crit.kl, sm.crit.clipped, *ts.opt.clip]).clone())
        out.append(torch.stack(seen))
    assert ts.stats['replayed'] >= 5, ts.stats
    assert torch.equal(out[0], out[1]) and len({tuple(r) for r in out[0].tolist()}) == 8


def test_policy_module_loss_and_gradient():
    """loss and d loss / d scores through the module against float64"""
    from mit_semseg.models import PolicyLoss
    sm = make(PolicyLoss(0.1, 0.3, kl_weight=0.2))
    f = images(5)
    g = torch.Generator().manual_seed(2)
    kept = {}
    sm.decoder.register_forward_hook(lambda m, i, o: (o.retain_grad(), kept.update(z=o))[1])
    f.update(advantage=torch.randn(2, 8, 12, generator=g).to(dev()), old_logp=(-5 + 0.3 * torch.randn(2, 8, 12, generator=g)).to(dev()),
             ref_logp=(-5 + 0.3 * torch.randn(2, 8, 12, generator=g)).to(dev()))
    loss, acc = sm(f)
    loss.backward()
    z = kept['z']
    want, err, grad, eg, (logp, x, top, valid) = reference_policy(z.detach(), f['seg_label'], f['advantage'], f['old_logp'], f['ref_logp'],
                                                                  0.1, 0.3, 0.2)
    assert abs(float(loss.detach()) - float(want[0])) <= float(err[0]) + 2 * U32 * abs(float(want[0]))
    hit = torch.zeros_like(logp)
    hit[valid, f['seg_label'].cpu().reshape(-1)[valid]] = 1.0
    wantz = grad.unsqueeze(1) * (hit - logp.exp())
    got = z.grad.permute(0, 2, 3, 1).reshape(-1, 150).cpu().double()
    # scores are log probabilities: their gradient is the loss's, before log_softmax's own.  The row's factor is off by eg, p by its
    # exponent's roundings (tests/test_gpu_finetune.py, check_gradient)
    p, d = logp.exp(), (x - top.unsqueeze(1)).abs()
    err_p = p * U32 * (3 * d + 3 * (logp - (x - top.unsqueeze(1))).abs() + log_sum_roundings(150) + 6)
    assert torch.all((got - wantz).abs() <= (eg + 6 * U32 * grad.abs()).unsqueeze(1) + (grad.abs() + eg).unsqueeze(1) * err_p)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in sm.parameters())


def test_train_command_with_adamw(tmp_path):
    """train.py with TRAIN.optim AdamW8bit and clipping writes its checkpoints"""
    data, ckpt = str(tmp_path / 'data'), str(tmp_path / 'ckpt')
    _dataset(data)
    sys.path.insert(0, PKG)
    from mit_semseg.models import resnet
    from mit_semseg.models.models import ResnetDilated
    torch.manual_seed(1)
    enc0 = str(tmp_path / 'enc0.pth')
    torch.save(ResnetDilated(resnet.resnet18(pretrained=False), dilate_scale=8).state_dict(), enc0)
    env = dict(os.environ, SEMSEG_TUNE='0', PYTHONPATH=PKG + os.pathsep + os.environ.get('PYTHONPATH', ''))
    out = _run('train.py', ['--cfg', 'preset:ade20k-resnet18dilated-ppm_deepsup', '--gpus', '0', 'DIR', ckpt, 'DATASET.root_dataset', data,
                            'DATASET.list_train', os.path.join(data, 'train.odgt'), 'DATASET.list_val', os.path.join(data, 'val.odgt'),
                            'DATASET.imgSizes', '(64, 96)', 'DATASET.imgMaxSize', '160', 'TRAIN.epoch_iters', '4', 'TRAIN.num_epoch', '1',
                            'TRAIN.disp_iter', '1', 'MODEL.weights_encoder', enc0, 'TRAIN.optim', 'AdamW8bit', 'TRAIN.clip_grad_norm', '1.0',
                            'TRAIN.lr_encoder', '1e-4', 'TRAIN.lr_decoder', '1e-3'], env)
    assert out.count('Epoch: [1]') == 4 and 'Training Done!' in out
    sd = torch.load(os.path.join(ckpt, 'encoder_epoch_1.pth'), weights_only=True)
    start = torch.load(enc0, weights_only=True)
    assert all(torch.isfinite(v).all() for v in sd.values()) and not torch.equal(sd['conv1.weight'].cpu(), start['conv1.weight'])
