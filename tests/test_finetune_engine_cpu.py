"""Host logic of the AdamW optimisers and of the policy criterion inside TrainStep (CPU): the C ABI is the stub of
test_host_logic_dryrun that checks every call's arguments against the declared signature."""
import pytest
import torch
import torch.nn as nn

from tests.test_host_logic_dryrun import stub  # noqa: F401  (fixture)


def make(crit=None, dss=0.4, arch='c1_deepsup'):
    from mit_semseg.models import ModelBuilder, SegmentationModule, resnet
    from mit_semseg.models.models import ResnetDilated
    enc = ResnetDilated(resnet.resnet18(pretrained=False), 8)
    dec = ModelBuilder.build_decoder(arch, fc_dim=512, num_class=150)
    return SegmentationModule(enc, dec, crit or nn.NLLLoss(ignore_index=-1), dss).train()


def feed(policy=False):
    f = {'img_data': torch.randn(2, 3, 64, 64), 'seg_label': torch.randint(-1, 150, (2, 8, 8))}
    if policy:
        f.update(advantage=torch.randn(2), old_logp=torch.randn(2, 8, 8), ref_logp=torch.randn(2, 8, 8))
    return f


@pytest.mark.parametrize('optim,clip', [('AdamW', None), ('adamw8bit', None), ('AdamW', 1.0), ('AdamW8bit', float('inf'))])
def test_train_step_calls_adamw(stub, optim, clip):  # noqa: F811
    from mit_semseg.engine import FusedAdamW, TrainStep
    sm = make()
    ts = TrainStep(sm, max_iters=10, optim=optim, clip_grad_norm=clip, lr_encoder=1e-3, lr_decoder=2e-3, beta2=0.95)
    assert isinstance(ts.opt, FusedAdamW) and ts.opt.betas == (0.9, 0.95)
    ts.step(feed())
    names = stub.calls
    assert 'semseg_adamw_step' in names and ('semseg_adamw8_step' in names) == ('8' in optim)
    assert 'semseg_sgd_step_fused' not in names and 'semseg_sgd_step' not in names
    assert names.count('semseg_grad_norm') == (0 if clip is None else 1)
    # the deferred weight gradients are summed before anything reads them, the weight planes rebuilt afterwards
    first = names.index('semseg_grad_norm' if clip is not None else 'semseg_adamw_step')
    assert 'semseg_reduce_slabs_multi' in names[:first]
    assert 'semseg_weights_prepare_h2_after_sgd' in names[first:]
    assert 'semseg_reduce_slabs_multi' not in names[first:]


def test_states_by_size(stub):  # noqa: F811
    from mit_semseg import ops
    from mit_semseg.engine import FusedAdamW
    ps = [nn.Parameter(torch.zeros(4096)), nn.Parameter(torch.zeros(4095))]
    opt = FusedAdamW([dict(params=ps, lr=0.1, weight_decay=0.0)], bits=8)
    assert isinstance(opt.state[ps[0]][1], ops.AdamW8State) and not isinstance(opt.state[ps[1]][1], ops.AdamW8State)
    opt.step()                                              # no gradients: nothing to do
    assert not stub.calls
    ps[1].grad = torch.zeros(4095)
    opt.step()
    assert 'semseg_adamw_step' in stub.calls and 'semseg_adamw8_step' not in stub.calls


def test_optimiser_refusals(stub):  # noqa: F811
    from mit_semseg.engine import FusedAdamW, TrainStep, build_optimiser
    groups = [dict(params=[nn.Parameter(torch.zeros(3))], lr=0.1, weight_decay=0.0)]
    with pytest.raises(ValueError, match='TRAIN.optim'):
        build_optimiser('Adagrad', groups)
    with pytest.raises(ValueError, match='clip_grad_norm'):
        build_optimiser('SGD', groups, clip_grad_norm=1.0)
    with pytest.raises(ValueError):
        FusedAdamW(groups, bits=16)
    with pytest.raises(ValueError):
        FusedAdamW(groups, max_norm=-1.0)
    with pytest.raises(ValueError):
        FusedAdamW(groups, max_norm=float('nan'))
    with pytest.raises(ValueError):
        TrainStep(make(), optim='adam')


@pytest.mark.parametrize('dss,arch', [(0.4, 'c1_deepsup'), (None, 'c1_deepsup'), (None, 'c1')])
def test_policy_criterion(stub, dss, arch):  # noqa: F811
    from mit_semseg.engine import TrainStep
    from mit_semseg.models import PolicyLoss
    sm = make(PolicyLoss(kl_weight=0.1), dss, arch)
    with torch.no_grad():
        lp = sm.label_log_prob(feed())
    assert lp.shape == (2, 8, 8) and 'semseg_label_logp_fwd' in stub.calls
    ts = TrainStep(sm, max_iters=10, optim='AdamW')
    loss, acc = ts.step(feed(policy=True))
    assert loss.shape == acc.shape == () and sm.crit.kl.shape == sm.crit.clipped.shape == ()
    assert 'semseg_policy_loss_fwd' in stub.calls and 'semseg_label_logp_bwd' in stub.calls
    with_grad = {n for n, p in sm.named_parameters() if p.grad is not None}
    aux = {n for n, _ in sm.named_parameters() if 'deepsup' in n}
    assert not (aux & with_grad) and with_grad == {n for n, _ in sm.named_parameters()} - aux
    with pytest.raises(ValueError):
        ts.step({k: v for k, v in feed(policy=True).items() if k != 'ref_logp'})
    with pytest.raises(KeyError):
        ts.step(feed())


def test_config_names_the_optimiser():
    from mit_semseg.config import load
    c = load('preset:ade20k-resnet18dilated-ppm_deepsup', ['TRAIN.optim', 'AdamW8bit', 'TRAIN.clip_grad_norm', '1', 'TRAIN.beta2', '0.98'])
    assert (c.TRAIN.optim, c.TRAIN.clip_grad_norm, c.TRAIN.beta2, c.TRAIN.eps) == ('AdamW8bit', 1.0, 0.98, 1e-8)
