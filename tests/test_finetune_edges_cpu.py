"""The fine-tuning operators without a GPU: calls that lie beside the documented ones (layouts that only look alike, memory that is read and
written in one call, forward-mode derivatives, numbers at the ends of float32's range), and the host code around them."""
import math

import pytest
import torch

from tests.test_finetune_cpu import U32, emulated, emulator, host  # noqa: F401  (fixtures)
from tests.test_host_logic_dryrun import stub  # noqa: F401  (fixture)


def one(ops, bits, p, g, m=None, v=None, copy=None, more=()):
    """an AdamW step over p (and `more` whole parameters)"""
    ps = [p, *more]
    gs = [g] + [torch.zeros_like(q) for q in more]
    steps, wds = list(torch.zeros(len(ps), dtype=torch.int32).unbind()), [0.0] * len(ps)
    copies = None if copy is None else [copy] + [None] * len(more)
    if bits == 8:
        return ops.adamw8_step(ps, gs, [ops.adamw8_state(q) for q in ps], steps, wds, torch.zeros(1), copies=copies)
    ms = [torch.zeros_like(p) if m is None else m] + [torch.zeros_like(q) for q in more]
    vs = [torch.zeros_like(p) if v is None else v] + [torch.zeros_like(q) for q in more]
    return ops.adamw_step(ps, gs, ms, vs, steps, wds, torch.zeros(1), copies=copies)


@pytest.mark.parametrize('bits', [32, 8])
def test_layouts_that_share_only_their_strides_are_refused(host, bits):  # noqa: F811
    """[8, 2] and a [2, 8] view with the same strides (2, 1): the view covers 10 elements of memory, the parameter 16"""
    p = torch.zeros(8, 2)
    alike = torch.zeros(10).as_strided((2, 8), (2, 1))
    apart = torch.zeros(8).as_strided((3, 2), (3, 1))                # not dense: [2, 3] has the same strides and 6 elements in 6 places
    for q, g in ((p, alike), (torch.zeros(2, 3), apart)):
        with pytest.raises(RuntimeError, match='layout'):
            one(host, bits, q, g)
    with pytest.raises(RuntimeError, match='copy'):
        one(host, bits, p, torch.zeros(8, 2), copy=torch.zeros(10, dtype=torch.bfloat16).as_strided((2, 8), (2, 1)))
    if bits == 32:
        for k in ('m', 'v'):
            with pytest.raises(RuntimeError, match='layout'):
                one(host, bits, p, torch.zeros(8, 2), **{k: alike})


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_that_the_call_writes_are_refused(host, bits):  # noqa: F811
    """a gradient that is (part of) a parameter, a state or a copy: which values are read would depend on which block runs first"""
    p, q, w = torch.zeros(600), torch.zeros(600), torch.zeros(1000, dtype=torch.bfloat16)
    both = torch.zeros(1000)
    for a, g, more, copy in ((p, q, (q,), None), (p, p, (), None), (both[:600], both[400:], (), None), (both[400:], both[:600], (), None),
                             (p, w[:600], (), w[400:]), (p, w[400:], (), w[:600])):
        with pytest.raises(ValueError, match='gradient shares memory'):
            one(host, bits, a, g, copy=copy, more=more)
    if bits == 32:
        m = torch.zeros(600)
        with pytest.raises(ValueError, match='gradient shares memory'):
            one(host, bits, p, m, m=m)
    # neighbours in one buffer are no overlap: the call gets as far as the library
    with pytest.raises(AssertionError, match='was reached'):
        one(host, bits, both[:500], both[500:])


def test_forward_mode_derivatives_are_refused(stub):  # noqa: F811
    """a tangent that an operator does not carry on raises, as in the other operators: an output without one stands for a derivative of 0"""
    import torch.autograd.forward_ad as fwd
    from mit_semseg import ops
    z, label, adv, rows = torch.randn(2, 5, 3, 4), torch.zeros(2, 3, 4, dtype=torch.long), torch.zeros(2), torch.zeros(2, 3, 4)
    flat = torch.zeros(6)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t.clone(), torch.ones_like(t))           # noqa: E731
        calls = [lambda: ops.label_log_prob(dual(z), label), lambda: ops.policy_loss(dual(z), label, adv, rows),
                 lambda: ops.label_log_prob(dual(z.clone().requires_grad_(True)), label),
                 lambda: ops.policy_loss(z, label, dual(adv), rows), lambda: ops.policy_loss(z, label, adv, dual(rows)),
                 lambda: ops.policy_loss(z, label, adv, rows, dual(rows)), lambda: ops.grad_norm([flat, dual(flat)]),
                 lambda: one(ops, 32, dual(flat), flat), lambda: one(ops, 32, flat, dual(flat)), lambda: one(ops, 8, flat, dual(flat)),
                 lambda: one(ops, 32, flat, flat.clone(), m=dual(flat)), lambda: ops.log_softmax(dual(z))]
        for grad in (True, False):
            for call in calls if grad else calls[:-1]:
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call()
        # tensors without a tangent are taken inside the level too
        assert ops.label_log_prob(z, label).shape == label.shape
        ops.grad_norm([flat])
    ops.label_log_prob(z, label)


@pytest.mark.parametrize('eps', [1e-40, 1e-45, 2.0 ** 127])
def test_adamw8_refuses_an_eps_that_has_no_reciprocal(host, eps):  # noqa: F811
    """the 8-bit step multiplies by the hardware's reciprocal, which is 0 or infinite there; the 32-bit step divides and takes it"""
    p = torch.zeros(6)
    a = [[p], [torch.zeros(6)], [host.adamw8_state(p)], [torch.zeros((), dtype=torch.int32)], [0.0], torch.zeros(1)]
    with pytest.raises(ValueError, match='eps'):
        host.adamw8_step(*a, eps=eps)
    for fine in (0.0, 2.0 ** -126, 2.0 ** 126):
        with pytest.raises(AssertionError, match='was reached'):
            host.adamw8_step(*a, eps=fine)
    with pytest.raises(AssertionError, match='was reached'):
        host.adamw_step([p], [torch.zeros(6)], [torch.zeros(6)], [torch.zeros(6)], *a[3:], eps=eps)


def test_a_failed_host_job_does_not_leave_a_stale_library(tmp_path, monkeypatch):
    """both kinds of job are stale, the host extension's fails after the kernels' objects are in place: the next build links them"""
    import importlib.util
    import os
    import subprocess
    import time
    from tests.conftest import PKG
    spec = importlib.util.spec_from_file_location('build_native_under_test', os.path.join(PKG, 'build_native.py'))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    for name in ('a.hip', 'b.hip', 'host_ext.cpp'):
        (tmp_path / name).write_text('')
    for name, value in dict(CSRC=str(tmp_path), OUT_DIR=str(tmp_path), LIB=str(tmp_path / 'lib.so'), SOURCES=['a.hip', 'b.hip'],
                            HOST_SRC=str(tmp_path / 'host_ext.cpp'), HOST_LIB=str(tmp_path / '_host.so')).items():
        monkeypatch.setattr(b, name, value)
    ran, broken, clock = [], [], [time.time() + 100.0]

    def touch(path):                                                  # every file written is a second younger than the one before
        clock[0] += 1.0
        with open(path, 'a'):
            os.utime(path, (clock[0], clock[0]))

    def run(cmd, verbose):
        out = cmd[cmd.index('-o') + 1]
        what = os.path.basename(out).split('.tmp')[0]
        ran.append(what)
        if what in broken:
            raise subprocess.CalledProcessError(1, cmd)
        touch(out)
        if '-MF' in cmd:
            with open(cmd[cmd.index('-MF') + 1], 'w') as f:
                f.write('x: %s\n' % (cmd[cmd.index('-c') + 1] if '-c' in cmd else b.HOST_SRC))
    monkeypatch.setattr(b, '_run', run)
    monkeypatch.setattr(b.os, 'cpu_count', lambda: 1)                 # one job after the other

    def build(fails=()):
        ran.clear()
        broken[:] = fails
        if fails:
            with pytest.raises(subprocess.CalledProcessError):
                b.build(verbose=False)
        else:
            b.build(verbose=False)
        return sorted(ran)
    assert build() == ['_host.so', 'a.o', 'b.o', 'lib.so'] and build() == []
    for name in ('a.hip', 'host_ext.cpp'):
        touch(str(tmp_path / name))
    assert build(['_host.so']) == ['_host.so', 'a.o']
    assert build() == ['_host.so', 'lib.so'] and build() == []        # the object that is newer than the library goes into it
    touch(str(tmp_path / 'b.hip'))
    assert build(['lib.so']) == ['b.o', 'lib.so']                     # a link that failed is tried again
    assert build() == ['lib.so'] and build() == []
    touch(str(tmp_path / 'host_ext.cpp'))
    assert build() == ['_host.so']                                    # the extension alone needs no link


def _module(crit, arch='ppm_deepsup'):
    from mit_semseg.models import ModelBuilder, SegmentationModule, resnet
    from mit_semseg.models.models import ResnetDilated
    enc = ResnetDilated(resnet.resnet18(pretrained=False), 8)
    return SegmentationModule(enc, ModelBuilder.build_decoder(arch, fc_dim=512, num_class=150), crit, 0.4).train()


def _feed():
    return {'img_data': torch.randn(2, 3, 64, 64), 'seg_label': torch.randint(-1, 150, (2, 8, 8)), 'advantage': torch.randn(2),
            'old_logp': torch.randn(2, 8, 8), 'ref_logp': torch.randn(2, 8, 8)}


def test_log_probabilities_leave_the_module_as_it_was(stub, monkeypatch):  # noqa: F811
    """in training mode: the running statistics that the kernels get are not the module's, no dropout mask is drawn, and everything is
    back in its place afterwards, after an error too"""
    from mit_semseg import ops
    from mit_semseg.models import PolicyLoss
    sm = _module(PolicyLoss())
    own = {k: (t, t.clone()) for k, t in sm.named_buffers()}
    statistics = {t.data_ptr() for k, (t, _) in own.items() if 'running' in k or 'num_batches' in k}
    seen, real = [], ops._p
    monkeypatch.setattr(ops, '_p', lambda t: (seen.append(t.data_ptr()) if t is not None else None, real(t))[1])
    for call in (lambda: sm.label_log_prob(_feed()), lambda: sm.label_log_prob([_feed()])):
        with torch.no_grad():
            assert call().shape == (2, 8, 8)
    assert seen and not statistics & set(seen)
    assert not any('dropout' in n or 'scale_nc' in n for n in stub.calls)

    def back():
        for k, t in sm.named_buffers():
            assert t is own[k][0] and torch.equal(t, own[k][1]), k
        assert all(m.training for m in sm.modules())
    back()
    sm.encoder.other = torch.nn.BatchNorm2d(4)                        # a module of the user's with fewer statistics
    del sm.encoder.other.num_batches_tracked
    with torch.no_grad():
        sm.label_log_prob(_feed())
    del sm.encoder.other
    monkeypatch.setattr(sm.decoder, 'forward', lambda *a, **k: 1 // 0)
    with pytest.raises(ZeroDivisionError):
        sm.label_log_prob(_feed())
    back()
    monkeypatch.undo()


def test_dropout_takes_no_part_in_a_policy_step(stub):  # noqa: F811
    import torch.nn as nn
    from mit_semseg.engine import TrainStep
    from mit_semseg.models import PolicyLoss
    for crit, dropped in ((PolicyLoss(), False), (nn.NLLLoss(ignore_index=-1), True)):
        sm = _module(crit)
        stub.calls.clear()
        TrainStep(sm, max_iters=10, optim='AdamW', lr_encoder=1e-4, lr_decoder=1e-4).step(_feed())
        assert any('scale_nc' in n for n in stub.calls) == dropped
        assert all(m.training for m in sm.modules())


def test_changed_numbers_are_another_recording(monkeypatch):
    """what the criterion and AdamW hand to the kernels as numbers is part of what a recorded step is looked up by"""
    import torch.nn as nn
    from mit_semseg.models import PolicyLoss
    from tests import test_graph_policy_cpu as policy
    ts, log = policy._step(monkeypatch, True)
    from mit_semseg.engine import FusedAdamW
    p = [[nn.Parameter(torch.zeros(3))] for _ in range(2)]
    ts.sm.crit = PolicyLoss(kl_weight=0.1)
    ts.opt = FusedAdamW([dict(params=q, lr=0.1, weight_decay=0.0) for q in p], max_norm=1.0)
    changes = [(ts.sm.crit, 'kl_weight', 0.2), (ts.sm.crit, 'clip_low', 0.3), (ts.sm.crit, 'clip_high', 0.1), (ts.sm.crit, 'ignore_index', 255),
               (ts.opt, 'max_norm', 2.0), (ts.opt, 'betas', (0.8, 0.999)), (ts.opt, 'eps', 1e-6), (ts.opt.groups[1], 'weight_decay', 0.5)]
    for _ in range(4):
        policy._run(ts, log, [(4, 4)])
    recorded = [e for e in log if e[0] == 'capture']
    assert len(recorded) == 1 and log[-1][0] == 'replay'
    for k, (of, name, value) in enumerate(changes):
        old = of[name] if isinstance(of, dict) else getattr(of, name)
        put = of.__setitem__ if isinstance(of, dict) else lambda n, v: setattr(of, n, v)
        put(name, value)
        policy._run(ts, log, [(4, 4), (4, 4)])
        assert len([e for e in log if e[0] == 'capture']) == 2 + k, name
        put(name, old)
        policy._run(ts, log, [(4, 4)])                                # the first recording still stands for the first numbers
        assert len([e for e in log if e[0] == 'capture']) == 2 + k and log[-1][0] == 'replay', name
    ts.opt.set_lr(0, 0.7)
    policy._run(ts, log, [(4, 4)])
    assert len([e for e in log if e[0] == 'capture']) == 1 + len(changes)         # the learning rate is device memory


@pytest.mark.parametrize('name,taken', [('SGD', 'SGD'), ('AdamW8bit', 'AdamW8bit'), ('adamw', 'adamw'), ('Adam', 'SGD'), ('', 'SGD')])
def test_configurations_that_trained_before_still_do(stub, name, taken, capsys):  # noqa: F811
    """the reference ignores TRAIN.optim, and so did train.py: a name that is not built here means SGD, with a line that says so"""
    from mit_semseg import drivers
    from mit_semseg.config import load
    from mit_semseg.engine import TrainStep
    cfg = load('preset:ade20k-resnet18dilated-ppm_deepsup', ['TRAIN.optim', name])
    assert drivers.optimiser_of(cfg) == taken
    said = capsys.readouterr().out
    assert ('training with SGD' in said) == (name in ('Adam', ''))
    drivers.optimiser_of(cfg, 1)
    assert capsys.readouterr().out == ''
    TrainStep(_module(None), optim=drivers.optimiser_of(cfg, 1))


def test_one_address_per_entry_point(stub, monkeypatch):  # noqa: F811
    """as many losses as one likes: nothing is added after the first"""
    from mit_semseg import _native, ops
    monkeypatch.setattr(_native, '_addresses', {})
    z, label = torch.randn(2, 5, 3, 4, requires_grad=True), torch.zeros(2, 3, 4, dtype=torch.long)
    counts = []
    for _ in range(3):
        torch.autograd.grad(ops.label_log_prob(z, label).sum(), z)
        counts.append(sum(len(v) if isinstance(v, list) else 1 for v in _native._addresses.values()))
    assert counts == [2, 2, 2]


def test_addresses_of_the_built_library():
    import ctypes
    import os
    from mit_semseg import _native
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip('the library is not built')
    for name in ('semseg_label_logp_bwd', 'semseg_scale_by'):
        first = _native.address(name)
        assert first == _native.address(name) == ctypes.cast(getattr(_native.lib(), name), ctypes.c_void_p).value
