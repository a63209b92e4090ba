"""Cases for measuring the fine-tuning operators: the log probability of chosen labels, the clipped policy loss, the norm of many
gradients, and the AdamW step with states in 32 and in 8 bits.

`run` computes them from elementary torch operations, or, where `own` is set, through mit_semseg's entry points.  A case is a dict
of plain values; the state of the optimiser cases keeps every parameter as a view of one flat buffer whose tensors start at
multiples of 256 elements (zeros between them, which stay zeros)."""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'semantic-segmentation-pytorch_amd')
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
BLOCK = 256                 # elements of one scale of the 8-bit states
BETAS, EPS, SEED = (0.9, 0.999), 1e-8, 304
MASK = 0xFFFFFFFF


def _ops():
    from mit_semseg import ops
    return ops


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    r50 = {'tensors': 168, 'largest': 18874368, 'smallest': 64, 'layout': 1}       # 168 tensors, ~50 M elements: ResNet50dilated + PPM_deepsup
    return [
        # the head of a decoder alone is tuned: a few small tensors, the call's latency counts
        {'name': 'adamw_head', 'op': 'adamw', 'tensors': 5, 'largest': 76800, 'smallest': 150, 'layout': 2, 'grad': 'f32', 'copy': ''},
        {'name': 'adamw_r50', 'op': 'adamw', **r50, 'grad': 'f32', 'copy': ''},
        # gradients and working copies in 16 bits, f32 master weights, large matrices
        {'name': 'adamw_large_bf16', 'op': 'adamw', 'tensors': 24, 'largest': 67108864, 'smallest': 4096, 'layout': 3, 'grad': 'bf16', 'copy': 'bf16'},
        {'name': 'adamw8_head', 'op': 'adamw8', 'tensors': 5, 'largest': 76800, 'smallest': 150, 'layout': 2, 'grad': 'f32', 'copy': ''},
        {'name': 'adamw8_r50', 'op': 'adamw8', **r50, 'grad': 'f32', 'copy': ''},
        {'name': 'adamw8_large_bf16', 'op': 'adamw8', 'tensors': 24, 'largest': 67108864, 'smallest': 4096, 'layout': 3, 'grad': 'bf16', 'copy': 'bf16'},
        {'name': 'norm_r50', 'op': 'norm', **r50, 'grad': 'f32'},
        {'name': 'norm_large_bf16', 'op': 'norm', 'tensors': 24, 'largest': 67108864, 'smallest': 4096, 'layout': 3, 'grad': 'bf16'},
        # a training batch of the framework: 2 images of 512 x 512, labels at 1/8, 150 classes
        {'name': 'policy_64x64x150', 'op': 'policy', 'n': 2, 'h': 64, 'w': 64, 'c': 150, 'pad': 0, 'type': 'f32', 'ref': True, 'back': True},
        # full-resolution score maps
        {'name': 'policy_512x512x150', 'op': 'policy', 'n': 2, 'h': 512, 'w': 512, 'c': 150, 'pad': 0, 'type': 'f32', 'ref': True, 'back': True},
        # log probabilities under the reference model: forward alone, an odd size, 16-bit logits
        {'name': 'logp_375x501x150_f16', 'op': 'logp', 'n': 2, 'h': 375, 'w': 501, 'c': 150, 'pad': 0, 'type': 'f16', 'back': False},
        # one categorical over a large vocabulary per position
        {'name': 'logp_2048x32000_bf16', 'op': 'logp', 'n': 1, 'h': 1, 'w': 2048, 'c': 32000, 'pad': 0, 'type': 'bf16', 'back': True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['adamw', 'adamw8', 'norm', 'policy', 'policy', 'logp', 'logp'])
    if op in ('adamw', 'adamw8', 'norm'):
        smallest = _log(rng, 1, 5000)
        case = {'op': op, 'tensors': _log(rng, 1, 400), 'largest': _log(rng, smallest, 20000000), 'smallest': smallest,
                'layout': rng.randrange(1 << 20), 'grad': rng.choice(['f32', 'bf16', 'f16'])}
        if op != 'norm':
            case['copy'] = rng.choice(['', '', 'bf16', 'f16'])
        while sum(_sizes(case)) > 200000000:
            case['largest'] = max(case['smallest'], case['largest'] // 2)
        return case
    c = rng.choice([2, 19, 21, 150, _log(rng, 1, 300), _log(rng, 300, 60000)])
    rows = _log(rng, 1, max(1, min(600000, 80000000 // c)))
    n = rng.randint(1, 4)
    h = max(1, min(_log(rng, 1, 800), rows // n))
    w = max(1, rows // n // h)
    case = {'op': op, 'n': n, 'h': h, 'w': w, 'c': c, 'pad': rng.choice([0, 0, 0, 1, 6, 8]), 'type': rng.choice(['f32', 'f32', 'bf16', 'f16']),
            'back': rng.random() < 0.7}
    if op == 'policy':
        case['ref'] = rng.random() < 0.7
    return case


def _sizes(case):
    """the tensors of a case: the largest one, the others spread over the logarithm of the range"""
    r = random.Random(case['layout'])
    lo, hi = math.log(case['smallest']), math.log(case['largest'])
    # most of a network's tensors are far smaller than its largest
    return [case['largest']] + [int(math.exp(lo + (hi - lo) * r.random() * 0.87)) or 1 for _ in range(case['tensors'] - 1)]


def _padded(case):
    return [-(-s // BLOCK) * BLOCK for s in _sizes(case)]


# -------------------------------------------------------------------------------------------------------------- inputs
def _views(flat, case):
    out, at = [], 0
    for s, full in zip(_sizes(case), _padded(case)):
        out.append(flat[at:at + s])
        at += full
    return out


def _random(case, gen, scale, dtype=torch.float32, positive=False):
    """a flat buffer of normal values, zeros in the gaps"""
    sizes, full = _sizes(case), _padded(case)
    flat = torch.randn(sum(full), generator=gen, device='cuda')
    if positive:
        flat = flat.abs_()
    flat = flat.mul_(scale).to(dtype)
    at = 0
    for s, f in zip(sizes, full):
        flat[at + s:at + f] = 0
        at += f
    return flat


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op = case['op']
    if op in ('policy', 'logp'):
        n, h, w, c = case['n'], case['h'], case['w'], case['c']
        buf = torch.randn(n, h, w, c + case['pad'], generator=gen, device='cuda').mul_(2.0).to(TYPES[case['type']])
        z = buf[..., :c].permute(0, 3, 1, 2)                     # logical NCHW over NHWC memory, as every map of the framework
        label = torch.randint(0, c, (n, h, w), generator=gen, device='cuda')
        label[torch.rand(n, h, w, generator=gen, device='cuda') < 0.1] = -1          # unlabelled pixels
        s = {'case': case, 'z': z.requires_grad_(case['back']), 'label': label}
        if op == 'logp':
            s['g'] = torch.randn(n, h, w, generator=gen, device='cuda')
            return s
        with torch.no_grad():
            lp = _plain_logp(z, label)[0]
        s['advantage'] = torch.randn(n, generator=gen, device='cuda')
        d = 0.2 * torch.randn(n, h, w, generator=gen, device='cuda')
        # no ratio on the border of the clip, where the last bit of a 32-bit sum decides between two different answers
        for border in (0.8, 1.2):
            d = torch.where((d + math.log(border)).abs() < 2e-5, torch.zeros_like(d), d)
        s['old'] = lp + d
        s['refp'] = lp + 0.2 * torch.randn(n, h, w, generator=gen, device='cuda') if case['ref'] else None
        s['kl_weight'] = 0.05 if case['ref'] else 0.0
        return s
    s = {'case': case, 'g': _random(case, gen, 1e-3, TYPES[case['grad']])}
    s['grads'] = _views(s['g'], case)
    if op == 'norm':
        s['max_norm'] = 0.5
        return s
    sizes, full = _sizes(case), _padded(case)
    s['p'] = _random(case, gen, 0.05)
    s['params'] = _views(s['p'], case)
    s['lr'] = torch.full((1,), 2e-4, device='cuda')
    s['wd'] = [1e-4 if i % 3 else 0.0 for i in range(len(sizes))]
    s['wd_t'] = torch.tensor(s['wd'], device='cuda')
    s['steps'] = torch.randint(0, 1000, (len(sizes),), generator=gen, device='cuda', dtype=torch.int32)
    s['step_list'] = list(s['steps'].unbind())
    s['of_block'] = torch.repeat_interleave(torch.arange(len(sizes), device='cuda'), torch.tensor([f // BLOCK for f in full], device='cuda'))
    s['copy'] = torch.zeros_like(s['p'], dtype=TYPES[case['copy']]) if case['copy'] else None
    s['copies'] = _views(s['copy'], case) if case['copy'] else None
    if op == 'adamw':
        s['m'], s['v'] = _random(case, gen, 3e-4), _random(case, gen, 1e-3).square_()
        s['ms'], s['vs'] = _views(s['m'], case), _views(s['v'], case)
        return s
    blocks = sum(full) // BLOCK
    s['m'] = _random(case, gen, 100.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
    s['r'] = _random(case, gen, 100.0, positive=True).clamp_(0, 448).to(torch.float8_e4m3fn)
    s['m_scale'] = 3e-6 * (0.5 + torch.rand(blocks, generator=gen, device='cuda'))
    s['r_scale'] = 1e-5 * (0.5 + torch.rand(blocks, generator=gen, device='cuda'))
    at, states = 0, []
    for m, r, f in zip(_views(s['m'], case), _views(s['r'], case), full):
        b = slice(at // BLOCK, (at + f) // BLOCK)
        states.append((m, s['m_scale'][b], r, s['r_scale'][b]))
        at += f
    s['states'] = states
    # where each element's counter starts: its place in its tensor
    starts = torch.tensor([0] + full[:-1], device='cuda').cumsum(0)
    s['start'] = starts[s['of_block']]
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_logp(z, label, ignore_index=-1):
    """([N,H,W] log probability of the label, valid rows, exp-sum-normalised logits)"""
    x = z.detach().float()
    x = x - x.amax(dim=1, keepdim=True)
    logp = x - x.exp().sum(dim=1, keepdim=True).log()
    valid = (label != ignore_index) & (label >= 0) & (label < z.shape[1])
    at = torch.where(valid, label, torch.zeros_like(label))
    lp = logp.gather(1, at.unsqueeze(1)).squeeze(1)
    return torch.where(valid, lp, torch.zeros_like(lp)), valid, logp, at


def _plain_dz(logp, at, g, dtype):
    d = -g.unsqueeze(1) * logp.exp()
    d.scatter_add_(1, at.unsqueeze(1), g.unsqueeze(1))
    return d.to(dtype)


def _policy(s, case):
    lp, valid, logp, at = _plain_logp(s['z'], s['label'])
    adv = s['advantage'].view(-1, 1, 1)
    count = valid.sum().clamp(min=1).float()
    ratio = (lp - s['old']).exp()
    full, cut = ratio * adv, ratio.clamp(0.8, 1.2) * adv
    clipped = (cut < full) & valid
    loss, dlp, kl = -torch.minimum(full, cut), -torch.where(clipped, torch.zeros_like(full), full), torch.zeros_like(lp)
    if s['refp'] is not None:
        d = s['refp'] - lp
        kl = d.exp() - d - 1
        loss = loss + s['kl_weight'] * kl
        dlp = dlp + s['kl_weight'] * (1 - d.exp())
    zero = torch.zeros_like(lp)
    out = [torch.where(valid, x, zero).double().sum().div(count).float() for x in (loss, kl)] + [clipped.sum() / count]
    if case['back']:
        out.append(_plain_dz(logp, at, torch.where(valid, dlp, zero) / count, s['z'].dtype))
    return out


def _coefficients(s):
    """per block [blocks, 1]: step size, 1 / sqrt(1 - b2^t), lr * weight decay"""
    t = s['steps'].double()
    lr = s['lr'].double()
    size = lr / (1 - BETAS[0] ** t)
    root = 1 / (1 - BETAS[1] ** t).sqrt()
    return [x.float()[s['of_block']].unsqueeze(1) for x in (size, root, lr.float() * s['wd_t'])]


def _moved(p, m, r, size, root, decay):
    return p - (size * (m / (r * root + EPS)) + decay * p)


def _adamw(s):
    s['steps'] += 1
    size, root, decay = _coefficients(s)
    p, g, m, v = (s[k].view(-1, BLOCK) for k in ('p', 'g', 'm', 'v'))
    g = g.float()
    m.copy_(BETAS[0] * m + (1 - BETAS[0]) * g)
    v.copy_(BETAS[1] * v + ((1 - BETAS[1]) * g) * g)
    p.copy_(_moved(p, m, v.sqrt(), size, root, decay))
    if s['copy'] is not None:
        s['copy'].copy_(s['p'])
    return [s['p'], s['m'], s['v'], s['steps']] + ([s['copy']] if s['copy'] is not None else [])


def _mix(x):
    """32 bits scrambled, held in int64"""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & MASK
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & MASK
    return x ^ (x >> 16)


def _rounded(a, random16):
    """stochastic rounding of 0 <= a <= 448 to e4m3: random bits added below the last kept one, then cut off"""
    low = torch.where(a < 2.0 ** -6, torch.full_like(a, 2.0 ** -6), torch.zeros_like(a))
    bits = (a + low).view(torch.int32) + (random16 << 4).int()
    return (bits & ~0xFFFFF).view(torch.float32) - low


def _coded(x, random16, positive):
    """(codes, scale per block) of [blocks, 256] values"""
    top = x.abs().amax(dim=1, keepdim=True)
    scale = torch.where(top < 2.0 ** -100, torch.zeros_like(top), top * (1.0 / 448))
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    a = _rounded((x.abs() * inv).clamp(max=448.0), random16)
    if positive:
        a = torch.where((x > 0) & (a < 2.0 ** -9) & (scale > 0), torch.full_like(a, 2.0 ** -9), a)
    return torch.copysign(a, x).to(torch.float8_e4m3fn), scale.squeeze(1)


def _adamw8(s):
    s['steps'] += 1
    size, root, decay = _coefficients(s)
    p, g, mc, rc = (s[k].view(-1, BLOCK) for k in ('p', 'g', 'm', 'r'))
    g = g.float()
    r = rc.float() * s['r_scale'].unsqueeze(1)
    m = BETAS[0] * (mc.float() * s['m_scale'].unsqueeze(1)) + (1 - BETAS[0]) * g
    r = (BETAS[1] * (r * r) + ((1 - BETAS[1]) * g) * g).sqrt()
    p.copy_(_moved(p, m, r, size, root, decay))
    # the counter hash of (seed, step, tensor, element)
    base = _mix(SEED ^ _mix(s['steps'].long() ^ _mix(torch.arange(len(s['wd']), device=p.device))))[s['of_block']]
    place = torch.arange(s['p'].numel(), device=p.device).view(-1, BLOCK) - s['start'].unsqueeze(1)
    bits = _mix((place + base.unsqueeze(1)) & MASK)
    mc2, ms = _coded(m, bits & 0xFFFF, False)
    rc2, rs = _coded(r, bits >> 16, True)
    mc.copy_(mc2), rc.copy_(rc2), s['m_scale'].copy_(ms), s['r_scale'].copy_(rs)
    if s['copy'] is not None:
        s['copy'].copy_(s['p'])
    return [s['p'], s['m'], s['m_scale'], s['r'], s['r_scale'], s['steps']] + ([s['copy']] if s['copy'] is not None else [])


def _norm(s):
    n = s['g'].double().square().sum().sqrt()
    return torch.stack([n, torch.clamp(s['max_norm'] / (n + 1e-6), max=1.0)]).float()


def _run_plain(s):
    case = s['case']
    op = case['op']
    if op == 'logp':
        lp, valid, logp, at = _plain_logp(s['z'], s['label'])
        if not case['back']:
            return lp
        return lp, _plain_dz(logp, at, torch.where(valid, s['g'], torch.zeros_like(s['g'])), s['z'].dtype)
    return {'policy': lambda: _policy(s, case), 'adamw': lambda: _adamw(s), 'adamw8': lambda: _adamw8(s), 'norm': lambda: _norm(s)}[op]()


def _run_own(s):
    ops, case = _ops(), s['case']
    op = case['op']
    if op == 'logp':
        lp = ops.label_log_prob(s['z'], s['label'])
        return (lp, torch.autograd.grad(lp, s['z'], s['g'])[0]) if case['back'] else lp
    if op == 'policy':
        loss, kl, clipped = ops.policy_loss(s['z'], s['label'], s['advantage'], s['old'], s['refp'], kl_weight=s['kl_weight'])
        return [loss, kl, clipped] + ([torch.autograd.grad(loss, s['z'])[0]] if case['back'] else [])
    if op == 'norm':
        return ops.grad_norm(s['grads'], max_norm=s['max_norm'])
    more = [s['copy']] if s['copy'] is not None else []
    if op == 'adamw':
        ops.adamw_step(s['params'], s['grads'], s['ms'], s['vs'], s['step_list'], s['wd'], s['lr'], BETAS, EPS, copies=s['copies'])
        return [s['p'], s['m'], s['v'], s['steps']] + more
    ops.adamw8_step(s['params'], s['grads'], s['states'], s['step_list'], s['wd'], s['lr'], BETAS, EPS, copies=s['copies'], seed=SEED)
    return [s['p'], s['m'], s['m_scale'], s['r'], s['r_scale'], s['steps']] + more


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------------- work and values
def work(case):
    op = case['op']
    if op in ('policy', 'logp'):
        rows, e = case['n'] * case['h'] * case['w'], BYTES[case['type']]
        small = 8 + 4 if op == 'logp' else 8 + 4 + (4 if case['ref'] else 0)
        back = rows * case['c'] * e + (4 * rows if op == 'logp' else 0) if case['back'] else 0
        return {'bytes': rows * (case['c'] * e + small) + back, 'flops': rows * case['c'] * (7 if case['back'] else 4)}
    n = sum(_sizes(case))
    eg = BYTES[case['grad']]
    if op == 'norm':
        return {'bytes': n * eg, 'flops': 2 * n}
    ec = BYTES[case['copy']] if case['copy'] else 0
    if op == 'adamw':
        return {'bytes': n * (24 + eg + ec), 'flops': 15 * n}
    return {'bytes': n * (12 + eg + ec) + 16 * sum(_padded(case)) // BLOCK, 'flops': 25 * n}


def exact(case, seed):
    """the operators' definitions in 64 bits, tensor by tensor and image by image"""
    s = prepare(case, seed)
    op = case['op']
    if op == 'norm':
        total = sum(float(g.double().pow(2).sum()) for g in s['grads'])
        return torch.tensor([math.sqrt(total), min(1.0, 0.5 / (math.sqrt(total) + 1e-6))], dtype=torch.float64)
    if op in ('policy', 'logp'):
        z, label = s['z'].detach(), s['label']
        valid = label >= 0
        count = max(1, int(valid.sum()))
        lps, dzs, loss, kl, cut = [], [], 0.0, 0.0, 0
        for i in range(z.shape[0]):
            q = torch.log_softmax(z[i].double(), dim=0)
            hit = torch.zeros_like(q).scatter_(0, label[i].clamp(min=0).unsqueeze(0), 1.0)
            lp = (q * hit).sum(0)
            if op == 'logp':
                up = s['g'][i].double()
            else:
                a = s['advantage'][i].double()
                ratio = torch.exp(lp - s['old'][i].double())
                inside = torch.where(a >= 0, ratio <= 1.2, ratio >= 0.8)
                value = torch.where(inside, ratio * a, (1.2 if a >= 0 else 0.8) * a)
                up = -ratio * a * inside
                cut += int((~inside & valid[i]).sum())
                loss -= float(value[valid[i]].sum())
                if s['refp'] is not None:
                    d = s['refp'][i].double() - lp
                    k = torch.expm1(d) - d
                    kl += float(k[valid[i]].sum())
                    up = up - s['kl_weight'] * torch.expm1(d)
                up = up / count
            lps.append(lp * valid[i])
            if case['back']:
                dzs.append((hit - q.exp()) * (up * valid[i]))
        dz = [torch.stack(dzs)] if case['back'] else []
        if op == 'logp':
            return (torch.stack(lps), dz[0]) if dz else torch.stack(lps)
        kl /= count
        return [torch.tensor(x, dtype=torch.float64) for x in (loss / count + s['kl_weight'] * kl, kl, cut / count)] + dz
    out = {k: torch.zeros(s[k].numel(), dtype=torch.float64, device='cuda') for k in ('p', 'm', 'v' if op == 'adamw' else 'r')}
    scales = {k: torch.zeros(sum(_padded(case)) // BLOCK, dtype=torch.float64, device='cuda') for k in ('m_scale', 'r_scale')}
    at = 0
    for i, (size, full) in enumerate(zip(_sizes(case), _padded(case))):
        t = int(s['steps'][i]) + 1
        p, g = s['params'][i].double(), s['grads'][i].double()
        if op == 'adamw':
            m, v = s['ms'][i].double(), s['vs'][i].double()
        else:
            m, ms, r, rs = (x.double() for x in s['states'][i])
            m, v = m * ms.repeat_interleave(BLOCK)[:size], (r * rs.repeat_interleave(BLOCK)[:size]) ** 2
        m = BETAS[0] * m + (1 - BETAS[0]) * g
        v = BETAS[1] * v + (1 - BETAS[1]) * g * g
        lr = float(s['lr'])
        wd = float(s['wd_t'][i])
        out['p'][at:at + size] = p * (1 - lr * wd) - lr * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
        if op == 'adamw':
            out['m'][at:at + size], out['v'][at:at + size] = m, v
        else:
            h = _exact_hash(t, i, size)
            for key, x, u in (('m', m, h & 0xFFFF), ('r', v.sqrt(), h >> 16)):
                x = torch.nn.functional.pad(x, (0, full - size)).view(-1, BLOCK)
                u = torch.nn.functional.pad(u.double() / 65536, (0, full - size)).view(-1, BLOCK)
                sc = x.abs().amax(1) / 448
                y = x.abs() / sc.clamp(min=1e-300).unsqueeze(1)
                quantum = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
                y = torch.floor(y / quantum + u) * quantum
                if key == 'r':
                    y = torch.where((x > 0) & (y == 0), torch.full_like(y, 2.0 ** -9), y)
                out[key][at:at + full] = (y * torch.sign(x)).view(-1)
                scales[key + '_scale'][at // BLOCK:(at + full) // BLOCK] = sc
        at += full
    more = [out['p']] if s['copy'] is not None else []
    if op == 'adamw':
        return [out['p'], out['m'], out['v'], None] + more
    return [out['p'], out['m'], scales['m_scale'], out['r'], scales['r_scale'], None] + more


def _exact_hash(t, tensor, size):
    def mix(x):
        x ^= x >> 16
        x = x * 0x6A09E667 % (1 << 32)
        x ^= x >> 15
        x = x * 0xBB67AE85 % (1 << 32)
        return x ^ (x >> 16)
    base = mix(SEED ^ mix(t ^ mix(tensor)))
    return mix((torch.arange(size, device='cuda') + base) % (1 << 32))
