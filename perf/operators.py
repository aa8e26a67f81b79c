"""Cases that the speed of the operators of language models is measured on: the parts of a net over tokens that work on
one column of a features x tokens matrix at a time, forward and backward, through the Python entry points.

A case is a dict of plain values; ``prepare`` makes what a program holds before the call, ``run`` is one pass.  Tensors
are the transposes of the matrices (a row of a tensor is a column of a matrix, the memory is the same).  Where ``own`` is
false, ``run`` computes the operators in their plain form with elementary torch operations.

  norm        cm.layer_norm: every column to mean 0 and variance 1, times gain, plus bias
  norm_grad   cm.layer_norm_grad: gradients of the inputs, of gain and of bias
  gated       cm.dot_gated: act(gate) * up of the two halves of w^T x + bias
  gated_grad  cm.dot_gated_grad: gradients of the halves, the weights, the inputs and the bias
  dropout     cm.counter_dropout: entries are dropped by a counter-based generator (Philox4x32-10, Salmon et al. 2011), alone
              or onto a residual; the backward pass is the same call on the derivative
  logp        cm.log_probs: log probabilities of given tokens, entropies, log partitions and the best alternatives
  logp_grad   cm.log_probs_grad: gradient of weighted log probabilities and entropies
"""
import ctypes
import math

import numpy as np
import torch

own = False

EPS = 1e-5

# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one step of decoding for a few sequences: latency counts
        dict(name='norm_1024x4', kind='norm', rows=1024, cols=4),
        # the tokens of a training batch, streamed from memory
        dict(name='norm_4096x8192', kind='norm', rows=4096, cols=8192),
        # backward on odd sides: columns start at any 4-byte boundary, gradients of gain and bias over all tokens
        dict(name='norm_grad_4098x4099', kind='norm_grad', rows=4098, cols=4099),
        # the feed-forward half of a block for one new token: bound by the weights' bytes
        dict(name='gated_2048x5632_b1', kind='gated', inputs=2048, units=5632, cols=1, act='silu', bias=False, keep=False),
        # an ordinary layer with odd sides, its inputs to the activation kept for the backward pass
        dict(name='gated_1001x1500_b300', kind='gated', inputs=1001, units=1500, cols=300, act='gelu', bias=True, keep=True),
        # a prompt or a training batch on a wide layer: bound by the products
        dict(name='gated_4096x8192_b4096', kind='gated', inputs=4096, units=8192, cols=4096, act='silu', bias=False, keep=False),
        # the backward pass of a training step
        dict(name='gated_grad_2048x4096_b2048', kind='gated_grad', inputs=2048, units=4096, cols=2048, act='silu', bias=True),
        # a small layer's state at its batch size
        dict(name='dropout_1024x100', kind='dropout', rows=1024, cols=100, prob=0.5, residual=False),
        # what a block adds to the residual stream of a training batch
        dict(name='dropout_4096x8192', kind='dropout', rows=4096, cols=8192, prob=0.1, residual=True),
        # answers of a few sequences over a large vocabulary, with the alternatives that a server reports
        dict(name='logp_50000x4_top20', kind='logp', rows=50000, cols=4, top=20),
        # scoring a batch of tokens
        dict(name='logp_32768x2048', kind='logp', rows=32768, cols=2048, top=0),
        # the gradient of a policy's objective (log probabilities weighted by advantages, an entropy term), odd vocabulary
        dict(name='logp_grad_32003x1000', kind='logp_grad', rows=32003, cols=1000),
    ]


def _log(rng, lo, hi):
    """A whole number, spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _cols(rng, rows, lo, hi, most):
    return _log(rng, lo, max(lo, min(hi, most // rows)))


def _aligned(rng, n, to):
    """n as it is, or (as often) the next multiple of ``to``."""
    return n if rng.random() < 0.5 else -(-n // to) * to


def draw(rng):
    kind = rng.choice(['norm', 'norm_grad', 'gated', 'gated', 'gated_grad', 'dropout', 'logp', 'logp', 'logp_grad'])
    if kind in ('norm', 'norm_grad'):
        rows = _aligned(rng, _log(rng, 8, 16384), 8)
        return dict(kind=kind, rows=rows, cols=_cols(rng, rows, 1, 32768, 1 << 25))
    if kind in ('gated', 'gated_grad'):
        most = 4.0 * 4096 * 8192 * 4096 if kind == 'gated' else 2.0 * 4096 * 8192 * 4096
        act = rng.choice(['silu', 'gelu', 'sigmoid', 'relu'])
        while True:
            c = dict(kind=kind, inputs=_aligned(rng, _log(rng, 64, 4096), 32), units=_aligned(rng, _log(rng, 64, 8192), 32),
                     cols=rng.choice([1, _log(rng, 2, 64), _log(rng, 64, 4096), _log(rng, 64, 4096)]), act=act,
                     bias=rng.random() < 0.5)
            if kind == 'gated':
                c['keep'] = rng.random() < 0.5
            if work(c)['flops'] <= most:
                return c
    if kind == 'dropout':
        rows = _aligned(rng, _log(rng, 8, 16384), 8)
        return dict(kind=kind, rows=rows, cols=_cols(rng, rows, 1, 32768, 1 << 25), prob=rng.choice([0.1, 0.2, 0.5]),
                    residual=rng.random() < 0.5)
    rows = _aligned(rng, _log(rng, 10, 131072), 64)
    c = dict(kind=kind, rows=rows, cols=_cols(rng, rows, 1, 8192, 1 << 26 if kind == 'logp' else 1 << 25))
    if kind == 'logp':
        c['top'] = min(rows // 2, rng.choice([0, 0, 1, 5, 20, 50]))
    return c


def work(case):
    """Bytes: every input read once, every output written once.  Operations: those of the products, else those of the formulas
    for an entry, an exponential or the like as one."""
    k = case['kind']
    if k in ('norm', 'norm_grad', 'dropout', 'logp', 'logp_grad'):
        h, w = case['rows'], case['cols']
        n = float(h) * w
    if k == 'norm':
        return dict(bytes=4 * (2 * n + 2 * h), flops=8 * n)
    if k == 'norm_grad':
        return dict(bytes=4 * (3 * n + 3 * h), flops=18 * n)
    if k == 'dropout':
        return dict(bytes=4 * (3 if case['residual'] else 2) * n, flops=2 * n)
    if k == 'logp':
        return dict(bytes=4 * (n + 4 * w + 2 * case['top'] * w), flops=6 * n)
    if k == 'logp_grad':
        return dict(bytes=4 * (2 * n + 5 * w), flops=7 * n)
    d, f, w = case['inputs'], case['units'], case['cols']
    wb = 2 * f if case['bias'] else 0
    if k == 'gated':
        return dict(bytes=4.0 * (2 * f * d + d * w + f * w + (2 * f * w if case['keep'] else 0) + wb), flops=4.0 * d * f * w)
    return dict(bytes=4.0 * (2 * 2 * f * d + 2 * d * w + (1 + 2 + 2) * f * w + wb), flops=8.0 * d * f * w)


# ------------------------------------------------------------------ what a program has in hand


class _State(object):
    """``t``: tensors by name, ``m``: the matrices over their memory (where the framework computes), ``case`` and plain values."""

    def __init__(self, case):
        self.case, self.kind, self.t, self.m, self.cm = case, case['kind'], {}, {}, None


def _inputs(case, seed):
    """The inputs as tensors by name, and plain values."""
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    k = case['kind']

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.empty(shape, device='cuda').normal_(shift, scale, generator=gen)

    t, v = {}, {}
    if k in ('norm', 'norm_grad'):
        h, w = case['rows'], case['cols']
        # a residual stream: columns of different size, a few features far from the others
        x = normal(w, h) * torch.exp(0.5 * normal(w, 1)) + 0.5 * normal(1, h)
        x[:, :: 97] += 5.0
        t['x'], t['gain'] = x, normal(h, scale=0.2, shift=1.0)
        if k == 'norm':
            t['bias'] = normal(h, scale=0.2)
        else:
            t['dy'] = normal(w, h, scale=0.01)
    elif k in ('gated', 'gated_grad'):
        d, f, w = case['inputs'], case['units'], case['cols']
        t['x'] = normal(w, d)
        t['w'] = normal(2 * f, d, scale=1.0 / math.sqrt(d))
        if k == 'gated' and case['bias']:
            t['bias'] = normal(2 * f, scale=0.3)
        if k == 'gated_grad':
            t['dy'] = normal(w, f, scale=0.01)
            t['pre'] = normal(w, 2 * f)
    elif k == 'dropout':
        h, w = case['rows'], case['cols']
        t['x'] = normal(w, h)
        if case['residual']:
            t['residual'] = normal(w, h)
        t['step'] = torch.randint(0, 100000, (1, 1), generator=gen, device='cuda').float()
        v['seed'] = (seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 64)
        v['stream'] = seed % 96
    else:
        h, w = case['rows'], case['cols']
        x = normal(w, h) * (0.5 + 3.0 * torch.rand((w, 1), generator=gen, device='cuda'))
        # in every eighth column only part of the vocabulary is allowed, and the tokens are from it; one in sixteen is padding
        x[:: 8, h // 2 + 1: h - h // 4] = -math.inf
        labels = torch.randint(0, h, (w, 1), generator=gen, device='cuda')
        labels = torch.where((labels > h // 2) & (labels < h - h // 4), labels // 2, labels).float()
        labels[torch.rand((w, 1), generator=gen, device='cuda') < 1 / 16] = -1.0
        t['x'], t['labels'] = x, labels
        if k == 'logp_grad':
            m = x.max(dim=1, keepdim=True)[0]
            z = torch.exp(x - m).sum(dim=1, keepdim=True)
            p = torch.exp(x - m) / z
            t['log_z'] = m + torch.log(z)
            t['entropy'] = -torch.where(p > 0, p * (x - t['log_z']), torch.zeros_like(p)).sum(dim=1, keepdim=True)
            t['weight'] = normal(w, 1, scale=1.0 / w)
            t['entropy_weight'] = torch.full((w, 1), 0.01 / w, device='cuda')
    return t, v


def _outputs(case):
    """Shapes of the tensors that the framework writes, by name."""
    k = case['kind']
    if k in ('gated', 'gated_grad'):
        d, f, w = case['inputs'], case['units'], case['cols']
        if k == 'gated':
            return dict(y=(w, f), pre=(w, 2 * f)) if case['keep'] else dict(y=(w, f))
        out = dict(dpre=(w, 2 * f), dw=(2 * f, d), dx=(w, d))
        if case['bias']:
            out['dbias'] = (2 * f,)
        return out
    h, w = case['rows'], case['cols']
    if k == 'norm' or k == 'dropout':
        return dict(y=(w, h))
    if k == 'norm_grad':
        return dict(dx=(w, h), dgain=(h,), dbias=(h,))
    if k == 'logp_grad':
        return dict(dx=(w, h))
    out = dict(logp=(w, 1), entropy=(w, 1), log_z=(w, 1))
    if case['top']:
        out.update(top=(w, case['top']), top_labels=(w, case['top']))
    return out


def _matrix(cm, tensor):
    """The matrix over the memory of a tensor: (w, h) seen as h x w, a vector as one column."""
    handle = cm.cudamat()
    handle.data_device = ctypes.cast(tensor.data_ptr(), type(handle.data_device))
    handle.on_device, handle.owns_data = 1, 0
    handle.size[0], handle.size[1] = (tensor.shape[1], tensor.shape[0]) if tensor.dim() == 2 else (tensor.shape[0], 1)
    return cm.CUDAMatrix(handle)


def prepare(case, seed):
    s = _State(case)
    s.t, values = _inputs(case, seed)
    s.__dict__.update(values)
    if own:
        from deepnet_amd import cudamat as cm
        if not isinstance(cm.CUDAMatrix.ones, cm.CUDAMatrix):
            cm.cublas_init()
        s.cm = cm
        s.out = list(_outputs(case))
        s.t.update((name, torch.empty(shape, device='cuda')) for name, shape in _outputs(case).items())
        s.m = {name: _matrix(cm, tensor) for name, tensor in s.t.items()}
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    return _run_own(state) if own else _PLAIN[state.kind](state, state.case, state.t)


def _run_own(s):
    cm, m, c, k = s.cm, s.m, s.case, s.kind
    if k == 'norm':
        cm.layer_norm(m['x'], m['gain'], m['bias'], target=m['y'], eps=EPS)
    elif k == 'norm_grad':
        cm.layer_norm_grad(m['dy'], m['x'], m['gain'], target=m['dx'], gain_grad=m['dgain'], bias_grad=m['dbias'], eps=EPS)
    elif k == 'gated':
        cm.dot_gated(m['w'].T, m['x'], m.get('bias'), target=m['y'], act=c['act'], pre=m.get('pre'))
    elif k == 'gated_grad':
        cm.dot_gated_grad(m['dy'], m['w'].T, m['x'], m['pre'], target=m['dpre'], m1_grad=m['dw'], m2_grad=m['dx'],
                          bias_grad=m.get('dbias'), act=c['act'], mult=1.0 / c['cols'])
    elif k == 'dropout':
        cm.counter_dropout(m['x'], c['prob'], s.seed, stream=s.stream, step=m['step'], residual=m.get('residual'), target=m['y'])
    elif k == 'logp':
        cm.log_probs(m['x'], m['labels'], logp=m['logp'], entropy=m['entropy'], log_z=m['log_z'], top=m.get('top'),
                     top_labels=m.get('top_labels'))
    else:
        cm.log_probs_grad(m['x'], m['labels'], m['log_z'], logp_weight=m['weight'], entropy=m['entropy'],
                          entropy_weight=m['entropy_weight'], target=m['dx'])
    return [s.t[name] for name in s.out]


# ------------------------------------------------------------------ plain forms


def _act(name, g):
    if name == 'silu':
        return g * torch.sigmoid(g)
    if name == 'gelu':
        return 0.5 * g * torch.erfc(g * -math.sqrt(0.5))
    return torch.sigmoid(g) if name == 'sigmoid' else torch.clamp(g, min=0.0)


def _act_deriv(name, g):
    if name == 'relu':
        return (g > 0).to(g.dtype)
    if name == 'gelu':
        return 0.5 * torch.erfc(g * -math.sqrt(0.5)) + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    s = torch.sigmoid(g)
    return s * (1.0 - s) if name == 'sigmoid' else s * (1.0 + g * (1.0 - s))


def _plain_norm(s, c, t):
    x = t['x']
    x = x - x.mean(dim=1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS)
    return [x * r * t['gain'] + t['bias']]


def _plain_norm_grad(s, c, t):
    x, dy = t['x'], t['dy']
    x = x - x.mean(dim=1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS)
    x = x * r
    g = dy * t['gain']
    dx = r * (g - g.mean(dim=1, keepdim=True) - x * (g * x).mean(dim=1, keepdim=True))
    return [dx, (dy * x).sum(dim=0), dy.sum(dim=0)]


def _plain_gated(s, c, t):
    f = c['units']
    pre = t['x'] @ t['w'].t()
    if c['bias']:
        pre = pre + t['bias']
    y = _act(c['act'], pre[:, :f]) * pre[:, f:]
    return [y, pre] if c['keep'] else [y]


def _plain_gated_grad(s, c, t):
    f = c['units']
    gate, up = t['pre'][:, :f], t['pre'][:, f:]
    dpre = torch.cat([t['dy'] * up * _act_deriv(c['act'], gate), t['dy'] * _act(c['act'], gate)], dim=1)
    mult = 1.0 / c['cols']
    out = [dpre, (dpre.t() @ t['x']) * mult, dpre @ t['w']]
    if c['bias']:
        out.append(dpre.sum(dim=0) * mult)
    return out


_M32 = 0xFFFFFFFF


def _philox(groups, step, stream, seed):
    """Four 32-bit words for each of the numbers in ``groups`` (64-bit whole numbers; products of two words wrap)."""
    c = [groups & _M32, groups >> 32, torch.full_like(groups, 0) + step, torch.full_like(groups, stream)]
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & _M32) ^ c[1] ^ k0, b & _M32, ((a >> 32) & _M32) ^ c[3] ^ k1, a & _M32]
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack(c, dim=1)


def _border(prob):
    """A word below this drops its entry."""
    return int(math.floor(float(np.float32(prob)) * 2.0 ** 32))


def _factor(prob):
    return float(np.float32(1.0 / (1.0 - prob)))


def _plain_dropout(s, c, t):
    n = c['rows'] * c['cols']
    step = t['step'].view(torch.int32).long().view(1) & _M32
    words = _philox(torch.arange((n + 3) // 4, device='cuda'), step, s.stream, s.seed).view(-1)[:n]
    keep = (words >= _border(c['prob'])).view(c['cols'], c['rows'])
    y = torch.where(keep, t['x'] * _factor(c['prob']), torch.zeros_like(t['x']))
    return [y + t['residual']] if c['residual'] else [y]


def _plain_logp(s, c, t):
    x = t['x']
    m = x.max(dim=1, keepdim=True)[0]
    x0 = x - m
    e = torch.exp(x0)
    z = e.sum(dim=1, keepdim=True)
    log_z = m + torch.log(z)
    entropy = torch.log(z) - torch.where(e > 0, e * x0, torch.zeros_like(e)).sum(dim=1, keepdim=True) / z
    label = t['labels'].long()
    logp = x0.gather(1, label.clamp(min=0)) - torch.log(z)
    out = [torch.where(label >= 0, logp, torch.zeros_like(logp)), entropy, log_z]
    if c['top']:
        best, index = torch.sort(x, dim=1, descending=True, stable=True)
        out += [best[:, :c['top']] - log_z, index[:, :c['top']].float()]
    return out


def _plain_logp_grad(s, c, t):
    lp = t['x'] - t['log_z']
    p = torch.exp(lp)
    label = t['labels'].long()
    delta = torch.zeros_like(p).scatter_(1, label.clamp(min=0), (label >= 0).float())
    valid = (label >= 0).float()
    spread = torch.where(p > 0, p * (lp + t['entropy']), torch.zeros_like(p))
    return [t['weight'] * (delta - p * valid) - t['entropy_weight'] * spread]


_PLAIN = dict(norm=_plain_norm, norm_grad=_plain_norm_grad, gated=_plain_gated, gated_grad=_plain_gated_grad,
              dropout=_plain_dropout, logp=_plain_logp, logp_grad=_plain_logp_grad)


# ------------------------------------------------------------------ definitions in 64 bits


def exact(case, seed):
    t, v = _inputs(case, seed)
    t = {name: tensor.double() for name, tensor in t.items()}
    k = case['kind']
    if k in ('norm', 'norm_grad'):
        h = case['rows']
        mu = torch.sum(t['x'], 1) / h
        var = torch.sum(torch.square(t['x'] - mu[:, None]), 1) / h
        std = torch.sqrt(var + float(np.float32(EPS)))
        xh = (t['x'] - mu[:, None]) / std[:, None]
        if k == 'norm':
            return [torch.addcmul(t['bias'][None, :], xh, t['gain'][None, :])]
        g = t['dy'] * t['gain'][None, :]
        a, b = torch.sum(g, 1) / h, torch.sum(g * xh, 1) / h
        return [(g - a[:, None] - xh * b[:, None]) / std[:, None], torch.sum(xh * t['dy'], 0), torch.sum(t['dy'], 0)]
    if k == 'gated':
        f = case['units']
        halves = [torch.mm(t['w'][i * f:(i + 1) * f], t['x'].t().contiguous()).t() for i in (0, 1)]
        if case['bias']:
            halves = [z + t['bias'][i * f:(i + 1) * f][None, :] for i, z in enumerate(halves)]
        y = _gate_exact(case['act'], halves[0])[0] * halves[1]
        return [y.contiguous(), torch.cat(halves, 1)] if case['keep'] else [y.contiguous()]
    if k == 'gated_grad':
        f, n = case['units'], case['cols']
        value, slope = _gate_exact(case['act'], t['pre'][:, :f])
        parts = [t['dy'] * slope * t['pre'][:, f:], t['dy'] * value]
        dw = [torch.mm(part.t().contiguous(), t['x']) / n for part in parts]
        dx = torch.mm(parts[0], t['w'][:f]) + torch.mm(parts[1], t['w'][f:])
        out = [torch.cat(parts, 1), torch.cat(dw, 0), dx]
        if case['bias']:
            out.append(torch.cat([torch.sum(part, 0) / n for part in parts]))
        return out
    if k == 'dropout':
        return _dropout_exact(case, t, v)
    x = t['x']
    no_token = t['labels'] < 0
    label = torch.where(no_token, torch.zeros_like(t['labels']), t['labels']).long()
    if k == 'logp':
        log_z = torch.logsumexp(x, 1, keepdim=True)
        lp = x - log_z
        logp = torch.where(no_token, torch.zeros_like(log_z), torch.gather(lp, 1, label))
        entropy = torch.sum(torch.special.entr(torch.exp(lp)), 1, keepdim=True)
        out = [logp, entropy, log_z]
        if case['top']:
            # the best, one after the other: the greatest value, of equal ones the first
            left, values, places = x.clone(), [], []
            gone = torch.zeros_like(left, dtype=torch.bool)
            at = torch.arange(x.shape[1], device='cuda')[None, :]
            for _ in range(case['top']):
                best = torch.amax(left.masked_fill(gone, -math.inf), 1, keepdim=True)
                index = torch.amin(torch.where((left == best) & ~gone, at, x.shape[1]), 1, keepdim=True)
                gone.scatter_(1, index, True)
                values.append(best - log_z)
                places.append(index.double())
            out += [torch.cat(values, 1), torch.cat(places, 1)]
        return out
    lp = x - t['log_z']
    p = torch.exp(lp)
    grad = torch.special.entr(p) * t['entropy_weight'] - p * t['entropy'] * t['entropy_weight']
    weight = torch.where(no_token, torch.zeros_like(t['weight']), t['weight'])
    grad -= p * weight
    return [torch.scatter_add(grad, 1, label, weight)]


def _gate_exact(name, g):
    """An activation and its slope."""
    if name == 'relu':
        return torch.relu(g), torch.heaviside(g, torch.zeros_like(g))
    if name == 'gelu':
        share = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        return g * share, share + g * torch.exp(-g * g / 2.0) / math.sqrt(2.0 * math.pi)
    s = 1.0 / (1.0 + torch.exp(-g))
    up = 1.0 / (1.0 + torch.exp(g))
    return (s, s * up) if name == 'sigmoid' else (g * s, s + g * s * up)


def _dropout_exact(case, t, v):
    """Word by word from the generator's definition, products of 32-bit words put together from halves of 16 bits."""
    def product(word, factor):
        lo, hi = word & 0xFFFF, word >> 16
        flo, fhi = factor & 0xFFFF, factor >> 16
        low, mid = lo * flo, hi * flo + lo * fhi
        total = low + ((mid & 0xFFFF) << 16)
        return hi * fhi + (mid >> 16) + (total >> 32), total & 0xFFFFFFFF

    h, w = case['rows'], case['cols']
    count = h * w
    step = int(np.float32(t['step'].item()).view(np.uint32))
    keep = torch.empty(count, dtype=torch.bool, device='cuda')
    border = math.floor(float(np.float32(case['prob'])) * 4294967296.0)
    block = 1 << 22
    for first in range(0, (count + 3) // 4, block):
        g = torch.arange(first, min(first + block, (count + 3) // 4), device='cuda')
        x0, x1, x2, x3 = g % (1 << 32), torch.div(g, 1 << 32, rounding_mode='floor'), torch.full_like(g, step), torch.full_like(g, v['stream'])
        key = [v['seed'] % (1 << 32), v['seed'] // (1 << 32)]
        for r in range(10):
            hi0, lo0 = product(x0, 0xD2511F53)
            hi1, lo1 = product(x2, 0xCD9E8D57)
            x0, x1, x2, x3 = hi1 ^ x1 ^ key[0], lo1, hi0 ^ x3 ^ key[1], lo0
            key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
        words = torch.stack((x0, x1, x2, x3), 1).reshape(-1)
        keep[4 * first:4 * first + words.numel()] = (words >= border)[:count - 4 * first]
    y = t['x'] * keep.view(w, h) * float(np.float32(1.0 / (1.0 - case['prob'])))
    return [y + t['residual'] if case['residual'] else y]
