"""Cases that the speed of further operators of language models is measured on: the two ends of a net over tokens and what goes
along them, forward and backward, through the Python entry points.

A case is a dict of plain values; ``prepare`` makes what a program holds before the call, ``run`` is one pass.  Tensors
are the transposes of the matrices (a row of a tensor is a column of a matrix, the memory is the same).  Where ``own`` is
false, ``run`` computes the operators in their plain form with elementary torch operations.

  embed       cm.embed: columns of a table by token, scaled; columns of no token (padding) are 0
  embed_grad  cm.embed_grad: gradient of the table
  scan        cm.gated_scan: h_t = a_t h_{t-1} + (1 - a_t) u_t with a = sigmoid(g), over the columns of each sequence, from a state
              to a last state
  scan_grad   cm.gated_scan_grad: gradients of gates, inputs and states
  sample      cm.sample_tokens: tokens drawn by given random numbers with temperature, top-k, min-p and top-p, and their log
              probabilities
"""
import ctypes
import math

import numpy as np
import torch

own = False

# ------------------------------------------------------------------ the cases


def listed():
    return [
        # the tokens that a few sequences have drawn, on their way into the next step: latency counts
        dict(name='embed_1024x4_v50000', kind='embed', rows=1024, cols=4, vocab=50000),
        # the tokens of a training batch
        dict(name='embed_4096x8192_v32768', kind='embed', rows=4096, cols=8192, vocab=32768),
        # the gradient of a table over a batch: most of it is zeros, frequent tokens have hundreds of columns
        dict(name='embed_grad_1024x16384_v32003', kind='embed_grad', rows=1024, cols=16384, vocab=32003),
        # tokens that are bytes, odd sides: every token has many columns
        dict(name='embed_grad_1001x4099_v256', kind='embed_grad', rows=1001, cols=4099, vocab=256),
        # one step of decoding for a few sequences
        dict(name='scan_2048x4_s4', kind='scan', units=2048, cols=4, sequences=4, ragged=False, states=True),
        # one long text
        dict(name='scan_1024x32768_s1', kind='scan', units=1024, cols=32768, sequences=1, ragged=False, states=False),
        # a packed batch of texts of any lengths, with padding behind them
        dict(name='scan_1001x4099_s37', kind='scan', units=1001, cols=4099, sequences=37, ragged=True, states=True),
        # the backward pass of a training step
        dict(name='scan_grad_2048x8192_s8', kind='scan_grad', units=2048, cols=8192, sequences=8, ragged=False, states=False),
        # ... of a packed batch cut from longer texts: states go in and out
        dict(name='scan_grad_515x10007_s11', kind='scan_grad', units=515, cols=10007, sequences=11, ragged=True, states=True),
        # the answer of one sequence: the usual limits, latency counts
        dict(name='sample_50000x1', kind='sample', rows=50000, cols=1, mode='limits'),
        # many answers at once from the whole distribution (rollouts)
        dict(name='sample_32768x512', kind='sample', rows=32768, cols=512, mode='plain'),
        # a server's batch: every request has its own settings, some are greedy
        dict(name='sample_128003x64', kind='sample', rows=128003, cols=64, mode='requests'),
    ]


def _log(rng, lo, hi):
    """A whole number, spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _aligned(rng, n, to):
    """n as it is, or (as often) the next multiple of ``to``."""
    return n if rng.random() < 0.5 else -(-n // to) * to


# of the largest listed ones
_MOST = dict(embed=1.85e8, embed_grad=1.9e8, scan=4.02e8, scan_grad=4.02e8, sample=6.71e7)


def draw(rng):
    kind = rng.choice(['embed', 'embed_grad', 'scan', 'scan_grad', 'sample', 'sample'])
    while True:
        if kind in ('embed', 'embed_grad'):
            c = dict(kind=kind, rows=_aligned(rng, _log(rng, 8, 8192), 8), cols=_log(rng, 1, 32768), vocab=_log(rng, 16, 131072))
            if c['rows'] * c['vocab'] > 1 << 27:
                continue
        elif kind in ('scan', 'scan_grad'):
            cols = _log(rng, 1, 65536)
            c = dict(kind=kind, units=_aligned(rng, _log(rng, 16, 8192), 8), cols=cols,
                     sequences=rng.choice([1, _log(rng, 1, min(cols, 512)), _log(rng, 1, min(cols, 512))]),
                     ragged=rng.random() < 0.5, states=rng.random() < 0.5)
            if not c['ragged']:
                c['cols'] = max(1, cols // c['sequences']) * c['sequences']
        else:
            c = dict(kind=kind, rows=_aligned(rng, _log(rng, 10, 131072), 64), cols=_log(rng, 1, 1024),
                     mode=rng.choice(['limits', 'plain', 'requests', 'requests']))
        if work(c)['bytes'] <= _MOST[kind]:
            return c


def _distinct(vocab, cols):
    """How many different tokens are among as many (see ``_tokens``), on average."""
    t = np.arange(1, vocab + 1, dtype=np.float64)
    return float(np.sum(1.0 - np.exp(cols * 15 / 16 * np.log1p(-np.log1p(1.0 / t) / math.log(vocab + 1)))))


def work(case):
    """Bytes: every input read once (of a table the columns of the tokens that are there), every output written once.  Operations: those
    of the formulas for an entry, an exponential or the like as one."""
    k = case['kind']
    if k in ('embed', 'embed_grad'):
        h, w, v = case['rows'], case['cols'], case['vocab']
        if k == 'embed':
            return dict(bytes=4.0 * (h * w + h * _distinct(v, w) + w), flops=1.0 * h * w)
        return dict(bytes=4.0 * (h * w * 15 / 16 + h * v + w), flops=1.0 * h * w)
    if k in ('scan', 'scan_grad'):
        f, w, n = case['units'], case['cols'], case['sequences']
        used = _used(case)
        states = 2.0 * f * n if case['states'] else 0.0
        return dict(bytes=4.0 * ((3.0 if k == 'scan' else 6.0) * f * used + states * (1 if k == 'scan' else 1.5)),
                    flops=(6.0 if k == 'scan' else 12.0) * f * used)
    h, w = case['rows'], case['cols']
    return dict(bytes=4.0 * (h * w + 7 * w), flops=5.0 * h * w)


# ------------------------------------------------------------------ what a program has in hand


class _State(object):
    """``t``: tensors by name, ``m``: the matrices over their memory (where the framework computes), ``case`` and plain values."""

    def __init__(self, case):
        self.case, self.kind, self.t, self.m, self.cm = case, case['kind'], {}, {}, None


def _used(case):
    """Columns that belong to a sequence: behind the last one of a packed batch there is padding."""
    w = case['cols']
    return w - w // 64 if case['ragged'] else w


def _tokens(gen, vocab, cols):
    """Token t about as often as 1 / (t + 1); one in sixteen is padding."""
    r = torch.rand((cols, 1), generator=gen, device='cuda', dtype=torch.float64)
    t = (torch.exp(r * math.log(vocab + 1)).long() - 1).clamp(0, vocab - 1).float()
    t[torch.rand((cols, 1), generator=gen, device='cuda') < 1 / 16] = -1.0
    return t


def _inputs(case, seed):
    """The inputs as tensors by name, and plain values."""
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    k = case['kind']

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.empty(shape, device='cuda').normal_(shift, scale, generator=gen)

    def uniform(*shape, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(shape, generator=gen, device='cuda')

    t, v = {}, {}
    if k in ('embed', 'embed_grad'):
        h, w, n = case['rows'], case['cols'], case['vocab']
        t['labels'] = _tokens(gen, n, w)
        v['mult'] = float(np.float32(math.sqrt(h)))
        if k == 'embed':
            t['table'] = normal(n, h, scale=0.02)
        else:
            t['dy'] = normal(w, h, scale=0.01)
    elif k in ('scan', 'scan_grad'):
        f, w, n = case['units'], case['cols'], case['sequences']
        # units that forget at once beside units that keep for hundreds of columns
        t['pre'] = torch.cat([normal(w, f) + uniform(1, f, lo=-1.0, hi=6.0), normal(w, f)], dim=1)
        if case['ragged']:
            used = _used(case)
            cuts = torch.randint(0, used + 1, (n - 1,), generator=gen, device='cuda').sort()[0]
            t['offsets'] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), used)]).float().view(n + 1, 1)
        if case['states']:
            t['state'] = normal(n, f, scale=0.5)
        if k == 'scan_grad':
            t['dy'] = normal(w, f, scale=0.01)
            t['y'] = torch.zeros(w, f, device='cuda')
            if case['states']:
                t['dlast'] = normal(n, f, scale=0.01)
            t['y'] = _forward(case, t, torch.float32)[0]
    else:
        h, w = case['rows'], case['cols']
        x = normal(w, h) * uniform(w, 1, lo=0.5, hi=3.5)
        # in every eighth column only part of the vocabulary is allowed
        x[:: 8, h // 2 + 1: h - h // 4] = -math.inf
        t['x'], t['uniform'] = x, torch.rand((w, 1), generator=gen, device='cuda')
        if case['mode'] == 'requests':
            t['temperature'] = uniform(w, 1, lo=0.4, hi=1.5)
            t['temperature'][3:: 8] = 0.0
            t['top_k'] = torch.randint(0, max(2, min(h, 1000)), (w, 1), generator=gen, device='cuda').float()
            t['top_k'][1:: 4] = 0.0
            t['top_p'] = uniform(w, 1, lo=0.5, hi=1.0)
            t['top_p'][2:: 4] = 1.0
            t['min_p'] = uniform(w, 1, lo=0.0, hi=0.1)
            t['min_p'][:: 2] = 0.0
        else:
            v['temperature'], v['top_k'], v['top_p'], v['min_p'] = (0.7, 50, 0.95, 0.02) if case['mode'] == 'limits' else (0.9, 0, 1.0, 0.0)
    return t, v


def _outputs(case):
    """Shapes of the tensors that the framework writes, by name."""
    k = case['kind']
    if k == 'embed':
        return dict(y=(case['cols'], case['rows']))
    if k == 'embed_grad':
        return dict(dtable=(case['vocab'], case['rows']))
    if k == 'sample':
        return dict(tokens=(case['cols'], 1), logp=(case['cols'], 1))
    f, w, n = case['units'], case['cols'], case['sequences']
    out = dict(y=(w, f)) if k == 'scan' else dict(dpre=(w, 2 * f))
    if case['states']:
        out['last' if k == 'scan' else 'dstate'] = (n, f)
    return out


def _matrix(cm, tensor):
    """The matrix over the memory of a tensor: (w, h) seen as h x w."""
    handle = cm.cudamat()
    handle.data_device = ctypes.cast(tensor.data_ptr(), type(handle.data_device))
    handle.on_device, handle.owns_data = 1, 0
    handle.size[0], handle.size[1] = tensor.shape[1], tensor.shape[0]
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
        # (columns behind the last sequence stay as they are)
        s.t.update((name, torch.zeros(shape, device='cuda')) for name, shape in _outputs(case).items())
        s.m = {name: _matrix(cm, tensor) for name, tensor in s.t.items()}
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    return _run_own(state) if own else _PLAIN[state.kind](state, state.case, state.t)


def _run_own(s):
    cm, m, k = s.cm, s.m, s.kind
    if k == 'embed':
        cm.embed(m['table'], m['labels'], target=m['y'], mult=s.mult)
    elif k == 'embed_grad':
        cm.embed_grad(m['dy'], m['labels'], target=m['dtable'], mult=s.mult)
    elif k == 'scan':
        cm.gated_scan(m['pre'], target=m['y'], offsets=m.get('offsets'), sequences=s.case['sequences'], state=m.get('state'),
                      last=m.get('last'))
    elif k == 'scan_grad':
        cm.gated_scan_grad(m['dy'], m['pre'], m['y'], target=m['dpre'], offsets=m.get('offsets'), sequences=s.case['sequences'],
                           state=m.get('state'), last_deriv=m.get('dlast'), state_grad=m.get('dstate'))
    elif s.case['mode'] == 'requests':
        cm.sample_tokens(m['x'], m['uniform'], target=m['tokens'], temperature=m['temperature'], top_k=m['top_k'], top_p=m['top_p'],
                         min_p=m['min_p'], logp=m['logp'])
    else:
        cm.sample_tokens(m['x'], m['uniform'], target=m['tokens'], temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p,
                         logp=m['logp'])
    return [s.t[name] for name in s.out]


# ------------------------------------------------------------------ plain forms


def _plain_embed(s, c, t):
    label = t['labels'].view(-1).long()
    y = t['table'][label.clamp(min=0)] * s.mult
    return [torch.where((label >= 0)[:, None], y, torch.zeros_like(y))]


def _plain_embed_grad(s, c, t):
    label = t['labels'].view(-1).long()
    token = (label >= 0)[:, None]
    dy = torch.where(token, t['dy'], torch.zeros_like(t['dy']))
    return [torch.zeros(c['vocab'], c['rows'], device='cuda').index_add_(0, label.clamp(min=0), dy) * s.mult]


def _places(c, t):
    """Of every column its sequence, whether it belongs to one, and whether it is the first of it; the borders of the sequences."""
    w, n = c['cols'], c['sequences']
    pos = torch.arange(w, device='cuda')
    if c['ragged']:
        borders = t['offsets'].view(-1).long()
    else:
        borders = torch.arange(n + 1, device='cuda') * (w // n)
    seq = torch.searchsorted(borders[1:].contiguous(), pos, right=True).clamp(max=n - 1)
    return seq, pos < borders[n], pos == borders[seq], borders


def _scan(a, b):
    """x_t = a_t x_{t-1} + b_t along the rows, in doubling steps."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _forward(c, t, dtype):
    f, n = c['units'], c['sequences']
    seq, inside, first, borders = _places(c, t)
    g, u = t['pre'][:, :f].to(dtype), t['pre'][:, f:].to(dtype)
    a, b = torch.sigmoid(g), torch.sigmoid(-g) * u
    state = t['state'].to(dtype) if c['states'] else torch.zeros(n, f, device='cuda', dtype=dtype)
    zero = torch.zeros((), device='cuda', dtype=dtype)
    b = torch.where(first[:, None], a * state[seq] + b, b)
    y = _scan(torch.where(first[:, None], zero, a), b)
    y = torch.where(inside[:, None], y, zero)
    last = torch.where((borders[1:] > borders[:-1])[:, None], y[(borders[1:] - 1).clamp(min=0)], state)
    return y, last


def _plain_scan(s, c, t):
    y, last = _forward(c, t, torch.float32)
    return [y, last] if c['states'] else [y]


def _plain_scan_grad(s, c, t):
    f, n, w = c['units'], c['sequences'], c['cols']
    seq, inside, first, borders = _places(c, t)
    g, u = t['pre'][:, :f], t['pre'][:, f:]
    a, na = torch.sigmoid(g), torch.sigmoid(-g)
    state = t['state'] if c['states'] else torch.zeros(n, f, device='cuda')
    dlast = t['dlast'] if c['states'] else torch.zeros(n, f, device='cuda')
    zero = torch.zeros((), device='cuda')
    end = inside & (torch.arange(w, device='cuda') == borders[seq + 1] - 1)
    b = torch.where(end[:, None], t['dy'] + dlast[seq], t['dy'])
    # the gate of the next column carries what comes from behind
    carry = torch.where(end[:, None], zero, torch.cat([a[1:], a.new_zeros(1, f)]))
    back = _scan(torch.flip(carry, [0]), torch.flip(b, [0]))
    back = torch.where(inside[:, None], torch.flip(back, [0]), zero)
    before = torch.where(first[:, None], state[seq], torch.cat([a.new_zeros(1, f), t['y'][:-1]]))
    out = [torch.cat([a * na * (before - u) * back, na * back], dim=1)]
    if c['states']:
        at = borders[:-1].clamp(max=w - 1)
        out.append(torch.where((borders[1:] > borders[:-1])[:, None], (a * back)[at], dlast))
    return out


def _settings(s, c, t):
    """temperature, top_k, top_p, min_p as columns of 64-bit numbers (numbers that are given to the call are 32-bit ones there)."""
    if c['mode'] == 'requests':
        return [t[name].double() for name in ('temperature', 'top_k', 'top_p', 'min_p')]
    return [torch.full((c['cols'], 1), float(np.float32(v)), device='cuda', dtype=torch.float64)
            for v in (s.temperature, s.top_k, s.top_p, s.min_p)]


def _plain_sample(s, c, t):
    # (in 64 bits: which token it is turns on borders between sums of weights)
    h = c['rows']
    temperature, top_k, top_p, min_p = _settings(s, c, t)
    greedy = temperature <= 0
    temperature = torch.where(greedy, torch.ones_like(temperature), temperature)
    best, index = torch.sort(t['x'], dim=1, descending=True, stable=True)
    z = (best.double() - best[:, :1].double()) / temperature
    e = torch.exp(z)
    rank = torch.arange(h, device='cuda')[None, :]
    keep = ((top_k < 1) | (rank < top_k)) & (e >= min_p)
    e = torch.where(keep, e, torch.zeros_like(e))
    up_to = torch.cumsum(e, dim=1)
    total = up_to[:, -1:]
    keep = keep & ((top_p >= 1) | (up_to - e < top_p * total) | (rank == 0))
    e = torch.where(keep, e, torch.zeros_like(e))
    place = torch.zeros_like(e).scatter_(1, index, e)
    up_to = torch.cumsum(place, dim=1)
    total = up_to[:, -1:]
    token = (up_to <= t['uniform'].double() * total).sum(dim=1, keepdim=True).clamp(max=h - 1)
    logp = torch.log(place.gather(1, token) / total)
    return [torch.where(greedy, index[:, :1], token).float(), torch.where(greedy, torch.zeros_like(logp), logp).float()]


_PLAIN = dict(embed=_plain_embed, embed_grad=_plain_embed_grad, scan=_plain_scan, scan_grad=_plain_scan_grad, sample=_plain_sample)


# ------------------------------------------------------------------ definitions in 64 bits


def exact(case, seed):
    t, v = _inputs(case, seed)
    k = case['kind']
    if k == 'embed':
        y = torch.zeros(case['cols'], case['rows'], device='cuda', dtype=torch.float64)
        for c, l in enumerate(t['labels'].view(-1).tolist()):
            if l >= 0:
                y[c] = v['mult'] * t['table'][int(l)].double()
        return [y]
    if k == 'embed_grad':
        # columns in the order of their tokens, sums up to each, differences between the borders of the tokens
        order = torch.argsort(t['labels'].view(-1))
        sums = torch.cumsum(t['dy'][order].double(), 0)
        sums = torch.cat([sums.new_zeros(1, case['rows']), sums])
        borders = torch.searchsorted(t['labels'].view(-1)[order].contiguous(), torch.arange(case['vocab'] + 1, device='cuda').float() - 0.5)
        return [v['mult'] * (sums[borders[1:]] - sums[borders[:-1]])]
    if k in ('scan', 'scan_grad'):
        return _scan_exact(case, t)
    return _sample_exact(case, t, v)


def _borders(case, t):
    if case['ragged']:
        return [int(b) for b in t['offsets'].view(-1).tolist()]
    each = case['cols'] // case['sequences']
    return [i * each for i in range(case['sequences'] + 1)]


def _scan_exact(case, t):
    """Column after column."""
    f, w, n = case['units'], case['cols'], case['sequences']
    borders = _borders(case, t)
    pre = t['pre'].double()
    a = 1.0 / (1.0 + torch.exp(-pre[:, :f]))
    na = torch.exp(-pre[:, :f]) * a
    u = pre[:, f:]
    if case['kind'] == 'scan':
        y = torch.zeros(w, f, device='cuda', dtype=torch.float64)
        last = torch.zeros(n, f, device='cuda', dtype=torch.float64)
        b = na * u
        for q in range(n):
            if case['states']:
                last[q] = t['state'][q].double()
            h = last[q]
            for c in range(borders[q], borders[q + 1]):
                h = torch.addcmul(b[c], a[c], h)
                y[c] = h
            last[q] = h
        return [y, last] if case['states'] else [y]
    dpre = torch.zeros(w, 2 * f, device='cuda', dtype=torch.float64)
    dstate = torch.zeros(n, f, device='cuda', dtype=torch.float64)
    y, dy = t['y'].double(), t['dy'].double()
    for q in range(n):
        back = t['dlast'][q].double() if case['states'] else torch.zeros(f, device='cuda', dtype=torch.float64)
        lo, hi = borders[q], borders[q + 1]
        if hi > lo:
            total = torch.empty(hi - lo, f, device='cuda', dtype=torch.float64)
            for c in range(hi - 1, lo - 1, -1):
                total[c - lo] = dy[c] + back
                back = total[c - lo] * a[c]
            start = t['state'][q: q + 1].double() if case['states'] else torch.zeros(1, f, device='cuda', dtype=torch.float64)
            before = torch.cat([start, y[lo: hi - 1]])
            dpre[lo: hi, f:] = total * na[lo: hi]
            dpre[lo: hi, :f] = dpre[lo: hi, f:] * a[lo: hi] * (before - u[lo: hi])
        dstate[q] = back
    return [dpre, dstate] if case['states'] else [dpre]


def _sample_exact(case, t, v):
    """Column after column, on the host."""
    h, w = case['rows'], case['cols']
    tokens, logp = np.empty((w, 1)), np.empty((w, 1))
    rows = {name: (t[name].view(-1).double().cpu().numpy() if name in t else np.full(w, float(np.float32(v[name]))))
            for name in ('temperature', 'top_k', 'top_p', 'min_p')}
    u = t['uniform'].view(-1).double().cpu().numpy()
    for c in range(w):
        x = t['x'][c].double().cpu().numpy()
        best = int(np.argmax(x))
        if rows['temperature'][c] <= 0:
            tokens[c], logp[c] = best, 0.0
            continue
        p = np.exp((x - x[best]) / rows['temperature'][c])
        order = np.argsort(-x, kind='stable')
        n = h if rows['top_k'][c] < 1 else min(h, int(rows['top_k'][c]))
        n = min(n, int(np.count_nonzero(p >= rows['min_p'][c])))
        if rows['top_p'][c] < 1:
            sums = np.cumsum(p[order[:n]])
            n = min(n, 1 + int(np.searchsorted(sums, rows['top_p'][c] * sums[-1], side='left')))
        kept = np.sort(order[:n])
        sums = np.cumsum(p[kept])
        i = min(n - 1, int(np.searchsorted(sums, u[c] * sums[-1], side='right')))
        tokens[c], logp[c] = kept[i], math.log(p[kept[i]] / sums[-1])
    return [torch.from_numpy(tokens).cuda(), torch.from_numpy(logp).cuda()]
