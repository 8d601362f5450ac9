"""
The sequence operators and the constraint of scores, as cases that can be timed and compared: real sizes, their inputs, their plain
form in elementary torch operations, and their definition in 64 bits.  ``own`` chooses between the plain form and the library's kernels.
"""
import math
import random

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a page's 256 lines behind the convolution stack (2 x 200 features, 150 steps, ragged), read right to left
        {'name': 'conv lines', 'op': 'conv', 'n': 256, 't': 150, 'd': 400, 'k': 4, 'dtype': 'f32', 'ragged': True, 'reverse': True, 'silu': True},
        # one long scroll per row: the largest call, memory bound
        {'name': 'conv long', 'op': 'conv', 'n': 2, 't': 16384, 'd': 4096, 'k': 4, 'dtype': 'bf16', 'ragged': False, 'reverse': False, 'silu': True},
        # one column at a time for a few streamed lines: latency
        {'name': 'conv step', 'op': 'conv_step', 'n': 8, 'd': 800, 'k': 4, 'dtype': 'f16', 'silu': True},
        # the page's lines through a state space layer
        {'name': 'scan lines', 'op': 'scan', 'n': 256, 't': 150, 'd': 400, 's': 16, 'g': 1, 'dtype': 'f32', 'ragged': True, 'reverse': True, 'gate': False},
        # one long row, gated, as a language model over labels has it: few channels, many steps
        {'name': 'scan long', 'op': 'scan', 'n': 1, 't': 8191, 'd': 2048, 's': 16, 'g': 1, 'dtype': 'bf16', 'ragged': False, 'reverse': False, 'gate': True},
        # the same layer, one label a call
        {'name': 'scan step', 'op': 'scan_step', 'n': 64, 'd': 1600, 's': 16, 'g': 1, 'dtype': 'bf16', 'gate': True},
        # self-attention over the page's lines: odd head width, distance bias, ragged
        {'name': 'attention lines', 'op': 'attention', 'n': 256, 't': 150, 'h': 8, 'hk': 8, 'e': 50, 'dtype': 'f32', 'ragged': True, 'causal': False,
         'prefix': 0, 'documents': 0, 'cap': 0.0, 'slopes': True},
        # a page's lines packed behind one another on one axis, every line a document of its own
        {'name': 'attention documents', 'op': 'attention', 'n': 1, 't': 8192, 'h': 16, 'hk': 4, 'e': 128, 'dtype': 'bf16', 'ragged': False, 'causal': True,
         'prefix': 0, 'documents': 24, 'cap': 0.0, 'slopes': False},
        # long rows, capped scores, a prefix that every step sees
        {'name': 'attention capped prefix', 'op': 'attention', 'n': 2, 't': 4000, 'h': 16, 'hk': 16, 'e': 64, 'dtype': 'f16', 'ragged': True, 'causal': True,
         'prefix': 700, 'documents': 0, 'cap': 30.0, 'slopes': False},
        # one new step against long caches: keys and values from memory once
        {'name': 'attention step', 'op': 'attention_step', 'n': 16, 't': 8192, 'h': 32, 'hk': 8, 'e': 128, 'dtype': 'bf16', 'ragged': True, 'cap': 0.0,
         'slopes': True},
        # the scores of a page's lines in front of the decoder, an alphabet for each line
        {'name': 'constrain lines', 'op': 'constrain', 'n': 256, 't': 150, 'c': 256, 'dtype': 'f32', 'history': 0, 'bias': True},
        # one step of a label model with a large inventory: penalties of what was written, biases, a grammar's mask
        {'name': 'constrain step', 'op': 'constrain', 'n': 64, 't': 1, 'c': 128000, 'dtype': 'bf16', 'history': 1024, 'bias': True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['conv', 'conv', 'conv_step', 'scan', 'scan', 'scan_step', 'attention', 'attention', 'attention', 'attention_step',
                     'constrain', 'constrain'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if op in ('conv', 'scan'):
        d = _log(rng, 24, 4096)
        t = _log(rng, 1, 8192)
        n = max(1, min(_log(rng, 1, 256), (64 << 20 if op == 'conv' else 16 << 20) // (t * d)))
        case = {'op': op, 'n': n, 't': t, 'd': d, 'dtype': dtype, 'ragged': rng.random() < 0.6, 'reverse': rng.random() < 0.4}
        if op == 'conv':
            case.update(k=rng.randint(2, 8), silu=rng.random() < 0.7)
        else:
            g = rng.choice([1, 1, 2])
            case.update(d=d - d % g, s=rng.choice([4, 8, 13, 16, 16]), g=g, gate=rng.random() < 0.5)
        return case
    if op == 'conv_step':
        return {'op': op, 'n': _log(rng, 1, 512), 'd': _log(rng, 64, 4096), 'k': rng.randint(2, 8), 'dtype': dtype, 'silu': rng.random() < 0.7}
    if op == 'scan_step':
        return {'op': op, 'n': _log(rng, 1, 256), 'd': 2 * _log(rng, 32, 2048), 's': rng.choice([8, 16, 16, 40]), 'g': rng.choice([1, 2]), 'dtype': dtype,
                'gate': rng.random() < 0.5}
    if op == 'attention':
        hk = rng.choice([1, 2, 4, 8])
        h, e = hk * rng.choice([1, 1, 2, 4]), rng.choice([32, 50, 64, 64, 80, 128, 128, 200])
        t = _log(rng, 1, 4096)
        n = max(1, min(_log(rng, 1, 64), (1 << 29) // (t * t * h)))
        docs = rng.choice([0, 0, 1 + _log(rng, 1, 16)])
        causal = rng.random() < 0.6
        return {'op': op, 'n': n, 't': t, 'h': h, 'hk': hk, 'e': e, 'dtype': dtype, 'ragged': rng.random() < 0.5, 'causal': causal,
                'prefix': _log(rng, 1, t) if causal and rng.random() < 0.4 else 0, 'documents': docs, 'cap': rng.choice([0.0, 0.0, 20.0, 50.0]),
                'slopes': rng.random() < 0.4}
    if op == 'attention_step':
        hk = rng.choice([1, 2, 4, 8])
        t, e = _log(rng, 1, 16384), rng.choice([32, 50, 64, 128, 128, 200])
        h = hk * rng.choice([1, 2, 4, 8])
        n = max(1, min(_log(rng, 1, 64), (128 << 20) // (t * hk * e)))
        return {'op': op, 'n': n, 't': t, 'h': h, 'hk': hk, 'e': e, 'dtype': dtype, 'ragged': rng.random() < 0.7, 'cap': rng.choice([0.0, 0.0, 30.0]),
                'slopes': rng.random() < 0.4}
    t = rng.choice([1, 1, _log(rng, 2, 300)])
    c = _log(rng, 30, 150000 if t == 1 else 8000)
    return {'op': op, 'n': max(1, min(_log(rng, 1, 256), (8 << 20) // (t * c))), 't': t, 'c': c, 'dtype': dtype, 'history': rng.choice([0, _log(rng, 1, 4096)]),
            'bias': rng.random() < 0.6}


def _lens(case, low=0.3):
    """The valid lengths of the rows: a property of the case, so that its work is known without a seed."""
    if not case.get('ragged'):
        return [case['t']] * case['n']
    rng = random.Random(case['n'] * 100003 + case['t'])
    return [case['t'] if i == 0 else max(1, int(case['t'] * rng.uniform(low, 1.0))) for i in range(case['n'])]


def _documents(case):
    """Lengths of the documents on the time axis, ragged, one behind the other."""
    rng = random.Random(case['t'] * 31 + case['documents'])
    cuts = sorted(rng.randint(0, case['t']) for _ in range(case['documents'] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [case['t']])]


# ----------------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    dev = 'cuda'
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case['dtype']]
    op = case['op']

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device=dev) * (hi - lo) + lo

    st = dict(case)
    if 'ragged' in case:
        st['lens'] = torch.tensor(_lens(case), dtype=torch.int32, device=dev) if case['ragged'] or op == 'attention_step' else None
    if op in ('conv', 'conv_step'):
        n, d, k = case['n'], case['d'], case['k']
        st['x'] = normal(n, case['t'], d) if op == 'conv' else normal(n, d)
        st['weight'], st['bias'] = normal(d, k, scale=k ** -0.5), normal(d, scale=0.2)
        st['state'] = normal(n, k - 1, d)
    elif op in ('scan', 'scan_step'):
        n, d, s, gr = case['n'], case['d'], case['s'], case['g']
        rows = (n, case['t']) if op == 'scan' else (n,)
        st['x'], st['dt'] = normal(*rows, d), normal(*rows, d, scale=0.5)
        st['b'], st['c'] = normal(*rows, gr, s), normal(*rows, gr, s)
        st['z'] = normal(*rows, d) if case['gate'] else None
        # decays between 1/1000 and 1/10 of a step, as such layers are initialised; softplus(bias) is that step
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), d))
        st['dt_bias'] = step + torch.log(-torch.expm1(-step))
        st['a'] = -(torch.arange(1, s + 1, device=dev, dtype=torch.float32) * uniform(0.9, 1.1, d, 1)).contiguous()
        st['skip'] = uniform(0.5, 1.5, d)
        st['state'] = normal(n, d, s, dtype=torch.float32)
    elif op in ('attention', 'attention_step'):
        n, t, h, hk, e = case['n'], case['t'], case['h'], case['hk'], case['e']
        st['q'] = normal(n, t, h, e) if op == 'attention' else normal(n, h, e)
        st['k'], st['v'] = normal(n, t, hk, e), normal(n, t, hk, e)
        st['slopes_t'] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device=dev) if case['slopes'] else None
        st['prefix_t'] = st['docs_t'] = None
        if case.get('prefix'):
            st['prefix_t'] = torch.tensor([max(0, case['prefix'] - 3 * i) for i in range(n)], dtype=torch.int32, device=dev)
        if case.get('documents'):
            ids = [i for i, w in enumerate(_documents(case)) for _ in range(w)]
            st['docs_t'] = torch.tensor(ids, dtype=torch.int32, device=dev).expand(n, t).contiguous()
    else:
        n, t, c = case['n'], case['t'], case['c']
        st['logits'] = normal(n, t, c, scale=3.0)
        allowed = torch.rand(n, (c + 31) // 32 * 32, generator=g, device=dev) < 0.7
        bits = (allowed.view(n, -1, 32).long() << torch.arange(32, device=dev)).sum(-1)
        st['mask'] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
        st['bias_t'] = normal(c, dtype=torch.float32) if case['bias'] else None
        st['seen'] = st['penalties'] = None
        if case['history']:
            # labels that a text repeats: squares of uniform numbers favour the low ones
            st['seen'] = (uniform(0.0, 1.0, n, case['history']).square() * c).int().clamp_(max=c - 1)
            st['seen_lens'] = torch.tensor([max(1, case['history'] * (i + 1) // n) for i in range(n)], dtype=torch.int32, device=dev)
            st['penalties'] = [uniform(1.05, 1.3, n), uniform(0.1, 0.5, n), uniform(0.05, 0.3, n)]
    return st


# ------------------------------------------------------------------------------------------------------------- the plain form
def _valid(lens, n, t, dev):
    if lens is None:
        return torch.ones(n, t, dtype=torch.bool, device=dev)
    return torch.arange(t, device=dev) < lens.long()[:, None]


def _order(lens, n, t, reverse, dev):
    """Position of the i-th processed step of every row."""
    i = torch.arange(t, device=dev).expand(n, t)
    if not reverse:
        return i
    lens = torch.full((n, 1), t, device=dev) if lens is None else lens.long()[:, None]
    return torch.where(i < lens, lens - 1 - i, i)


def _pick(x, order):
    return x.gather(1, order.view(*order.shape, *[1] * (x.dim() - 2)).expand_as(x))


def _silu(p):
    return p / (1 + torch.exp(-p))


def _plain_conv(st):
    n, t, d = st['x'].shape
    k, dev = st['k'], st['x'].device
    order, valid = _order(st['lens'], n, t, st['reverse'], dev), _valid(st['lens'], n, t, dev)
    x = _pick(st['x'], order) if st['reverse'] else st['x']
    x = torch.cat([st['state'], x], 1).float()
    w = st['weight'].float()
    p = sum(x[:, i:i + t] * w[:, i] for i in range(k)) + st['bias'].float()
    p = _silu(p) if st['silu'] else p
    p = torch.where(valid[..., None], p, torch.zeros((), device=dev))
    p = _pick(p, order) if st['reverse'] else p
    last = valid.sum(1)[:, None] + torch.arange(k - 1, device=dev)
    last = x.gather(1, last[..., None].expand(n, k - 1, d))
    return p.to(st['x'].dtype), last.to(st['x'].dtype)


def _plain_conv_step(st):
    x = torch.cat([st['state'], st['x'][:, None]], 1)
    p = (x.float() * st['weight'].float().t()).sum(1) + st['bias'].float()
    st['state'].copy_(x[:, 1:])
    return (_silu(p) if st['silu'] else p).to(st['x'].dtype), st['state']


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(torch.clamp(v, max=20.0))))


def _plain_scan(st):
    n, t, d = st['x'].shape
    s, gr, dev = st['s'], st['g'], st['x'].device
    order, valid = _order(st['lens'], n, t, st['reverse'], dev), _valid(st['lens'], n, t, dev)
    x, dt, b, c = (_pick(v, order).float() if st['reverse'] else v.float() for v in (st['x'], st['dt'], st['b'], st['c']))
    dt = torch.where(valid[..., None], _softplus(dt + st['dt_bias']), torch.zeros((), device=dev))
    decay = torch.exp(dt[..., None] * st['a'])
    h = (dt * x).view(n, t, gr, d // gr, 1) * b.view(n, t, gr, 1, s)
    h = h.view(n, t, d, s)
    h[:, 0] += decay[:, 0] * st['state']
    step = 1
    while step < t:        # after each turn every place holds the states of twice as many steps before it
        h = torch.cat([h[:, :step], h[:, step:] + decay[:, step:] * h[:, :-step]], 1)
        decay = torch.cat([decay[:, :step], decay[:, step:] * decay[:, :-step]], 1)
        step *= 2
    y = (h.view(n, t, gr, d // gr, s) * c.view(n, t, gr, 1, s)).sum(-1).view(n, t, d) + x * st['skip']
    y = _pick(y, order) if st['reverse'] else y
    if st['z'] is not None:
        y = y * _silu(st['z'].float())
    y = torch.where(valid[..., None], y, torch.zeros((), device=dev))
    return y.to(st['x'].dtype), h[:, -1].contiguous()


def _plain_scan_step(st):
    n, d = st['x'].shape
    s, gr = st['s'], st['g']
    x, dt = st['x'].float(), _softplus(st['dt'].float() + st['dt_bias'])
    b, c = (v.float().view(n, gr, 1, s) for v in (st['b'], st['c']))
    h = st['state'] * torch.exp(dt[..., None] * st['a']) + ((dt * x).view(n, gr, d // gr, 1) * b).view(n, d, s)
    st['state'].copy_(h)
    y = (h.view(n, gr, d // gr, s) * c).sum(-1).view(n, d) + x * st['skip']
    if st['z'] is not None:
        y = y * _silu(st['z'].float())
    return y.to(st['x'].dtype), st['state']


def _softmax_times(s, allow, v):
    low = torch.full((), -math.inf, device=s.device, dtype=s.dtype)
    s = torch.where(allow, s, low)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == low, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_attention(st):
    n, t, h, e = st['q'].shape
    dev, rep = st['q'].device, h // st['hk']
    q = st['q'].float().transpose(1, 2).contiguous()
    k = st['k'].float().permute(0, 2, 3, 1).repeat_interleave(rep, 1).contiguous()
    v = st['v'].float().transpose(1, 2).repeat_interleave(rep, 1).contiguous()
    s = torch.matmul(q, k) * e ** -0.5
    if st['cap']:
        s = st['cap'] * torch.tanh(s / st['cap'])
    i, j = torch.arange(t, device=dev)[:, None], torch.arange(t, device=dev)[None]
    if st['slopes_t'] is not None:
        s = s - st['slopes_t'][:, None, None] * (i - j).abs()
    valid = _valid(st['lens'], n, t, dev)
    allow = valid[:, None, :] & valid[:, :, None]
    if st['causal']:
        seen = (j <= i).expand(n, t, t)
        if st['prefix_t'] is not None:
            seen = seen | (j < st['prefix_t'].long()[:, None, None])
        allow = allow & seen
    if st['docs_t'] is not None:
        allow = allow & (st['docs_t'][:, :, None] == st['docs_t'][:, None, :])
    return _softmax_times(s, allow[:, None], v).transpose(1, 2).contiguous().to(st['q'].dtype)


def _plain_attention_step(st):
    n, h, e = st['q'].shape
    t, hk, dev = st['t'], st['hk'], st['q'].device
    q = st['q'].float().view(n, hk, h // hk, e)
    k, v = st['k'].float().permute(0, 2, 3, 1).contiguous(), st['v'].float().transpose(1, 2).contiguous()
    s = torch.matmul(q, k) * e ** -0.5
    if st['cap']:
        s = st['cap'] * torch.tanh(s / st['cap'])
    j, lens = torch.arange(t, device=dev), st['lens'].long()[:, None, None, None]
    if st['slopes_t'] is not None:
        s = s - st['slopes_t'].view(hk, h // hk, 1) * (lens - 1 - j).abs()
    return _softmax_times(s, j < lens, v).reshape(n, h, e).to(st['q'].dtype)


def _plain_constrain(st):
    n, t, c = st['logits'].shape
    dev = st['logits'].device
    v = st['logits'].float()
    if st['seen'] is not None:
        used = _valid(st['seen_lens'], n, st['history'], dev)
        count = torch.zeros(n, c + 1, device=dev).scatter_add_(1, torch.where(used, st['seen'].long(), c), used.float())[:, None, :c]
        r, p, f = (w[:, None, None] for w in st['penalties'])
        v = torch.where(count > 0, torch.where(v > 0, v / r, v * r), v)
        v = v - f * count
        v = torch.where(count > 0, v - p, v)
    if st['bias_t'] is not None:
        v = v + st['bias_t']
    bits = (st['mask'][..., None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1
    allowed = bits.view(n, 1, -1)[..., :c] != 0
    return torch.where(allowed, v, torch.full((), -math.inf, device=dev)).to(st['logits'].dtype)


PLAIN = {'conv': _plain_conv, 'conv_step': _plain_conv_step, 'scan': _plain_scan, 'scan_step': _plain_scan_step, 'attention': _plain_attention,
         'attention_step': _plain_attention_step, 'constrain': _plain_constrain}


# ------------------------------------------------------------------------------------------------------- the library's calls
def _own(st):
    from kraken_amd import constraints, sequence
    op = st['op']
    if op == 'conv':
        return sequence.causal_conv(st['x'], st['weight'], st['bias'], st['lens'], state=st['state'], reverse=st['reverse'],
                                    activation='silu' if st['silu'] else 'linear')
    if op == 'conv_step':
        y = sequence.causal_conv_step(st['x'], st['weight'], st['bias'], state=st['state'], activation='silu' if st['silu'] else 'linear')
        return y, st['state']
    if op == 'scan':
        return sequence.selective_scan(st['x'], st['dt'], st['a'], st['b'], st['c'], st['skip'], z=st['z'], dt_bias=st['dt_bias'], dt_softplus=True,
                                       seq_lens=st['lens'], reverse=st['reverse'], state=st['state'])
    if op == 'scan_step':
        y = sequence.selective_scan_step(st['x'], st['dt'], st['a'], st['b'], st['c'], st['skip'], z=st['z'], dt_bias=st['dt_bias'], dt_softplus=True,
                                         state=st['state'])
        return y, st['state']
    if op == 'attention':
        return sequence.attention(st['q'], st['k'], st['v'], st['lens'], causal=st['causal'], prefix_lens=st['prefix_t'], documents=st['docs_t'],
                                  slopes=st['slopes_t'], cap=st['cap'])
    if op == 'attention_step':
        return sequence.attention_step(st['q'], st['k'], st['v'], st['lens'], slopes=st['slopes_t'], cap=st['cap'])
    r, p, f = st['penalties'] or (1.0, 0.0, 0.0)
    return constraints.constrain_logits(st['logits'], mask=st['mask'], bias=st['bias_t'], history=st['seen'],
                                        history_lens=st['seen_lens'] if st['seen'] is not None else None, repetition=r, presence=p, frequency=f)


def run(state):
    return _own(state) if own else PLAIN[state['op']](state)


# ------------------------------------------------------------------------------------------------------------------- the work
def _pairs(case):
    """(query, key) pairs that the masks leave, all rows."""
    docs = _documents(case) if case['documents'] else [case['t']]
    total = 0
    for n, length in enumerate(_lens(case)):
        prefix, begin = max(0, case['prefix'] - 3 * n) if case['prefix'] else 0, 0
        for w in docs:
            lo, hi = begin, min(begin + w, length)
            begin += w
            m = max(0, hi - lo)
            if not case['causal']:
                total += m * m
            else:      # query lo + i sees its own document up to itself, and up to the prefix
                p = max(0, min(prefix, hi) - lo)
                total += p * p + (m * (m + 1) - p * (p + 1)) // 2
    return total


def work(case):
    op, size, n = case['op'], BYTES[case['dtype']], case['n']
    if op == 'conv':
        rows, d, k = sum(_lens(case)), case['d'], case['k']
        return {'bytes': size * (rows * d + n * case['t'] * d + 2 * n * (k - 1) * d + d * (k + 1)), 'flops': rows * d * (2 * k + (4 if case['silu'] else 0))}
    if op == 'conv_step':
        d, k = case['d'], case['k']
        return {'bytes': size * (2 * n * d + 2 * n * (k - 1) * d + d * (k + 1)), 'flops': n * d * (2 * k + 4)}
    if op in ('scan', 'scan_step'):
        d, s, g = case['d'], case['s'], case['g']
        rows, written = (sum(_lens(case)), n * case['t']) if op == 'scan' else (n, n)
        read = rows * (d * (3 if case['gate'] else 2) + 2 * g * s)
        return {'bytes': size * (read + written * d) + 8 * n * d * s + 4 * d * (s + 2), 'flops': rows * d * (6 * s + 10)}
    if op == 'attention':
        h, hk, e = case['h'], case['hk'], case['e']
        rows = sum(_lens(case))
        return {'bytes': size * e * (rows * (h + 2 * hk) + n * case['t'] * h), 'flops': 4 * e * h * _pairs(case)}
    if op == 'attention_step':
        h, hk, e = case['h'], case['hk'], case['e']
        rows = sum(_lens(case))
        return {'bytes': size * e * (2 * rows * hk + 2 * n * h), 'flops': 4 * e * h * rows}
    t, c = case['t'], case['c']
    return {'bytes': 2 * size * n * t * c + 4 * n * ((c + 31) // 32) + 4 * (c if case['bias'] else 0) + 4 * n * case['history'],
            'flops': n * t * c * (6 if case['history'] else 2)}


# ------------------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op, n = case['op'], case['n']
    dev = st['state'].device if 'state' in st else st['q'].device if 'q' in st else st['logits'].device

    def sigmoid(v):
        return torch.sigmoid(v)

    if op in ('conv', 'conv_step'):
        x = st['x'].double() if op == 'conv' else st['x'].double()[:, None]
        t, k = x.shape[1], case['k']
        lens = _lens(case) if op == 'conv' else [1] * n
        y, after = torch.zeros_like(x), torch.zeros(n, k - 1, case['d'], dtype=torch.float64, device=dev)
        for i, length in enumerate(lens):
            row = x[i, :length].flip(0) if case.get('reverse') else x[i, :length]
            row = torch.cat([st['state'][i].double(), row])
            windows = row.unfold(0, k, 1)                                # (length, d, k)
            p = (windows * st['weight'].double()).sum(-1) + st['bias'].double()
            p = p * sigmoid(p) if case['silu'] else p
            y[i, :length] = p.flip(0) if case.get('reverse') else p
            after[i] = row[length:]
        return (y if op == 'conv' else y[:, 0]), after
    if op in ('scan', 'scan_step'):
        one = op == 'scan_step'
        x, dt, b, c = (st[v].double()[:, None] if one else st[v].double() for v in ('x', 'dt', 'b', 'c'))
        t, per = x.shape[1], case['d'] // case['g']
        lens = [1] * n if one else _lens(case)
        step = torch.nn.functional.softplus(dt + st['dt_bias'].double())
        h, a = st['state'].double(), st['a'].double()
        y = torch.zeros_like(x)
        length = torch.tensor(lens, device=dev)
        every = torch.arange(n, device=dev)
        for i in range(t):
            live = i < length
            at = torch.where(live, length - 1 - i, torch.full_like(length, i)) if case.get('reverse') else torch.full_like(length, i)
            d_t, x_t = step[every, at], x[every, at]
            b_t, c_t = (v[every, at].repeat_interleave(per, 1) for v in (b, c))
            h = torch.where(live[:, None, None], torch.exp(d_t[..., None] * a) * h + (d_t * x_t)[..., None] * b_t, h)
            y[every, at] = torch.where(live[:, None], (h * c_t).sum(-1) + st['skip'].double() * x_t, torch.zeros_like(x_t))
        if st['z'] is not None:
            z = st['z'].double()[:, None] if one else st['z'].double()
            y = y * z * sigmoid(z)
        return (y[:, 0] if one else y), h
    if op in ('attention', 'attention_step'):
        one = op == 'attention_step'
        q = (st['q'][:, None] if one else st['q']).double()
        t, h, e = case['t'], case['h'], case['e']
        out = torch.zeros_like(q)
        places = torch.arange(t, device=dev)
        for i, length in enumerate(_lens(case)):
            p = torch.tensor([length - 1], device=dev) if one else places[:length]
            keys = places[:length]
            bad = torch.zeros(len(p), length, dtype=torch.bool, device=dev)
            if case.get('causal'):
                limit = 0 if st['prefix_t'] is None else max(0, case['prefix'] - 3 * i)
                bad = (keys[None] > p[:, None]) & (keys[None] >= limit)
            if st['docs_t'] is not None:
                bad = bad | (st['docs_t'][i, :length][:, None] != st['docs_t'][i, :length][None])
            for head in range(h):
                k, v = (st[m][i, :length, head * case['hk'] // h].double() for m in ('k', 'v'))
                s = q[i, :len(p), head] @ k.t().contiguous() / math.sqrt(e)
                s = case['cap'] * torch.tanh(s / case['cap']) if case['cap'] else s
                if case['slopes']:
                    s = s - 2.0 ** (-8.0 * (head + 1) / h) * (p[:, None] - keys[None]).abs()
                out[i, :len(p), head] = torch.softmax(s.masked_fill(bad, -math.inf), -1) @ v
        return out[:, 0] if one else out
    v = st['logits'].double()
    for i in range(n):
        if case['history']:
            seen = torch.bincount(st['seen'][i, :int(st['seen_lens'][i])].long(), minlength=case['c']).double()
            r, p, f = (float(w[i]) for w in st['penalties'])
            hit = seen > 0
            v[i] = torch.where(hit, torch.where(v[i] > 0, v[i] / r, v[i] * r), v[i]) - f * seen - p * hit.double()
        if case['bias']:
            v[i] += st['bias_t'].double()
        words = st['mask'][i].long() & 0xffffffff
        ids = torch.arange(case['c'], device=dev)
        v[i].masked_fill_((words[ids // 32] >> (ids % 32)) & 1 == 0, -math.inf)
    return v
