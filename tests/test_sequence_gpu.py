"""
The operators on sequence rows and the constraint of scores against their definitions in 64 bits, on the device.

Tolerances are counted: a result may be off by half a step of its own type (eps / 2 of its value, and half a subnormal step), and by the
roundings of the fp32 arithmetic behind it, 2^-24 of the sum of the ABSOLUTE terms for each rounding on the way.  The counts stand at each
reference, which returns (result, bound).
"""
import math

import pytest
import torch

from kraken_amd.constraints import constrain_logits, label_mask
from kraken_amd.sequence import attention, attention_step, causal_conv, causal_conv_step, selective_scan, selective_scan_step

pytestmark = pytest.mark.gpu

DEV = 'cuda'
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def check(got, want, bound, what=''):
    info = torch.finfo(got.dtype)
    tol = want.abs() * (info.eps / 2) * 1.001 + info.smallest_normal * info.eps / 2 + bound * (1 + info.eps)
    off = (got.double() - want).abs() - tol
    assert got.isfinite().all(), f'{what}: not finite'
    assert off.numel() == 0 or off.max().item() <= 0, f'{what}: {off.max().item():.3e} over the bound, at {off.flatten().argmax().item()}'


def ragged(n, t, seed=1):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, t + 1, (n,), generator=g)
    if n:
        lens[0] = t
    if n > 1:
        lens[1] = 0
    return lens


# ------------------------------------------------------------------------------------------------------------- convolution
def conv_ref(x, w, b, lens, state, silu, reverse):
    """K products and sums, the bias: 2 K + 2 roundings of sum |w x| + |b|; sigmoid's exponential and reciprocal: 8 more (|p| <= that sum
    adds |p| 2^-24 to the exponent, times p sigmoid' <= 0.23 p: within the 8 up to |p| = 20)."""
    n, t, d = x.shape
    k = w.shape[1]
    x, w = x.double(), w.double()
    b = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    after = torch.zeros(n, k - 1, d, dtype=torch.float64, device=x.device)
    for i in range(n):
        m = t if lens is None else int(lens[i])
        row = x[i, :m].flip(0) if reverse else x[i, :m]
        row = torch.cat([torch.zeros(k - 1, d, dtype=torch.float64, device=x.device) if state is None else state[i].double(), row])
        after[i] = row[m:]
        if m:
            win = row.unfold(0, k, 1)
            p, a = (win * w).sum(-1) + b, (win * w).abs().sum(-1) + b.abs()
            a = a * (2 * k + 10) * U
            p = p * torch.sigmoid(p) if silu else p
            y[i, :m], bound[i, :m] = (p.flip(0), a.flip(0)) if reverse else (p, a)
    return y, bound, after


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,t,d,k,lens,reverse,silu,state', [
    (1, 1, 1, 1, False, False, False, False), (1, 1, 5, 4, False, False, True, True), (3, 2, 7, 4, True, True, False, True),
    (4, 37, 33, 3, True, False, True, False), (4, 37, 33, 4, True, True, True, True), (2, 130, 400, 4, False, True, False, False),
    (2, 65, 257, 8, True, True, True, True), (5, 9, 64, 2, True, False, False, True), (2, 1000, 24, 5, False, False, True, True),
    (70000, 1, 3, 3, False, False, True, True), (3, 5, 16, 6, True, True, False, False), (1, 300, 2049, 7, False, False, True, False)])
def test_causal_conv(dtype, n, t, d, k, lens, reverse, silu, state):
    x, w, b = rand(n, t, d, dtype=dtype), rand(d, k, dtype=dtype, seed=1, scale=0.5), rand(d, dtype=dtype, seed=2)
    st = rand(n, k - 1, d, dtype=dtype, seed=3) if state else None
    ls = ragged(n, t) if lens else None
    got, after = causal_conv(x, w, b, ls, activation='silu' if silu else 'linear', reverse=reverse, state=st)
    if n > 100:            # the reference goes line by line
        pick = [0, 1, n - 1, 65534, 65535, 65536]
        x, got, after, st, n = x[pick], got[pick], after[pick], None if st is None else st[pick], len(pick)
    want, bound, want_after = conv_ref(x, w, b, ls, st, silu, reverse)
    check(got, want, bound, 'y')
    assert torch.equal(after.double(), want_after)


@pytest.mark.parametrize('reverse', [False, True])
def test_causal_conv_padding_is_neither_read_nor_left(reverse):
    x, w = rand(4, 50, 40), rand(40, 4, seed=1)
    lens = torch.tensor([50, 0, 17, 3])
    want, state = causal_conv(x, w, None, lens, reverse=reverse)
    dirty = x.clone()
    for i, m in enumerate(lens.tolist()):
        dirty[i, m:] = float('nan')
    for ls in (lens, lens.to(DEV), lens.int().to(DEV), lens.tolist()):
        got, st = causal_conv(dirty, w, None, ls, reverse=reverse)
        assert torch.equal(got, want) and torch.equal(st, state)
        for i, m in enumerate(lens.tolist()):
            assert not got[i, m:].any()
    alone, _ = causal_conv(x[2:3, :17], w, None, reverse=reverse)
    assert torch.equal(alone[0], want[2, :17])


def test_causal_conv_device_lengths_are_clamped():
    x, w = rand(3, 9, 8), rand(8, 4, seed=1)
    got, _ = causal_conv(x, w, None, torch.tensor([-4, 1000, 9], device=DEV))
    want, _ = causal_conv(x, w, None, [0, 9, 9])
    assert torch.equal(got, want)
    got, _ = causal_conv(x, w, None, torch.tensor([-2 ** 40, 2 ** 40 + 3, 9], device=DEV))
    assert torch.equal(got, want)


@pytest.mark.parametrize('dtype', TYPES)
def test_causal_conv_in_pieces_and_in_steps(dtype):
    x, w, b = rand(3, 41, 50, dtype=dtype), rand(50, 4, dtype=dtype, seed=1), rand(50, dtype=dtype, seed=2)
    want, last = causal_conv(x, w, b, activation='silu')
    state, parts = None, []
    for lo, hi in ((0, 1), (1, 3), (3, 4), (4, 30), (30, 41)):
        y, state = causal_conv(x[:, lo:hi], w, b, activation='silu', state=state)
        parts.append(y)
    assert torch.equal(torch.cat(parts, 1), want) and torch.equal(state, last)
    pool = torch.full((5, 3, 70), 9.0, dtype=dtype, device=DEV)       # the states are rows and columns of a larger buffer
    state = pool[1:4, :, 10:60]
    state.zero_()
    for i in range(41):
        assert torch.equal(causal_conv_step(x[:, i], w, b, state=state, activation='silu'), want[:, i])
    assert torch.equal(state, last)
    assert (pool[0] == 9).all() and (pool[4] == 9).all() and (pool[:, :, :10] == 9).all() and (pool[:, :, 60:] == 9).all()


def test_causal_conv_strides():
    w, b = rand(40, 4, seed=1), rand(40, seed=2)
    big = rand(6, 30, 100)
    want, last = causal_conv(big[::2, 3:25, 7:47].contiguous(), w, b)
    for x in (big[::2, 3:25, 7:47], big[::2, 3:25, 7:47].transpose(1, 2).contiguous().transpose(1, 2)):
        got, st = causal_conv(x, w, b)
        assert torch.equal(got, want) and torch.equal(st, last)
    one = big[:1, 3:25, 7:47]
    got, _ = causal_conv(one.expand(4, -1, -1), w, b)
    assert torch.equal(got, causal_conv(one.contiguous(), w, b)[0].expand(4, -1, -1))
    st = rand(3, 3, 40, seed=5)
    a, _ = causal_conv(big[:3, :9, :40], w, b, state=st)
    c, _ = causal_conv(big[:3, :9, :40], w, b, state=st.permute(1, 0, 2).contiguous().permute(1, 0, 2))
    assert torch.equal(a, c)


def test_causal_conv_nothing_to_do():
    w = rand(8, 4)
    st = rand(2, 3, 8, seed=1)
    y, out = causal_conv(torch.empty(2, 0, 8, device=DEV), w, state=st)
    assert y.shape == (2, 0, 8) and torch.equal(out, st)
    y, out = causal_conv(torch.empty(0, 5, 8, device=DEV), w)
    assert y.shape == (0, 5, 8) and out.shape == (0, 3, 8)
    assert causal_conv_step(torch.empty(0, 8, device=DEV), w, state=torch.empty(0, 3, 8, device=DEV)).shape == (0, 8)


# ------------------------------------------------------------------------------------------------------------------------ scan
def scan_inputs(n, t, d, s, g, dtype, gate, bias=True, seed=0):
    c = dict(x=rand(n, t, d, dtype=dtype, seed=seed), dt=rand(n, t, d, dtype=dtype, seed=seed + 1, scale=0.5),
             A=-(rand(d, s, seed=seed + 2).abs() * 4 + 0.1), B=rand(n, t, g, s, dtype=dtype, seed=seed + 3),
             C=rand(n, t, g, s, dtype=dtype, seed=seed + 4), D=rand(d, seed=seed + 5))
    k = dict(z=rand(n, t, d, dtype=dtype, seed=seed + 6) if gate else None, dt_bias=rand(d, seed=seed + 7) - 3 if bias else None)
    return c, k


def scan_ref(x, dt, A, B, C, D, z=None, dt_bias=None, softplus=True, lens=None, reverse=False, state=None):
    """Per step the decay, two products and a sum: 6 roundings of what the states hold in absolute terms, over up to T steps; the step width 8
    (softplus) and the exponent's |s A| 2^-24, which the decay itself outweighs (x e^-x < 0.4); S + 4 for the output, 8 for the gate.
    Together (6 T + S + 40) 2^-24 of the absolute sums."""
    n, t, d = x.shape
    g, s = B.shape[-2:]
    x, dt, A, B, C = x.double(), dt.double(), A.double(), B.double(), C.double()
    h = torch.zeros(n, d, s, dtype=torch.float64, device=x.device) if state is None else state.double()
    habs = h.abs()
    dt = dt if dt_bias is None else dt + dt_bias.double()
    dt = torch.nn.functional.softplus(dt) if softplus else dt
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    every = torch.arange(n, device=x.device)
    lens = torch.full((n,), t, device=x.device) if lens is None else lens.to(x.device)
    for i in range(t):
        live = i < lens
        at = torch.where(live, lens - 1 - i, i) if reverse else torch.full_like(lens, i)
        b, c = (v[every, at].repeat_interleave(d // g, 1) for v in (B, C))
        u, w = (dt[every, at] * x[every, at])[..., None] * b, torch.exp(dt[every, at][..., None] * A)
        h = torch.where(live[:, None, None], w * h + u, h)
        habs = torch.where(live[:, None, None], w * habs + u.abs(), habs)
        o, ob = (h * c).sum(-1), (habs * c.abs()).sum(-1)
        if D is not None:
            o, ob = o + D.double() * x[every, at], ob + (D.double() * x[every, at]).abs()
        y[every, at], bound[every, at] = o * live[:, None], ob * live[:, None]
    if z is not None:
        z = z.double()
        y, bound = y * z * torch.sigmoid(z), bound * (z * torch.sigmoid(z)).abs()
    c = (6 * t + s + 40) * U
    return y, bound * c, h, habs * c


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,t,d,s,g,lens,reverse,gate,state', [
    (1, 1, 1, 1, 1, False, False, False, False), (1, 1, 7, 16, 1, False, True, True, True), (3, 40, 20, 4, 2, True, False, True, True),
    (3, 40, 33, 13, 1, True, True, False, True), (2, 150, 400, 16, 1, True, True, True, False), (1, 700, 65, 16, 1, False, False, True, True),
    (1, 515, 130, 16, 2, False, True, False, True), (2, 33, 10, 40, 1, True, False, True, True), (1, 20, 6, 256, 3, False, True, True, True),
    (2, 300, 6, 100, 1, True, False, False, True), (1, 1100, 64, 8, 1, False, False, False, False), (5, 257, 192, 16, 3, True, True, True, True),
    (2, 64, 257, 17, 1, True, False, True, True)])
def test_selective_scan(dtype, n, t, d, s, g, lens, reverse, gate, state):
    c, k = scan_inputs(n, t, d, s, g, dtype, gate)
    st = rand(n, d, s, seed=9) if state else None
    ls = ragged(n, t) if lens else None
    got, after = selective_scan(**c, **k, dt_softplus=True, seq_lens=ls, reverse=reverse, state=st)
    want, bound, want_after, bound_after = scan_ref(**c, **k, lens=ls, reverse=reverse, state=st)
    check(got, want, bound, 'y')
    check(after, want_after, bound_after, 'state')


def test_selective_scan_bare_arguments():
    """No skip, no bias, no softplus, B and C without a group axis, steps that are large or zero."""
    c, _ = scan_inputs(2, 50, 12, 8, 1, torch.float32, False)
    c['dt'] = c['dt'].abs() * 3
    c['dt'][0, :10] = 0
    c['D'] = None
    flat = dict(c, B=c['B'][:, :, 0], C=c['C'][:, :, 0])
    got, after = selective_scan(**flat)
    want, bound, want_after, bound_after = scan_ref(**c, softplus=False)
    check(got, want, bound)
    check(after, want_after, bound_after)


def test_selective_scan_small_steps_keep_their_digits():
    """softplus far below zero is exp: log(1 + e) would lose it.  y = s x (one state, first step): 24 roundings of it."""
    v = torch.linspace(-30, 30, 601, device=DEV)
    one = torch.ones(1, 1, 601, device=DEV)
    y, _ = selective_scan(one, v.view(1, 1, -1), -torch.ones(601, 1, device=DEV), torch.ones(1, 1, 1, device=DEV), torch.ones(1, 1, 1, device=DEV),
                          dt_softplus=True)
    want = torch.nn.functional.softplus(v.double(), threshold=100)
    assert ((y[0, 0].double() - want).abs() / want).max().item() <= (24 + 30) * U    # 30: |v| 2^-24 in the exponent


@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('t', [60, 900])
def test_selective_scan_padding_is_neither_read_nor_left(reverse, t):
    c, k = scan_inputs(4, t, 48, 16, 1, torch.float32, True)
    lens = torch.tensor([t, 0, t // 3, 3])
    want, after = selective_scan(**c, **k, dt_softplus=True, seq_lens=lens, reverse=reverse)
    dirty = {m: (v.clone() if v.dim() > 2 else v) for m, v in c.items()}
    z = k['z'].clone()
    for i, m in enumerate(lens.tolist()):
        for name in ('x', 'dt', 'B', 'C'):
            dirty[name][i, m:] = float('nan')
        z[i, m:] = float('inf')
    got, st = selective_scan(**dirty, z=z, dt_bias=k['dt_bias'], dt_softplus=True, seq_lens=lens.to(DEV), reverse=reverse)
    assert torch.equal(got, want) and torch.equal(st, after)
    for i, m in enumerate(lens.tolist()):
        assert not got[i, m:].any()
    assert not st[1].any()


@pytest.mark.parametrize('dtype', TYPES)
def test_selective_scan_in_pieces_and_in_steps(dtype):
    """Pieces and steps carry the same fp32 state: within the whole call's own bound."""
    c, k = scan_inputs(3, 41, 50, 16, 2, dtype, True)
    want, bound, want_after, bound_after = scan_ref(**c, **k)
    cut = lambda lo, hi: {m: (v[:, lo:hi] if v is not None and v.dim() > 2 else v) for m, v in {**c, **k}.items()}  # noqa: E731
    state, parts = None, []
    for lo, hi in ((0, 1), (1, 3), (3, 30), (30, 41)):
        y, state = selective_scan(**cut(lo, hi), dt_softplus=True, state=state)
        parts.append(y)
    check(torch.cat(parts, 1), want, bound, 'pieces')
    check(state, want_after, bound_after, 'state of the pieces')
    pool = torch.full((5, 60, 16), 9.0, device=DEV)
    state = pool[1:4, 5:55]
    state.zero_()
    for i in range(41):
        step = {m: (v[:, i] if v is not None and v.dim() > 2 else v) for m, v in {**c, **k}.items()}
        y = selective_scan_step(**step, dt_softplus=True, state=state)
        check(y, want[:, i], bound[:, i], f'step {i}')
    check(state, want_after, bound_after, 'state of the steps')
    assert (pool[0] == 9).all() and (pool[4] == 9).all() and (pool[:, :5] == 9).all() and (pool[:, 55:] == 9).all()


@pytest.mark.parametrize('s', [1, 3, 16, 40, 256])
def test_selective_scan_step_sizes(s):
    c, k = scan_inputs(5, 1, 34, s, 2, torch.bfloat16, True, seed=3)
    st = rand(5, 34, s, seed=8)
    want, bound, want_after, bound_after = scan_ref(**c, **k, state=st)
    one = {m: (v[:, 0] if v is not None and v.dim() > 2 else v) for m, v in {**c, **k}.items()}
    check(selective_scan_step(**one, dt_softplus=True, state=st), want[:, 0], bound[:, 0])
    check(st, want_after, bound_after)


@pytest.mark.parametrize('t', [40, 900])
def test_selective_scan_growth_from_nothing(t):
    """A state of zero stays zero however large its factor: exp(10 * 17 steps) is infinite in fp32, and 0 times that no number."""
    x = torch.zeros(1, t, 32, device=DEV)
    A, bc = torch.full((32, 16), 10.0, device=DEV), torch.ones(1, t, 16, device=DEV)
    y, state = selective_scan(x, torch.ones_like(x), A, bc, bc)
    assert not y.any() and not state.any()


def test_selective_scan_strides():
    c, k = scan_inputs(2, 70, 48, 16, 1, torch.float32, True)
    want, after = selective_scan(**c, **k, dt_softplus=True)
    packed = torch.cat([c['x'], c['dt'], k['z'], c['B'][:, :, 0], c['C'][:, :, 0]], -1)       # one projection's columns
    x, dt, z, b, cc = packed.split([48, 48, 48, 16, 16], -1)
    got, st = selective_scan(x, dt, c['A'], b, cc, c['D'], z=z, dt_bias=k['dt_bias'], dt_softplus=True)
    assert torch.equal(got, want) and torch.equal(st, after)
    got, _ = selective_scan(c['x'].transpose(1, 2).contiguous().transpose(1, 2), dt, c['A'].t().contiguous().t(), b, cc, c['D'], z=z,
                            dt_bias=k['dt_bias'], dt_softplus=True)
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------------------------- attention
def attention_ref(q, k, v, q_lens=None, k_lens=None, causal=False, align='start', prefix=None, documents=None, slopes=None, cap=0.0, scale=None):
    """A weight's relative error: its score's absolute one.  E + 8 roundings of scale sum |q k| for the product, 16 of cap for the tanh,
    8 of the score's own size (at most 88 below the top before it vanishes); the sums of up to Tk weights: 2 Tk roundings.  Each counts
    twice (numerator and denominator).  With 16-bit values the weights are rounded to that type for the product with them: half a step
    each, and fp16 weights below 2^-14 lose up to 2^-25 of the largest."""
    n, tq, h, e = q.shape
    tk, hk = k.shape[1:3]
    dt = q.dtype
    scale = e ** -0.5 if scale is None else scale
    q, k, v = q.double().cpu(), k.double().cpu().repeat_interleave(h // hk, 2), v.double().cpu().repeat_interleave(h // hk, 2)
    out, bound = torch.zeros(n, tq, h, e, dtype=torch.float64), torch.zeros(n, tq, h, e, dtype=torch.float64)
    for i in range(n):
        ql, kl = tq if q_lens is None else int(q_lens[i]), tk if k_lens is None else int(k_lens[i])
        if not ql or not kl:
            continue
        p = torch.arange(ql) + (kl - ql if align == 'end' else 0)
        j = torch.arange(kl)
        seen = torch.ones(ql, kl, dtype=torch.bool)
        if causal:
            seen = (j[None] <= p[:, None]) | (j[None] < (0 if prefix is None else int(prefix[i])))
        if documents is not None:
            d = documents[i].cpu()
            seen = seen & (d[:ql, None] == d[None, :kl])
        qi, ki, vi = (m[i, :m_len].transpose(0, 1) for m, m_len in ((q, ql), (k, kl), (v, kl)))
        s, size = scale * qi @ ki.transpose(1, 2), abs(scale) * qi.abs() @ ki.abs().transpose(1, 2)
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - slopes.double().cpu()[:, None, None] * (p[:, None] - j[None]).abs()
        s = s.masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1).masked_fill(~seen, 0.0).nan_to_num(0.0)
        size = size.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        c = 2 * U * ((e + 8) * size + 16 * cap + 8 * 88 + 2 * kl)
        part = w @ vi.abs()
        b = c * part
        if dt != torch.float32:
            b = b + torch.finfo(dt).eps * part
        if dt == torch.float16:
            b = b + (2.0 ** -25) * w.amax(-1, keepdim=True) * (seen.double() @ vi.abs())
        out[i, :ql], bound[i, :ql] = (w @ vi).transpose(0, 1), b.transpose(0, 1)
    return out.to(DEV), bound.to(DEV)


def qkv(n, tq, tk, h, hk, e, dtype, seed=0):
    return rand(n, tq, h, e, dtype=dtype, seed=seed), rand(n, tk, hk, e, dtype=dtype, seed=seed + 1), rand(n, tk, hk, e, dtype=dtype, seed=seed + 2)


def slopes_of(h):
    return torch.tensor([2.0 ** (-8 * (i + 1) / h) for i in range(h)], device=DEV)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,t,h,hk,e,lens,causal,prefix,docs,slopes,cap', [
    (1, 1, 1, 1, 1, False, False, 0, 0, False, 0.0), (2, 2, 2, 1, 5, True, True, 0, 0, True, 0.0), (3, 33, 4, 2, 50, True, False, 0, 0, True, 0.0),
    (2, 64, 2, 2, 64, False, True, 0, 0, False, 20.0), (2, 65, 8, 1, 32, True, True, 20, 0, False, 0.0), (1, 200, 3, 1, 128, False, True, 0, 5, False, 0.0),
    (2, 129, 4, 4, 80, True, False, 0, 4, True, 5.0), (1, 300, 12, 4, 64, True, True, 150, 3, True, 30.0), (1, 140, 2, 1, 256, False, False, 0, 0, False, 0.0),
    (1, 257, 2, 2, 200, False, True, 0, 0, True, 0.0), (9, 31, 5, 5, 17, True, True, 7, 2, False, 2.0), (1, 1030, 2, 1, 128, False, True, 0, 0, False, 0.0),
    (2, 513, 16, 2, 32, True, False, 0, 0, False, 0.0), (1, 640, 1, 1, 96, False, True, 300, 0, False, 0.0)])
def test_attention(dtype, n, t, h, hk, e, lens, causal, prefix, docs, slopes, cap):
    q, k, v = qkv(n, t, t, h, hk, e, dtype)
    ls = ragged(n, t) if lens else None
    pf = torch.tensor([max(0, prefix - 3 * i) for i in range(n)]) if prefix else None
    ids = torch.sort(torch.randint(0, docs, (n, t), generator=torch.Generator().manual_seed(4)), 1)[0].int().to(DEV) if docs else None
    sl = slopes_of(h) if slopes else None
    got = attention(q, k, v, ls, causal=causal, prefix_lens=pf, documents=ids, slopes=sl, cap=cap)
    want, bound = attention_ref(q, k, v, ls, ls, causal, 'start', pf, ids, sl, cap)
    check(got, want, bound)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,tq,tk,h,hk,e,ql,kl,causal,align,prefix', [
    (2, 7, 100, 4, 2, 64, None, [100, 60], False, 'start', 0), (3, 20, 130, 4, 1, 48, [20, 5, 0], [130, 77, 20], True, 'end', 0),
    (2, 100, 40, 2, 2, 64, None, [40, 1], True, 'start', 0), (2, 50, 300, 8, 2, 128, [50, 31], [300, 31], True, 'end', 40),
    (2, 9, 5, 2, 1, 33, None, [5, 3], True, 'end', 0), (2, 3, 900, 8, 1, 64, None, [900, 0], True, 'end', 0)])
def test_attention_of_other_keys(dtype, n, tq, tk, h, hk, e, ql, kl, causal, align, prefix):
    """Cross attention and chunks behind older keys; queries in front of the first key (a chunk longer than its cache) see nothing."""
    q, k, v = qkv(n, tq, tk, h, hk, e, dtype)
    pf = [prefix] * n if prefix else None
    got = attention(q, k, v, ql, key_lens=kl, causal=causal, align=align, prefix_lens=pf)
    want, bound = attention_ref(q, k, v, ql, kl, causal, align, pf)
    check(got, want, bound)


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_documents_in_any_order(dtype):
    """Ids need not be sorted or dense, and a document of one step sees itself."""
    q, k, v = qkv(2, 200, 200, 2, 1, 64, dtype)
    ids = torch.randint(-3, 3, (2, 200), generator=torch.Generator().manual_seed(1)).int() * 1000003
    ids[0, 77] = 2 ** 31 - 1
    ids[1, 5] = -2 ** 31
    ids = ids.to(DEV)
    got = attention(q, k, v, documents=ids)
    want, bound = attention_ref(q, k, v, documents=ids)
    check(got, want, bound)
    assert torch.equal(got[0, 77], v[0, 77].expand(2, 64))


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_rows_that_see_nothing_are_zero(dtype):
    q, k, v = qkv(2, 90, 90, 2, 2, 64, dtype)
    got = attention(q, k, v, [90, 40], key_lens=[0, 90])
    assert not got[0].any() and not got[1, 40:].any() and got[1, :40].any()
    assert not attention(q, k[:, :0], v[:, :0]).any()
    assert attention(q[:, :0], k, v).shape == (2, 0, 2, 64)
    assert attention(q[:0], k[:0], v[:0]).shape == (0, 90, 2, 64)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('t,e', [(150, 64), (300, 50), (150, 13), (300, 128), (150, 200), (150, 3)])
def test_attention_what_may_not_be_seen_does_not_matter(dtype, bad, t, e):
    """Behind the valid keys, in other documents, and behind the query's position: whatever stands there."""
    q, k, v = qkv(2, t, t, 4, 2, e, dtype)
    ids = (torch.arange(t) // 47).int().expand(2, t).contiguous().to(DEV)
    lens = torch.tensor([t, 70])
    want = attention(q, k, v, lens, causal=True, documents=ids)
    for at in ((0, 100), (0, 47), (0, 149), (1, 69)):
        k2, v2 = k.clone(), v.clone()
        k2[1, 70:], v2[1, 70:] = bad, bad
        k2[at], v2[at] = bad, bad
        got = attention(q, k2, v2, lens, causal=True, documents=ids)
        same = torch.ones(2, t, dtype=torch.bool)
        same[at[0], at[1]:] = False
        same[at[0], (ids[at[0]] != ids[at]).cpu()] = True
        assert torch.equal(got[same.to(DEV)], want[same.to(DEV)]), at
        assert not got[at].isfinite().all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('e', [64, 37])
def test_attention_one_odd_value(dtype, e):
    """A single infinity among the values reaches its channel of the queries that see it, and nothing else."""
    t = 140
    q, k, v = qkv(1, t, t, 2, 1, e, dtype)
    want = attention(q, k, v, causal=True)
    for j, c, bad in ((0, 0, math.inf), (100, e - 1, -math.inf), (139, 5, math.nan), (63, 31, math.inf)):
        v2 = v.clone()
        v2[0, j, 0, c] = bad
        got = attention(q, k, v2, causal=True)
        hit = torch.zeros(1, t, 2, e, dtype=torch.bool, device=DEV)
        hit[:, j:, :, c] = True
        assert torch.equal(got[~hit], want[~hit])
        assert got[hit].isnan().all() if bad != bad else (got[hit] == bad).all()
    v2 = v.clone()
    v2[0, 10, 0, 3], v2[0, 90, 0, 3] = math.inf, -math.inf
    got = attention(q, k, v2, causal=True)
    assert (got[0, 10:90, :, 3] == math.inf).all() and got[0, 90:, :, 3].isnan().all() and torch.equal(got[0, :10], want[0, :10])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('scale', [0.0, -0.3, 2.0])
@pytest.mark.parametrize('tq', [1, 70])
def test_attention_scales(dtype, scale, tq):
    q, k, v = qkv(2, tq, 70, 4, 2, 40, dtype)
    got = attention(q, k, v, scale=scale)
    want, bound = attention_ref(q, k, v, scale=scale)
    check(got, want, bound)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('tq', [1, 70])
def test_attention_cap_far_above_the_scores(dtype, tq):
    """cap tanh(s / cap) = s (1 - (s / cap)^2 / 3 + ...): at 1e7 the scores themselves.  Eleven roundings of a score behind its product (two of the
    scale, two of 1 / log2 e, the product with both, 1 / cap and the product with it, the polynomial, cap, two of log2 e) are three more than the
    bound's E + 8 have: 3 x 40 steps at the sizes here, well within its 8 x 88, of which scores below 10 take 8 x 10."""
    q, k, v = qkv(2, tq, 200, 4, 2, 48, dtype, seed=5)
    check(attention(q, k, v, cap=1e7), *attention_ref(q, k, v), 'a cap that does nothing')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('tq', [1, 70, 300])
@pytest.mark.parametrize('e', [13, 50, 64, 100, 200])
def test_attention_keys_of_minus_infinity(dtype, tq, e):
    """Keys whose score is -inf have no weight: the result is the one without them, in any channel of a head."""
    q, k, v = qkv(2, tq, 150, 4, 2, e, dtype, seed=6)
    q = q.abs() + 0.125
    kept = [j for j in range(150) if j not in (3, 70, 149)]
    want, bound = attention_ref(q, k[:, kept], v[:, kept])
    k[:, 3, :, e - 1] = k[:, 70, :, 0] = k[:, 149, :, max(0, e - 6)] = -math.inf
    check(attention(q, k, v), want, bound, 'keys of -inf')


def test_attention_large_scores():
    """Scores of thousands: one key takes all, and growing ones move the reference point again and again."""
    t = 200
    q = torch.ones(1, t, 1, 64, device=DEV)
    k = (torch.arange(t, device=DEV).float() - 100)[None, :, None, None].expand(1, t, 1, 64).contiguous()
    v = rand(1, t, 1, 64)
    got = attention(q, k, v, causal=True)                              # scores 8 (j - 100): the next one is e^-8 of the last
    want, bound = attention_ref(q, k, v, causal=True)
    check(got, want, bound)
    # the reference point is a rounded score, so the one weight p is 2^(its rounding), not 1: fl(fl(p v) fl(1 / p)) is v within three roundings
    got = attention(q, k.flip(1) * 40, v)[0, 0]
    assert ((got - v[0, 0]).abs() <= 3 * U * 1.001 * v[0, 0].abs()).all()


def test_attention_strides():
    q, k, v = qkv(2, 70, 70, 4, 2, 64, torch.bfloat16)
    want = attention(q, k, v, causal=True)
    packed = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)       # one projection's columns
    qs, ks, vs = packed.split([256, 128, 128], -1)
    heads = lambda x: x.unflatten(-1, (-1, 64))  # noqa: E731
    assert torch.equal(attention(heads(qs), heads(ks), heads(vs), causal=True), want)
    first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]                   # (N, H, T, E) in memory
    assert torch.equal(attention(*first, causal=True), want)
    last = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)]                    # channels not adjacent
    assert torch.equal(attention(*last, causal=True), want)
    odd = torch.zeros(2 * 70 * 4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 70, 4, 64).copy_(q)
    assert torch.equal(attention(odd, k, v, causal=True), want)
    one = attention(q[:1].expand(3, -1, -1, -1), k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), causal=True)
    assert torch.equal(one, want[:1].expand(3, -1, -1, -1))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,t,h,hk,e,slopes,cap', [
    (1, 1, 1, 1, 1, False, 0.0), (3, 50, 8, 2, 50, True, 0.0), (2, 700, 8, 1, 64, False, 10.0), (4, 2048, 32, 8, 128, True, 0.0),
    (2, 3001, 6, 2, 80, True, 30.0), (1, 5000, 3, 1, 200, False, 0.0), (2, 300, 16, 1, 256, False, 0.0), (40, 257, 4, 4, 33, False, 0.0)])
def test_attention_step(dtype, n, t, h, hk, e, slopes, cap):
    q, k, v = qkv(n, 1, t, h, hk, e, dtype)
    ls = ragged(n, t)
    sl = slopes_of(h) if slopes else None
    got = attention_step(q[:, 0], k, v, ls, slopes=sl, cap=cap)
    want, bound = attention_ref(q, k, v, None, ls, align='end', slopes=sl, cap=cap)
    check(got, want[:, 0], bound[:, 0])
    k2, v2 = k.clone(), v.clone()
    for i, m in enumerate(ls.tolist()):
        k2[i, m:], v2[i, m:] = float('nan'), float('inf')
    assert torch.equal(attention_step(q[:, 0], k2, v2, ls.to(DEV), slopes=sl, cap=cap), got)


def test_attention_step_far_into_a_large_buffer():
    """Caches whose rows lie over 2^31 elements apart."""
    rows, t = 2 ** 31 // (2 * 64) + 5000, 600
    buf = torch.empty(2, rows, 2, 64, dtype=torch.bfloat16, device=DEV)
    q, k, v = qkv(2, 1, t, 4, 2, 64, torch.bfloat16)
    buf[:, -2 * t:-t], buf[:, -t:] = k, v
    ls = [t, 401]
    got = attention_step(q[:, 0], buf[:, -2 * t:-t], buf[:, -t:], ls)
    assert torch.equal(got, attention_step(q[:, 0], k, v, ls))
    got = attention(q.expand(-1, 3, -1, -1), buf[:, -2 * t:-t], buf[:, -t:], key_lens=ls)
    assert torch.equal(got, attention(q.expand(-1, 3, -1, -1), k, v, key_lens=ls))


def test_attention_many_lines():
    q, k, v = qkv(70000, 2, 2, 1, 1, 8, torch.float32)
    got = attention(q, k, v, causal=True)
    assert torch.equal(got[:, 0], v[:, 0])
    pick = [0, 1, 65535, 65536, 69999]
    want, bound = attention_ref(q[pick], k[pick], v[pick], causal=True)
    check(got[pick], want, bound)


def test_attention_step_follows_the_whole_line():
    """One step at a time over a growing cache = the causal call: within both bounds."""
    q, k, v = qkv(2, 40, 40, 4, 2, 64, torch.float32)
    sl = slopes_of(4)
    want, bound = attention_ref(q, k, v, causal=True, slopes=sl, cap=8.0)
    for i in range(40):
        check(attention_step(q[:, i], k, v, [i + 1] * 2, slopes=sl, cap=8.0), want[:, i], bound[:, i], f'step {i}')
    check(attention(q[:, 25:], k, v, key_lens=[40, 40], causal=True, align='end', slopes=sl, cap=8.0), want[:, 25:], bound[:, 25:], 'chunk')


# ------------------------------------------------------------------------------------------------------------------ constraint
def constrain_ref(x, mask=None, bias=None, history=None, lens=None, rep=1.0, pres=0.0, freq=0.0):
    """In fp32 and in the kernel's order, each operation rounded on its own: equal bit for bit."""
    n, t, c = x.shape
    v = x.float().cpu().clone()
    for i in range(n):
        if history is not None:
            row = history[i].cpu()
            row = row if lens is None else row[:int(lens[i])]
            row = row[(row >= 0) & (row < c)]
            cnt = torch.bincount(row.long(), minlength=c).float()
            r, p, f = (w[i].cpu() if isinstance(w, torch.Tensor) else torch.tensor(w) for w in (rep, pres, freq))
            hit = cnt > 0
            u = torch.where(v[i] > 0, v[i] / r, v[i] * r) - f * cnt - p
            v[i] = torch.where(hit, u, v[i])
        if bias is not None:
            v[i] = v[i] + (bias if bias.dim() == 1 else bias[i]).cpu()
        if mask is not None:
            w = mask if mask.dim() == 3 else mask[:, None]
            w = w[i if w.shape[0] > 1 else 0].cpu().long() & 0xffffffff
            ok = ((w[:, torch.arange(c) // 32] >> (torch.arange(c) % 32)) & 1) != 0
            v[i] = torch.where(ok.expand(t, c), v[i], torch.tensor(-math.inf))
    return v.to(x.dtype).to(x.device)


def random_mask(n, t, c, seed=0):
    w = torch.randint(-2 ** 31, 2 ** 31, (n, t, (c + 31) // 32), generator=torch.Generator().manual_seed(seed))
    return w.int().to(DEV)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,t,c,hist,mask_t,per_line', [
    (1, 1, 1, 0, 1, False), (3, 7, 33, 5, 7, True), (2, 150, 256, 0, 1, False), (4, 1, 5000, 300, 1, True), (2, 3, 4097, 64, 1, False),
    (1, 40, 9001, 1000, 40, True), (5, 2, 31, 2000, 1, True), (2, 300, 95, 12, 1, False), (1, 1, 130001, 4096, 1, False)])
def test_constrain_logits(dtype, n, t, c, hist, mask_t, per_line):
    x = rand(n, t, c, dtype=dtype, scale=4.0)
    g = torch.Generator().manual_seed(3)
    mask = random_mask(n, mask_t, c)
    bias = rand(n, c, seed=2) if per_line else rand(c, seed=2)
    kw, ref = {}, {}
    if hist:
        h = (torch.rand(n, hist, generator=g).square() * (c + 4)).long() - 2          # some labels outside [0, c)
        lens = ragged(n, hist)
        pen = [torch.rand(n, generator=g).to(DEV) + lo for lo in (1.05, 0.1, 0.05)] if per_line else [1.25, 0.4, 0.15]
        kw = dict(history=h.to(DEV), history_lens=lens, repetition=pen[0], presence=pen[1], frequency=pen[2])
        ref = dict(history=h, lens=lens, rep=pen[0], pres=pen[1], freq=pen[2])
    want = constrain_ref(x, mask, bias, **ref)
    assert torch.equal(constrain_logits(x, mask=mask, bias=bias, **kw), want)
    if hist:
        assert torch.equal(constrain_logits(x, mask=mask, bias=bias, **dict(kw, history=kw['history'].int())), want)
    out = x.clone()
    assert constrain_logits(out, mask=mask, bias=bias, out=out, **kw) is out
    assert torch.equal(out, want)
    if t == 1:
        assert torch.equal(constrain_logits(x[:, 0], mask=mask[:, 0], bias=bias, **kw), want[:, 0])


def test_constrain_logits_masked_scores_do_not_matter():
    x = rand(2, 3, 70)
    x[0, 0, 3], x[0, 1, 4], x[1, 2, 69] = float('nan'), float('inf'), torch.finfo(torch.float32).min
    mask = label_mask([[c for c in range(70) if c not in (3, 4)], []], 70, blank=False)
    y = constrain_logits(x, mask=mask)
    assert (y[0, :, 3:5] == -math.inf).all() and y[0, :, :3].isfinite().all() and y[0, :, 5:].isfinite().all()
    assert (y[1] == -math.inf).all()
    assert torch.equal(constrain_logits(x[:, :, :3]), x[:, :, :3])


def test_constrain_logits_broadcast_and_strides():
    x = rand(4, 6, 100)
    mask = random_mask(1, 1, 100, seed=2)
    want = constrain_ref(x, mask.expand(4, 1, 4))
    assert torch.equal(constrain_logits(x, mask=mask), want)
    assert torch.equal(constrain_logits(x, mask=mask[:, 0]), want)
    assert torch.equal(constrain_logits(x, mask=mask.expand(4, 6, 4)), want)
    big = torch.full((4, 9, 140), 5.0, device=DEV)
    view = big[:, 2:8, 11:111]
    view.copy_(x)
    got = constrain_logits(view, mask=mask, out=view)
    assert torch.equal(got, want)
    big[:, 2:8, 11:111] = 5.0
    assert (big == 5).all()
    assert torch.equal(constrain_logits(x.transpose(1, 2).contiguous().transpose(1, 2), mask=mask), want)


def test_constrain_logits_many_lines():
    x = rand(70000, 9)
    h = torch.randint(0, 9, (70000, 4), generator=torch.Generator().manual_seed(1)).to(DEV)
    got = constrain_logits(x, history=h, presence=0.5)
    hit = torch.zeros(70000, 9, dtype=torch.bool, device=DEV).scatter_(1, h, True)
    assert torch.equal(got, torch.where(hit, x - 0.5, x))


def test_constrain_logits_nothing_to_do():
    assert constrain_logits(torch.empty(0, 4, 5, device=DEV)).shape == (0, 4, 5)
    assert constrain_logits(torch.empty(2, 0, 5, device=DEV)).shape == (2, 0, 5)
    x = rand(2, 5)
    assert torch.equal(constrain_logits(x, history=torch.empty(2, 0, dtype=torch.int64, device=DEV), repetition=2.0), x)
    assert torch.equal(constrain_logits(x, history=torch.zeros(2, 4, dtype=torch.int64, device=DEV), history_lens=[0, 0], repetition=2.0), x)


# ---------------------------------------------------------------------------------------------------------- how they are called
def everything(seed=0, dtype=torch.bfloat16):
    """One call of each operator, on lengths that live on the device: (function of no arguments -> list of results, inputs)."""
    n, t, d = 3, 300, 96
    lens = torch.tensor([300, 120, 7], dtype=torch.int32, device=DEV)
    x, w = rand(n, t, d, dtype=dtype, seed=seed), rand(d, 4, dtype=dtype, seed=seed + 1)
    c, k = scan_inputs(n, t, d, 16, 1, dtype, True, seed=seed)
    q, kk, vv = qkv(n, t, t, 4, 2, 64, dtype, seed=seed)
    q1, kc, vc = qkv(n, 1, 2000, 4, 2, 64, dtype, seed=seed + 5)
    cl = torch.tensor([2000, 1, 1313], dtype=torch.int32, device=DEV)
    sc, mask = rand(n, t, 200, dtype=dtype, seed=seed), random_mask(n, 1, 200, seed)
    hist = torch.randint(0, 200, (n, 40), generator=torch.Generator().manual_seed(seed)).to(DEV)

    def run():
        y, s = causal_conv(x, w, None, lens, activation='silu', reverse=True)
        z, h = selective_scan(**c, **k, dt_softplus=True, seq_lens=lens)
        return [y, s, z, h, attention(q, kk, vv, lens, causal=True), attention_step(q1[:, 0], kc, vc, cl),
                constrain_logits(sc, mask=mask, history=hist, repetition=1.3, presence=0.2, frequency=0.1)]
    return run, (x, c['x'], q, q1, sc)


def test_operators_on_another_stream():
    run, _ = everything()
    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_give_the_same_bits_twice():
    run, _ = everything(seed=3)
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_operators_captured_and_replayed():
    """Two graphs, whose workspaces must not be one another's, replayed with eager work between and new inputs."""
    runs = [everything(seed=s) for s in (0, 50)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for run, _ in runs:
            run()
    side.synchronize()
    graphs, outs = [], []
    for run, _ in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for turn in range(4):
        for _, inputs in runs:
            for x in inputs:
                x.mul_(0.9)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (run, _), out in zip(runs, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, run())), turn


def test_sequence_block_to_strings():
    """The operators as they are used: a block over ragged lines (convolution, scan, attention), scores, an alphabet per line, the decoder."""
    from kraken_amd.ctc_decoder import greedy_decoder
    n, t, d, classes = 4, 60, 64, 40
    lens = torch.tensor([60, 41, 1, 23])
    x = rand(n, t, d, scale=1.0)
    w, proj, head = rand(d, 4, seed=1), rand(d, 2 * 16, seed=2, scale=0.2), rand(d, classes, seed=3)
    A, heads = -(torch.arange(1, 17, device=DEV).float().expand(d, 16)).contiguous(), lambda v: v.unflatten(-1, (4, 16))
    allowed = [list(range(1, 9)), list(range(20, 40)), [5], None]

    def block(rows, ls):
        u, _ = causal_conv(rows, w, None, ls, activation='silu')
        b, c = (u @ proj).split(16, -1)
        y, _ = selective_scan(u, u - 2, A, b, c, dt_softplus=True, seq_lens=ls, reverse=True)
        y = y + attention(heads(y), heads(u), heads(u), ls, slopes=slopes_of(4)).flatten(2)
        return y @ head
    scores = block(x, lens)
    lines = greedy_decoder(constrain_logits(scores, mask=label_mask(allowed, classes)).transpose(1, 2), lens)
    assert [len(line) > 0 for line in lines][:2] == [True, True]
    for line, labels, m in zip(lines, allowed, lens.tolist()):
        assert all((labels is None or lab in labels) and 0 < lab < classes and end < m for lab, _, end, _ in line)
    for i, m in enumerate(lens.tolist()):           # a line does not depend on its batch: fp32 matrix products of other shapes sum in other orders
        alone = block(x[i:i + 1, :m].contiguous(), None)
        scale = scores[i, :m].abs().max().item()
        assert (alone[0] - scores[i, :m]).abs().max().item() <= 1e-4 * scale + 1e-6
        assert not scores[i, m:].any()


# ------------------------------------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_recurrences():
    x, w = rand(2, 9, 8), rand(8, 4)
    st = rand(2, 3, 8)
    for bad in (lambda: causal_conv(x.cpu(), w), lambda: causal_conv(x.double(), w), lambda: causal_conv(x[0], w), lambda: causal_conv(x, w.half()),
                lambda: causal_conv(x, rand(8, 9)), lambda: causal_conv(x, w[:4]), lambda: causal_conv(x, w, rand(7)), lambda: causal_conv(x, w.cpu()),
                lambda: causal_conv(x, w, None, [9]), lambda: causal_conv(x, w, None, [9, 10]), lambda: causal_conv(x, w, None, [-1, 3]),
                lambda: causal_conv(x, w, None, [1.5, 3]), lambda: causal_conv(x, w, activation='relu'), lambda: causal_conv(x, w, state=st[:1]),
                lambda: causal_conv(x, w, state=st.half()), lambda: causal_conv(x.requires_grad_(), w),
                lambda: causal_conv_step(x.detach()[:, 0], w, state=st[:1].expand(2, 3, 8)),
                lambda: causal_conv_step(x.detach()[:, 0], w, state=st.transpose(1, 2).contiguous().transpose(1, 2)),
                lambda: causal_conv_step(st[:, 2], w, state=st), lambda: causal_conv_step(x.detach()[:, 0], w, state=st.double())):
        with pytest.raises(ValueError):
            bad()
    c, k = scan_inputs(2, 9, 12, 4, 2, torch.float32, True)
    one = {m: (v[:, 0] if v.dim() > 2 else v) for m, v in {**c, **k}.items()}
    st = rand(2, 12, 4)
    for bad in (dict(c, dt=c['dt'].half()), dict(c, A=c['A'].half()), dict(c, A=rand(12, 257)), dict(c, B=c['B'][..., :3]), dict(c, C=c['C'][:, :, :1]),
                dict(c, B=rand(2, 9, 5, 4), C=rand(2, 9, 5, 4)), dict(c, D=c['D'][:3]), dict(c, x=c['x'].cpu()), dict(c, z=c['x'][:1]),
                dict(c, dt_bias=c['D'].double()), dict(c, state=st[:1]), dict(c, seq_lens=[10, 1]), dict(c, seq_lens=torch.zeros(3, device=DEV).int())):
        with pytest.raises(ValueError):
            selective_scan(**bad)
    for state in (st[:1].expand(2, 12, 4), st.transpose(1, 2).contiguous().transpose(1, 2), st.half(), st[:, :3]):
        with pytest.raises(ValueError):
            selective_scan_step(**one, state=state)
    shared = rand(2, 60)
    with pytest.raises(ValueError):
        selective_scan_step(**dict(one, x=shared[:, :12]), state=shared.as_strided((2, 12, 4), (60, 4, 1)))


def test_refusals_of_attention():
    q, k, v = qkv(2, 9, 9, 4, 2, 16, torch.float32)
    for bad in (dict(q=q.cpu()), dict(q=q.double()), dict(q=q[0]), dict(k=k.half()), dict(v=v[:, :8]), dict(q=q[:, :, :3]), dict(k=k[..., :8], v=v[..., :8]),
                dict(seq_lens=[9]), dict(seq_lens=[10, 1]), dict(key_lens=[1, 10]), dict(align='left'), dict(prefix_lens=[1, 1]), dict(cap=-1.0),
                dict(cap=float('nan')), dict(scale=float('inf')), dict(slopes=slopes_of(3)), dict(slopes=slopes_of(4).half()),
                dict(documents=torch.zeros(2, 9, device=DEV).long()), dict(documents=torch.zeros(1, 9, device=DEV).int()),
                dict(q=q[:, :5], documents=torch.zeros(2, 5, device=DEV).int()), dict(q=rand(2, 9, 4, 257), k=rand(2, 9, 2, 257), v=rand(2, 9, 2, 257)),
                dict(k=k[:, :, :0], v=v[:, :, :0]), dict(k=k.clone().requires_grad_())):
        with pytest.raises(ValueError):
            attention(**{**dict(q=q, k=k, v=v), **bad})
    with torch.no_grad():
        attention(q, k.clone().requires_grad_(), v)
    with pytest.raises(ValueError):
        attention_step(q, k, v, [1, 1])
    with pytest.raises(ValueError):
        attention_step(q[:, 0], k, v, [1, 10])


def test_refusals_of_constrain_logits():
    x = rand(2, 3, 40)
    h = torch.zeros(2, 5, dtype=torch.int64, device=DEV)
    for bad in (dict(logits=x.cpu()), dict(logits=x.double()), dict(logits=x[0, 0]), dict(mask=random_mask(2, 1, 65)), dict(mask=random_mask(3, 1, 40)),
                dict(mask=random_mask(2, 2, 40)), dict(mask=random_mask(2, 1, 40).long()), dict(bias=rand(39)), dict(bias=rand(40).half()), dict(bias=rand(3, 40)),
                dict(history=h.float()), dict(history=h[:1]), dict(history=h, history_lens=[6, 0]), dict(history_lens=[1, 1]), dict(history=h, repetition=0.0),
                dict(history=h, repetition=float('nan')), dict(history=h, presence=rand(3)), dict(history=h, frequency=rand(2).half()), dict(out=rand(2, 3, 41)),
                dict(out=x.half()), dict(out=x[:1].expand(2, 3, 40)), dict(out=rand(2, 40, 3).transpose(1, 2))):
        with pytest.raises(ValueError):
            constrain_logits(**{**dict(logits=x), **bad})
    big = rand(3, 3, 40)
    with pytest.raises(ValueError):
        constrain_logits(big[:2], out=big[1:])
    with pytest.raises(ValueError):
        label_mask([[40]], 40)


# ------------------------------------------------------------------------------------------- weights of 16-bit attention keep their digits
def whole_weights_ref(q, k, v, *args, **kw):
    """`attention_ref` without its allowance for weights in 16 bits.  They are taken as the sum of two 16-bit numbers: half a step of half a
    step off, 2^-16 (bf16) or 2^-22 (fp16) of the weight, and fp16's absolute half step of 2^-25 where the row's largest weight is 2^7 or more:
    2^-32 of it, for every key."""
    want, bound = attention_ref(q.float(), k.float(), v.float(), *args, **kw)
    if q.dtype != torch.float32:
        part, _ = attention_ref(q.float(), k.float(), v.float().abs(), *args, **kw)
        bound = bound + part * (2.0 ** -16 if q.dtype == torch.bfloat16 else 2.0 ** -22)
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -32 * k.shape[1] * v.float().abs().max().item()
    return want, bound


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,t,h,hk,e,lens,causal,prefix,docs,slopes,cap', [
    (2, 3, 2, 1, 16, True, True, 0, 0, False, 0.0), (3, 150, 4, 4, 50, True, False, 0, 0, True, 0.0), (1, 300, 4, 2, 64, False, True, 90, 0, False, 30.0),
    (1, 300, 4, 1, 128, False, True, 0, 5, False, 0.0), (1, 140, 2, 2, 200, False, False, 0, 0, False, 0.0), (2, 130, 2, 1, 13, True, True, 0, 3, True, 5.0),
    (1, 1030, 2, 1, 96, False, True, 0, 0, False, 0.0)])
def test_attention_is_rounded_once(dtype, n, t, h, hk, e, lens, causal, prefix, docs, slopes, cap):
    q, k, v = qkv(n, t, t, h, hk, e, dtype, seed=11)
    ls = ragged(n, t) if lens else None
    pf = [prefix] * n if prefix else None
    ids = torch.sort(torch.randint(0, docs, (n, t), generator=torch.Generator().manual_seed(4)), 1)[0].int().to(DEV) if docs else None
    sl = slopes_of(h) if slopes else None
    got = attention(q, k, v, ls, causal=causal, prefix_lens=pf, documents=ids, slopes=sl, cap=cap)
    check(got, *whole_weights_ref(q, k, v, ls, ls, causal, 'start', pf, ids, sl, cap))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,t,h,hk,e,slopes,cap', [(3, 50, 8, 2, 50, True, 0.0), (2, 700, 8, 1, 64, False, 10.0), (1, 3001, 6, 2, 80, True, 0.0)])
def test_attention_step_is_rounded_once(dtype, n, t, h, hk, e, slopes, cap):
    q, k, v = qkv(n, 1, t, h, hk, e, dtype, seed=12)
    ls = ragged(n, t)
    sl = slopes_of(h) if slopes else None
    want, bound = whole_weights_ref(q, k, v, None, ls, align='end', slopes=sl, cap=cap)
    check(attention_step(q[:, 0], k, v, ls, slopes=sl, cap=cap), want[:, 0], bound[:, 0])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('causal', [False, True])
def test_attention_infinite_values_that_every_query_sees(dtype, causal):
    """A weight whose lower part is zero or negative must not turn an infinity into no number."""
    q, k, v = qkv(1, 200, 200, 2, 1, 64, dtype, seed=14)
    want = attention(q, k, v, causal=causal)
    v[0, 0, 0, 7], v[0, 1, 0, 9] = math.inf, -math.inf
    got = attention(q, k, v, causal=causal)
    assert (got[..., 7] == math.inf).all() and (got[:, 1:, :, 9] == -math.inf).all()
    rest = [c for c in range(64) if c not in (7, 9)]
    assert torch.equal(got[..., rest], want[..., rest])


# ---------------------------------------------------------------------------------------- the scan's range does not depend on how it is cut
@pytest.mark.parametrize('n', [1, 800])
def test_selective_scan_small_state_under_growth(n):
    """exp(6) a step for 20 steps, exp(-6) for 20: the state goes from 1e-30 to 1e22 and back, a chunk's factor passes float32's range.  One row is
    cut into chunks, 800 rows are not.  Each of the up to 200 exponents is off by 6 / ln 2 steps of 2^-24 and the sums of a chunk's by as much again:
    2 x 9 a step on top of the reference's 6."""
    t, d, s = 200, 64, 4
    dt = (torch.where(torch.arange(t) % 40 < 20, 1.0, -1.0) * torch.linspace(0.9, 1.0, d)[:, None]).t()[None].to(DEV).contiguous()
    x, bc = torch.zeros(1, t, d, device=DEV), torch.ones(1, t, 1, s, device=DEV)
    A, st = torch.full((d, s), 6.0, device=DEV), torch.full((1, d, s), 1e-30, device=DEV)
    want, bound, want_after, bound_after = scan_ref(x, dt, A, bc, bc, None, softplus=False, state=st)
    y, after = selective_scan(*(v.expand(n, -1, -1) for v in (x, dt)), A, *(bc.expand(n, -1, -1, -1),) * 2, state=st.expand(n, -1, -1))
    for i in (0, n - 1):
        check(y[i:i + 1], want, bound * 4)
        check(after[i:i + 1], want_after, bound_after * 4)


@pytest.mark.parametrize('n', [1, 800])
def test_selective_scan_infinite_state_under_decay(n):
    """An infinite state stays infinite as step by step, although its factor over a chunk is zero in float32."""
    x, bc = torch.zeros(n, 200, 64, device=DEV), torch.ones(n, 200, 4, device=DEV)
    y, after = selective_scan(x, torch.ones_like(x), torch.full((64, 4), -7.0, device=DEV), bc, bc, state=torch.full((n, 64, 4), math.inf, device=DEV))
    assert (y == math.inf).all() and (after == math.inf).all()


@pytest.mark.parametrize('t', [1, 3, 8, 13, 200])
def test_selective_scan_state_that_forgets_at_once(t):
    """A = -inf: exp(s A) is 0 in every step, the state is s x B of the last one, whatever number of steps is computed together."""
    c, _ = scan_inputs(2, t, 40, 4, 1, torch.float32, False)
    c['A'][:20] = -math.inf
    lens = torch.tensor([t, (t + 1) // 2])
    want, bound, want_after, bound_after = scan_ref(**c, lens=lens)
    y, after = selective_scan(**c, dt_softplus=True, seq_lens=lens)
    check(y, want, bound)
    check(after, want_after, bound_after)


def test_selective_scan_no_step_of_a_state_that_forgets_at_once():
    """A step of width zero leaves such a state too, in whole lines (cut and not) as in single steps."""
    for n, t in ((2, 13), (1, 200)):
        x, bc = torch.zeros(n, t, 8, device=DEV), torch.ones(n, t, 4, device=DEV)
        A, st = torch.full((8, 4), -math.inf, device=DEV), rand(n, 8, 4)
        y, after = selective_scan(x, x, A, bc, bc, state=st)
        assert torch.equal(after, st) and y.isfinite().all()
        one = st.clone()
        selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], state=one)
        assert torch.equal(one, st)


def test_forward_mode_is_refused():
    """A dual tensor has requires_grad False: its tangent would be lost in silence."""
    import torch.autograd.forward_ad as fwd
    x, w = rand(2, 9, 8), rand(8, 4)
    q, k, v = qkv(2, 9, 9, 4, 2, 16, torch.float32)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for bad in (lambda: causal_conv(dual(x), w), lambda: causal_conv(x, dual(w)), lambda: attention(q, dual(k), v), lambda: attention_step(dual(q[:, 0]), k, v, [9, 9]),
                    lambda: constrain_logits(dual(x)), lambda: constrain_logits(x, bias=dual(rand(8))), lambda: causal_conv_step(x[:, 0], w, state=dual(rand(2, 3, 8)))):
            with pytest.raises(ValueError, match='gradient'):
                bad()
        assert torch.equal(causal_conv(x, w)[0], causal_conv(x, w)[0])
    c, _ = scan_inputs(2, 9, 12, 4, 1, torch.float32, False)
    with fwd.dual_level(), pytest.raises(ValueError, match='gradient'):
        selective_scan(**dict(c, A=fwd.make_dual(c['A'], c['A'])))


# ------------------------------------------------------------------------------------------------- long key axes, many rows, a plan's output
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('h,e', [(1, 64), (2, 40)])
def test_attention_documents_over_a_split_axis(dtype, h, e):
    """Few heads on a long axis: it is split, and the documents' id ranges lie behind the partial sums in the workspace."""
    q, k, v = qkv(2, 1500, 1500, h, 1, e, dtype)
    ids = torch.randint(0, 5, (2, 1500), generator=torch.Generator().manual_seed(2)).int()
    ids[1] = ids[1].sort()[0]
    ids, lens = ids.to(DEV), [1401, 1500]
    got = attention(q, k, v, lens, causal=True, documents=ids)
    check(got, *attention_ref(q, k, v, lens, lens, True, documents=ids))


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_more_tiles_than_bits(dtype):
    """Enough workgroups that nothing is split, and more key tiles than the 64 whose masks are looked at together."""
    q, k, v = qkv(64, 33, 4300, 8, 1, 16, dtype)
    got = attention(q, k, v, key_lens=[4300] * 63 + [4097])
    pick = [0, 31, 63]
    check(got[pick], *attention_ref(q[pick], k[pick], v[pick], None, [4300, 4300, 4097]))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shuffled', [False, True])
def test_attention_documents_of_more_tiles_than_bits(dtype, shuffled):
    t, pick = 4300, [0, 9]
    q, k, v = qkv(1, t, t, 16, 1, 16, dtype)
    ids = torch.randint(0, 3, (1, t), generator=torch.Generator().manual_seed(5)).int()
    ids = (ids if shuffled else ids.sort()[0]).to(DEV)
    got = attention(q, k, v, [4291], documents=ids)
    check(got[:, :, pick], *attention_ref(q[:, :, pick], k, v, [4291], [4291], documents=ids))


@pytest.mark.parametrize('dtype', TYPES)
def test_selective_scan_many_rows(dtype):
    """More rows than a grid holds along one axis, and more than one step: the loop over rows."""
    n, pick = 65600, [0, 1, 65534, 65535, 65536, 65599]
    c, k = scan_inputs(n, 2, 3, 2, 1, dtype, True)
    lens = torch.full((n,), 2)
    lens[65536] = 1
    y, after = selective_scan(**c, **k, dt_softplus=True, seq_lens=lens)
    few = {m: (v[pick] if v.dim() > 2 else v) for m, v in {**c, **k}.items()}
    want, bound, want_after, bound_after = scan_ref(**few, lens=lens[pick])
    check(y[pick], want, bound)
    check(after[pick], want_after, bound_after)


def test_a_plans_output_through_the_operators():
    """What a network gives goes in as it is, a view of time-major rows, with the lengths that the network gives: the decoder's classes are those
    allowed, and scores that nothing constrains decode as they did."""
    from tests.helpers import build_model, synth_input
    from kraken_amd.ctc_decoder import greedy_decoder
    from kraken_amd.specs import BENCH_A, bench_codec
    m = build_model(BENCH_A, codec=bench_codec(), seed=0).to(DEV)
    scores, lens = m.nn(synth_input(3, 400).to(DEV), torch.tensor([400, 250, 96]))
    rows = scores.squeeze(2).transpose(1, 2)                             # (N, C, 1, T) -> (N, T, C), no copy
    assert rows.stride(-1) == 1
    classes = rows.shape[-1]
    free = constrain_logits(rows, mask=label_mask([None] * 3, classes))
    assert torch.equal(free, rows)
    assert greedy_decoder(free.transpose(1, 2), lens) == greedy_decoder(scores.squeeze(2), lens)
    allowed = [list(range(1, 40)), list(range(100, 200)), [7]]
    lines = greedy_decoder(constrain_logits(rows, mask=label_mask(allowed, classes)).transpose(1, 2), lens)
    assert any(lines) and all(lab in labels for line, labels in zip(lines, allowed) for lab, *_ in line)
    heads = lambda v: v.unflatten(-1, (8, -1))  # noqa: E731
    u, _ = causal_conv(rows, rand(classes, 4, seed=1, scale=0.5), None, lens)
    want, bound, _ = conv_ref(rows, rand(classes, 4, seed=1, scale=0.5), None, lens, None, False, False)
    check(u, want, bound)
    check(attention(heads(rows), heads(u), heads(u), lens, causal=True), *attention_ref(heads(rows), heads(u), heads(u), lens, lens, True))


def test_selective_scan_steps_within_ten_roundings():
    """softplus over its whole range, y = s x of one state's first step: exp2 2 steps of 2^-24, its correction 1, 2 + e 1/3, the reciprocal 2, their
    product 1, the series 1.3 and the last sum 1."""
    v = torch.cat([torch.linspace(-80, 80, 16001), torch.linspace(-4, 4, 8001), torch.tensor([0.0, -300.0, 300.0, math.inf, -math.inf])]).to(DEV)
    one, d = torch.ones(1, 1, len(v), device=DEV), len(v)
    unit = torch.ones(1, 1, 1, device=DEV)
    y, _ = selective_scan(one, v.view(1, 1, -1), -torch.ones(d, 1, device=DEV), unit, unit, dt_softplus=True)
    y2 = selective_scan(one.expand(1, 20, d), v.expand(1, 20, d), torch.full((d, 1), -math.inf, device=DEV), unit.expand(1, 20, 1), unit.expand(1, 20, 1),
                        dt_softplus=True)[0][:, -1:]
    want = torch.nn.functional.softplus(v.double(), threshold=1000)
    # an infinite width leaves its channel without a finite result: infinity, or none at all (times the zeros that fill a lane's set of states up)
    assert not y[0, 0][want == math.inf].isfinite().any()
    for got in (y, y2):
        got = got[0, 0].double()
        low = want < 1e-36                                                                        # results without full precision
        assert ((got - want).abs()[~low & want.isfinite()] <= 10 * U * want[~low & want.isfinite()]).all()
        assert (got[low].abs() <= 2e-36).all()
    bad = torch.full((1, 1, 4), math.nan, device=DEV)
    assert selective_scan(torch.ones_like(bad), bad, -torch.ones(4, 1, device=DEV), unit, unit, dt_softplus=True)[0].isnan().all()
