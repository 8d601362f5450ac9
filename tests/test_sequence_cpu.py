"""The operators on sequence rows without a device: what the C entry points refuse, the checks of arguments, masks made on the host."""
import ctypes

import numpy as np
import pytest
import torch

from kraken_amd import _lib, constraints, sequence

PTR = 4096           # stands for a device address: nothing is read before the arguments are checked


def conv(**kw):
    a = _lib.KrkConvArgs(x=PTR, weight=PTR, y=PTR, N=1, T=4, D=8, K=4, type=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.load().krk_causal_conv(ctypes.byref(a), None)


def scan_args(**kw):
    a = _lib.KrkScanArgs(x=PTR, dt=PTR, B=PTR, C=PTR, A=PTR, y=PTR, N=1, T=4, D=8, S=16, G=1, type=1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attention_args(**kw):
    a = _lib.KrkAttentionArgs(q=PTR, k=PTR, v=PTR, out=PTR, N=1, Tq=4, Tk=4, H=4, Hk=2, E=64, type=2, scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def constrain(**kw):
    a = _lib.KrkConstrainArgs(logits=PTR, out=PTR, N=1, T=1, C=8, type=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.load().krk_constrain_logits(ctypes.byref(a), None)


def test_c_entries_refuse_null():
    lib = _lib.load()
    assert lib.krk_causal_conv(None, None) == lib.krk_selective_scan(None, None) == _lib.KRK_E_INVALID
    assert lib.krk_attention(None, None) == lib.krk_constrain_logits(None, None) == _lib.KRK_E_INVALID
    assert lib.krk_selective_scan_workspace(None) < 0 and lib.krk_attention_workspace(None) < 0


@pytest.mark.parametrize('bad,code', [(dict(x=None), -1), (dict(y=None), -1), (dict(D=0), -1), (dict(N=-1), -1), (dict(T=-1), -1), (dict(type=3), -1),
                                      (dict(K=0), -4), (dict(K=9), -4), (dict(T=2 ** 30 + 1), -4), (dict(state=PTR, state_out=PTR), -1)])
def test_c_conv_refusals(bad, code):
    assert conv(**bad) == code
    assert b'krk_causal_conv' in _lib.load().krk_last_error()


@pytest.mark.parametrize('bad,code', [(dict(dt=None), -1), (dict(A=None), -1), (dict(S=0), -4), (dict(S=257), -4), (dict(G=3), -1), (dict(G=0), -1),
                                      (dict(D=-8), -1), (dict(type=-1), -1), (dict(state=PTR, state_out=PTR), -1)])
def test_c_scan_refusals(bad, code):
    lib = _lib.load()
    assert lib.krk_selective_scan(ctypes.byref(scan_args(**bad)), None) == code
    assert lib.krk_selective_scan_workspace(ctypes.byref(scan_args(**bad))) == code
    assert b'krk_selective_scan' in lib.krk_last_error()


@pytest.mark.parametrize('bad,code', [(dict(k=None), -1), (dict(H=3), -1), (dict(Hk=0), -1), (dict(E=257), -4), (dict(E=0), -4), (dict(Tq=-1), -1),
                                      (dict(documents=PTR, Tq=3), -1), (dict(Tk=2 ** 30 + 1), -4), (dict(cap=-1.0), -1), (dict(cap=float('nan')), -1), (dict(type=7), -1)])
def test_c_attention_refusals(bad, code):
    lib = _lib.load()
    assert lib.krk_attention(ctypes.byref(attention_args(**bad)), None) == code
    assert lib.krk_attention_workspace(ctypes.byref(attention_args(**bad))) == code
    assert b'krk_attention' in lib.krk_last_error()


@pytest.mark.parametrize('bad', [dict(logits=None), dict(out=None), dict(C=0), dict(L=-1), dict(type=5), dict(T=-2)])
def test_c_constrain_refusals(bad):
    assert constrain(**bad) == _lib.KRK_E_INVALID


@pytest.mark.skipif(_lib.device_count() > 0, reason='a GPU is present')
def test_operators_fail_loudly_without_gpu():
    x = torch.rand(2, 5, 8)
    for call in (lambda: sequence.causal_conv(x, torch.rand(8, 4)), lambda: sequence.selective_scan(x, x, -torch.rand(8, 4), x[..., :4], x[..., :4]),
                 lambda: sequence.attention(x[:, :, None], x[:, :, None], x[:, :, None]), lambda: constraints.constrain_logits(x)):
        with pytest.raises(_lib.KrakenAmdError):
            call()
    assert conv() == _lib.KRK_E_HIP and constrain() == _lib.KRK_E_HIP


def test_long_axes_ask_for_a_workspace_and_short_ones_do_not():
    lib = _lib.load()
    assert lib.krk_attention_workspace(ctypes.byref(attention_args(N=512, Tk=200))) == 0
    one = attention_args(N=1, Tq=1, Tk=1 << 20, E=128)
    need = lib.krk_attention_workspace(ctypes.byref(one))
    assert need > 0
    one.workspace, one.workspace_bytes = PTR, need - 1
    if _lib.device_count() == 0:
        assert lib.krk_attention(ctypes.byref(one), None) == _lib.KRK_E_HIP
    assert lib.krk_selective_scan_workspace(ctypes.byref(scan_args(N=512, D=800, T=64))) == 0


def test_lengths_on_the_host_are_checked():
    dev = torch.device('cpu')
    assert sequence._lengths(None, 'lens', 3, 9, dev) is None
    got = sequence._lengths([0, 9, 4], 'lens', 3, 9, dev)
    assert got.dtype == torch.int32 and got.tolist() == [0, 9, 4]
    for bad in ([1, 2], [0, 10, 1], [-1, 0, 0], [0.5, 1, 1], [[1, 2, 3]], torch.ones(3, dtype=torch.bool)):
        with pytest.raises(ValueError):
            sequence._lengths(bad, 'lens', 3, 9, dev)


def test_tensors_that_are_updated_in_place():
    t = torch.zeros(5, 6, 7)
    for ok in (t, t[1:3], t[:, 2:4], t[:, :, 3:], t.transpose(0, 1), t[:1].expand(1, 6, 7)):
        sequence._own_memory(ok, 'state', ())
    for bad in (t[:1].expand(3, 6, 7), t.flatten().as_strided((3, 4), (2, 1)), t.flatten().as_strided((2, 2, 2), (3, 2, 1))):
        with pytest.raises(ValueError):
            sequence._own_memory(bad, 'state', ())
    with pytest.raises(ValueError):
        sequence._own_memory(t[2], 'state', (None, t[1:3]))
    with pytest.raises(ValueError):
        sequence._own_memory(t[4], 'state', (t[::4, :1, :1],))           # few elements, far apart
    sequence._own_memory(t[2], 'state', (t[:2], t[3:], torch.zeros(4)))


def test_tensors_that_go_together():
    x = torch.zeros(2, 3, 8)
    t = torch.zeros(4, 3, 16)[:2, :, 4:12]
    assert sequence._like(t, 't', (2, 3, 8), x) is t                    # adjacent channels: as it is
    copy = sequence._like(t.transpose(1, 2).contiguous().transpose(1, 2), 't', (2, 3, 8), x)
    assert copy.is_contiguous()
    assert sequence._like(t, 't', (2, 3, 8), x, inner=2).is_contiguous()
    for bad in (t.double(), t[:1], 3, None):
        with pytest.raises(ValueError):
            sequence._like(bad, 't', (2, 3, 8), x)
    with pytest.raises(ValueError):
        sequence._like(torch.zeros(2, 3, 8, requires_grad=True), 't', (2, 3, 8), x)
    with torch.no_grad():
        sequence._like(torch.zeros(2, 3, 8, requires_grad=True), 't', (2, 3, 8), x)


def test_label_mask():
    m = constraints.label_mask([[1, 5], None, [33], []], 40, device='cpu')
    assert m.dtype == torch.int32 and m.tolist() == [[0b100011, 0], [-1, 0xff], [1, 2], [1, 0]]
    assert constraints.label_mask([[]], 32, blank=False, device='cpu').tolist() == [[0]]
    assert constraints.label_mask([[31]], 32, blank=False, device='cpu').tolist() == [[-2 ** 31]]
    assert constraints.label_mask([], 33, device='cpu').shape == (0, 2)
    bits = np.random.RandomState(0).rand(5, 100) < 0.5
    m = constraints.label_mask([np.nonzero(b)[0] for b in bits], 100, blank=False, device='cpu').numpy().view(np.uint32)
    assert (((m[:, np.arange(100) // 32] >> (np.arange(100) % 32)) & 1) == bits).all()
    for bad in ([-1], [40]):
        with pytest.raises(ValueError):
            constraints.label_mask([bad], 40, device='cpu')


def test_lengths_of_an_empty_batch():
    """An empty list has no whole numbers that its type could show: a batch of no lines takes it."""
    got = sequence._lengths([], 'seq_lens', 0, 5, torch.device('cpu'))
    assert got.shape == (0,) and got.dtype == torch.int32
    with pytest.raises(ValueError, match='whole number'):
        sequence._lengths([], 'seq_lens', 1, 5, torch.device('cpu'))
    with pytest.raises(ValueError, match='whole number'):
        sequence._lengths([1.0], 'seq_lens', 1, 5, torch.device('cpu'))


@pytest.mark.parametrize('value,least', [(1e39, 0), (-1e39, -float('inf')), (float('nan'), 0), (-1.0, 0)])
def test_numbers_that_float32_does_not_hold(value, least):
    """The kernels take them as float32: 1e39 is infinite there."""
    with pytest.raises(ValueError):
        sequence._finite(value, 'scale', least)


def test_caps_below_float32s_normal_range():
    """1 / cap would be infinite, and a score of zero times it no number."""
    for cap in (1e-39, 1e-60):
        with pytest.raises(ValueError, match='cap'):
            sequence._scores(None, 2, 4, None, cap, None)
    assert sequence._scores(None, 2, 4, None, 1e-37, None)[1] > 0
    assert sequence._scores(None, 2, 4, None, 0.0, None) == (None, 0.0, 0.5)


@pytest.mark.parametrize('bad', [dict(cap=float('inf')), dict(cap=1e-39), dict(scale=float('inf')), dict(scale=float('nan'))])
def test_c_attention_refuses_numbers_that_it_cannot_use(bad):
    assert _lib.load().krk_attention(ctypes.byref(attention_args(**bad)), None) == _lib.KRK_E_INVALID


def test_penalties_that_float32_does_not_hold():
    """1e-60 is zero as float32, a divisor: the score would be infinite or no number."""
    for value, positive in ((1e-60, True), (1e39, True), (1e39, False), (-1e39, False)):
        with pytest.raises(ValueError):
            constraints._penalty(value, 'penalty', 2, None, positive)
    assert constraints._penalty(1.5, 'penalty', 2, None, True) == (None, 1.5)


def test_forward_mode_is_refused():
    """A dual tensor has requires_grad False: its tangent would be lost in silence."""
    from torch.autograd import forward_ad
    x = torch.rand(2, 3, 8)
    with forward_ad.dual_level():
        for t in (x, x[:, :, ::2].contiguous(), torch.rand(8)):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(ValueError, match='gradient'):
                sequence._like(dual, 't', t.shape, x)
            with torch.no_grad(), pytest.raises(ValueError, match='gradient'):
                sequence._like(dual, 't', t.shape, x)
            assert sequence._like(t, 't', t.shape, x) is t
            assert sequence._like(torch.zeros(2, dtype=torch.int32), 't', (2,), x, torch.int32).dtype == torch.int32
    assert sequence._like(x, 't', x.shape, x) is x


def test_scales_whose_exponent_float32_does_not_hold():
    """The kernels' exponentials have the base 2: 3e38 times log2 e is infinite, and a score of zero times it no number."""
    for scale in (3e38, -3e38):
        with pytest.raises(ValueError, match='scale'):
            sequence._scores(None, 2, 4, None, 0.0, scale)
        assert _lib.load().krk_attention_workspace(ctypes.byref(attention_args(scale=scale))) == _lib.KRK_E_INVALID
    assert sequence._scores(None, 2, 4, None, 0.0, -2.0 ** 127)[2] == -2.0 ** 127
    assert _lib.load().krk_attention_workspace(ctypes.byref(attention_args(scale=2.0 ** 127))) >= 0


def test_label_masks_of_what_is_no_label():
    """1.7 is not label 1; whole numbers of any kind are labels."""
    for bad in ([1.7], ['3'], [None]):
        with pytest.raises(ValueError, match='whole numbers'):
            constraints.label_mask([bad], 40, device='cpu')
    want = constraints.label_mask([[1, 5]], 40, device='cpu')
    for labels in (np.array([1, 5], dtype=np.int16), torch.tensor([1, 5]), {1, 5}, (5, 1), range(1, 6, 4), iter([1, 5])):
        assert torch.equal(constraints.label_mask([labels], 40, device='cpu'), want)
    with pytest.raises(ValueError, match='whole numbers'):
        constraints.label_mask([torch.tensor([1.0])], 40, device='cpu')
