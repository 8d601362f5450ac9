"""
Operators on sequence rows: a short causal convolution, a selective state space scan, and attention -- the mixers of a sequence block over a
line's time axis, next to the LSTM layers of :mod:`kraken_amd.vgsl` (the reference's only one, kraken/lib/vgsl/layers.py:462-547).

They take and give what a network's sequence layers do here: time-major rows ``(N, T, channels)``, right-padded, with ``seq_lens`` valid
steps per line.  Padding is never used, whatever it holds, and is zero in the result, so a line does not depend on what else is in its
batch; on how MANY lines there are the last bits of a scan or of attention may depend, since few lines are cut along their axis.  A recurrence
runs in either direction and carries its state from call to call; the ``_step`` forms take one step per line and update the state in
place.  Tensors are float32, bfloat16 or float16 on a HIP device, all of one type; sums, softmax statistics and states are float32, and a
16-bit result is rounded once.  Channels that are not adjacent in memory are laid out first (a copy); every other stride is taken as it is.

Work goes to the current stream of the tensors' device; nothing synchronises, so calls with lengths on the device may be captured into a
graph.  Lengths given on the host are checked; on the device they are clamped.  There is no backward pass: the library does not train, and a
tensor that asks for a gradient, or carries one in forward mode, is refused.  There is no CPU implementation here: without a HIP device every call raises.
"""
import ctypes as C
import math
from typing import Optional, Sequence, Union

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ['causal_conv', 'causal_conv_step', 'selective_scan', 'selective_scan_step', 'attention', 'attention_step']

Lens = Union[torch.Tensor, Sequence[int], None]

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}


def _no_gradient(t, name):
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f'{name} requires a gradient: there is no backward pass, call under torch.no_grad()')
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:      # a dual tensor requires none itself
        raise ValueError(f'{name} carries a forward gradient: there is no forward mode either')


def _first(x, name, dim):
    """The tensor that sets device and type of a call."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _lib.require_gpu()
        raise ValueError(f'{name} has to be a tensor on a HIP device')
    if x.dtype not in _TYPES:
        raise ValueError(f'{name} has to be float32, bfloat16 or float16, not {x.dtype}')
    if x.dim() != dim:
        raise ValueError(f'{name} has to have {dim} axes, got {tuple(x.shape)}')
    _no_gradient(x, name)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _like(t, name, shape, first, dtype=None, inner=1):
    """A tensor that goes with `first`: shape, type (first's unless given), device; its last `inner` axes adjacent (else a copy)."""
    if dtype is None:
        dtype = first.dtype
    if (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype is dtype and t.device == first.device and not t.requires_grad
            and forward_ad._current_level < 0 and t.is_contiguous()):
        return t                                    # what a step of a stream passes, in one condition: it is called for every label
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        raise ValueError(f'{name} has to be a tensor of shape {tuple(shape)}, got {tuple(t.shape) if isinstance(t, torch.Tensor) else type(t)}')
    if t.dtype != dtype:
        raise ValueError(f'{name} has to be {dtype}, not {t.dtype}')
    if t.device != first.device:
        raise ValueError(f'{name} is on {t.device}, the call on {first.device}')
    _no_gradient(t, name)
    if t.is_contiguous():
        return t
    want = 1
    for size, stride in zip(t.shape[:-inner - 1:-1], t.stride()[:-inner - 1:-1]):
        if size != 1 and stride != want:
            return t.contiguous()
        want *= size
    return t


def _lengths(lens, name, n, top, dev):
    """Lengths of n rows as int32 on the device: checked where they are on the host, clamped by the kernels where they are not."""
    if lens is None:
        return None
    if isinstance(lens, torch.Tensor) and lens.is_cuda:
        if lens.shape != (n,) or lens.device != dev or lens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f'{name} has to be {n} int32 or int64 on {dev}')
        if lens.dtype == torch.int64:
            lens = lens.clamp(0, top).int()
        return lens.contiguous()
    lens = torch.as_tensor(lens)
    if lens.shape != (n,) or (n and (lens.is_floating_point() or lens.dtype == torch.bool)):
        raise ValueError(f'{name} needs one whole number per line')
    if n and (int(lens.min()) < 0 or int(lens.max()) > top):
        raise ValueError(f'{name} outside [0, {top}]')
    return lens.to(device=dev, dtype=torch.int32)


def _extent(t):
    """Bytes from a tensor's first element to behind its last one."""
    if t.is_contiguous():
        return t.nbytes
    return (1 + sum((sz - 1) * st for st, sz in zip(t.stride(), t.shape))) * t.element_size() if t.numel() else 0


def _own_memory(t, name, others):
    """A tensor that a call updates in place: no element twice, and nothing shared with the inputs."""
    end = t.numel()
    if not t.is_contiguous():
        end = 1
        for st, sz in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
            if st < end:
                raise ValueError(f'{name} overlaps itself: it is updated in place')
            end += (sz - 1) * st
    lo = t.data_ptr()
    hi = lo + end * t.element_size()
    for o in others:
        if o is not None and o.data_ptr() < hi and lo < o.data_ptr() + _extent(o):
            raise ValueError(f'{name} shares memory with another argument: it is updated in place')


def _ptr(t):
    return None if t is None else t.data_ptr()


def _current_stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


# the handle alone, without an object around it: a third of what a step costs the host otherwise
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _call(fn, args, dev):
    """The entry point on the device's current stream; a device that is not the current one is made it for the launch."""
    if dev.index == torch.cuda.current_device():
        rc = fn(C.byref(args), _raw_stream(dev.index) if _raw_stream else _current_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(C.byref(args), _current_stream(dev))
    if rc:
        _lib.check(rc)


def _silu(activation):
    if activation not in ('linear', 'silu'):
        raise ValueError(f"activation has to be 'linear' or 'silu', not {activation!r}")
    return activation == 'silu'


# ------------------------------------------------------------------------------------------------------- causal convolution
def _conv_weights(x, weight, bias):
    d = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError('weight has to be (channels, kernel steps)')
    k = weight.shape[1]
    if not 1 <= k <= 8:
        raise ValueError(f'a kernel of {k} steps: 1 to 8 are supported')
    return k, _like(weight, 'weight', (d, k), x, inner=2), None if bias is None else _like(bias, 'bias', (d,), x)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, seq_lens: Lens = None, *,
                activation: str = 'linear', reverse: bool = False,
                state: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """
    Depthwise convolution of every channel with its own short kernel over the steps up to the present one.

    ``x`` (N, T, D); ``weight`` (D, K), K <= 8, the last column on the present step; ``bias`` (D); ``activation`` 'linear' or 'silu'.
    ``reverse`` runs from a line's last valid step to its first.  ``state`` (N, K-1, D): the inputs in front of the first step, oldest
    first (zeros without it).  Returns the result (N, T, D) and the new state, the last K-1 inputs in processing order.
    """
    x = _first(x, 'x', 3)
    n, t, d = x.shape
    k, weight, bias = _conv_weights(x, weight, bias)
    silu = _silu(activation)
    lens = _lengths(seq_lens, 'seq_lens', n, t, x.device)
    if state is not None:
        state = _like(state, 'state', (n, k - 1, d), x)
    y = x.new_empty((n, t, d))
    out = x.new_empty((n, k - 1, d))
    if n == 0 or d == 0 or t == 0:
        return y, out.zero_() if state is None else out.copy_(state)
    has = k > 1
    sn, sk, _ = state.stride() if state is not None else (0, 0, 0)
    a = _lib.KrkConvArgs(x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(state) if has else None, y.data_ptr(), out.data_ptr() if has else None,
                         _ptr(lens), x.stride(0), x.stride(1), t * d, d, sn, sk, (k - 1) * d, d, n, t, d, k, _TYPES[x.dtype], silu, bool(reverse))
    _call(_lib.load().krk_causal_conv, a, x.device)
    return y, out


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, state: torch.Tensor,
                     activation: str = 'linear') -> torch.Tensor:
    """
    One step per line of :func:`causal_conv`: ``x`` (N, D), ``state`` (N, K-1, D), which is moved on by one step IN PLACE (it may be a
    strided view of a larger buffer, but its channels are adjacent and nothing else is in its memory).  Returns (N, D).
    """
    x = _first(x, 'x', 2)
    n, d = x.shape
    k, weight, bias = _conv_weights(x, weight, bias)
    silu = _silu(activation)
    if _like(state, 'state', (n, k - 1, d), x) is not state:
        raise ValueError('state is updated in place: its channels have to be adjacent')
    y = x.new_empty((n, d))
    if n == 0 or d == 0:
        return y
    at = None
    if k > 1:
        _own_memory(state, 'state', (x, weight, bias))
        at = state.data_ptr()
    sn, sk, _ = state.stride()
    a = _lib.KrkConvArgs(x.data_ptr(), weight.data_ptr(), _ptr(bias), at, y.data_ptr(), at, None, x.stride(0), 0, d, 0, sn, sk, sn, sk, n, 1, d, k,
                         _TYPES[x.dtype], silu, 0)
    _call(_lib.load().krk_causal_conv, a, x.device)
    return y


# ------------------------------------------------------------------------------------------------------ selective state space scan
def _scan_args(x, dt, A, B, Cc, D, z, dt_bias):
    """The checks that the whole call and the step share; x (..., D) -> the call's tensors, states, groups."""
    rows, d = x.shape[:-1], x.shape[-1]
    f32 = torch.float32
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= 256:
        raise ValueError('A has to be (channels, states), 1 to 256 states')
    s = A.shape[1]
    if not isinstance(B, torch.Tensor) or not isinstance(Cc, torch.Tensor):
        raise ValueError('B and C have to be tensors')
    if B.dim() == len(rows) + 1:
        B = B.unsqueeze(-2)
    if Cc.dim() == len(rows) + 1:
        Cc = Cc.unsqueeze(-2)
    g = B.shape[-2] if B.dim() == len(rows) + 2 else 0
    if g < 1 or d % g:
        raise ValueError(f'B of shape {tuple(B.shape)}: its groups have to divide the {d} channels')
    return (_like(dt, 'dt', x.shape, x), _like(A, 'A', (d, s), x, f32, 2), _like(B, 'B', (*rows, g, s), x, inner=2),
            _like(Cc, 'C', (*rows, g, s), x, inner=2), None if D is None else _like(D, 'D', (d,), x, f32),
            None if z is None else _like(z, 'z', x.shape, x), None if dt_bias is None else _like(dt_bias, 'dt_bias', (d,), x, f32), s, g)


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None, *,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False, seq_lens: Lens = None,
                   reverse: bool = False, state: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """
    The recurrence ``h = exp(dt A) h + dt x B``, ``y = C . h + D x``, every channel with states of its own, all of it chosen by the input.

    ``x``, ``dt`` (N, T, D'); ``A`` (D', S) float32, S <= 256; ``B``, ``C`` (N, T, S), or (N, T, G, S) for G groups of channels; ``D`` (D') float32;
    ``z`` (N, T, D') gates the result by ``z sigmoid(z)``; ``dt_bias`` (D') float32 is added to ``dt``, ``dt_softplus`` applies softplus after
    it.  ``reverse`` runs from a line's last valid step to its first.  ``state`` (N, D', S) float32 starts the recurrence (zeros without it).
    Returns the result (N, T, D') and the state behind every line's last valid step.
    """
    x = _first(x, 'x', 3)
    n, t, d = x.shape
    dt, A, B, C, D, z, dt_bias, s, g = _scan_args(x, dt, A, B, C, D, z, dt_bias)
    lens = _lengths(seq_lens, 'seq_lens', n, t, x.device)
    if state is not None:
        state = _like(state, 'state', (n, d, s), x, torch.float32, 2)
    y = x.new_empty((n, t, d))
    out = torch.empty((n, d, s), dtype=torch.float32, device=x.device)
    if n == 0 or d == 0 or t == 0:
        return y, out.zero_() if state is None else out.copy_(state)
    zs = z.stride() if z is not None else (0, 0)
    a = _lib.KrkScanArgs(x.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z), A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(state),
                         y.data_ptr(), out.data_ptr(), _ptr(lens), None, 0, x.stride(0), x.stride(1), dt.stride(0), dt.stride(1), B.stride(0),
                         B.stride(1), C.stride(0), C.stride(1), zs[0], zs[1], t * d, d, state.stride(0) if state is not None else 0, d * s,
                         n, t, d, s, g, _TYPES[x.dtype], bool(dt_softplus), bool(reverse))
    lib = _lib.load()
    scratch = _scratch(lib.krk_selective_scan_workspace, a, x.device)       # noqa: F841 (alive until the launch is enqueued)
    _call(lib.krk_selective_scan, a, x.device)
    return y, out


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None, *,
                        state: torch.Tensor, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                        dt_softplus: bool = False) -> torch.Tensor:
    """
    One step per line of :func:`selective_scan`: ``x``, ``dt``, ``z`` (N, D'), ``B``, ``C`` (N, S) or (N, G, S), ``state`` (N, D', S) float32,
    updated IN PLACE (rows of a larger buffer will do).  Returns (N, D').
    """
    x = _first(x, 'x', 2)
    n, d = x.shape
    dt, A, B, C, D, z, dt_bias, s, g = _scan_args(x, dt, A, B, C, D, z, dt_bias)
    if _like(state, 'state', (n, d, s), x, torch.float32, 2) is not state:
        raise ValueError('state is updated in place: the states of a line have to be adjacent')
    y = x.new_empty((n, d))
    if n == 0 or d == 0:
        return y
    _own_memory(state, 'state', (x, dt, A, B, C, D, z, dt_bias))
    at, sn = state.data_ptr(), state.stride(0)
    a = _lib.KrkScanArgs(x.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z), A.data_ptr(), _ptr(D), _ptr(dt_bias), at,
                         y.data_ptr(), at, None, None, 0, x.stride(0), 0, dt.stride(0), 0, B.stride(0), 0, C.stride(0), 0,
                         z.stride(0) if z is not None else 0, 0, d, 0, sn, sn, n, 1, d, s, g, _TYPES[x.dtype], bool(dt_softplus), 0)
    _call(_lib.load().krk_selective_scan, a, x.device)
    return y


def _scratch(fn, args, dev):
    """The call's workspace, from torch's stream-ordered allocator (a captured graph gets its own); held by the caller until the launch."""
    need = fn(C.byref(args))
    if need < 0:
        _lib.check(int(need))
    if need == 0:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = ws.data_ptr(), need
    return ws


# -------------------------------------------------------------------------------------------------------------------- attention
def _finite(v, name, least):
    v = C.c_float(v).value                          # what the kernel gets: 1e39 is infinite there
    if not math.isfinite(v) or v < least:
        raise ValueError(f'{name} has to be finite{" and not negative" if least == 0 else ""}, got {v}')
    return v


def _keys(q, n, h, e, k, v):
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError('k has to be (N, Tk, Hk, E)')
    tk, hk = k.shape[1], k.shape[2]
    k, v = _like(k, 'k', (n, tk, hk, e), q), _like(v, 'v', (n, tk, hk, e), q)
    if h == 0 or hk == 0 or h % hk:
        raise ValueError(f'{hk} key heads have to divide {h} query heads')
    if not 1 <= e <= 256:
        raise ValueError(f'heads of {e} channels: 1 to 256 are supported')
    return k, v, tk, hk


def _scores(q, h, e, slopes, cap, scale):
    if slopes is not None:
        slopes = _like(slopes, 'slopes', (h,), q, torch.float32)
    if 0 < cap < 2.0 ** -126:
        raise ValueError(f'cap has to be 0 or a normal float32, got {cap}')
    scale = e ** -0.5 if scale is None else _finite(scale, 'scale', -math.inf)
    if abs(scale) > 2.0 ** 127:                     # its product with log2 e, the exponentials' base, has to be finite too
        raise ValueError(f'scale has to be within 2^127, got {scale}')
    return slopes, _finite(cap, 'cap', 0), scale


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seq_lens: Lens = None, *, key_lens: Lens = None, causal: bool = False,
              align: str = 'start', prefix_lens: Lens = None, documents: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None,
              cap: float = 0.0, scale: Optional[float] = None) -> torch.Tensor:
    """
    Softmax attention with masks that come as lengths and ids, never as a matrix.

    ``q`` (N, Tq, H, E), ``k``, ``v`` (N, Tk, Hk, E), E <= 256; Hk divides H, neighbouring query heads share a key head.  ``seq_lens``: valid
    queries; ``key_lens``: valid keys (``seq_lens`` when Tq == Tk, else all).  Query i stands at position i of the keys, or, with
    ``align='end'``, so that the last valid query stands at the last valid key (a chunk of new steps behind older ones).

    A key is seen if it is valid, of the query's document (``documents`` (N, T) int32 ids, Tq == Tk), and, when ``causal``, not behind the
    query's position or within the line's first ``prefix_lens`` keys.  Scores are ``scale q.k`` (E^-1/2), squashed to ``cap tanh(score / cap)``
    when ``cap`` > 0, less ``slopes[h] |distance|`` (``slopes`` (H) float32).  A query that sees nothing gives zeros.  Returns (N, Tq, H, E).
    """
    q = _first(q, 'q', 4)
    n, tq, h, e = q.shape
    k, v, tk, hk = _keys(q, n, h, e, k, v)
    if align not in ('start', 'end'):
        raise ValueError(f"align has to be 'start' or 'end', not {align!r}")
    dev = q.device
    q_lens = _lengths(seq_lens, 'seq_lens', n, tq, dev)
    k_lens = q_lens if key_lens is None and tq == tk else _lengths(key_lens, 'key_lens', n, tk, dev)
    prefix = _lengths(prefix_lens, 'prefix_lens', n, tk, dev)
    if prefix is not None and not causal:
        raise ValueError('prefix_lens without causal: every key is seen already')
    if documents is not None:
        if tq != tk:
            raise ValueError('documents need as many queries as keys')
        documents = _like(documents, 'documents', (n, tq), q, torch.int32)
    slopes, cap, scale = _scores(q, h, e, slopes, cap, scale)
    return _attend(q, (n, tq, h, e), k, v, tk, hk, q_lens, k_lens, prefix, documents, slopes, bool(causal), align == 'end', scale, cap)


def _attend(q, shape, k, v, tk, hk, q_lens, k_lens, prefix, documents, slopes, causal, at_end, scale, cap):
    """The call itself, its arguments checked: q (N, Tq, H, E), or (N, H, E) for one step."""
    n, tq, h, e = shape
    out = q.new_empty(q.shape)
    if n == 0 or tq == 0:
        return out
    if tk == 0:
        return out.zero_()
    if q.dim() == 4:
        qs, os = q.stride()[:3], (tq * h * e, h * e, e)
    else:
        qs, os = (q.stride(0), 0, q.stride(1)), (h * e, 0, e)
    a = _lib.KrkAttentionArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(q_lens), _ptr(k_lens), _ptr(prefix), _ptr(documents),
                              _ptr(slopes), None, 0, *qs, *k.stride()[:3], *v.stride()[:3], *os,
                              documents.stride(0) if documents is not None else 0, n, tq, tk, h, hk, e, _TYPES[q.dtype], causal, at_end, scale, cap)
    lib = _lib.load()
    scratch = _scratch(lib.krk_attention_workspace, a, q.device)            # noqa: F841 (alive until the launch is enqueued)
    _call(lib.krk_attention, a, q.device)
    return out


def attention_step(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_lens: Lens, *, slopes: Optional[torch.Tensor] = None,
                   cap: float = 0.0, scale: Optional[float] = None) -> torch.Tensor:
    """
    One new step per line of :func:`attention`: ``q`` (N, H, E) against the first ``cache_lens`` steps of ``k_cache``, ``v_cache`` (N, Tk, Hk, E), the
    last of which is the step's own.  The caches may be strided views of larger ones.  Returns (N, H, E); zeros for an empty cache.
    """
    q = _first(q, 'q', 3)
    n, h, e = q.shape
    k, v, tk, hk = _keys(q, n, h, e, k_cache, v_cache)
    lens = _lengths(cache_lens, 'cache_lens', n, tk, q.device)
    slopes, cap, scale = _scores(q, h, e, slopes, cap, scale)
    return _attend(q, (n, 1, h, e), k, v, tk, hk, None, lens, None, None, slopes, False, True, scale, cap)
