"""
Constraint of a network's scores in front of a decoder: the labels a line may hold, biases, and penalties of what was written already.

``constrain_logits`` stands between a network's scores and :func:`kraken_amd.ctc_decoder.greedy_decoder` (reference
kraken/lib/ctc_decoder.py:35-72, which takes the scores as they are): a form field that holds digits only, a page in one script, or the next
label of a label model.  It is for a loop of one's own over a network's ``nn(x)``; ``rpred`` and ``predict`` decode on the
device and hand a custom decoder softmax values on the host, not scores.  Like the decoder it has no CPU implementation: without a HIP device
the call raises.
"""
import ctypes as C
import operator
from typing import Iterable, Optional, Union

import numpy as np
import torch

from . import _lib
from .sequence import _TYPES, _call, _first, _lengths, _like, _own_memory, _ptr

__all__ = ['constrain_logits', 'label_mask']

Penalty = Union[float, torch.Tensor]


def label_mask(allowed: Iterable[Optional[Iterable[int]]], classes: int, *, blank: bool = True, device='cuda') -> torch.Tensor:
    """
    The mask words of lines that may hold only certain labels: ``allowed`` has one collection of labels per line (None: all of them);
    ``blank`` allows label 0 besides, which a CTC network needs.  Returns (lines, ceil(classes / 32)) int32 on ``device``: bit c % 32 of word
    c / 32 stands for class c.
    """
    rows = []
    for labels in allowed:
        bits = np.zeros((classes + 31) // 32 * 32, dtype=np.uint8)
        if labels is None:
            bits[:classes] = 1
        else:
            try:
                labels = np.asarray([operator.index(label) for label in labels], dtype=np.int64)
            except TypeError as e:
                raise ValueError(f'labels have to be whole numbers: {e}') from None
            if labels.size and (labels.min() < 0 or labels.max() >= classes):
                raise ValueError(f'labels outside [0, {classes})')
            bits[labels] = 1
        if blank and classes:
            bits[0] = 1
        rows.append(np.packbits(bits, bitorder='little').view('<i4'))
    words = np.stack(rows) if rows else np.zeros((0, (classes + 31) // 32), dtype='<i4')
    return torch.from_numpy(words.astype(np.int32)).to(device)


def _penalty(p, name, n, first, positive=False):
    """(tensor or None, value): a number for all lines, or one per line."""
    if isinstance(p, torch.Tensor) and p.dim() == 1:
        return _like(p, name, (n,), first, torch.float32).contiguous(), 0.0
    p = C.c_float(float(p)).value                   # what the kernel gets: 1e-60 is zero there
    if not np.isfinite(p) or (positive and p <= 0):
        raise ValueError(f'{name} has to be finite{" and positive" if positive else ""}, got {p}')
    return None, p


def constrain_logits(logits: torch.Tensor, *, mask: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                     history: Optional[torch.Tensor] = None, history_lens=None, repetition: Penalty = 1.0, presence: Penalty = 0.0,
                     frequency: Penalty = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    ``logits`` (N, T, C), or (N, C) for one step, float32, bfloat16 or float16.  In this order, each rounded to float32 on its own, the
    result once to the logits' type:

    * a label that ``history`` (N, L) holds ``count`` times within its first ``history_lens`` entries: ``v / repetition`` if v > 0, else
      ``v * repetition``; then ``- frequency * count``; then ``- presence``.  Each of the three is a number or a float32 tensor (N).  Entries outside
      [0, C) count for nothing.  int32 or int64; the lengths as everywhere: checked on the host, clamped on the device.
    * ``+ bias``, float32 (C) or (N, C).
    * ``mask`` (N, W), (1, W), (N, T, W) or (1, T, W) int32 words, W = ceil(C / 32) (:func:`label_mask`): -inf where a class' bit is 0, whatever
      the score holds, NaN too.  A line that may hold nothing is -inf throughout.

    Returns a new tensor, or ``out``, which may be ``logits``.  No gradient, like the decoder; the current stream; nothing synchronises.
    """
    shape = getattr(logits, 'shape', ())
    step = isinstance(logits, torch.Tensor) and logits.dim() == 2
    x = _first(logits, 'logits', 2 if step else 3)
    n, t, c = (shape[0], 1, shape[1]) if step else shape
    words = (c + 31) // 32
    if bias is not None:
        bias = _like(bias, 'bias', (c,) if isinstance(bias, torch.Tensor) and bias.dim() == 1 else (n, c), x, torch.float32)
    mn = mt = 0
    if mask is not None:
        lead = tuple(getattr(mask, 'shape', ()))[:-1]
        if len(lead) not in (1, 2) or lead[0] not in (n, 1) or lead[1:] not in ((), (1,), (t,)):
            raise ValueError(f'mask has to be (lines or 1, words) or (lines or 1, steps, words), got {tuple(getattr(mask, "shape", ()))}')
        mask = _like(mask, 'mask', (*lead, words), x, torch.int32)
        mn, mt = (mask.stride(0) if lead[0] > 1 else 0), (mask.stride(1) if len(lead) == 2 and lead[1] > 1 else 0)
    length, lens, wide = 0, None, 0
    rep, pres, freq = (_penalty(p, s, n, x, s == 'repetition') for p, s in
                       ((repetition, 'repetition'), (presence, 'presence'), (frequency, 'frequency')))
    if history is not None:
        if not isinstance(history, torch.Tensor) or history.dim() != 2 or history.dtype not in (torch.int32, torch.int64):
            raise ValueError('history has to be (lines, entries) int32 or int64')
        length, wide = history.shape[1], history.dtype == torch.int64
        history = _like(history, 'history', (n, length), x, history.dtype)
        lens = _lengths(history_lens, 'history_lens', n, length, x.device)
        if length == 0:
            history = None
    elif history_lens is not None:
        raise ValueError('history_lens without history')
    if out is None:
        out = x.new_empty(x.shape)
    else:
        if _like(out, 'out', shape, x) is not out:
            raise ValueError('out is written in place: its classes have to be adjacent')
        same = out.data_ptr() == x.data_ptr() and all(i == j or s == 1 for i, j, s in zip(out.stride(), x.stride(), x.shape))
        _own_memory(out, 'out', (None if same else x, mask, bias, history, lens, rep[0], pres[0], freq[0]))
    if n == 0 or t == 0 or c == 0:
        return out
    a = _lib.KrkConstrainArgs(x.data_ptr(), out.data_ptr(), _ptr(mask), _ptr(bias), _ptr(history), _ptr(lens), _ptr(rep[0]), _ptr(pres[0]),
                              _ptr(freq[0]), x.stride(0), 0 if step else x.stride(1), out.stride(0), 0 if step else out.stride(1), mn, mt,
                              bias.stride(0) if bias is not None and bias.dim() == 2 else 0, history.stride(0) if history is not None else 0,
                              n, t, c, length, _TYPES[x.dtype], wide, rep[1], pres[1], freq[1])
    _call(_lib.load().krk_constrain_logits, a, x.device)
    return out
