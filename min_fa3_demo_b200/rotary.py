"""Rotary positions with one or several axes (text; height and width of an image; time, height and width of a clip).

No counterpart in the reference, which takes q and k as they are (``bindings.cpp:240-363``).
"""

from __future__ import annotations

import ctypes
from fractions import Fraction
from math import isfinite
from typing import Optional, Sequence, Tuple

import torch

from . import _cabi
from .min_fa3_op import _check, _check_device_capability, _on_device, _SM100, _stream_ptr

__all__ = ["RotaryAxes", "rotary"]

_TURN = round(2**192 / (2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")))
_MAX_PAIRS = 64
_NONE3 = (0, 0, 0)


def _turn(freq: float) -> int:
    """``freq / (2 pi)`` in units of 2^-64 modulo a turn: a float is an integer over a power of two."""
    num, den = freq.as_integer_ratio()
    shift = 127 + den.bit_length()                      # 2^128, which _TURN has too much, times den
    return ((num * _TURN + (1 << shift - 1)) >> shift) % 2**64


class RotaryAxes:
    """Which angle each pair of a head's 128 dimensions turns by.

    Pair ``i`` turns by ``positions[axis[i]] * inv_freq[i]``; there are 8, 16, ... or 64 pairs, and the dimensions behind the
    first ``2 * pairs`` stay as they are.  ``adjacent``: pair ``i`` is dimensions ``(2 i, 2 i + 1)``, otherwise
    ``(i, i + pairs)``.  Frequencies are taken as the 64-bit floats they are.  An angle is within 1.1e-7 for
    positions up to 2^36, and 1.7e-19 times the position more beyond (2^45: 6e-6).
    """

    def __init__(self, inv_freq: Sequence[float], axis: Optional[Sequence[int]] = None, *, adjacent: bool = False):
        inv_freq = [float(f) for f in inv_freq]
        axis = [0] * len(inv_freq) if axis is None else [int(a) for a in axis]
        pairs = len(inv_freq)
        _check(pairs % 8 == 0 and 8 <= pairs <= _MAX_PAIRS,
               f"the number of pairs must be a multiple of 8 between 8 and {_MAX_PAIRS}, got {pairs}")
        _check(len(axis) == pairs, f"inv_freq and axis must have the same length. Got {pairs} vs {len(axis)}")
        _check(all(0 <= a < _MAX_PAIRS for a in axis), f"an axis must be between 0 and {_MAX_PAIRS - 1}")
        _check(all(isfinite(f) for f in inv_freq), "inv_freq must be finite")
        self.axes = max(axis) + 1
        self.pairs = pairs
        c = _cabi.RotaryAxes()
        c.turn[:pairs] = [_turn(f) for f in inv_freq]
        c.axis[:pairs] = axis
        c.pairs, c.axes, c.adjacent = pairs, self.axes, int(bool(adjacent))
        self._c = c
        # The same as plain values, which an operator's schema can hold: turns as signed numbers of 64 bits.
        self._plain = ([t - 2**64 if t >= 2**63 else t for t in c.turn[:pairs]], axis, bool(adjacent))

    @classmethod
    def _from_plain(cls, turn: Sequence[int], axis: Sequence[int], adjacent: bool) -> "RotaryAxes":
        self = cls.__new__(cls)
        self.axes, self.pairs = max(axis) + 1, len(axis)
        self._c = c = _cabi.RotaryAxes()
        c.turn[:self.pairs] = [t % 2**64 for t in turn]
        c.axis[:self.pairs] = axis
        c.pairs, c.axes, c.adjacent = self.pairs, self.axes, int(adjacent)
        self._plain = (list(turn), list(axis), bool(adjacent))
        return self

    @property
    def _at(self) -> int:
        # Asked for at each call: a copy or an unpickled object has a structure of its own, elsewhere.
        return ctypes.addressof(self._c)

    @classmethod
    def from_sections(cls, sections: Sequence[int], base: float = 10000.0, *, restart: bool = False,
                      adjacent: bool = False) -> "RotaryAxes":
        """The first ``sections[0]`` pairs follow axis 0, the next ``sections[1]`` axis 1, and so on.  Pair ``i`` of ``n`` has
        frequency ``base ** (-i / n)``, counted over all sections, or, with ``restart``, within its own."""
        _check(all(int(n) >= 0 for n in sections), "sections must not be negative")
        total = sum(int(n) for n in sections)
        freq, axis = [], []
        for a, n in enumerate(int(n) for n in sections):
            for j in range(n):
                freq.append(float(base) ** (-(j / n if restart else len(freq) / total)))
                axis.append(a)
        return cls(freq, axis, adjacent=adjacent)


_BF16, _INT32, _INT64 = torch.bfloat16, torch.int32, torch.int64


def _rows(t: torch.Tensor) -> Tuple[int, int, int]:
    """Elements from sequence to sequence, token to token, head to head; 0 where there is only one."""
    st = t.stride()
    three = st[:3] if len(st) == 4 else (0, st[0], st[1])
    if (three[0] | three[1] | three[2]) & 7:
        size = t.shape if len(st) == 4 else (1, *t.shape)
        three = tuple(0 if n == 1 else s for n, s in zip(size, three))
    return three


def _is_rows(t: torch.Tensor, dim: int, index: int) -> bool:
    """Whether t is heads of 128 adjacent values, 16 bytes aligned (in one expression; _check_heads says what is wrong)."""
    if t.dtype is not _BF16 or t.get_device() != index:
        return False
    size, st = t.shape, t.stride()
    return (len(size) == dim and size[-1] == 128 and size[-2] > 0 and st[-1] == 1 and (st[0] | st[1] | st[-2]) & 7 == 0
            and t.data_ptr() & 15 == 0)


def _check_heads(t: torch.Tensor, name: str, dim: int) -> None:
    _check(t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.dtype == torch.bfloat16, f"{name} must have dtype torch.bfloat16")
    _check(t.dim() == dim, f"{name} must have shape " + ("[B, S, H, D]" if dim == 4 else "[total_tokens, H, D]"))
    _check(t.size(-1) == 128, f"{name} must have head_dim D=128")
    _check(t.size(-2) > 0, f"{name} must have heads")
    _check(t.stride(-1) == 1 and not any(s & 7 for s in _rows(t)) and t.data_ptr() % 16 == 0,
           f"{name} must be 16-byte aligned, with adjacent values in a head and other strides multiples of 8")


def _check_positions(positions: torch.Tensor, axes: RotaryAxes, shape, device) -> None:
    _check(isinstance(axes, RotaryAxes), "axes must be a RotaryAxes")
    _check(positions.device == device, "positions must be on the same CUDA device")
    _check(positions.dtype in (torch.int32, torch.int64), "positions must have dtype torch.int32 or torch.int64")
    _check(tuple(positions.shape) == (axes.axes, *shape),
           f"positions must have shape {[axes.axes, *shape]}. Got {list(positions.shape)}")


def _are_positions(positions: torch.Tensor, axes: RotaryAxes, shape, index: int) -> bool:
    return (type(axes) is RotaryAxes and positions.get_device() == index and positions.dtype in (_INT64, _INT32)
            and positions.shape == (axes.axes, *shape))


def _position_strides(positions: torch.Tensor) -> Tuple[int, int, int]:
    s = positions.stride()
    return s if len(s) == 3 else (s[0], 0, s[1])


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _check_rotary(q, k, positions, axes, dim) -> None:
    _check(dim in (3, 4), "q must have shape [B, S, H, D] or [total_tokens, H, D]")
    _check_heads(q, "q", dim)
    if k is not None:
        _check_heads(k, "k", dim)
        _check(k.device == q.device, "q and k must be on the same CUDA device")
        _check(k.shape[:-2] == q.shape[:-2], "q and k must have the same tokens")
    _check_positions(positions, axes, q.shape[:-2], q.device)
    _check_device_capability(q.device, "min_fa3_demo_b200 rotary")


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, axes: RotaryAxes, *,
           inverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q and k turned by their positions.

    q ``[B, S, QH, 128]``, k ``[B, S, KVH, 128]`` or None, positions ``[axes, B, S]`` (packed tokens: ``[T, H, 128]`` and
    ``[axes, T]``), int32 or int64, of any strides (``expand`` one row of positions over a batch).  q and k may be slices of
    one projection: only the 128 values of a head have to be adjacent.  Returns new contiguous tensors.  ``inverse``
    turns the other way, which is what the gradients want; ``autograd.rotary`` does it by itself.
    """
    index, qs, q_at = q.get_device(), q.shape, q.data_ptr()
    dim = len(qs)
    # As in min_fa3_op: a few expressions ask whether everything is as it should be, and _check_rotary says what is not.
    fine = (dim in (3, 4) and index in _SM100 and q.dtype is _BF16 and type(axes) is RotaryAxes
            and positions.dtype in (_INT64, _INT32) and positions.get_device() == index and positions.dim() == dim - 1)
    if fine:
        q_step, batch, seqlen, heads_q = q.stride(), 1 if dim == 3 else qs[0], qs[-3], qs[-2]
        q_rows = (0, q_step[0], q_step[1]) if dim == 3 else q_step[:3]
        fine = (qs[-1] == 128 and q_step[-1] == 1 and (q_rows[0] | q_rows[1] | q_rows[2]) & 7 == 0 and q_at & 15 == 0 and heads_q > 0
                and positions.shape == ((axes.axes, seqlen) if dim == 3 else (axes.axes, batch, seqlen)))
    k_at, k_rows, heads_k = 0, _NONE3, 0
    if fine and k is not None:
        ks, k_step, k_at = k.shape, k.stride(), k.data_ptr()
        fine = len(ks) == dim and k.dtype is _BF16 and k.get_device() == index and k_at & 15 == 0 and ks[-3] == seqlen
        if fine:
            heads_k = ks[-2]
            k_rows = (0, k_step[0], k_step[1]) if dim == 3 else k_step[:3]
            fine = (ks[-1] == 128 and k_step[-1] == 1 and heads_k > 0 and (k_rows[0] | k_rows[1] | k_rows[2]) & 7 == 0
                    and (dim == 3 or ks[0] == batch))
    if not fine:
        _check_rotary(q, k, positions, axes, dim)
        q_rows, batch, seqlen, heads_q = _rows(q), 1 if dim == 3 else qs[0], qs[-3], qs[-2]
        if k is not None:
            k_at, k_rows, heads_k = k.data_ptr(), _rows(k), k.size(-2)
    q_out = _like(q)
    k_out = None if k is None else _like(k)
    if batch * seqlen == 0:
        return q_out, k_out
    args = _cabi.ROTARY.pack(axes._at, q_at, k_at, q_out.data_ptr(), 0 if k is None else k_out.data_ptr(), positions.data_ptr(),
                             *q_rows, *k_rows, *_position_strides(positions), positions.dtype is _INT64, batch, seqlen, heads_q,
                             heads_k, bool(inverse))
    device = q.device
    with _on_device(device):
        _cabi.check(_cabi.load().b2a_rotary(args, _stream_ptr(device)))
    return q_out, k_out
