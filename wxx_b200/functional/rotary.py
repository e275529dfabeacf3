"""Rotary positions (no reference counterpart; kernel in ``csrc/rotary.cu``).

The first ``rotary_dim`` channels of every head are pairs (a, b) that a position
turns by its angle, so that products of queries and keys depend on how far apart
they are:

    a' = m (a cos t - b sin t)    b' = m (a sin t + b cos t)    t = position f_i
"""

import ctypes
import math

from ._common import F, check, compact, empty, finite32, ptr_or_none

_MOST = 512
_SCALINGS = ("linear", "ntk", "yarn")


class RotaryFrequencies:
    """What ``rotary`` turns by: ``frequencies``, the angle a position of each pair
    (radians), and ``gain``, the factor m on the turned channels."""

    def __init__(self, frequencies, gain=1.0):
        self.frequencies = tuple(float(f) for f in frequencies)
        self.gain = float(gain)
        if not 1 <= len(self.frequencies) <= _MOST // 2:
            raise ValueError(f"rotary: 1 to {_MOST // 2} frequencies, got {len(self.frequencies)}")
        if not all(math.isfinite(f) for f in self.frequencies) or not finite32(self.gain):
            raise ValueError("rotary: the frequencies and the gain must be finite")
        self.dim = 2 * len(self.frequencies)
        self._turns = (ctypes.c_double * len(self.frequencies))(
            *(f / (2 * math.pi) for f in self.frequencies))

    def __repr__(self):
        return f"RotaryFrequencies(dim={self.dim}, gain={self.gain:g})"


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None):
    """The frequencies ``base ** (-2 i / rotary_dim)`` of ``rotary_dim`` / 2 pairs, scaled
    to reach ``factor`` times further than they were made for:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base raised so that the slowest pair slows by ``factor`` and the
      fastest stays, ``base * factor ** (dim / (dim - 2))``;
    * ``"yarn"``: pairs that turn less than once over ``original_length`` positions are
      divided by ``factor``, those that turn more than 32 times stay, in between by their
      number of turns; the turned channels grow by ``0.1 log(factor) + 1``.
    """
    dim = int(rotary_dim)
    if dim != rotary_dim or not 2 <= dim <= _MOST or dim % 2:
        raise ValueError(f"rotary_frequencies: an even number of channels up to {_MOST}, got "
                         f"{rotary_dim}")
    base, factor = float(base), float(factor)
    if not 0.0 < base < math.inf:
        raise ValueError(f"rotary_frequencies: the base must be positive, got {base}")
    if scaling is not None and scaling not in _SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling must be one of {_SCALINGS}, got {scaling!r}")
    if not 1.0 <= factor < math.inf:
        raise ValueError(f"rotary_frequencies: the factor must be at least 1, got {factor}")
    if scaling == "ntk" and dim > 2:
        base *= factor ** (dim / (dim - 2))
    f = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        return RotaryFrequencies([v / factor for v in f])
    if scaling != "yarn":
        return RotaryFrequencies(f)
    if original_length is None or not 0 < original_length < math.inf:
        raise ValueError(f"rotary_frequencies: yarn scaling needs the original length, got "
                         f"{original_length}")

    def kept(v):
        turns = original_length * v / (2 * math.pi)
        return min(1.0, max(0.0, (turns - 1) / (32 - 1)))

    return RotaryFrequencies([v * kept(v) + v / factor * (1 - kept(v)) for v in f],
                             0.1 * math.log(factor) + 1)


def _rotate(what, x, n_heads, frequencies, positions, offset, layout, back):
    if x.type != "f32":
        raise TypeError(f"{what} expects an f32 tensor, got {x.type!r}")
    if len(x.shape) != 3:
        raise ValueError(f"{what} expects (batch, time, channels), got {tuple(x.shape)}")
    if not isinstance(frequencies, RotaryFrequencies):
        raise TypeError(f"{what} expects RotaryFrequencies, got {type(frequencies).__name__}")
    B, T, D = x.shape
    n_heads = int(n_heads)
    if n_heads < 1 or D % n_heads:
        raise ValueError(f"{what}: {D} channels cannot be split over {n_heads} heads")
    if D and frequencies.dim > D // n_heads:
        raise ValueError(f"{what}: {frequencies.dim} channels to turn in heads of {D // n_heads}")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"{what}: layout must be 'half' or 'interleaved', got {layout!r}")
    offset = int(offset)
    if not 0 <= offset < 1 << 32:
        raise ValueError(f"{what}: the offset must be between 0 and 2^32, got {offset}")
    p_bs = 0
    if positions is not None:
        if positions.type != "u32":
            raise TypeError(f"{what} expects u32 positions, got {positions.type!r}")
        if tuple(positions.shape) not in ((T,), (B, T)):
            raise ValueError(f"{what}: positions {tuple(positions.shape)} are neither {(T,)} nor "
                             f"{(B, T)}")
        p_bs = T if len(positions.shape) == 2 else 0
        positions = compact(positions)
    if D > 1 and (x.stride[-1] != 1 or min(x.stride) < 0):
        x = compact(x)
    y = empty((B, T, D))
    check(F.wxx_rotary(y.buffer.ptr, x.ptr, x.stride[0], x.stride[1], ptr_or_none(positions), p_bs,
                       offset, frequencies._turns, frequencies.dim, frequencies.gain, B, T,
                       n_heads, D // n_heads, int(layout == "half"), int(back)), what)
    return y


def rotary(x, n_heads, frequencies, positions=None, offset=0, layout="half"):
    """``x`` (batch, time, channels) with the first ``frequencies.dim`` channels of each of
    its ``n_heads`` heads turned by their positions, the others copied.

    ``positions``: u32, (time) or (batch, time); without them a row's positions count from
    0.  ``offset`` is added to them.  ``layout``: a pair is a head's channels i and i +
    dim / 2 (``"half"``) or 2 i and 2 i + 1 (``"interleaved"``).  Queries and keys next to
    each other in one tensor are one call with the heads of both.  Angles are made in 64
    bits, so positions may be far; the rows of ``x`` may be strided."""
    return _rotate("rotary", x, n_heads, frequencies, positions, offset, layout, False)


def rotary_backward(grad, n_heads, frequencies, positions=None, offset=0, layout="half"):
    """The gradient of ``rotary``'s input from that of its output: the map with the
    angles' signs turned (positions receive none)."""
    return _rotate("rotary_backward", grad, n_heads, frequencies, positions, offset, layout, True)
