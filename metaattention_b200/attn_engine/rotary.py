"""Rotary positions of queries and keys (csrc/rotary.cu), in front of any of the engines and of a paged cache.

The first ``rotary_dim`` columns of every head are pairs that turn with the token's position, pair i by
``position * frequencies[i]`` radians: ``(a, b) -> magnitude * (a cos - b sin, b cos + a sin)``.  The reference has no such
operator: its examples take q and k with positions in them.
"""

from __future__ import annotations

import math

import torch

from core.native import lib as native

_TURN = 2 * math.pi   # radians of a full turn as the frequencies' own type has them


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(radians per position of each of the ``rotary_dim / 2`` pairs, magnitude), in 64 bits.

    ``scaling`` for contexts ``factor`` times as long as the ``original_length`` that a model was trained on: None;
    "linear" divides every frequency by ``factor``; "ntk" takes the base to ``base * factor ** (d / (d - 2))``, which leaves
    the highest frequency and divides the lowest by ``factor``; "yarn" leaves pairs that turn more than ``beta_fast`` times
    in ``original_length``, divides those that turn less than ``beta_slow`` times, blends between, and multiplies by the
    magnitude ``0.1 ln(factor) + 1``."""
    if rotary_dim <= 0 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be positive and even (got {rotary_dim})")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"base must be finite and larger than 1 (got {base})")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn' (got {scaling!r})")
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"factor must be finite and at least 1 (got {factor})")
    n = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("scaling 'ntk' needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2.0))
    f = [base ** (-2.0 * i / rotary_dim) for i in range(n)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        if original_length <= 0 or not beta_fast > beta_slow > 0.0:
            raise ValueError("scaling 'yarn' needs a positive original_length and beta_fast > beta_slow > 0")
        low, high = (rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (beta_fast, beta_slow))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rotary_dim - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(n)]
        f = [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)]
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


class RotaryEmbedding:
    """Turns q and k by their positions: ``rope(q, k, positions) -> (q', k')``, or ``rope(q) -> q'``.

    ``interleaved``: pairs of neighbouring columns (2 i, 2 i + 1) instead of (i, i + rotary_dim / 2); columns from
    ``rotary_dim`` on stay as they are.  The frequencies are those of ``rotary_frequencies``, or ``frequencies``
    (``rotary_dim / 2`` values in radians per position) with ``magnitude``.  The first call on a device lays them out there:
    make it before capturing a CUDA graph.  Calls on any stream and captured graphs keep what they read, also when the
    RotaryEmbedding itself is gone."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: str | None = None, factor: float = 1.0,
                 original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0, frequencies=None, magnitude: float | None = None):
        f, m = rotary_frequencies(rotary_dim, base, scaling, factor, original_length, beta_fast, beta_slow)
        if frequencies is not None:
            f, m = [float(x) for x in frequencies], 1.0
            if len(f) != rotary_dim // 2 or not all(math.isfinite(x) for x in f):
                raise ValueError(f"frequencies must be {rotary_dim // 2} finite values")
        self.rotary_dim, self.interleaved, self.frequencies = int(rotary_dim), bool(interleaved), f
        self.magnitude = m if magnitude is None else float(magnitude)
        if not math.isfinite(self.magnitude):
            raise ValueError(f"magnitude must be finite (got {magnitude})")
        self._turns = {}   # device -> the native form
        self._table = self.turns()

    def __getstate__(self):
        """Copies and pickles lay their frequencies out again at their first call."""
        return {**self.__dict__, "_turns": {}}

    def turns(self) -> list[int]:
        """The frequencies as 64-bit fractions of a full turn, as signed integers."""
        whole = 1 << 64
        top, bottom = _TURN.as_integer_ratio()
        values = []
        for x in self.frequencies:
            n, d = x.as_integer_ratio()
            n, d = n * bottom * whole, d * top
            values.append((2 * n + d) // (2 * d) % whole)   # the nearest
        return [x - whole if x >= whole // 2 else x for x in values]

    def native_on(self, device: torch.device):
        made = self._turns.get(device)
        if made is None:
            index = device.index if device.index is not None else torch.cuda.current_device()
            with torch.cuda.device(index), torch.inference_mode(False):   # the stream that is asked and waited for is that device's
                if torch.cuda.is_current_stream_capturing():
                    raise native.NativeError("the first call of a RotaryEmbedding on a device lays its frequencies out there: make it before the capture")
                table = torch.tensor(self._table, dtype=torch.int64).to(torch.device("cuda", index))
                torch.cuda.current_stream().synchronize()   # other streams use it too
            made = self._turns[device] = native.host().make_turns(table, self.rotary_dim, self.interleaved, self.magnitude)
        return made

    def __call__(self, q, k=None, positions=None, inplace: bool = False):
        """q: [batch, seq, heads, head_dim] or packed [tokens, heads, head_dim], k the same with heads of its own; float16,
        bfloat16 or float32, any strides with a contiguous last dimension.  ``positions``: int32 or int64 [batch, seq] or
        [seq] (packed: [tokens]), default 0, 1, ... along seq; negative ones turn backwards.  Computed in 32 bits and rounded
        once.  Differentiable in q and k (twice too; tangents of forward mode are refused); ``inplace`` writes over q and k
        instead and keeps no graph.
        In a captured training step, as with every operation of torch, no graph made outside of the capture may still hold the leaves."""
        if not q.is_cuda:
            raise native.NativeError("rotary positions need CUDA tensors: there is no CPU path")
        made = self._turns.get(q.device)
        return native.host().rotary(made if made is not None else self.native_on(q.device), q, k, positions, inplace)
