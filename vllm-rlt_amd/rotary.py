"""Rotary positions: the rotation that a model applies to queries and keys before attention.

The reference leaves it to its model layers (``vllm_rlt/layers/``), in torch operations around
the writer and the attention of every layer.  Here ``Rotary`` holds a model's frequencies and
``apply_rotary`` turns queries and keys in one launch; ``kv_write.append_kv`` does the same on
the way into the paged cache.
"""

import math

import torch

from . import _lib

SCALINGS = (None, "none", "linear", "ntk", "yarn", "bands")


class Rotary:
    """The rotation of one model: made once, on the device that it runs on.

    Pair i of the head's first ``rotary_dim`` dims turns by ``position * f_i`` radians,
    ``f_i = base ** (-2 i / rotary_dim)``, or scaled for contexts ``factor`` times longer than
    the ``original_length`` that was trained:

    * ``"linear"``: ``f_i / factor``;
    * ``"ntk"``: the base times ``factor ** (rotary_dim / (rotary_dim - 2))``, so that the first
      pair keeps its frequency and the last one's is divided by ``factor``;
    * ``"yarn"``: ``f_i`` up to the pair that turns ``fast`` (32) times within
      ``original_length``, ``f_i / factor`` from the one that turns ``slow`` (1) times on, a
      ramp over the pair's index between (both bounds rounded outwards to whole pairs), and
      sines and cosines times ``0.1 ln(factor) + 1`` where ``amplitude`` gives nothing else;
    * ``"bands"``: ``f_i`` where the pair turns ``fast`` (4) times or more within
      ``original_length``, ``f_i / factor`` at ``slow`` (1) or less, a ramp over the number of
      turns between.

    ``divisors`` (``rotary_dim / 2`` numbers) divide the frequencies further, pair by pair.
    ``interleaved``: pair i is dims (2 i, 2 i + 1); otherwise (i, i + rotary_dim / 2).
    ``turns`` (float64 ``[rotary_dim / 2]``) are the frequencies in turns per position.
    """

    def __init__(self, rotary_dim, base=10000.0, *, interleaved=False, scaling=None, factor=1.0,
                 original_length=None, fast=None, slow=1.0, divisors=None, amplitude=None,
                 device="cuda"):
        if type(rotary_dim) is not int or rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 256:
            raise ValueError("rotary_dim must be an even number from 2 to 256")
        if not (base > 0 and math.isfinite(base)):
            raise ValueError("base must be a positive number")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}")
        if not (factor > 0 and math.isfinite(factor)):
            raise ValueError("factor must be a positive number")
        r, half = rotary_dim, rotary_dim // 2
        if scaling == "ntk":
            if r < 4:
                raise ValueError("ntk scaling needs a rotary_dim of 4 or more")
            base = base * factor ** (r / (r - 2))
        f = [base ** (-2.0 * i / r) for i in range(half)]
        if scaling == "linear":
            f = [x / factor for x in f]
        elif scaling in ("yarn", "bands"):
            if original_length is None or not 0 < original_length < math.inf:
                raise ValueError(f"{scaling} scaling needs original_length")
            fast = (32.0 if scaling == "yarn" else 4.0) if fast is None else fast
            if not math.inf > fast > slow > 0:
                raise ValueError("fast must be above slow, both positive")
            if scaling == "yarn":
                if base == 1.0:
                    raise ValueError("yarn scaling needs a base other than 1")
                low, high = (r * math.log(original_length / (2 * math.pi * n)) /
                             (2 * math.log(base)) for n in (fast, slow))
                low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
                width = max(high - low, 0.001)
                divided = [min(max((i - low) / width, 0.0), 1.0) for i in range(half)]
                if amplitude is None:
                    amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
            else:
                turns = [original_length * x / (2 * math.pi) for x in f]
                divided = [1.0 - min(max((n - slow) / (fast - slow), 0.0), 1.0) for n in turns]
            f = [x * (1.0 - d) + x / factor * d for x, d in zip(f, divided)]
        if divisors is not None:
            if len(divisors) != half or not all(0 < d < math.inf for d in divisors):
                raise ValueError("divisors must be rotary_dim / 2 positive numbers")
            f = [x / float(d) for x, d in zip(f, divisors)]
        if amplitude is not None and not math.isfinite(amplitude):
            raise ValueError("amplitude must be a number")
        self.rotary_dim = rotary_dim
        self.interleaved = bool(interleaved)
        self.amplitude = 1.0 if amplitude is None else float(amplitude)
        self.turns = torch.tensor([x / (2 * math.pi) for x in f], dtype=torch.float64,
                                  device=device)


# (shapes, dtypes and devices are the operators' checks; what they read as it is, is made so here)
def _heads(x):
    return x if x.ndim != 3 or x.stride(2) == 1 else x.contiguous()


def _positions(positions):
    p = positions if positions.dtype == torch.int64 else positions.long()
    return p if p.is_contiguous() else p.contiguous()


def apply_rotary(q, k, positions, rotary, *, inverse=False, inplace=False):
    """Queries ``[rows, heads, head_dim]`` and keys ``[rows, kv_heads, head_dim]`` (or None)
    turned by ``positions`` (``[rows]``), in one launch: ``(q', k')``.

    Any row and head strides; ``head_dim`` up to 256, of which the first ``rotary.rotary_dim``
    turn and the rest is copied.  ``inverse`` turns back (the transpose of the rotation times
    the amplitude, so that it takes a gradient of the outputs to one of the inputs);
    ``inplace`` writes q and k themselves.  Angles are reduced in float64, sums are float32,
    rounded once.  Runs ``torch.ops.rlt_mi355x.rotary`` (``rotary_`` in place).
    """
    _lib.require_gpu(q, k, positions, rotary.turns)
    rest = (_positions(positions), rotary.turns, rotary.amplitude, rotary.interleaved, bool(inverse))
    if inplace:
        _lib.ops().rotary_(q, k, *rest)
        return q, k
    if k is None:
        return _lib.ops().rotary(_heads(q), None, *rest)[0], None
    return _lib.ops().rotary(_heads(q), _heads(k), *rest)
