"""Rotary positions on the sm_100a kernel: queries and keys of an attention
call turned by their positions, with a backward pass.

``apply_rotary(query, key, positions, frequencies)`` turns the first
``2 * len(frequencies)`` elements of every row and copies the rest.  Its
results are contiguous [B, H, N, D], the layout the attention calls take, so a
projection's output viewed as [B, N, H, D] goes in transposed and needs no copy
of its own.  ``rotary_frequencies`` gives the frequencies, stretched for
contexts longer than the trained one if asked to.

The reference has no positions; there is no CPU path.
"""

from __future__ import annotations

import math

import torch

from ._native import ext

LAYOUTS = ("half", "interleaved")
SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None,
                       factor: float = 1.0, trained_length: int | None = None,
                       fast_turns: float = 32.0, slow_turns: float = 1.0, device=None):
    """(frequencies, attention_factor): radians a position of the ``rotary_dim / 2`` pairs,
    ``base ** (-2 i / rotary_dim)``, as a float64 tensor, and the factor that
    ``apply_rotary`` multiplies with.

    ``scaling`` serves contexts ``factor`` times as long as the trained one:

    * ``"linear"`` divides every frequency by ``factor``;
    * ``"ntk"`` raises the base to ``base * factor ** (r / (r - 2))``, which divides the
      lowest frequency by ``factor`` and leaves the highest;
    * ``"yarn"`` divides the pairs that turn fewer than ``slow_turns`` times over
      ``trained_length`` positions, leaves those that turn more than ``fast_turns`` times
      and blends linearly between them; its attention factor is ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError("base must be above 1 and finite")
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError("factor must be at least 1 and finite")
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    frequencies = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    attention_factor = 1.0
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "yarn":
        if trained_length is None or trained_length < 1:
            raise ValueError("yarn scaling needs the trained_length")
        if not 0 < slow_turns < fast_turns:
            raise ValueError("slow_turns must be positive and below fast_turns")

        def pair_of(turns):  # the pair that turns so often over the trained length
            return rotary_dim * math.log(trained_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_of(fast_turns)), 0)
        high = min(math.ceil(pair_of(slow_turns)), rotary_dim - 1)
        ramp = (torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)
        ramp = ramp.clamp(0, 1)
        frequencies = frequencies / factor * ramp + frequencies * (1 - ramp)
        attention_factor = 0.1 * math.log(factor) + 1.0
    return frequencies.to(device), attention_factor


def apply_rotary(query, key, positions, frequencies, layout: str = "half",
                 attention_factor: float = 1.0, inverse: bool = False):
    """(query', key'): both turned by ``positions * frequencies`` and multiplied by
    ``attention_factor`` where turned.

    query: [B, H, N, D], key: [B, H_k, N, D] or None (then key' is None); float16, bfloat16 or
    float32 CUDA tensors of any strides with dense rows.  positions: int32 or int64 [N] or
    [B, N].  frequencies: float64, 1 to D / 2 of them.  ``layout``: pair i is (i, i + R / 2)
    for ``"half"`` and (2i, 2i + 1) for ``"interleaved"``, R = 2 * len(frequencies).
    ``inverse`` turns the other way.  Differentiable in query and key, any number of times, by
    reverse mode (positions and frequencies get no gradient); forward mode, ``torch.func``
    transforms and ``vmap`` end in an error, and ``torch.compile`` breaks its graph here.
    """
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}")
    return ext().rotary(query, key, positions, frequencies, layout == "interleaved",
                        attention_factor, inverse)
