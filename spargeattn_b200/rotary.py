"""Rotary positions of queries and keys: the step in front of the attention of every model whose attention this package serves.

The reference's operators begin behind it (its model patches rotate q and k with the models' own code).
"""
import math

import torch

from ._cabi import _binding

# the tracing compiler leaves these frames alone, which costs a call nothing
_skip_frame = torch.compiler.disable(recursive=False)

SCALINGS = (None, "linear", "ntk", "llama3", "yarn")


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low=None, high=None, device="cuda"):
    """(frequencies, magnitude) for `dim` rotated channels: float64 [dim / 2], radians per position, and the factor of the
    rotated values (1.0 but for "yarn"). The unscaled frequency of pair i is base ** (-2 i / dim).

    `scaling` stretches them for contexts `factor` times as long as the ones the model was trained on (`original_length`):

    "linear"   every frequency by 1 / factor.
    "ntk"      a larger base, base * factor ** (dim / (dim - 2)): the first pair keeps its frequency, the last gets 1 / factor.
    "yarn"     pairs that turn more than `high` (32) times over the original length keep their frequency, pairs that turn less
               than `low` (1) times get 1 / factor, in between a ramp that is linear in the pair's number; the magnitude is
               0.1 ln(factor) + 1.
    "llama3"   the same by wavelength: more than `high` (4) turns keep, less than `low` (1) turns get 1 / factor, in between a
               ramp that is linear in the number of turns.
    """
    if dim <= 0 or dim % 2:
        raise ValueError(f"dim must be even and positive, is {dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, is {scaling!r}")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    pair = torch.arange(dim // 2, dtype=torch.float64)
    magnitude = 1.0
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling needs dim of at least 4")
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-2.0 * pair / dim)
    if scaling == "linear":
        f = f / factor
    elif scaling in ("yarn", "llama3"):
        if not original_length or original_length <= 0:
            raise ValueError(f"{scaling} scaling needs original_length")
        low = 1.0 if low is None else float(low)
        high = (32.0 if scaling == "yarn" else 4.0) if high is None else float(high)
        if not 0 < low < high:
            raise ValueError("low and high must be positive, low below high")
        if scaling == "llama3":
            keep = ((original_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        else:   # the pair that turns t times over the original length, as a real number
            at = lambda t: dim * math.log(original_length / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            first, last = max(math.floor(at(high)), 0), min(math.ceil(at(low)), dim - 1)
            keep = 1 - ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
            magnitude = 0.1 * math.log(factor) + 1.0
        f = f * keep + f / factor * (1 - keep)
    return f.to(device), magnitude


@_skip_frame
def apply_rotary(q, k, positions, frequencies, interleaved=False, sections=None, magnitude=1.0, tensor_layout="HND"):
    """Turns pairs of channels of q and k by position * frequency and returns (q', k'), or q' where k is None.

    q, k: [B, H, N, D] ("HND") or [B, N, H, D] ("NHD"), or without the batch, fp16, bf16 or fp32, any strides with a dense last
    dimension; k may have another number of heads. `frequencies`: float64 [pairs] (`rotary_frequencies`), 2 pairs <= D; the
    channels behind them are copied. `interleaved`: pairs are neighbours (2 i, 2 i + 1), else (i, i + pairs). `positions`: int32 or
    int64 [N] or [B, N]. With `sections` (pairs per axis, in order) positions have an axis of that length in front, and a
    pair turns by the position on its axis: frame, row and column of a video. Angles are formed in 64 bits, so far
    positions lose nothing. Differentiable in q and k; the gradient is turned back by the same kernel, and
    tangents of forward mode are turned like their values.

    Work is queued on the current stream. Shapes, types and ranges that do not fit are ValueError, CPU tensors RuntimeError."""
    return _binding.rotary(q, k, positions, frequencies, interleaved, sections, magnitude, tensor_layout)
