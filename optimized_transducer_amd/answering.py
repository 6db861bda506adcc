"""Answering with a joiner: its output layer in 8 bits, and symbols drawn from its logits.

A step of decoding (or a pass over all packed rows, to score a batch or to draw
alignments for sequence training) is::

    q, s = quantize_blocks(x)                               # joiner activations (rows, D)
    logits, den = project_joiner_fp8(q, s, wq, ws, bias)    # wq, ws = quantize_blocks(weight, 128)
    symbols, log_probs = sample_symbols(logits, uniform, temperature=0.8, top_p=0.95)

All three are serving forms: they carry no gradient (:func:`project_joiner` is the
projection to train with).
"""
from typing import Optional, Tuple, Union

import torch

from . import _optimized_transducer


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad() or pass detached tensors"
                           % name)


def quantize_blocks(x: torch.Tensor, block_rows: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` in 8 bits, with a float32 scale for each block of 128.

    Args:
      x: (rows, D) float32, float16 or bfloat16 on a HIP device; any row pitch; rows may be 0.
      block_rows: 1 for activations (a scale for each 128 elements of a row), 128 for a
        weight (a scale for each 128 x 128 block).  The last blocks may be partial.
    Returns:
      (values, scale): ``scale`` (ceil(rows / block_rows), ceil(D / 128)) float32 is
      max|x| of the block / 448 (2^-126 at least), ``values`` (rows, D) float8_e4m3fn is
      x / scale, each rounded once to nearest even, so that ``values * scale`` is within
      2^-4 of x relative to it, or 2^-10 scales for the smallest.  A NaN or an infinity
      makes its block's scale NaN or infinite, and with it the logits it enters.
    """
    _no_gradient("quantize_blocks", x)
    return _optimized_transducer.quantize_blocks(x, block_rows)


def project_joiner_fp8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor,
                       weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       logits_dtype: torch.dtype = torch.float32,
                       denominators: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The joiner's output projection (:func:`project_joiner`) for operands in 8 bits, to
    decode and to score.

    Args:
      x, x_scale: ``quantize_blocks(activations)``: (rows, D) float8_e4m3fn, contiguous, D a
        multiple of 16, and (rows, ceil(D / 128)) float32.  rows may be 0.
      weight, weight_scale: ``quantize_blocks(linear.weight, 128)``: (V, D) and
        (ceil(V / 128), ceil(D / 128)).
      bias: (V,) or None.
      logits_dtype: torch.float32, torch.float16 or torch.bfloat16.
      denominators: False leaves the second result out.
    Returns:
      (logits, denominators): ``logits`` (rows, V) = (x * x_scale) @ (weight *
      weight_scale).T + bias on the matrix cores, accumulated in float32 and rounded once;
      ``denominators`` (rows,) float32 = the log-sum-exp of the float32 logits (before the
      rounding to ``logits_dtype``), for ``transducer_loss(..., denominators=...)``, or None.
    """
    _no_gradient("project_joiner_fp8", x, x_scale, weight, weight_scale, bias)
    return _optimized_transducer.joiner_project_blocks(x, x_scale, weight, weight_scale, bias,
                                                       logits_dtype, denominators)


def _setting(value):
    """(tensor or None, number) of a setting given for each row or for all."""
    return (value, 0) if isinstance(value, torch.Tensor) else (None, value)


def sample_symbols(logits: torch.Tensor, uniform: torch.Tensor,
                   temperature: Union[float, torch.Tensor] = 1.0,
                   top_k: Union[int, torch.Tensor] = 0,
                   top_p: Union[float, torch.Tensor] = 1.0,
                   min_p: Union[float, torch.Tensor] = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """A symbol drawn from each row of logits by a given random number.

    With m a row's largest entry, the weights are w_i = exp((x_i - m) / temperature), in an
    order of larger values first and equal values by lower index.  The first ``top_k`` entries
    remain; of those, the entries in front of which the weights sum to less than ``top_p``
    times the sum of all of them (the first always remains); of those, the entries with
    w_i >= ``min_p``.  The symbol is the first index, in index order, whose running sum of
    remaining weights exceeds ``uniform`` times their total.  Weights and sums behave as in
    64 bits: only where a border lies within a rounding of those can the symbol depend on how
    many rows are drawn from at once, and it is then one of the entries at that border.

    Args:
      logits: (rows, V) float32, float16 or bfloat16 on a HIP device; any row pitch (columns
        ``[:V]`` of padded logits, say); masked entries are -inf; rows may be 0.
      uniform: (rows,) float32 numbers of [0, 1), e.g. ``torch.rand(rows, device=...)``; small ones
        count as they are, whatever the entries in front of which they fall.
      temperature: >= 0; 0 takes the first of the largest entries.
      top_k: >= 0; 0 leaves it out.
      top_p: [0, 1]; 1 leaves it out.
      min_p: [0, 1]; 0 leaves it out.
        Each setting is one number or a tensor of shape (rows,) (float32; ``top_k`` int32); numbers are
        taken as float32 too, so that a temperature below its smallest value is 0.
        Numbers out of range are refused; in a tensor a temperature that is not positive
        counts as 0, top_k < 0 as 0, top_p as clamped to [0, 1] and min_p too.
    Returns:
      (symbols, log_probs): (rows,) int32 and (rows,) float32 = log(w_symbol / total) under
      the distribution drawn from (0 at temperature 0), rounded once, without a gradient.  A row without a
      largest finite entry (all -inf, a NaN, +inf), or whose number is NaN, gives -1 and -inf.
    """
    t, t_value = _setting(temperature)
    k, k_value = _setting(top_k)
    p, p_value = _setting(top_p)
    m, m_value = _setting(min_p)
    return _optimized_transducer.sample_symbols(logits, uniform, t, t_value, k, k_value, p, p_value,
                                                m, m_value)
