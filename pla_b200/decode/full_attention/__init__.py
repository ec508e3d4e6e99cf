"""The full-attention layers of a hybrid stack's serving step, next to the linear ones of :mod:`pla_b200.decode`.

``build_block_tables`` gives every new token its page and slot, ``qk_norm_rotary_cache`` norms and rotates queries and
keys and puts keys and values into their slots, ``paged_attention_decode`` attends over the cache with one new token
per request::

    plan = build_block_tables(table, context_lens, query_start_loc, free_blocks, 64, num_tokens=T)
    q = qk_norm_rotary_cache(q, k, v, q_weight, k_weight, plan.positions, inv_freq, k_cache, v_cache, plan.slot_mapping)
    out = paged_attention_decode(q, k_cache, v_cache, plan.block_table, plan.seq_lens)

``apply_rotary`` and ``qk_norm_rotary`` are the rotation alone and without a cache. Activations and caches are bf16 or fp16, sums
and softmax statistics 32-bit, one rounding at the end. All work goes to the current stream, nothing synchronises, scratch
comes from torch's allocator, and calls can be captured into CUDA graphs. Inference only: no gradients.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from ..._ops import ops

# The overloads themselves: half a microsecond less per call than looking them up through their packets. Arguments that are
# not given are left out of the calls below for the same reason.
_block_tables = ops.build_block_tables.default
_rotary = ops.apply_rotary.default
_norm_rotary = ops.qk_norm_rotary.default
_norm_rotary_cache = ops.qk_norm_rotary_cache.default
_paged_decode = ops.paged_attention_decode.default

__all__ = [
    "BlockPlan",
    "apply_rotary",
    "build_block_tables",
    "paged_attention_decode",
    "qk_norm_rotary",
    "qk_norm_rotary_cache",
    "rotary_frequencies",
]


class BlockPlan(NamedTuple):
    """What ``build_block_tables`` returns; ``block_table`` is the caller's own tensor, updated."""
    block_table: torch.Tensor    # [N, columns] int32
    slot_mapping: torch.Tensor   # [num_tokens] int64: page * block_size + offset, -1 = store nothing
    positions: torch.Tensor      # [num_tokens] int64
    seq_lens: torch.Tensor       # [N] int32: context + new tokens
    free_next: torch.Tensor      # [1] int32: first entry of free_blocks that is still free


def build_block_tables(
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    free_blocks: torch.Tensor,
    block_size: int,
    *,
    num_tokens: int,
    free_start: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> BlockPlan:
    """Page and slot of every new token of a step, on the GPU.

    Request ``n`` has ``context_lens[n]`` tokens in the pages that ``block_table[n]`` lists and gets the tokens
    ``query_start_loc[n] .. query_start_loc[n + 1]``. Pages that it lacks are taken from ``free_blocks`` in request order, beginning at
    entry ``free_start[0]`` (0 by default), and entered into its row in place; the other entries keep their values.
    ``num_tokens`` is the row count of the step's token tensors: rows at or past ``query_start_loc[N]`` (padding) get slot
    -1 and position 0. Pass ``free_next`` as the next step's ``free_start`` to go on in the same list.

    ``status`` (int32[1]) gets 32 when the list ran out and 64 when a row has too few columns (the tokens without a page
    have slot -1), 1 for negative lengths, offsets that are negative or fall (such a request gets nothing) and for offsets past ``num_tokens`` (new tokens past it are left out: no page, not in
    ``seq_lens``).
    """
    if status is None:
        slots, positions, seq_lens, free_next = _block_tables(
            block_table, context_lens, query_start_loc, free_blocks, block_size, num_tokens, free_start)
    else:
        slots, positions, seq_lens, free_next = _block_tables(
            block_table, context_lens, query_start_loc, free_blocks, block_size, num_tokens, free_start, status)
    return BlockPlan(block_table, slots, positions, seq_lens, free_next)


def rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: Optional[str] = None,
    factor: float = 1.0,
    original_max_position: int = 4096,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    low_freq_factor: float = 1.0,
    high_freq_factor: float = 4.0,
    device=None,
) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, factor)`` for the rotation: frequencies in radians per position (float64, ``[rotary_dim / 2]``) and the number
    that multiplies the rotated channels. ``scaling`` stretches a context of ``original_max_position`` by ``factor``:

    * ``None``: ``base ** (-2 i / rotary_dim)``;
    * ``"linear"``: all frequencies divided by ``factor``;
    * ``"ntk"``: the base raised by ``factor ** (d / (d - 2))``, so that the slowest frequency is divided by ``factor``;
    * ``"bands"``: wavelengths above ``original / low_freq_factor`` divided, below ``original / high_freq_factor`` kept, linear in between;
    * ``"yarn"``: channels that turn more than ``beta_fast`` times over the original context kept, fewer than ``beta_slow`` divided, a
      linear ramp over the channel index in between; the rotated channels are multiplied by ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError("rotary_dim must be a positive even number")
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError("base must be finite and above 1")
    if scaling not in (None, "linear", "ntk", "bands", "yarn"):
        raise ValueError("scaling must be None, linear, ntk, bands or yarn")
    if not factor >= 1.0 or not math.isfinite(factor):
        raise ValueError("factor must be finite and at least 1")
    if scaling in ("bands", "yarn") and original_max_position < 1:
        raise ValueError("original_max_position must be positive")
    if scaling == "bands" and not 0.0 < low_freq_factor < high_freq_factor:
        raise ValueError("bands needs 0 < low_freq_factor < high_freq_factor")
    if scaling == "yarn" and not 0.0 < beta_slow < beta_fast:
        raise ValueError("yarn needs 0 < beta_slow < beta_fast")
    multiply = 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    index = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = base ** (-2.0 * index / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "bands":
        turns = original_max_position * freq / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
    elif scaling == "yarn":
        def channel(turns: float) -> float:          # where the frequency makes that many turns over the original context
            return rotary_dim * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(channel(beta_fast)), 0)
        high = min(math.ceil(channel(beta_slow)), rotary_dim - 1)
        keep = 1.0 - ((index - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        if channel(beta_slow) < 0.0:                 # even the first channel turns fewer than beta_slow times
            keep = torch.zeros_like(index)
        freq = freq * keep + freq / factor * (1.0 - keep)
        multiply = 0.1 * math.log(factor) + 1.0
    return freq.to(device), multiply


def apply_rotary(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    interleaved: bool = False,
    factor: float = 1.0,
    out_q: Optional[torch.Tensor] = None,
    out_k: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotates the first ``2 * len(inv_freq)`` channels of every head of ``q`` ``[tokens, heads, dim]`` and ``k``
    by ``positions[t] * inv_freq`` and multiplies them by ``factor``; the other channels are copied. Pairs are ``(i, i + R/2)``, or
    ``(2i, 2i + 1)`` with ``interleaved``. ``out_q=q`` / ``out_k=k`` rotate in place; outputs that overlap anything else are refused."""
    if out_q is None and out_k is None:
        return _rotary(q, k, positions, inv_freq, factor, interleaved)
    return _rotary(q, k, positions, inv_freq, factor, interleaved, out_q, out_k)


def qk_norm_rotary(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    q_weight: Optional[torch.Tensor],
    k_weight: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    eps: float = 1e-6,
    unit_offset: bool = False,
    interleaved: bool = False,
    factor: float = 1.0,
    out_q: Optional[torch.Tensor] = None,
    out_k: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm of every head of ``q`` and ``k`` (``x * rsqrt(mean(x^2) + eps) * weight``, ``1 + weight`` with ``unit_offset``; a
    ``None`` weight leaves that side as it is), then the rotation of :func:`apply_rotary`, in one pass."""
    if out_q is None and out_k is None:
        return _norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, eps, factor, interleaved, unit_offset)
    return _norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, eps, factor, interleaved, unit_offset, out_q, out_k)


def qk_norm_rotary_cache(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    q_weight: Optional[torch.Tensor],
    k_weight: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    eps: float = 1e-6,
    unit_offset: bool = False,
    interleaved: bool = False,
    factor: float = 1.0,
    out_q: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """:func:`qk_norm_rotary` whose keys go to ``k_cache[slot // block_size, slot % block_size]`` (``[blocks, block_size, kv heads, dim]``
    with any strides) and whose values are copied to ``v_cache`` likewise; returns the queries. A negative slot stores
    nothing; a slot outside the pool stores nothing and sets 8 in ``status``. The slots of a call must differ, and the caches must not
    overlap each other or the rows."""
    if out_q is None and status is None:
        return _norm_rotary_cache(q, k, v, q_weight, k_weight, positions, inv_freq, k_cache, v_cache, slot_mapping, eps, factor, interleaved,
                                  unit_offset)
    return _norm_rotary_cache(q, k, v, q_weight, k_weight, positions, inv_freq, k_cache, v_cache, slot_mapping, eps, factor, interleaved,
                              unit_offset, out_q, status)


def paged_attention_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    status: Optional[torch.Tensor] = None,
):
    """Attention of one new token per request, ``q`` ``[requests, heads, dim]``, over the first ``seq_lens[b]`` tokens (the new one among
    them) of the pages in ``block_table[b]``. Query head ``h`` reads key/value head ``h // (heads / kv heads)``. ``scale`` is
    ``dim ** -0.5`` by default. A request of length 0 gets zeros (and ``lse = -inf``). Returns ``out``, or ``(out, lse)`` with the
    natural log of the softmax sums in fp32.

    ``status`` (int32[1]) gets 1 for a length that is negative or past the table's row, 8 for a page outside the pool (its
    tokens are left out). ``out`` is contiguous; it may be ``q``."""
    if out is None and status is None:
        o, lse = _paged_decode(q, k_cache, v_cache, block_table, seq_lens, scale, return_lse)
    else:
        o, lse = _paged_decode(q, k_cache, v_cache, block_table, seq_lens, scale, return_lse, out, status)
    return (o, lse) if return_lse else o
