"""Rotary positions and cache append of a serving step's new tokens (``fgw_rotary_append`` of ``libfgw_mha.so``).

``rotary_table`` builds the angles once (FP64, rounded to FP32); ``rotary_append`` turns the new tokens' queries and
keys and writes keys and values where ``paged_chunk_attention`` reads them, in one launch. FGW itself has neither: its
callers bring a filled cache.
"""
import math

import torch

from fgw_b200 import _native

SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_table(positions, rotary_dim, base=10000.0, scaling=None, factor=1.0, original_positions=None,
                 beta_fast=32.0, beta_slow=1.0, attention_factor=None, device="cuda"):
    """The angles of positions 0 .. positions - 1 as ``cos_sin`` [positions, rotary_dim] float32: cosines, then sines.

    Pair i of position p turns by p * f_i, f_i = base ** (-2 i / rotary_dim). For contexts longer than trained,
    ``scaling`` changes the frequencies by ``factor`` = new length / trained length:

    * ``"linear"``: f_i / factor (positions counted more densely);
    * ``"ntk"``: base * factor ** (rotary_dim / (rotary_dim - 2)) in place of base, so that the slowest pair slows
      down by ``factor`` and the fastest stays;
    * ``"yarn"``: per pair, by the turns it makes over ``original_positions``: f_i from ``beta_fast`` turns on, f_i /
      factor up to ``beta_slow`` turns, a linear blend over the pair index between; cosines and sines are multiplied
      by ``attention_factor`` (default 0.1 ln(factor) + 1), which scales the scores by its square.
    """
    if positions <= 0 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("positive positions and an even rotary_dim required")
    if scaling not in SCALINGS:
        raise ValueError("scaling must be None, linear, ntk or yarn")
    if not base > 1.0 or not factor >= 1.0 or (scaling is None and factor != 1.0):
        raise ValueError("base above 1 and factor of at least 1 required (1 without scaling)")
    if scaling == "yarn" and (original_positions is None or original_positions <= 0 or beta_fast <= beta_slow):
        raise ValueError("yarn needs original_positions and beta_fast above beta_slow")
    if attention_factor is not None and (scaling != "yarn" or not attention_factor > 0.0):
        raise ValueError("attention_factor is a positive number and goes with yarn")
    pairs = rotary_dim // 2
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2)) if rotary_dim > 2 else base
    index = torch.arange(pairs, dtype=torch.float64, device=device)
    freq = base ** (-index / pairs)
    size = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        def pair_of(turns):  # the (fractional) pair that makes `turns` turns over the original positions
            return pairs * math.log(original_positions / (turns * 2.0 * math.pi)) / math.log(base)

        low = max(math.floor(pair_of(beta_fast)), 0)
        # may lie past the last pair, whose blend then ends unfinished; the limit is the published one
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        slow = ((index - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        freq = freq * (1.0 - slow) + freq / factor * slow
        size = 0.1 * math.log(factor) + 1.0 if attention_factor is None else float(attention_factor)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos() * size, angle.sin() * size], 1).float().contiguous()


def rotary_append(q, k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q, cos_sin, page_size,
                  interleaved=False, out=None):
    """Turn ``q`` and ``k`` by their positions and append ``k`` and ``v`` to the cache; returns the turned queries.

    ``q`` is [T, H, D], ``k`` and ``v`` [T, Hkv, D] (each token's heads contiguous, any token stride that is a multiple
    of 8), ``cos_sin`` [positions, rotary_dim] float32 from ``rotary_table``; the other arguments are those of
    ``paged_chunk_attention``, which takes the result. The i-th of request b's n new tokens has position
    ``cache_seqlens[b] - n + i``. Pairs are values (i, i + rotary_dim / 2) of a head, or (2 i, 2 i + 1) when
    ``interleaved``; values from rotary_dim on pass. ``out`` may be ``q``. Rows of no request, and positions outside
    the page table or ``cos_sin``, give zeros and append nothing. Raises
    ValueError for tensors that do not fit this, before any launch.
    """
    return _native.torch_binding().rotary_append(q, k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens_q,
                                                 cos_sin, page_size, interleaved, out)
