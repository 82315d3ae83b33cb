"""NVFP4 KV cache: rotary positions and the scale-sweep quantizer in one write.

Between the qkv projection and attention, a decoder layer rotates its query
and key heads and stores keys and values.  This module does both in one
launch, holding the cache in the format of the framework's activations: E2M1
codes with one E4M3 scale per 16 elements, the scale chosen by the
``scalesweep_mse`` sweep.  The stored bytes are those of
``scalesweep_mse_nvfp4_quant`` on the rotated 16-bit keys and the values.

Layout (``alloc_kv_cache``): pages of ``page_size`` tokens,

* ``codes``  uint8 ``[num_pages, 2, kv_heads, page_size, head_size / 2]``,
* ``scales`` float8_e4m3fn ``[num_pages, 2, kv_heads, page_size, head_size / 16]``,

index 0 of the second axis holding keys and index 1 values.  The first axis
may be strided: ``codes[layer]`` of a cache allocated for all layers is a
layer's cache.  ``kv_input_scale`` is a float32 ``[2]`` tensor with the
multipliers (``256 * 6 / amax``) of the layer's keys and values; a stored value
stands for ``code * scale / multiplier``.  A token's slot is
``page * page_size + row``.
"""
from __future__ import annotations

import math

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)
HEAD_SIZES = (64, 128, 256)

# What a rope_scaling may hold, by rope_type, and what any may: names, and keys
# that do not change the frequencies of a given rotary_dim.
_SCALING_KEYS = {
    "default": (), "linear": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
    "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor",
             "mscale", "mscale_all_dim", "truncate")}
_SCALING_REQUIRED = {
    "default": (), "linear": ("factor",), "llama3": _SCALING_KEYS["llama3"],
    "yarn": ("factor", "original_max_position_embeddings")}
_SCALING_ANY = ("rope_type", "type", "rope_theta", "partial_rotary_factor", "max_position_embeddings",
                "original_max_position_embeddings", "mrope_section", "mrope_interleaved")


def alloc_kv_cache(num_pages: int, page_size: int, kv_heads: int, head_size: int,
                   device: torch.device | str = "cuda", num_layers: int | None = None):
    """(codes, scales) of an empty cache; with ``num_layers`` a leading layer
    axis.  Uninitialised, like the pages of any cache."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    if head_size not in HEAD_SIZES:
        raise ValueError(f"head_size must be one of {HEAD_SIZES}, got {head_size}")
    if num_pages < 1 or kv_heads < 1 or (num_layers is not None and num_layers < 1):
        raise ValueError("num_pages, kv_heads and num_layers must be positive")
    shape = ((num_layers,) if num_layers is not None else ()) + (num_pages, 2, kv_heads, page_size)
    return (torch.empty(shape + (head_size // 2,), dtype=torch.uint8, device=device),
            torch.empty(shape + (head_size // 16,), dtype=torch.float8_e4m3fn, device=device))


def rotary_cos_sin_cache(max_position: int, rotary_dim: int, base: float = 10000.0,
                         scaling: dict | None = None,
                         device: torch.device | str = "cuda") -> torch.Tensor:
    """float32 ``[max_position, rotary_dim]``: the cosines, then the sines, of
    ``position * frequency``, formed in binary64 (a binary32 angle is off by
    4e-3 at position 100000).

    ``scaling`` follows the ``rope_scaling`` of a model's configuration, by its
    ``rope_type``: ``linear`` (``factor``), ``llama3`` (``factor``,
    ``low_freq_factor``, ``high_freq_factor``,
    ``original_max_position_embeddings``) or ``yarn`` (``factor``,
    ``original_max_position_embeddings``, optionally ``beta_fast``,
    ``beta_slow`` and ``attention_factor``, which multiplies both tables).
    Other keys are refused, and so is a ``rope_theta`` that is not ``base``;
    a key that is None counts as absent.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if max_position < 1:
        raise ValueError(f"max_position must be positive, got {max_position}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    freq = float(base) ** (-i / rotary_dim)
    mult = 1.0
    scaling = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _SCALING_KEYS:
        raise ValueError(f"unsupported rope_type {kind!r}")
    missing = [k for k in _SCALING_REQUIRED[kind] if k not in scaling]
    if missing:
        raise ValueError(f"{kind}: scaling needs {', '.join(missing)}")
    unknown = sorted(set(scaling) - set(_SCALING_KEYS[kind]) - set(_SCALING_ANY))
    if unknown:
        raise ValueError(f"{kind}: unsupported keys {', '.join(unknown)}")
    if "rope_theta" in scaling and float(scaling["rope_theta"]) != float(base):
        raise ValueError(f"scaling has rope_theta {scaling['rope_theta']}, but base is {base}")
    if kind == "linear":
        freq = freq / float(scaling["factor"])
    elif kind == "llama3":
        factor, original = float(scaling["factor"]), float(scaling["original_max_position_embeddings"])
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        wave = 2 * math.pi / freq
        smooth = (original / wave - low) / (high - low)
        between = (1 - smooth) * freq / factor + smooth * freq
        freq = torch.where(wave > original / low, freq / factor,
                           torch.where(wave < original / high, freq, between))
    elif kind == "yarn":
        if scaling.get("mscale") or scaling.get("mscale_all_dim") or not scaling.get("truncate", True):
            raise ValueError("yarn: mscale, mscale_all_dim and truncate=False are not supported; "
                             "give attention_factor")
        factor, original = float(scaling["factor"]), float(scaling["original_max_position_embeddings"])

        def dim_of(turns):  # the pair that turns this often over the original length
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(dim_of(float(scaling.get("beta_fast", 32.0)))), 0)
        high = min(math.ceil(dim_of(float(scaling.get("beta_slow", 1.0)))), rotary_dim - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        mult = scaling.get("attention_factor")
        mult = 0.1 * math.log(factor) + 1.0 if mult is None else float(mult)
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos() * mult, angle.sin() * mult], dim=-1).float()


def rotary_scalesweep_mse_nvfp4_kv_write(query: torch.Tensor, key: torch.Tensor,
                                         value: torch.Tensor, positions: torch.Tensor,
                                         cos_sin_cache: torch.Tensor, slot_mapping: torch.Tensor,
                                         kv_input_scale: torch.Tensor, codes: torch.Tensor,
                                         scales: torch.Tensor, *, is_neox: bool = True,
                                         query_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate ``query`` [T, Hq, D] and ``key`` [T, Hkv, D], and quantize the
    rotated keys and ``value`` into the cache's rows ``slot_mapping`` [T].

    The three are bf16 or f16, and may be slices of a qkv projection's output
    (last dimension contiguous, other strides multiples of 8).  ``positions``
    and ``slot_mapping`` are int64 [T].  ``cos_sin_cache`` is float32
    ``[max_position, rotary_dim]`` (:func:`rotary_cos_sin_cache`), ``rotary_dim``
    a multiple of 16 up to D; elements past it are not rotated.  ``is_neox``
    pairs element i with i + rotary_dim / 2, otherwise 2i with 2i + 1.

    Returns the rotated query: ``query_out`` if given (``query`` itself rotates
    in place, any other overlaps no input), else a new contiguous tensor.
    ``key`` and ``value`` are only read.  Rows whose slot is negative or past the last page are padding: not
    stored.  Slots must be distinct.  A position outside the table gives NaN in
    the query, and that token is not stored.  There is no backward pass: inputs
    that require a gradient are refused outside ``torch.no_grad()``."""
    return _lib.kv_binding().write(query, key, value, positions, cos_sin_cache, slot_mapping,
                                   kv_input_scale, codes, scales, is_neox, query_out)


def nvfp4_kv_gather(codes: torch.Tensor, scales: torch.Tensor, kv_input_scale: torch.Tensor,
                    slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The keys and values stored at ``slot_mapping`` [T], as 16-bit floats:
    (key, value), each [T, kv_heads, head_size] and contiguous.  Zeros for a
    slot outside the cache.  For a cache's readers that want plain keys and
    values: another engine's cache, or a check of what the quantizer kept."""
    return _lib.kv_binding().gather(codes, scales, kv_input_scale, slot_mapping, dtype)
