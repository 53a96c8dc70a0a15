"""Serving a ragged batch from a cache in pages on CUDA torch tensors: rotary positions, keys and values into the cache and back, attention of
new tokens over it (the C entry points hipgpt_rotary*, hipgpt_cache_* and hipgpt_paged_attention in include/hipgpt_attn.h, which say what each computes).

Like launchers.py: outputs are given by the caller, calls are asynchronous on torch's current stream, torch holds the memory and nothing else.
Activations are float32 or bfloat16, one type per call and that of the cache; offsets, lengths, page numbers and positions int32.  All tensors are on the current device.
Tensors of tokens are contiguous, or views whose first dimension alone is spread (columns of a packed projection); what their rows hold must be heads * head_dim values.

A batch is given by offsets [B + 1] (rows of each sequence's new tokens), lengths [B] (tokens of each sequence with the new ones, which are its last), pages [B, most pages]
(page numbers), the number of new tokens T and of sequences B.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _capi, launchers

_check = _capi.check
FORMATS = {"plain": _capi.CACHE_PLAIN, "e4m3": _capi.CACHE_E4M3, "int8": _capi.CACHE_INT8}
SCALINGS = {None: _capi.ROTARY_UNSCALED, "linear": _capi.ROTARY_LINEAR, "base": _capi.ROTARY_BASE, "ramp": _capi.ROTARY_RAMP}


def rotary_frequencies(R: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0, original: float = 0.0, low: float = 1.0, high: float = 4.0):
    """Radians per position of the R / 2 pairs, a float64 CPU tensor: base^(-2i/R), slowed down for long contexts by `scaling` "linear", "base" or "ramp"."""
    (R,) = launchers._sizes(R)
    if scaling not in SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}")
    out = torch.empty(max(R, 0) // 2, dtype=torch.float64)
    _check(_capi.lib().hipgpt_rotary_frequencies(out.data_ptr(), R, base, SCALINGS[scaling], factor, original, low, high))
    return out


def rotary_words(frequencies, device="cuda"):
    """Frequencies (radians per position) as rotary takes them: an int64 tensor of 64-bit fractions of a turn on `device`.  Made once for a model."""
    f = torch.as_tensor(frequencies, dtype=torch.float64, device="cpu").contiguous()
    out = torch.empty(f.shape, dtype=torch.int64)
    _check(_capi.lib().hipgpt_rotary_words(f.data_ptr(), out.data_ptr(), f.numel()))
    return out.to(device)


def rotary(x, positions, words, out, T: int, H: int, D: int, R: int, *, interleaved: bool = False, magnitude: float = 1.0, inverse: bool = False):
    """out = magnitude * x with the first R values of each of H heads of D turned by their token's position; x [T, H, D] may be out.  Pairs (i, i + R/2), or
    neighbours (interleaved).  inverse: turned back, which is the gradient of x from that of out."""
    rc = launchers._native.rotary(x, positions, words, out, T, H, D, R, int(interleaved), int(inverse), magnitude)
    if rc:
        _check(rc)


class PagedCache:
    """Keys and values in pages: k, v [num_pages, heads, page_size, head_dim] of `dtype` (format "plain"), float8_e4m3fn ("e4m3") or int8 ("int8"), the latter two with scales
    k_scale, v_scale [num_pages, heads, page_size] float32.  What is not given is allocated (not set) on the current device.  The arrays are a cache's for good: another needs another PagedCache."""

    k, v = property(lambda self: self._arrays[0]), property(lambda self: self._arrays[1])
    k_scale, v_scale = property(lambda self: self._arrays[2]), property(lambda self: self._arrays[3])

    def __init__(self, num_pages: int, page_size: int, heads: int, head_dim: int, *, dtype=torch.float32, format: str = "plain", k=None, v=None, k_scale=None, v_scale=None):
        num_pages, page_size, heads, head_dim = launchers._sizes(num_pages, page_size, heads, head_dim)
        if format not in FORMATS:
            raise ValueError(f"unknown cache format {format!r}")
        if dtype not in launchers._TYPES:
            raise ValueError(f"expected float32 or bfloat16, not {dtype}")
        if min(num_pages, heads, head_dim) < 0 or page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"bad size: {num_pages} pages of {page_size} tokens, {heads} heads of {head_dim} values (pages hold a power of two from 16 to 1024 tokens)")
        shape = (num_pages, heads, page_size, head_dim)
        held = {"plain": dtype, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[format]
        device = next((t.device for t in (k, v, k_scale, v_scale) if isinstance(t, torch.Tensor)), None)

        def array(name, t, shape, dtype):
            if t is None:
                return torch.empty(shape, dtype=dtype, device=device if device is not None else "cuda")
            if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or not t.is_cuda or t.device != device:
                raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor of shape {list(shape)}, all of a cache on one device")
            return t

        if format == "plain" and (k_scale is not None or v_scale is not None):
            raise ValueError("a plain cache has no scales")
        self._arrays = array("k", k, shape, held), array("v", v, shape, held), None, None
        if format != "plain":
            self._arrays = *self._arrays[:2], array("k_scale", k_scale, shape[:3], torch.float32), array("v_scale", v_scale, shape[:3], torch.float32)
        self.num_pages, self.page_size, self.heads, self.head_dim, self.dtype, self.format = num_pages, page_size, heads, head_dim, dtype, format
        at = [t.data_ptr() if t is not None else None for t in self._arrays]
        self._struct = launchers._PagedCache(*at, num_pages, page_size, heads, head_dim, launchers._TYPES[dtype], FORMATS[format])
        self._address, self._device = C.addressof(self._struct), self.k.device.index


def _cache_of(cache):
    if not isinstance(cache, PagedCache):
        raise ValueError("cache: expected a PagedCache")
    return cache._address, cache._device


def cache_write(cache, k, v, offsets, lengths, pages, T: int, B: int):
    """Rows of k and v [T, heads, head_dim] to the pages of their sequences, in the cache's format."""
    rc = launchers._native.cache_move(*_cache_of(cache), k, v, offsets, lengths, pages, T, B, 1)
    if rc:
        _check(rc)


def cache_read(cache, k, v, offsets, lengths, pages, T: int, B: int):
    """The values that the cache holds for the batch's tokens, into k and v [T, heads, head_dim]."""
    rc = launchers._native.cache_move(*_cache_of(cache), k, v, offsets, lengths, pages, T, B, 0)
    if rc:
        _check(rc)


def paged_attention(cache, q, out, offsets, lengths, pages, T: int, B: int, H: int, *, causal: bool = True, scale: float | None = None):
    """Attention of each new token's H queries [T, H, head_dim] over the keys and values of its sequence, up to its own position (causal) or all of them; scale:
    1 / sqrt(head_dim) unless given.  H / heads queries in a row share a head of the cache."""
    rc = launchers._native.paged_attention(*_cache_of(cache), q, out, offsets, lengths, pages, T, B, H, int(causal), cache.head_dim ** -0.5 if scale is None else scale)
    if rc:
        _check(rc)
