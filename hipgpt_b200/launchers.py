"""Host-side mirror of the attention group of HipGPT's kernel API (include/hip_kernels.h:38-46
in the HipGPT tree) on top of the C ABI.  Names, argument order and meaning are the
reference's; arguments are CUDA float32 torch tensors (or raw device addresses) and the
calls are asynchronous on torch's current stream.  torch is used for device memory and
streams only; every kernel is the library's own.
"""
from __future__ import annotations

import ctypes
import threading
import warnings

import torch

from . import _capi


_FLOAT32 = torch.float32


def _ptr(t):
    if t is None or isinstance(t, int):
        return t
    if not (t.is_cuda and t.dtype is _FLOAT32 and t.is_contiguous()):
        raise ValueError("expected a contiguous CUDA float32 tensor")
    return t.data_ptr()


def _ptr_bf16(t):
    if not (t.is_cuda and t.dtype == torch.bfloat16 and t.is_contiguous()):
        raise ValueError("expected a contiguous CUDA bfloat16 tensor")
    return t.data_ptr()


_TYPES = {torch.float32: _capi.TYPE_F32, torch.bfloat16: _capi.TYPE_BF16}


def _storage(name, t):
    """The library's code of a tensor's type: float32 or bfloat16."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a CUDA tensor")
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise ValueError(f"expected float32 or bfloat16, not {t.dtype}") from None


def _sizes(*values):
    """Ints as the library takes them; more than one holds is refused (ctypes would pass its low bits)."""
    out = tuple(_int(v) for v in values)
    for v in out:
        if not -(1 << 31) <= v < 1 << 31:
            raise ValueError(f"{v} is beyond one call")
    return out


def _ptr_of(name, t, dtype, count, row=None):
    """The address of a tensor of at least `count` values on the current device, None for None; row: of two or more dimensions, the last of so many."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor")
    if row is not None and t.dim() >= 2 and t.shape[-1] != row:
        raise ValueError(f"{name} has rows of {t.shape[-1]} values, {row} are expected")
    if not (t.is_cuda and t.is_contiguous() and t.dtype == dtype):
        raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is {torch.cuda.current_device()}")
    if t.numel() < count:
        raise ValueError(f"{name} holds {t.numel()} values, {count} are needed")
    return t.data_ptr()


_TYPE_OF = {code: dtype for dtype, code in _TYPES.items()}


class _PagedCache(ctypes.Structure):
    """hipgpt_paged_cache"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + [(n, ctypes.c_int) for n in ("pages", "page_size", "heads", "head_dim", "type", "format")]


class _PagedBatch(ctypes.Structure):
    """hipgpt_paged_batch"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("offsets", "lengths", "page_table")] + [(n, ctypes.c_int) for n in ("sequences", "tokens", "most_pages")]


def _rows_of(name, t, dtype, T, H, D):
    """(address, values between rows) of a tensor of T rows of H * D values: contiguous, or its first dimension alone spread."""
    width = H * D
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a CUDA {dtype} tensor")
    inner = 1
    for n in t.shape[1:]:
        inner *= n
    whole = t.is_contiguous()
    # rows as one, or with the tokens in more dimensions than one: [...][width], [...][H][D], or heads one behind the other [T * H][D]
    heads = whole and t.dim() >= 2 and t.shape[-1] == D and (t.dim() == 2 or t.shape[-2] == H)
    if t.dim() >= 2 and not (inner == width or heads or (whole and t.shape[-1] == width)):
        raise ValueError(f"{name} has rows of {inner} values, {width} are expected")
    if not (t.is_cuda and t.dtype == dtype and (whole or (t.dim() >= 2 and t.shape[0] and t[0].is_contiguous()))):
        raise ValueError(f"{name}: expected a CUDA {dtype} tensor, contiguous but for its first dimension")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is {torch.cuda.current_device()}")
    if t.numel() < T * width:
        raise ValueError(f"{name} holds {t.numel()} values, {T * width} are needed")
    return t.data_ptr(), width if whole else t.stride(0)


def _batch_of(device, offsets, lengths, pages, T, B):
    if device != torch.cuda.current_device():
        raise ValueError(f"the cache is on cuda:{device}, the current device is {torch.cuda.current_device()}")
    if not isinstance(pages, torch.Tensor) or pages.dim() != 2:
        raise ValueError("pages: expected a contiguous CUDA int32 tensor of two dimensions")
    most = pages.shape[1]
    at = _ptr_of("offsets", offsets, torch.int32, B + 1), _ptr_of("lengths", lengths, torch.int32, B), _ptr_of("pages", pages, torch.int32, B * most)
    return _PagedBatch(*at, B, T, *_sizes(most))


# the current stream's handle without the Stream object around it (3.2 us of host time per call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = torch.cuda.current_device


def _stream():
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_current_device())


class ArgumentError(ctypes.ArgumentError, TypeError):
    """A size that is no integer."""


def _int(x):
    """What ctypes takes for an int: an int, a c_int, or what stands for one."""
    if isinstance(x, int):
        return x
    if isinstance(x, ctypes.c_int):
        return x.value
    if hasattr(x, "_as_parameter_"):
        return _int(x._as_parameter_)
    raise ArgumentError(f"int expected instead of {type(x).__name__} instance")


class _ThroughCtypes:
    """The extension's calls without it."""

    @staticmethod
    def attention(d_qkv, d_output, d_attn_probs, B, S, E, H, causal):
        return _capi.lib().hipgpt_mha_forward_planes(_ptr(d_qkv), _ptr(d_output), _ptr(d_attn_probs), _int(B), _int(S), _int(E), _int(H), causal, _stream())

    @staticmethod
    def attention_bf16(d_qkv, d_output, B, S, E, H, causal, variant):
        p, out = _ptr_bf16(d_qkv), _ptr_bf16(d_output)
        plane = B * S * E * 2                               # bytes
        return _capi.lib().hipgpt_mha_forward_bf16_ex(p, p + plane, p + 2 * plane, out, B, S, E, H, causal, variant, _stream())

    @staticmethod
    def decode(q, kcache, vcache, out, scratch, nbytes, B, H, D, ctx, cap):
        p = [_ptr(t) for t in (q, kcache, vcache, out, scratch)]
        if nbytes is None:
            nbytes = 0 if scratch is None else scratch.numel() * scratch.element_size()
        return _capi.lib().hipgpt_mha_decode(*p, nbytes, _int(B), _int(H), _int(D), _int(ctx), _int(cap), _stream())


    # training.py's
    @staticmethod
    def embedding_scaled(ids, tok, pos, out, scale, B, S, V, E):
        B, S, V, E = _sizes(B, S, V, E)
        type_, n, dt = _storage("out", out), B * S, out.dtype
        tables = _ptr_of("tok", tok, dt, V * E, E), _ptr_of("pos", pos, dt, S * E, E)
        return _capi.lib().hipgpt_embedding_scaled(_ptr_of("ids", ids, torch.int32, n), *tables, _ptr_of("out", out, dt, n * E), scale, B, S, V, E, type_, _stream())

    @staticmethod
    def embedding_backward(grad_out, ids, grad_tok, grad_pos, scale, accumulate, B, S, V, E):
        accumulate, B, S, V, E = _sizes(accumulate, B, S, V, E)
        n, table = B * S, grad_tok if grad_tok is not None else grad_pos
        type_, grad_type, gt = _storage("grad_out", grad_out), _storage("grad_tok", table), table.dtype
        tables = _ptr_of("grad_tok", grad_tok, gt, V * E, E), _ptr_of("grad_pos", grad_pos, gt, S * E, E)
        return _capi.lib().hipgpt_embedding_backward(_ptr_of("grad_out", grad_out, grad_out.dtype, n * E), _ptr_of("ids", ids, torch.int32, n), *tables, scale, accumulate, B, S, V, E,
                                                     type_, grad_type, _stream())

    @staticmethod
    def dropout_counter(x, residual, out, counter, p, seed, offset):
        type_ = _storage("out", out)
        n, dt, most = out.numel(), out.dtype, (1 << 64) - 1
        return _capi.lib().hipgpt_dropout_counter(_ptr_of("x", x, dt, n), _ptr_of("residual", residual, dt, n), _ptr_of("out", out, dt, n), p, seed & most, offset & most,
                                                  _ptr_of("counter", counter, torch.int64, 1), n, type_, _stream())

    @staticmethod
    def linear_cross_entropy(x, w, targets, loss, lse, N, E, V, layout):
        N, E, V, layout = _sizes(N, E, V, layout)
        type_, dt, f, row = _storage("x", x), x.dtype, _FLOAT32, V if layout == _capi.WEIGHTS_EV else E
        weights = _ptr_of("w", w, dt, V * E, row)
        return _capi.lib().hipgpt_linear_cross_entropy(_ptr_of("x", x, dt, N * E), weights, _ptr_of("targets", targets, torch.int32, N), _ptr_of("loss", loss, f, N),
                                                       _ptr_of("lse", lse, f, N), N, E, V, layout, type_, _stream())

    @staticmethod
    def linear_cross_entropy_backward(x, w, targets, lse, grad_loss, grad_x, grad_w, accumulate, N, E, V, layout):
        accumulate, N, E, V, layout = _sizes(accumulate, N, E, V, layout)
        type_, dt, f, row = _storage("x", x), x.dtype, _FLOAT32, V if layout == _capi.WEIGHTS_EV else E
        weights = _ptr_of("w", w, dt, V * E, row)
        return _capi.lib().hipgpt_linear_cross_entropy_backward(
            _ptr_of("x", x, dt, N * E), weights, _ptr_of("targets", targets, torch.int32, N), _ptr_of("lse", lse, f, N), _ptr_of("grad_loss", grad_loss, f, N),
            _ptr_of("grad_x", grad_x, dt, N * E), _ptr_of("grad_w", grad_w, dt, V * E, row), accumulate, N, E, V, layout, type_, _stream())

    # serving.py's
    @staticmethod
    def rotary(x, positions, words, out, T, H, D, R, interleaved, inverse, magnitude):
        T, H, D, R, interleaved, inverse = _sizes(T, H, D, R, interleaved, inverse)
        type_ = _storage("out", out)
        src, dst = _rows_of("x", x, out.dtype, T, H, D), _rows_of("out", out, out.dtype, T, H, D)
        return _capi.lib().hipgpt_rotary(*src, _ptr_of("positions", positions, torch.int32, T), _ptr_of("words", words, torch.int64, R // 2), *dst, magnitude, interleaved, inverse,
                                         T, H, D, R, type_, _stream())

    @staticmethod
    def cache_move(cache, device, k, v, offsets, lengths, pages, T, B, write):
        T, B = _sizes(T, B)
        c = _PagedCache.from_address(cache)
        dt = _TYPE_OF[c.type]
        rows = *_rows_of("k", k, dt, T, c.heads, c.head_dim), *_rows_of("v", v, dt, T, c.heads, c.head_dim)
        batch = _batch_of(device, offsets, lengths, pages, T, B)
        call = _capi.lib().hipgpt_cache_write if write else _capi.lib().hipgpt_cache_read
        return call(cache, ctypes.byref(batch), *rows, _stream())

    @staticmethod
    def paged_attention(cache, device, q, out, offsets, lengths, pages, T, B, H, causal, scale):
        T, B, H = _sizes(T, B, H)
        c = _PagedCache.from_address(cache)
        dt = _TYPE_OF[c.type]
        rows = *_rows_of("q", q, dt, T, H, c.head_dim), *_rows_of("out", out, dt, T, H, c.head_dim)
        batch = _batch_of(device, offsets, lengths, pages, T, B)
        return _capi.lib().hipgpt_paged_attention(cache, ctypes.byref(batch), *rows, H, causal, scale, _stream())


class _AtFirstCall:
    """Stands for the extension until it is needed, by the first of however many threads: importing this module builds and loads nothing."""

    _lock = threading.Lock()

    def __getattr__(self, name):
        global _native
        with self._lock:
            if _native is self:
                try:
                    native = _capi.native()
                    native.bind(_ptr, _ptr_bf16, _int)
                except (RuntimeError, ImportError, OSError) as e:       # no g++, no headers: the same library through ctypes
                    warnings.warn(f"the extension of the hot calls cannot be built or loaded, they go through ctypes (a few microseconds more each): {e}", RuntimeWarning, stacklevel=3)
                    native = _ThroughCtypes
                _native = native
        return getattr(_native, name)


_native = _AtFirstCall()


def launch_multihead_attention(d_qkv, d_output, d_attn_probs, B: int, S: int, E: int, H: int, *, causal: bool = False):
    """softmax(Q K^T / sqrt(E/H)) V per (batch, head).  d_qkv: three stacked [B*S, E] planes;
    d_output [B*S, E]; d_attn_probs [B, H, S, S] or None.  Not causal unless asked: the
    reference never masks (src/hip_kernels.cpp:287-319)."""
    if H <= 0 or E % H != 0:
        raise ValueError(f"Bad MHA config: E={E} H={H}")   # the reference aborts here
    rc = _native.attention(d_qkv, d_output, d_attn_probs, B, S, E, H, int(causal))
    if rc:
        _capi.check(rc)


def mha_forward(q, k, v, out, probs, B: int, S: int, E: int, H: int, *, causal: bool = False,
                algo: int = _capi.ALGO_AUTO, warps: int = 0):
    """The same on separate Q, K, V planes, with the kernel selector exposed."""
    _capi.check(_capi.lib().hipgpt_mha_forward_ex(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(probs),
                                                  B, S, E, H, int(causal), algo, warps, _stream()))


def mha_forward_bf16(d_qkv, d_output, B: int, S: int, E: int, H: int, *, causal: bool = False, variant: int = 0):
    """The launcher's contract with bf16 storage: d_qkv = three stacked [B*S, E] bf16 planes, d_output
    [B*S, E] bf16 (head_dim 64), fp32 accumulation."""
    rc = _native.attention_bf16(d_qkv, d_output, B, S, E, H, int(causal), int(variant))
    if rc:
        _capi.check(rc)


def launch_scaled_dot_product(Q, K, scores, B: int, S: int, D: int):
    _capi.check(_capi.lib().hipgpt_scaled_dot_product(_ptr(Q), _ptr(K), _ptr(scores), B, S, D, _stream()))


def launch_softmax(scores, softmax_out, B: int, S: int):
    _capi.check(_capi.lib().hipgpt_softmax(_ptr(scores), _ptr(softmax_out), B, S, _stream()))


def launch_attention_weighted_sum(softmax, V, output, B: int, S: int, D: int):
    _capi.check(_capi.lib().hipgpt_attention_weighted_sum(_ptr(softmax), _ptr(V), _ptr(output), B, S, D, _stream()))


def decode_scratch_bytes(B: int, H: int, D: int, ctx: int) -> int:
    return int(_capi.lib().hipgpt_mha_decode_scratch_bytes(B, H, D, ctx))


def mha_decode(q, kcache, vcache, out, scratch, B: int, H: int, D: int, ctx: int, cap: int):
    """One query row per (batch, head) over the first ctx rows of the caches."""
    nbytes = None if scratch is None or type(scratch) is torch.Tensor else scratch.numel() * scratch.element_size()
    rc = _native.decode(q, kcache, vcache, out, scratch, nbytes, B, H, D, ctx, cap)
    if rc:
        _capi.check(rc)


def mha_forward_host(h_qkv, h_out, h_probs, B: int, S: int, E: int, H: int, *, causal: bool = False):
    """Host buffers in, host buffers out (numpy float32 arrays or CPU torch tensors, ideally
    pinned): the copies and the kernel run inside the call, which returns when h_out is ready."""
    def hp(a):
        if a is None:
            return None
        if isinstance(a, torch.Tensor):
            assert not a.is_cuda and a.dtype == torch.float32 and a.is_contiguous()
            return a.data_ptr()
        assert a.dtype.name == "float32" and a.flags["C_CONTIGUOUS"]
        return a.ctypes.data
    _capi.check(_capi.lib().hipgpt_mha_forward_host(hp(h_qkv), hp(h_out), hp(h_probs), B, S, E, H, int(causal)))


def mha_forward_bf16_host(h_qkv, h_out, B: int, S: int, E: int, H: int, *, causal: bool = False):
    """The host-buffer call for bf16 planes: CPU torch.bfloat16 tensors (ideally pinned), h_qkv three
    stacked [B*S, E] planes, h_out [B*S, E]; head_dim 64."""
    for t in (h_qkv, h_out):
        if not (isinstance(t, torch.Tensor) and not t.is_cuda and t.dtype == torch.bfloat16 and t.is_contiguous()):
            raise ValueError("expected a contiguous CPU bfloat16 tensor")
    _capi.check(_capi.lib().hipgpt_mha_forward_bf16_host(h_qkv.data_ptr(), h_out.data_ptr(), B, S, E, H, int(causal)))
