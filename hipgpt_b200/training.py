"""The operators at the two ends of a training step on CUDA torch tensors: embedding and its gradient, dropout from a
counter, the loss and its gradient (the C entry points of the same names in include/hipgpt_attn.h, which say what each computes).

Like launchers.py: outputs are given by the caller, calls are asynchronous on torch's current stream, torch holds the memory and
nothing else.  Activations and weights are contiguous float32 or bfloat16 tensors, one type per call; ids and targets int32.  All
tensors are on the current device.  Sizes beyond what a tensor holds are refused.
"""
from __future__ import annotations

import torch

from . import _capi
from .launchers import _stream

_TYPES = {torch.float32: _capi.TYPE_F32, torch.bfloat16: _capi.TYPE_BF16}


def _type(t):
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise ValueError(f"expected float32 or bfloat16, not {t.dtype}") from None


def _ptr(name, t, dtype, count):
    """The address of a tensor of at least `count` values, None for None."""
    if t is None:
        return None
    if not (t.is_cuda and t.is_contiguous() and t.dtype == dtype):
        raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is {torch.cuda.current_device()}")
    if t.numel() < count:
        raise ValueError(f"{name} holds {t.numel()} values, {count} are needed")
    return t.data_ptr()


def embedding_scaled(ids, tok, pos, out, B: int, S: int, V: int, E: int, *, scale: float = 1.0):
    """out[t] = scale tok[id_t] + pos[t mod S]; pos may be None; zeros for an id outside [0, V)."""
    n, dt = B * S, out.dtype
    _capi.check(_capi.lib().hipgpt_embedding_scaled(_ptr("ids", ids, torch.int32, n), _ptr("tok", tok, dt, V * E), _ptr("pos", pos, dt, S * E), _ptr("out", out, dt, n * E),
                                                    scale, B, S, V, E, _type(out), _stream()))


def embedding_backward(grad_out, ids, grad_tok, grad_pos, B: int, S: int, V: int, E: int, *, scale: float = 1.0, accumulate: bool = False):
    """Gradients of the tables (float32 tables also for bfloat16 grad_out); either may be None."""
    n = B * S
    table = grad_tok if grad_tok is not None else grad_pos
    if table is None:
        return
    gt = table.dtype
    _capi.check(_capi.lib().hipgpt_embedding_backward(_ptr("grad_out", grad_out, grad_out.dtype, n * E), _ptr("ids", ids, torch.int32, n), _ptr("grad_tok", grad_tok, gt, V * E),
                                                      _ptr("grad_pos", grad_pos, gt, S * E), scale, int(accumulate), B, S, V, E, _type(grad_out), _type(table), _stream()))


def dropout_counter(x, residual, out, p: float, *, seed: int, offset: int = 0, counter=None):
    """out = [residual +] dropout(x); the same call on the gradient (residual None) is the backward pass.  counter: None, or an
    int64 CUDA tensor of one element that is added to `offset` when the kernel runs (for captured calls)."""
    n, dt, most = out.numel(), out.dtype, (1 << 64) - 1
    _capi.check(_capi.lib().hipgpt_dropout_counter(_ptr("x", x, dt, n), _ptr("residual", residual, dt, n), _ptr("out", out, dt, n), p, seed & most, offset & most,
                                                   _ptr("counter", counter, torch.int64, 1), n, _type(out), _stream()))


def linear_cross_entropy(x, w, targets, loss, lse, N: int, E: int, V: int, *, by_token: bool = True):
    """loss and log-sum-exp per row of softmax cross entropy of x W^T; w is [V, E] (by_token) or [E, V]; a row whose target is outside
    [0, V) gets zeros."""
    dt, f = x.dtype, torch.float32
    _capi.check(_capi.lib().hipgpt_linear_cross_entropy(_ptr("x", x, dt, N * E), _ptr("w", w, dt, V * E), _ptr("targets", targets, torch.int32, N), _ptr("loss", loss, f, N),
                                                        _ptr("lse", lse, f, N), N, E, V, _capi.WEIGHTS_VE if by_token else _capi.WEIGHTS_EV, _type(x), _stream()))


def linear_cross_entropy_backward(x, w, targets, lse, grad_loss, grad_x, grad_w, N: int, E: int, V: int, *, by_token: bool = True, accumulate: bool = False):
    """Gradients of x and w from that of each row's loss and the forward's lse; either may be None; accumulate: grad_w is added to."""
    dt, f = x.dtype, torch.float32
    _capi.check(_capi.lib().hipgpt_linear_cross_entropy_backward(
        _ptr("x", x, dt, N * E), _ptr("w", w, dt, V * E), _ptr("targets", targets, torch.int32, N), _ptr("lse", lse, f, N), _ptr("grad_loss", grad_loss, f, N),
        _ptr("grad_x", grad_x, dt, N * E), _ptr("grad_w", grad_w, dt, V * E), int(accumulate), N, E, V, _capi.WEIGHTS_VE if by_token else _capi.WEIGHTS_EV, _type(x), _stream()))
