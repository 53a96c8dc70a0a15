"""The operators at the two ends of a training step on CUDA torch tensors: embedding and its gradient, dropout from a
counter, the loss and its gradient (the C entry points of the same names in include/hipgpt_attn.h, which say what each computes).

Like launchers.py: outputs are given by the caller, calls are asynchronous on torch's current stream, torch holds the memory and
nothing else.  Activations and weights are contiguous float32 or bfloat16 tensors, one type per call; ids and targets int32.  All
tensors are on the current device.  Sizes beyond what a tensor holds are refused, and tables and weights of two dimensions whose
rows have another length than the sizes say.
"""
from __future__ import annotations

from . import _capi, launchers


def _check(rc):
    if rc:
        _capi.check(rc)


def embedding_scaled(ids, tok, pos, out, B: int, S: int, V: int, E: int, *, scale: float = 1.0):
    """out[t] = scale tok[id_t] + pos[t mod S]; pos may be None; zeros for an id outside [0, V)."""
    _check(launchers._native.embedding_scaled(ids, tok, pos, out, scale, B, S, V, E))


def embedding_backward(grad_out, ids, grad_tok, grad_pos, B: int, S: int, V: int, E: int, *, scale: float = 1.0, accumulate: bool = False):
    """Gradients of the tables (float32 tables also for bfloat16 grad_out); either may be None."""
    if grad_tok is not None or grad_pos is not None:
        _check(launchers._native.embedding_backward(grad_out, ids, grad_tok, grad_pos, scale, int(accumulate), B, S, V, E))


def dropout_counter(x, residual, out, p: float, *, seed: int, offset: int = 0, counter=None):
    """out = [residual +] dropout(x); the same call on the gradient (residual None) is the backward pass.  counter: None, or an
    int64 CUDA tensor of one element that is added to `offset` when the kernel runs (for captured calls)."""
    _check(launchers._native.dropout_counter(x, residual, out, counter, p, seed, offset))


def linear_cross_entropy(x, w, targets, loss, lse, N: int, E: int, V: int, *, by_token: bool = True):
    """loss and log-sum-exp per row of softmax cross entropy of x W^T; w is [V, E] (by_token) or [E, V]; a row whose target is outside
    [0, V) gets zeros."""
    _check(launchers._native.linear_cross_entropy(x, w, targets, loss, lse, N, E, V, _capi.WEIGHTS_VE if by_token else _capi.WEIGHTS_EV))


def linear_cross_entropy_backward(x, w, targets, lse, grad_loss, grad_x, grad_w, N: int, E: int, V: int, *, by_token: bool = True, accumulate: bool = False):
    """Gradients of x and w from that of each row's loss and the forward's lse; either may be None; accumulate: grad_w is added to."""
    _check(launchers._native.linear_cross_entropy_backward(x, w, targets, lse, grad_loss, grad_x, grad_w, int(accumulate), N, E, V,
                                                           _capi.WEIGHTS_VE if by_token else _capi.WEIGHTS_EV))
