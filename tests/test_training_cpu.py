"""Refusals of the operators at the two ends of a training step, and calls that do nothing: decided on the host, before any CUDA call."""
import ctypes as C

import pytest

from hipgpt_b200 import _capi

torch = pytest.importorskip("torch")
BAD, NULL, UNSUPPORTED = _capi.ERR_BAD_ARG, _capi.ERR_NULL, _capi.ERR_UNSUPPORTED
P = 0x7F0000000000                       # an address that is never followed


def _lib():
    return _capi.lib()


@pytest.mark.parametrize("args,code", [
    ((None, P, P, P, 1.0, 2, 3, 5, 8, 0), NULL), ((P, None, P, P, 1.0, 2, 3, 5, 8, 0), NULL), ((P, P, P, None, 1.0, 2, 3, 5, 8, 0), NULL),
    ((P, P, P, P, 1.0, -1, 3, 5, 8, 0), BAD), ((P, P, P, P, 1.0, 2, -3, 5, 8, 0), BAD), ((P, P, P, P, 1.0, 2, 3, -5, 8, 0), BAD), ((P, P, P, P, 1.0, 2, 3, 5, -8, 0), BAD),
    ((P, P, P, P, 1.0, 2, 3, 5, 8, 2), BAD), ((P, P, P, P, 1.0, 1 << 20, 1 << 20, 5, 8, 0), UNSUPPORTED),
    ((None, None, None, None, 1.0, 0, 3, 5, 8, 0), 0), ((None, None, None, None, 1.0, 2, 0, 5, 8, 1), 0), ((None, None, None, None, 1.0, 2, 3, 5, 0, 1), 0)])
def test_embedding(args, code):
    assert _lib().hipgpt_embedding_scaled(*args, None) == code


@pytest.mark.parametrize("args,code", [
    ((None, P, P, P, 1.0, 0, 2, 3, 5, 8, 0, 0), NULL), ((P, None, P, P, 1.0, 0, 2, 3, 5, 8, 0, 0), NULL),
    ((P, P, P, P, 1.0, 0, 2, 3, 5, 8, 3, 0), BAD), ((P, P, P, P, 1.0, 0, 2, 3, 5, 8, 0, -1), BAD), ((P, P, P, P, 1.0, 0, 2, 3, 5, 8, 0, 1), UNSUPPORTED),
    ((P, P, P, P, 1.0, 0, -2, 3, 5, 8, 0, 0), BAD), ((P, P, P, P, 1.0, 0, 1 << 16, 1 << 16, 5, 8, 0, 0), UNSUPPORTED),
    ((P, P, None, None, 1.0, 0, 2, 3, 5, 8, 0, 0), 0), ((None, None, P, P, 1.0, 0, 2, 3, 5, 0, 0, 0), 0), ((None, None, P, P, 1.0, 1, 0, 3, 5, 8, 0, 0), 0)])
def test_embedding_backward(args, code):
    assert _lib().hipgpt_embedding_backward(*args, None) == code


@pytest.mark.parametrize("args,code", [
    ((None, None, P, 0.1, 1, 0, None, 64, 0), NULL), ((P, None, None, 0.1, 1, 0, None, 64, 0), NULL),
    ((P, None, P, 1.0, 1, 0, None, 64, 0), BAD), ((P, None, P, -0.1, 1, 0, None, 64, 0), BAD), ((P, None, P, float("nan"), 1, 0, None, 64, 0), BAD),
    ((P, None, P, 0.1, 1, 0, None, -1, 0), BAD), ((P, None, P, 0.1, 1, 0, None, 64, 7), BAD),
    ((P, None, P + 4, 0.1, 1, 0, None, 64, 0), BAD), ((P, P + 252, P, 0.1, 1, 0, None, 64, 0), BAD),          # out overlaps an input without being it
    ((None, None, None, 0.1, 1, 0, None, 0, 0), 0)])
def test_dropout(args, code):
    assert _lib().hipgpt_dropout_counter(*args, None) == code


@pytest.mark.parametrize("which", range(5))
def test_loss_null(which):
    ptrs = [P] * 5
    ptrs[which] = None
    assert _lib().hipgpt_linear_cross_entropy(*ptrs, 4, 8, 16, 0, 0, None) == NULL
    assert _lib().hipgpt_linear_cross_entropy_backward(*ptrs, P, P, 0, 4, 8, 16, 0, 0, None) == NULL


@pytest.mark.parametrize("sizes,code", [((-1, 8, 16, 0, 0), BAD), ((4, 0, 16, 0, 0), BAD), ((4, 8, 0, 0, 0), BAD), ((4, 8, 16, 2, 0), BAD), ((4, 8, 16, 0, 2), BAD),
                                        ((1 << 27, 8, 16, 0, 0), UNSUPPORTED), ((4, 1 << 21, 16, 0, 0), UNSUPPORTED), ((4, 8, 1 << 29, 0, 0), UNSUPPORTED), ((0, 8, 16, 1, 1), 0)])
def test_loss_sizes(sizes, code):
    assert _lib().hipgpt_linear_cross_entropy(P, P, P, P, P, *sizes, None) == code
    assert _lib().hipgpt_linear_cross_entropy_backward(P, P, P, P, P, P, P, 1, *sizes, None) == code


def test_loss_backward_without_gradients_does_nothing():
    assert _lib().hipgpt_linear_cross_entropy_backward(P, P, P, P, P, None, None, 0, 4, 8, 16, 0, 0, None) == 0


def test_refusals_name_their_reason():
    _lib().hipgpt_dropout_counter(P, None, P, 1.5, 1, 0, None, 64, 0, None)
    assert b"outside [0, 1)" in _lib().hipgpt_last_error()


def test_the_python_calls_refuse_what_is_no_gpu_tensor():
    from hipgpt_b200 import training
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        training.dropout_counter(x, None, x, 0.1, seed=1)
    with pytest.raises(ValueError, match="float32 or bfloat16|CUDA"):
        training.embedding_scaled(torch.zeros(4, dtype=torch.int32), x.half(), None, x.half(), 1, 4, 4, 8)


def test_an_expiring_wait_can_be_asked_for_in_the_loss():
    assert _lib().hipgpt_debug_expire_wait(700, 0) == BAD
    assert _lib().hipgpt_debug_expire_wait(801, 0) == BAD


G = 1 << 32                              # addresses this far apart hold arrays that do not meet


@pytest.mark.parametrize("V,E", [((1 << 31) - 1, 1), (1 << 30, 8), (1, (1 << 31) - 1), (5, 1 << 30)])
def test_embedding_tables_beyond_the_index_range(V, E):
    assert _lib().hipgpt_embedding_scaled(P, P + G, None, P + 2 * G, 1.0, 1, 1, V, E, 1, None) == UNSUPPORTED
    assert _lib().hipgpt_embedding_backward(P, P + G, P + 2 * G, None, 1.0, 0, 1, 1, V, E, 1, 1, None) == UNSUPPORTED


def _with(arrays, which, at):
    return [at if i == which else a for i, a in enumerate(arrays)]


@pytest.mark.parametrize("which,size", [(0, 6 * 4), (1, 5 * 32), (2, 3 * 32)])
def test_embedding_into_its_own_inputs(which, size):
    for at in (P + 9 * G, P + 9 * G - size + 4, P + 9 * G + 6 * 32 - 4):
        ptrs = _with([P, P + G, P + 2 * G], which, at)
        assert _lib().hipgpt_embedding_scaled(*ptrs, P + 9 * G, 1.0, 2, 3, 5, 8, 0, None) == BAD


@pytest.mark.parametrize("out,other", [(2, 0), (2, 1), (3, 0), (3, 1), (2, 3)])
def test_embedding_gradient_into_its_own_inputs(out, other):
    ptrs = [P, P + G, P + 2 * G, P + 3 * G]
    assert _lib().hipgpt_embedding_backward(*_with(ptrs, out, ptrs[other]), 1.0, 0, 2, 3, 5, 8, 0, 0, None) == BAD


@pytest.mark.parametrize("out,other", [(3, 0), (3, 1), (3, 2), (4, 0), (4, 1), (4, 2), (3, 4)])
def test_loss_into_its_own_inputs(out, other):
    ptrs = [P + i * G for i in range(5)]
    assert _lib().hipgpt_linear_cross_entropy(*_with(ptrs, out, ptrs[other]), 4, 8, 16, 0, 0, None) == BAD


@pytest.mark.parametrize("out,other", [(5, i) for i in range(5)] + [(6, i) for i in range(6)])
def test_loss_gradient_into_its_own_inputs(out, other):
    ptrs = [P + i * G for i in range(7)]
    assert _lib().hipgpt_linear_cross_entropy_backward(*_with(ptrs, out, ptrs[other]), 0, 4, 8, 16, 0, 0, None) == BAD
