"""Arguments of training.py's calls that the counts of values cannot tell from right ones, refused before anything looks at the GPU: by the extension and by the calls through ctypes."""
import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import launchers, training  # noqa: E402


@pytest.fixture(params=["extension", "ctypes"])
def calls(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(launchers, "_native", launchers._ThroughCtypes)
    return training


def _loss_tensors(N, w_shape):
    return torch.zeros(N, 8), torch.zeros(w_shape), torch.zeros(N, dtype=torch.int32), torch.zeros(N), torch.zeros(N)


@pytest.mark.parametrize("by_token,shape", [(True, (8, 16)), (False, (16, 8)), (True, (2, 8, 8, 4))])
def test_weights_the_other_way_round(calls, by_token, shape):
    x, w, t, loss, lse = _loss_tensors(4, shape)
    with pytest.raises(ValueError, match="w has rows of"):
        calls.linear_cross_entropy(x, w, t, loss, lse, 4, 8, 16, by_token=by_token)
    with pytest.raises(ValueError, match="w has rows of"):
        calls.linear_cross_entropy_backward(x, w, t, lse, loss, x.clone(), w.clone(), 4, 8, 16, by_token=by_token)


@pytest.mark.parametrize("by_token,shape", [(True, (16, 8)), (False, (8, 16)), (True, (128,)), (False, (128,)), (True, (20, 8)), (False, (9, 16))])
def test_weights_that_are_right_or_say_nothing_are_looked_at_further(calls, by_token, shape):
    """... and refused here for not being on a GPU."""
    x, w, t, loss, lse = _loss_tensors(4, shape)
    with pytest.raises(ValueError, match="CUDA"):
        calls.linear_cross_entropy(x, w, t, loss, lse, 4, 8, 16, by_token=by_token)


def test_tables_the_other_way_round(calls):
    ids, out = torch.zeros(6, dtype=torch.int32), torch.zeros(6, 8)
    refused = pytest.raises(ValueError, match="tok has rows of")
    with refused:
        calls.embedding_scaled(ids, torch.zeros(8, 5), None, out, 2, 3, 5, 8)
    with refused:
        calls.embedding_backward(out, ids, torch.zeros(8, 5), None, 2, 3, 5, 8)


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("size", [(1 << 32) + 4, -(1 << 32) + 4, 1 << 31, 1 << 70])
def test_sizes_that_an_int_does_not_hold(calls, which, size):
    """(1 << 32) + 4 is not 4."""
    x, w, t, loss, lse = _loss_tensors(4, (4, 4))
    sizes = [4, 4, 4, 4]
    sizes[which] = size
    refused = pytest.raises(ValueError, match="beyond one call")
    with refused:
        calls.embedding_scaled(t, w, None, x, *sizes)
    with refused:
        calls.embedding_backward(x, t, w, None, *sizes)
    if which < 3:
        with refused:
            calls.linear_cross_entropy(x, w, t, loss, lse, *sizes[:3])
        with refused:
            calls.linear_cross_entropy_backward(x, w, t, lse, loss, x.clone(), w.clone(), *sizes[:3])


def test_what_is_no_tensor_is_named(calls):
    x, w, t, loss, lse = _loss_tensors(4, (16, 8))
    for bad in (None, 7, "x", [1.0]):
        with pytest.raises(ValueError, match="out"):
            calls.embedding_scaled(t, w, None, bad, 1, 4, 16, 8)
        with pytest.raises(ValueError, match="grad_out"):
            calls.embedding_backward(bad, t, w, None, 1, 4, 16, 8)
        with pytest.raises(ValueError, match="out"):
            calls.dropout_counter(x, None, bad, 0.1, seed=1)
        with pytest.raises(ValueError, match="x"):
            calls.linear_cross_entropy(bad, w, t, loss, lse, 4, 8, 16)
        with pytest.raises(ValueError, match="x"):
            calls.linear_cross_entropy_backward(bad, w, t, lse, loss, None, w.clone(), 4, 8, 16)
    with pytest.raises(ValueError, match="w"):
        calls.linear_cross_entropy(x, 3.0, t, loss, lse, 4, 8, 16)


def test_sizes_that_are_no_integers(calls):
    x, w, t, loss, lse = _loss_tensors(4, (16, 8))
    with pytest.raises(TypeError):
        calls.linear_cross_entropy(x, w, t, loss, lse, 4.0, 8, 16)


@pytest.mark.parametrize("at", [0, 8, 248])
def test_dropout_into_its_own_counter(at):
    """Blocks read the counter while others store."""
    from hipgpt_b200 import _capi
    P = 0x7F0000000000
    assert _capi.lib().hipgpt_dropout_counter(P + (1 << 32), None, P, 0.1, 1, 0, P + at, 64, 0, None) == _capi.ERR_BAD_ARG
