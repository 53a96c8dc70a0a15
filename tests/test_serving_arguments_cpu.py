"""Arguments of serving.py's calls and of the C entry points below them, refused before anything looks at the GPU."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import _capi, launchers, serving  # noqa: E402

P = 0x7F0000000000              # addresses that nothing looks at
GB = 1 << 30


@pytest.fixture(params=["extension", "ctypes"])
def calls(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(launchers, "_native", launchers._ThroughCtypes)
    return serving


def _cache(**kw):
    d = dict(k=P, v=P + GB, k_scale=P + 2 * GB, v_scale=P + 3 * GB, pages=4, page_size=16, heads=2, head_dim=32, type=0, format=1)
    d.update(kw)
    return launchers._PagedCache(*d.values())


def _batch(**kw):
    d = dict(offsets=P + 4 * GB, lengths=P + 5 * GB, page_table=P + 6 * GB, sequences=2, tokens=8, most_pages=3)
    d.update(kw)
    return launchers._PagedBatch(*d.values())


def _all(cache, batch, k=P + 7 * GB, v=P + 8 * GB, stride=64, H=4):
    lib, c, b = _capi.lib(), C.byref(cache), C.byref(batch)
    return [lib.hipgpt_cache_write(c, b, k, stride, v, stride, None), lib.hipgpt_cache_read(c, b, k, stride, v, stride, None),
            lib.hipgpt_paged_attention(c, b, k, 2 * stride, v, 2 * stride, H, 1, 0.1, None)]


@pytest.mark.parametrize("kw,code", [(dict(type=2), _capi.ERR_BAD_ARG), (dict(format=3), _capi.ERR_BAD_ARG), (dict(pages=-1), _capi.ERR_BAD_ARG), (dict(page_size=8), _capi.ERR_BAD_ARG),
                                     (dict(page_size=48), _capi.ERR_BAD_ARG), (dict(page_size=2048), _capi.ERR_BAD_ARG), (dict(heads=0), _capi.ERR_BAD_ARG), (dict(head_dim=0), _capi.ERR_BAD_ARG),
                                     (dict(head_dim=40), _capi.ERR_UNSUPPORTED), (dict(head_dim=256), _capi.ERR_UNSUPPORTED), (dict(k=None), _capi.ERR_NULL), (dict(v_scale=None), _capi.ERR_NULL),
                                     (dict(k=P + 8), _capi.ERR_BAD_ARG), (dict(k_scale=P + 2 * GB + 4), _capi.ERR_BAD_ARG)])
def test_caches_that_are_none(kw, code):
    assert _all(_cache(**kw), _batch()) == [code] * 3
    assert _capi.lib().hipgpt_last_error()


@pytest.mark.parametrize("kw,code", [(dict(sequences=-1), _capi.ERR_BAD_ARG), (dict(tokens=-1), _capi.ERR_BAD_ARG), (dict(most_pages=-1), _capi.ERR_BAD_ARG), (dict(most_pages=1 << 28), _capi.ERR_BAD_ARG),
                                     (dict(offsets=None), _capi.ERR_NULL), (dict(lengths=None), _capi.ERR_NULL), (dict(page_table=None), _capi.ERR_NULL)])
def test_batches_that_are_none(kw, code):
    assert _all(_cache(), _batch(**kw)) == [code] * 3


def test_nothing_to_do():
    for kw in (dict(tokens=0), dict(sequences=0)):
        assert _all(_cache(), _batch(**kw), k=None, v=None) == [_capi.OK] * 3
    assert _capi.lib().hipgpt_paged_attention(None, C.byref(_batch()), P, 64, P, 64, 2, 1, 0.1, None) == _capi.ERR_NULL


def test_rows_that_are_none():
    assert _all(_cache(), _batch(), k=None) == [_capi.ERR_NULL] * 3
    assert _all(_cache(), _batch(), stride=63) == [_capi.ERR_BAD_ARG] * 3
    assert _all(_cache(), _batch(), stride=-64) == [_capi.ERR_BAD_ARG] * 3
    for H in (0, -2, 3):
        assert _all(_cache(), _batch(), H=H)[2] == _capi.ERR_BAD_ARG
    lib = _capi.lib()
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert lib.hipgpt_paged_attention(C.byref(_cache()), C.byref(_batch()), P + 7 * GB, 128, P + 8 * GB, 128, 4, 1, scale, None) == _capi.ERR_BAD_ARG


def test_outputs_over_other_arrays():
    lib, c, b = _capi.lib(), _cache(), _batch()
    at = P + 7 * GB
    bad = _capi.ERR_BAD_ARG
    # (rows of q are 512 bytes, of k 256: the last of them ends at 512 * 7 + 256)
    assert lib.hipgpt_paged_attention(C.byref(c), C.byref(b), at, 128, at + 512 * 8 - 4, 128, 4, 1, 0.1, None) == bad
    assert lib.hipgpt_cache_read(C.byref(c), C.byref(b), at, 128, at + 512 * 7 + 252, 128, None) == bad
    for out in (P + 100, P + 2 * GB, P + 4 * GB + 4, P + 5 * GB, P + 6 * GB):
        assert lib.hipgpt_paged_attention(C.byref(c), C.byref(b), at, 128, out, 128, 4, 1, 0.1, None) == bad, hex(out)
        assert lib.hipgpt_cache_read(C.byref(c), C.byref(b), at, 128, out, 128, None) == bad, hex(out)
    # columns of one array: over each other
    assert lib.hipgpt_cache_read(C.byref(c), C.byref(b), at, 128, at + 63 * 4, 128, None) == bad
    assert lib.hipgpt_cache_read(C.byref(c), C.byref(b), at, 100, at + 64 * 4, 100, None) == bad
    # the cache over what is written to it
    assert lib.hipgpt_cache_write(C.byref(c), C.byref(b), P + 64, 64, at, 64, None) == bad
    assert lib.hipgpt_cache_write(C.byref(_cache(v=P + 1024)), C.byref(b), at, 64, at, 64, None) == bad
    assert lib.hipgpt_rotary(at, 64, P, P + GB, at + 256, 64, 1.0, 0, 0, 8, 1, 64, 64, 0, None) == bad
    assert lib.hipgpt_rotary(at, 64, P, P + GB, at, 128, 1.0, 0, 0, 8, 1, 64, 64, 0, None) == bad
    assert lib.hipgpt_rotary(at, 64, P, P + GB, P, 64, 1.0, 0, 0, 8, 1, 64, 64, 0, None) == bad


def test_rotations_that_are_none():
    lib, at, out = _capi.lib(), P + 7 * GB, P + 8 * GB
    for T, H, D, R, type_ in ((-1, 1, 64, 64, 0), (8, -1, 64, 64, 0), (8, 1, 64, 63, 0), (8, 1, 64, 66, 0), (8, 1, 64, -2, 0), (8, 1, 2000, 64, 0), (8, 1, 64, 64, 2), (8, 1 << 20, 64, 64, 0)):
        assert lib.hipgpt_rotary(at, 1 << 30, P, P + GB, out, 1 << 30, 1.0, 0, 0, T, H, D, R, type_, None) == _capi.ERR_BAD_ARG
    assert lib.hipgpt_rotary(at, 63, P, P + GB, out, 64, 1.0, 0, 0, 8, 1, 64, 64, 0, None) == _capi.ERR_BAD_ARG
    assert lib.hipgpt_rotary(None, 64, P, P + GB, out, 64, 1.0, 0, 0, 8, 1, 64, 64, 0, None) == _capi.ERR_NULL
    assert lib.hipgpt_rotary(at, 64, None, P + GB, out, 64, 1.0, 0, 0, 8, 1, 64, 64, 0, None) == _capi.ERR_NULL
    assert lib.hipgpt_rotary(None, 64, None, None, None, 64, 1.0, 0, 0, 0, 1, 64, 64, 0, None) == _capi.OK
    for kw in (dict(R=7), dict(R=-2), dict(R=8, base=0.0), dict(R=8, base=math.inf), dict(R=8, scaling="linear", factor=0.0), dict(R=8, scaling="ramp", factor=2.0),
               dict(R=8, scaling="ramp", factor=2.0, original=100.0, low=4.0, high=4.0)):
        with pytest.raises(_capi.HipGPTError):
            serving.rotary_frequencies(**kw)
    with pytest.raises(ValueError):
        serving.rotary_frequencies(8, scaling="other")
    with pytest.raises(_capi.HipGPTError):
        serving.rotary_words([1.0, math.nan], "cpu")


def test_words_are_fractions_of_a_turn():
    w = serving.rotary_words([0.0, math.pi, -math.pi / 2, 2 * math.pi * 5, 1.0], "cpu")
    turns = [int(x) % (1 << 64) / 2.0 ** 64 for x in w.tolist()]
    assert turns[0] == 0.0 and turns[1] == 0.5 and turns[2] == 0.75 and turns[3] == 0.0
    assert abs(turns[4] - 1 / (2 * math.pi)) < 2.0 ** -54


def _fake_cache():
    """A PagedCache of CPU tensors is refused, so one is put together without its checks."""
    c = serving.PagedCache.__new__(serving.PagedCache)
    c._struct = _cache(format=0)
    c._address, c._device, c.head_dim = C.addressof(c._struct), 0, 32
    return c


def test_what_is_no_cache_or_tensor_is_named(calls):
    z, i = torch.zeros(8, 64), torch.zeros(3, dtype=torch.int32)
    args = i, i, torch.zeros(2, 3, dtype=torch.int32), 8, 2
    for bad in (None, 7, z):
        with pytest.raises(ValueError, match="cache"):
            calls.cache_write(bad, z, z, *args)
        with pytest.raises(ValueError, match="cache"):
            calls.paged_attention(bad, z, z, *args, 2)
    c = _fake_cache()
    for bad in (None, 7, "x"):
        with pytest.raises(ValueError, match="k:"):
            calls.cache_write(c, bad, z, *args)
        with pytest.raises(ValueError, match="q:"):
            calls.paged_attention(c, bad, z, *args, 2)
        with pytest.raises(ValueError, match="out"):
            calls.rotary(z, i, i, bad, 8, 1, 64, 64)
        with pytest.raises(ValueError, match="x"):
            calls.rotary(bad, i, i, z, 8, 1, 64, 64)
    with pytest.raises(ValueError, match="q has rows of 64 values, 128"):
        calls.paged_attention(c, z, z, *args, 4)
    with pytest.raises(ValueError, match="k has rows of"):
        calls.cache_read(c, torch.zeros(64, 8), z, *args)
    with pytest.raises(ValueError, match="CUDA"):
        calls.cache_read(c, z, z, *args)


@pytest.mark.parametrize("size", [(1 << 32) + 2, 1 << 31, -(1 << 31) - 1])
def test_sizes_that_an_int_does_not_hold(calls, size):
    z, i, p = torch.zeros(8, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    c = _fake_cache()
    with pytest.raises(ValueError, match="beyond one call"):
        calls.cache_write(c, z, z, i, i, p, size, 2)
    with pytest.raises(ValueError, match="beyond one call"):
        calls.paged_attention(c, z, z, i, i, p, 8, size, 2)
    with pytest.raises(ValueError, match="beyond one call"):
        calls.rotary(z, i, i, z, 8, 1, size, 64)
    with pytest.raises(TypeError):
        calls.rotary(z, i, i, z, 8, 1, 64.0, 64)


def test_paged_caches_that_are_refused():
    for kw in (dict(format="fp4"), dict(dtype=torch.float16), dict(page_size=17), dict(page_size=8), dict(heads=-1), dict(num_pages=1 << 32)):
        full = dict(num_pages=2, page_size=16, heads=2, head_dim=32)
        full.update(kw)
        with pytest.raises(ValueError):
            serving.PagedCache(**full)
    with pytest.raises(ValueError):
        serving.PagedCache(2, 16, 2, 32, k=torch.zeros(2, 2, 16, 32), v=torch.zeros(2, 2, 16, 32))


def test_waits_that_no_kernel_has():
    for code in (1000, 1013, 1099, 1100):
        assert _capi.lib().hipgpt_debug_expire_wait(code, 0) == _capi.ERR_BAD_ARG


def test_rows_of_another_number_of_heads(calls):
    """A tensor of more heads than the call says is no tensor of its rows, although its heads have the right width."""
    i, p, c = torch.zeros(3, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32), _fake_cache()
    for shape in ((8, 5, 32), (2, 4, 6, 32), (8, 8, 32)):
        x = torch.zeros(shape)
        with pytest.raises(ValueError, match="q has rows of"):
            calls.paged_attention(c, x, x, i, i, p, 8, 2, 4)
        with pytest.raises(ValueError, match="x has rows of"):
            calls.rotary(x, i, i, x, 8, 4, 32, 32)
        with pytest.raises(ValueError, match="k has rows of"):
            calls.cache_write(c, x, x, i, i, p, 8, 2)
    for shape in ((8, 4, 32), (2, 4, 4, 32), (8, 128), (2, 4, 128), (32, 32), (1024,)):         # what their rows may be told as; CPU tensors are refused as such
        x = torch.zeros(shape)
        with pytest.raises(ValueError, match="q: expected a CUDA"):
            calls.paged_attention(c, x, x, i, i, p, 8, 2, 4)


def test_a_caches_arrays_stay_its_own():
    """What the library writes to is what the handle shows and keeps."""
    c = _fake_cache()
    c._arrays = tuple(torch.zeros(1) for _ in range(4))
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, torch.zeros(1))
    for bad in ([1.0], 7, "x"):
        with pytest.raises(ValueError, match="k: expected"):
            serving.PagedCache(2, 16, 2, 32, k=bad, v=torch.zeros(2, 2, 16, 32))
