"""Attention over a cache in pages and the cache's calls at the edges of their ranges (forms and bounds of tests/serving_util.py)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import _capi, serving  # noqa: E402
from tests import serving_util as su  # noqa: E402
from tests.serving_util import BF16, F32, Batch, within  # noqa: E402

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _status():
    st = C.c_int(-1)
    _capi.check(_capi.lib().hipgpt_kernel_status(C.byref(st)))
    return st.value


# ---- NaN codes --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_code_read_back(dtype):
    """A cache filled elsewhere: each of the 256 codes stands for the same value as torch's type, NaN among them."""
    for fmt, codes in su.CODES.items():
        heads, D, page = 2, 128, 16
        cache = serving.PagedCache(2, page, heads, D, dtype=dtype, format=fmt)
        raw = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(2 * heads * page * D // 256).view(2, heads, page, D)
        cache.k.view(torch.uint8).copy_(raw)
        cache.v.view(torch.uint8).copy_(raw.flip(-1))
        cache.k_scale.fill_(0.5)
        cache.v_scale.fill_(4.0)
        batch = Batch([(32, 32)], page, spare=0)
        back = [torch.zeros(32, heads, D, device="cuda", dtype=dtype) for _ in range(2)]
        serving.cache_read(cache, *back, *batch.args)
        at = batch.pages[0].long().repeat_interleave(page), torch.arange(page, device="cuda").repeat(2)
        for got, held, scale in ((back[0], cache.k, 0.5), (back[1], cache.v, 4.0)):
            want = (held.float() * scale)[at[0], :, at[1]].to(dtype)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
        assert (fmt == "e4m3") == bool(torch.isnan(back[0]).any())


@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("dtype,seqs,H", [(BF16, [(4, 60), (3, 200)], 4), (F32, [(4, 60), (3, 200)], 4), (BF16, [(12, 500)], 4), (F32, [(12, 500)], 4), (F32, [(300, 900), (70, 80)], 4),
                                          (BF16, [(1, 2), (300, 2000)], 4), (BF16, [(700, 900), (1000, 1200)], 8)], ids=["tokens", "tokens32", "rows", "rows32", "many32", "tcgen05", "widened"])
def test_a_nan_code_matters_to_the_rows_that_see_it(dtype, seqs, H, name):
    """A NaN code under a finite scale: the rows before its position are as they were without, the others are NaN."""
    batch = Batch(seqs, 16, seed=3)
    heads, D = 2, 32
    n, length = batch.seqs[-1]
    cache, k, v = su.filled_cache(batch, heads, D, dtype, "e4m3")
    p = length - 2                                                  # the last row but one sees it, the one before does not
    page, slot = int(batch.table[-1, p // 16]), p % 16
    getattr(cache, name).view(torch.uint8)[page, 1, slot, 3] = 0x7F if name == "k" else 0xFF
    (k if name == "k" else v)[page, 1, slot, 3] = float("nan")
    q = _normal(_gen(5), batch.T, H, D, dtype=dtype)
    out = torch.zeros_like(q)
    serving.paged_attention(cache, q, out, *batch.args, H)
    want, bound, _ = su.attention(batch, k, v, q, H, True, float(torch.tensor(D ** -0.5)), dtype, "e4m3")
    clean = torch.ones(batch.T, H, dtype=torch.bool, device="cuda")
    clean[batch.first[-2] + n - 2:, H // heads:] = False
    within(out[clean], want[clean], bound[clean], "rows that do not see it")
    seen = out[~clean]
    assert bool(torch.isnan(seen if name == "k" else seen[:, 3]).all()), "rows that do"


# ---- rows touched by what they do not see -------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,fmt,heads,H,D,seqs", [(BF16, "plain", 2, 4, 64, [(600, 140000), (40, 300)]), (BF16, "e4m3", 1, 2, 128, [(600, 140000), (40, 300)]), (BF16, "int8", 1, 4, 64, [(1000, 140000), (900, 950)]),
                                                      (F32, "plain", 2, 2, 32, [(500, 140000), (40, 300)]), (F32, "int8", 1, 2, 64, [(300, 140000), (40, 300)]), (BF16, "e4m3", 2, 2, 64, [(8, 200000), (8, 200)]),
                                                      (BF16, "plain", 8, 32, 128, [(1500, 20000), (900, 2000)]), (F32, "plain", 16, 32, 64, [(700, 9000), (300, 2000)])])
def test_an_infinity_that_long_rows_do_not_see(dtype, fmt, heads, H, D, seqs):
    """An infinity in the last value of a long sequence: the rows of its tile are worked out again, and no wait runs out for it in their block, so that everything else is as ever."""
    batch = Batch(seqs, 64, seed=3)
    n, length = seqs[0]
    page, slot = int(batch.table[0, (length - 1) // 64]), (length - 1) % 64

    def wild(name, x):
        if name == "v":
            x[page, :, slot, 3] = float("inf")
    cache, k, v = su.filled_cache(batch, heads, D, dtype, fmt, wild=wild)
    q = _normal(_gen(5), batch.T, H, D, dtype=dtype)
    out = torch.zeros_like(q)
    serving.paged_attention(cache, q, out, *batch.args, H)
    torch.cuda.synchronize()
    assert _status() == 0
    want, bound, _ = su.attention(batch, k, v, q, H, True, float(torch.tensor(D ** -0.5)), dtype, fmt)
    clean = torch.ones(batch.T, dtype=torch.bool, device="cuda")
    clean[n - 1] = False
    within(out[clean], want[clean], bound[clean])
    assert not bool(torch.isfinite(out[n - 1, :, 3]).any()), "the row that sees it"


# ---- the largest numbers ------------------------------------------------------------------------------------------------

# Each kernel of fp32 over a plain cache: single tokens, some rows, many cut by the warps, many cut before
FP32 = [([(1, 700), (2, 90)], 4, 64), ([(9, 300), (12, 77)], 2, 128), ([(40, 300), (25, 77)], 2, 32), ([(150, 300), (170, 400)], 2, 32), ([(200, 300), (170, 400)], 2, 128)]


@pytest.mark.parametrize("seqs,H,D", FP32, ids=["tokens", "some", "many", "cut32", "cut128"])
def test_fp32_next_to_its_largest_number(seqs, H, D):
    """Values, keys and queries beyond bf16's largest number, 3.39e38, are numbers; an infinite value makes infinities."""
    most = torch.finfo(F32).max
    batch, heads = Batch(seqs, 16, seed=5), 2
    n, length = batch.seqs[-1]
    page, slot = int(batch.table[-1, (length - 2) // 16]), (length - 2) % 16

    def run(wild, scale=None, spread=1.0, turn=None):
        cache, k, v = su.filled_cache(batch, heads, D, F32, "plain", wild=wild)
        q = _normal(_gen(5), batch.T, H, D, scale=spread)
        if turn is not None:
            turn(q)
        out = torch.zeros_like(q)
        serving.paged_attention(cache, q, out, *batch.args, H, scale=scale)
        want, bound, _ = su.attention(batch, k, v, q, H, True, float(torch.tensor(D ** -0.5 if scale is None else scale)), F32, "plain")
        return out, want, bound

    def values(name, x):
        if name == "v":
            x[page, :, slot, 3], x[page, :, slot, 4], x[page, :, slot, 5] = most, -3.4e38, 3.397e38
    within(*run(values), "values")

    def keys(name, x):
        if name == "k":
            x *= 1e-3
            x[page, :, slot, 3], x[page, :, slot, 7] = most, -3.398e38
    within(*run(keys, scale=1e-10, spread=1e-28), "keys")

    def small(name, x):
        if name == "k":
            x *= 1e-28

    def queries(q):
        q[-2:, :, 3], q[-1:, :, 7] = most, -3.398e38
    within(*run(small, scale=1e-10, turn=queries), "queries")

    def infinite(name, x):
        if name == "v":
            x[page, :, slot, 3], x[page, :, slot, 4] = float("inf"), float("-inf")
    out, want, bound = run(infinite)
    sees = torch.zeros(batch.T, dtype=torch.bool, device="cuda")
    sees[-2:] = True
    within(out[~sees], want[~sees], bound[~sees], "rows that do not see it")
    assert bool((out[sees][..., 3] == float("inf")).all()) and bool((out[sees][..., 4] == float("-inf")).all()) and bool(torch.isfinite(out[sees][..., 5:]).all())


@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("seqs,H", [([(1, 700), (2, 90)], 4), ([(12, 300), (9, 3000)], 4), ([(200, 500), (170, 400)], 4), ([(700, 5000), (900, 950)], 8)], ids=["tokens", "some", "many", "wide"])
def test_averages_of_the_largest_numbers(dtype, fmt, seqs, H):
    """Values of which a few pass fp32's range together: their average does not."""
    batch, heads, D = Batch(seqs, 64, seed=5), 2, 64

    def wild(name, x):
        if name == "v":
            x.clamp_(-1, 1)
            x[..., 3].fill_(3.0e38)
            x[..., 5].fill_(-2.9e38)
            x[..., 7] *= 3.0e38
    _cache, k, v = su.filled_cache(batch, heads, D, dtype, fmt, wild=wild)
    assert bool(torch.isfinite(v).all())
    q = _normal(_gen(5), batch.T, H, D, dtype=dtype, scale=0.25)
    out = torch.zeros_like(q)
    serving.paged_attention(_cache, q, out, *batch.args, H)
    want, bound, _ = su.attention(batch, k, v, q, H, True, float(torch.tensor(D ** -0.5)), dtype, fmt)
    within(out, want, bound)
    assert _status() == 0


# ---- sums over many keys --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("n,heads,H,D,copies", [(1, 16, 16, 32, 28), (1, 16, 192, 32, 28), (2400, 1, 16, 64, 1), (80, 2, 64, 64, 4)], ids=["tokens", "some", "wide", "many"])
def test_sums_over_a_million_keys(fmt, n, heads, H, D, copies):
    """Keys of zeros: every row is the average of all values.  What a sum in the tensor core's accumulators cuts off, always towards zero, must not add up over a long run of keys."""
    page, length = 1024, 1 << 20
    batch = Batch([(n, length)], page, seed=2)
    cache = serving.PagedCache(batch.num_pages, page, heads, D, dtype=BF16, format=fmt)
    cache.k.view(torch.uint8).zero_()
    gen = _gen(6)
    mean = torch.zeros(heads, D, dtype=torch.float64, device="cuda")
    lean = torch.rand(heads, 1, D, generator=gen, device="cuda") * 0.25
    used = torch.zeros(batch.num_pages, dtype=torch.float64)
    used[batch.table[0].long()] = 1.0
    for some in torch.arange(batch.num_pages, device="cuda").split(64):
        x = torch.rand(len(some), heads, page, D, generator=gen, device="cuda") * 0.7 + 1.0 + lean
        if fmt == "plain":
            cache.v[some] = x.to(BF16)
            x = x.to(BF16).double()
        else:
            code, unit = su.quantised(x, fmt)
            cache.v.view(torch.uint8)[some] = code.to(cache.v.dtype).view(torch.uint8)
            cache.v_scale[some], cache.k_scale[some] = unit.float(), 1.0
            x = code * unit[..., None]
        mean += torch.einsum("phkd,p->hd", x, used[some.cpu()].cuda())
    mean = (mean / length).repeat_interleave(H // heads, 0)
    offsets = torch.arange(0, n * copies + 1, n, dtype=torch.int32, device="cuda")          # (the sequences share their pages)
    lengths, pages = torch.full((copies,), length, dtype=torch.int32, device="cuda"), batch.pages.expand(copies, -1).contiguous()
    q = _normal(gen, n * copies, H, D, dtype=BF16)
    out = torch.zeros_like(q)
    serving.paged_attention(cache, q, out, offsets, lengths, pages, n * copies, copies, H, causal=False)
    # Half a step of the result (2^-8 where it is from 1 to 2), and on top of it: a value times its scale in fp16 (int8, the scale too: 2^-11 each, to nearest, 2^-17 on the average of these values); 2048 steps of
    # 2^-23 in an accumulator, 2^-12; sums and weights in fp32.  Values below 2.
    assert float((out.double() - mean).abs().max()) <= 2.0 ** -8 + 2.0 * (2.0 ** -12 + 2.0 ** -14)


# ---- waits that run out ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,fmt,seqs,H", [(BF16, "e4m3", [(1, 150000), (1, 60000), (1, 200)], 8), (F32, "plain", [(1, 90000), (1, 9000), (1, 200)], 8), (BF16, "plain", [(10, 80000), (8, 900)], 4),
                                              (F32, "int8", [(100, 20000), (60, 900)], 4), (F32, "plain", [(300, 5000), (200, 900)], 4)], ids=["tokens", "tokens32", "some", "many32", "cut"])
@pytest.mark.parametrize("code,block", [(1011, 0), (1011, 3), (1012, 1), (1012, 2)])
def test_an_expired_wait_of_few_rows_and_of_fp32(dtype, fmt, seqs, H, code, block):
    """Every row of the result is as ever, or nothing was stored there; the next call is as ever."""
    batch, heads, D = Batch(seqs, 64, seed=3), 2, 128
    cache, k, v = su.filled_cache(batch, heads, D, dtype, fmt)
    q = _normal(_gen(5), batch.T, H, D, dtype=dtype)
    out = torch.zeros_like(q)
    serving.paged_attention(cache, q, out, *batch.args, H)
    status = 0
    for _ in range(40):
        got = torch.full_like(out, -7.0)
        _capi.check(_capi.lib().hipgpt_debug_expire_wait(code, block))
        serving.paged_attention(cache, q, got, *batch.args, H)
        torch.cuda.synchronize()
        status = _status()
        same, left = (got == out).all(-1), (got == -7.0).all(-1)
        assert bool((same | left).all())
        if status:
            break
    assert status == code and _status() == 0
    assert bool(left.any()) and bool(same.any())
    serving.paged_attention(cache, q, got, *batch.args, H)
    assert torch.equal(got, out)


def test_the_status_is_of_launches_since_the_last_time():
    """Two kernels of attention gave up: the status says so once."""
    lib = _capi.lib()
    for dtype, code in ((BF16, 1003), (F32, 1011)):
        batch = Batch([(300, 3000)], 64, seed=3)
        cache, _, _ = su.filled_cache(batch, 2, 64, dtype, "plain")
        q = _normal(_gen(5), batch.T, 4, 64, dtype=dtype)
        _capi.check(lib.hipgpt_debug_expire_wait(code, 0))
        serving.paged_attention(cache, q, torch.empty_like(q), *batch.args, 4)
    assert _status() in (1003, 1011)
    assert _status() == 0


# ---- sizes ----------------------------------------------------------------------------------------------------------------

def test_as_many_tokens_as_an_int_holds():
    """The last block of tokens begins less than its own length before the largest int; the last tokens alone have a place."""
    torch.cuda.empty_cache()
    T, D = (1 << 31) - 5, 16
    if torch.cuda.mem_get_info()[0] < T * D * 2 + (8 << 30):
        pytest.skip("64 GB of rows do not fit beside what others hold")
    x = torch.empty(T, 1, D, device="cuda", dtype=BF16)
    x[-3:] = _normal(_gen(4), 3, 1, D, dtype=BF16)
    cache = serving.PagedCache(1, 16, 1, D, dtype=BF16, format="plain")
    offsets, lengths, pages = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, T], [3], [[0]]))
    serving.cache_write(cache, x, x, offsets, lengths, pages, T, 1)
    assert torch.equal(cache.k[0, 0, :3], x[-3:, 0]) and torch.equal(cache.v[0, 0, :3], x[-3:, 0])
    del x
    torch.cuda.empty_cache()


# ---- powers of two far from one another ----------------------------------------------------------------------------------

CODED = [(BF16, [(1, 900), (4, 500)], 4), (F32, [(1, 900), (4, 500)], 4), (BF16, [(20, 1700)], 4), (F32, [(20, 1700)], 4), (F32, [(70, 900)], 4), (BF16, [(300, 2000), (70, 80)], 4), (BF16, [(1000, 4000), (700, 800)], 8),
         (BF16, [(40, 20000)], 4)]
CODED_IDS = ["tokens", "tokens32", "some", "some32", "many32", "tcgen05", "widened", "parts"]


def _one(dtype, seqs, H, fmt, wild, spread=1.0, scale=None, turn=None):
    batch, heads, D = Batch(seqs, 64, seed=13), 2, 64
    cache, k, v = su.filled_cache(batch, heads, D, dtype, fmt, wild=wild)
    q = _normal(_gen(5), batch.T, H, D, dtype=dtype, scale=spread)
    if turn is not None:
        turn(q)
    out = torch.zeros_like(q)
    serving.paged_attention(cache, q, out, *batch.args, H, scale=scale)
    want, bound, _ = su.attention(batch, k, v, q, H, True, float(torch.tensor(D ** -0.5 if scale is None else scale)), dtype, fmt)
    within(out, want, bound)
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("powers", [(None, 60, None, -60), (60, None, None, 30), (None, 100, -100, 0), (-90, -20, 40, 110)])
@pytest.mark.parametrize("dtype,seqs,H", CODED, ids=CODED_IDS)
def test_values_of_powers_far_apart(dtype, seqs, H, fmt, powers):
    """Pages of zeros and of tiny and huge values beside each other: their keys keep their share of the probabilities, whatever their values count for."""
    def wild(name, x):
        if name == "v":
            for page in range(len(x)):
                p = powers[page % 4]
                x[page] *= 0.0 if p is None else 2.0 ** p
    _one(dtype, seqs, H, fmt, wild)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,seqs,H", CODED, ids=CODED_IDS)
def test_queries_and_keys_at_both_ends_of_the_range(dtype, seqs, H, fmt):
    def large(name, x):
        if name == "k":
            x *= 2.0 ** 115
    _one(dtype, seqs, H, fmt, large, spread=2.0 ** -115)

    def small(name, x):
        if name == "k":
            x *= 2.0 ** -100
    _one(dtype, seqs, H, fmt, small, spread=2.0 ** 100)

    def smaller(name, x):
        if name == "k":
            x *= 1e-28

    def largest(q):
        q[-2:, :, 3], q[-1:, :, 7] = 3.3e38, -3.2e38
    _one(dtype, seqs, H, fmt, smaller, scale=1e-10, turn=largest)
