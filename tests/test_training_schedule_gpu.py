"""The loss gradient's work as large calls divide it (tiles dealt out whole, shares of the rest, several pieces of the vocabulary), its waits made to run out, and
the forms of dropout and of the embedding's gradient that only large sizes take."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import _capi, training  # noqa: E402
from tests import training_util as tu  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _case(N, E, V, dtype, seed, outside):
    gen = _gen(seed)
    w = torch.randn(V, E, generator=gen, device="cuda") * (1.5 / E ** 0.5)
    targets = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
    x = torch.randn(N, E, generator=gen, device="cuda") + 1.5 * w[targets.long()]
    targets[torch.rand(N, generator=gen, device="cuda") < outside] = -1
    return x.to(dtype), w.to(dtype), targets, torch.rand(N, generator=gen, device="cuda") - 0.3


def _status():
    st = C.c_int(-1)
    _capi.check(_capi.lib().hipgpt_kernel_status(C.byref(st)))
    return st.value


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by_token", [True, False])
@pytest.mark.parametrize("N,E,V,outside", [(700, 776, 8001, 0.0), (700, 776, 8001, 0.3),       # 3 x 4 + 4 x 32 tiles, the last of each row narrow: a round of 74 dealt out whole, the rest shared
                                           (2050, 520, 6000, 0.0),                             # 9 x 3 + 3 x 24
                                           (5200, 520, 19000, 0.1)])                           # two pieces of the vocabulary, 21 x 3 + 3 x 38 tiles and more
def test_gradient_with_tiles_dealt_out_whole(dtype, by_token, N, E, V, outside):
    x, w, targets, g = _case(N, E, V, dtype, N + V, outside)
    ref = tu.Loss(x, w, targets, g, dtype)
    wl = w if by_token else w.t().contiguous()
    lse = ref.lse.float()
    (dx, dw), (ex, ew) = ref.gradients(lse)
    del ref
    runs = []
    for with_x, with_w in ((True, True), (True, True), (True, False), (False, True)):
        gx, gw = torch.full_like(x, NAN) if with_x else None, torch.full_like(wl, NAN) if with_w else None
        training.linear_cross_entropy_backward(x, wl, targets, lse, g, gx, gw, N, E, V, by_token=by_token)
        if with_x:
            tu.within(gx, dx, ex, "grad_x")
        if with_w:
            tu.within(gw if by_token else gw.t(), dw, ew, "grad_w")
        runs.append((gx, gw))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    del runs
    old = torch.randn(V, E, generator=_gen(3), device="cuda").to(dtype)
    gw = old.clone() if by_token else old.t().contiguous()
    training.linear_cross_entropy_backward(x, wl, targets, lse, g, None, gw, N, E, V, by_token=by_token, accumulate=True)
    full = old.double() + dw
    tu.within(gw if by_token else gw.t(), full, ew + (tu.HALF[dtype] + 2 * tu.HALF[F32]) * (full.abs() + ew), "accumulated grad_w")
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("code,block", [(701, 0), (702, 1), (703, 2), (703, 3), (704, 0)])
def test_an_expired_wait_of_the_gradient_stores_no_part_of_a_value(dtype, code, block):
    """The status names the wait; every value of the gradients is the old one or what it would be; the next call is as ever, whatever its predecessor left of the counters of shared
    tiles.  Where what is waited for had come before, nothing ran out: then once more."""
    N, E, V = (5200, 520, 19000) if dtype == BF16 else (3000, 264, 19000)          # two pieces of the vocabulary, tiles that several pairs share
    x, w, targets, g = _case(N, E, V, dtype, 5, 0.0)
    lse = torch.logsumexp(x.float() @ w.float().t(), 1)

    def run(gx, gw):
        training.linear_cross_entropy_backward(x, w, targets, lse, g, gx, gw, N, E, V)
        torch.cuda.synchronize()

    want = torch.full_like(x, -7.0), torch.full_like(w, -7.0)
    run(*want)
    for _ in range(20):
        got = torch.full_like(x, -7.0), torch.full_like(w, -7.0)
        _capi.check(_capi.lib().hipgpt_debug_expire_wait(code, block))
        run(*got)
        status = _status()
        if status:
            break
    assert status == code
    for a, b in zip(got, want):
        assert bool(((a == b) | (a == -7.0)).all())
    assert bool((got[1] == -7.0).any())
    again = torch.full_like(x, -7.0), torch.full_like(w, -7.0)
    run(*again)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1]) and _status() == 0


@pytest.mark.parametrize("residual", [False, True])
def test_dropout_of_many_16_bit_values(residual):
    n, p, seed, offset = (1 << 23) + 2048 * 3 + 5, 0.2, 77, 9
    gen = _gen(1)
    x = torch.randn(n, generator=gen, device="cuda").to(BF16)
    r = torch.randn(n, generator=gen, device="cuda").to(BF16) if residual else None
    out = torch.full_like(x, NAN)
    training.dropout_counter(x, r, out, p, seed=seed, offset=offset)
    for begin, count in ((0, 4096), (2048 * 4 - 512, 1024), (2048 * 4 * 100 + 2040, 4096), (n - 8 * 512 - n % 8, 8 * 512 + n % 8)):
        assert begin % 8 == 0
        keep, inv = tu.kept(count, p, seed, offset + begin // 8)
        y = torch.where(keep.cuda(), x[begin:begin + count].double() * inv, torch.zeros((), dtype=torch.float64, device="cuda"))
        z = r[begin:begin + count].double() if residual else torch.zeros_like(y)
        tu.within(out[begin:begin + count], y + z, 3 * tu.HALF[F32] * (y.abs() + z.abs()) + tu.HALF[BF16] * ((y + z).abs() + 2.0 ** -22 * (y.abs() + z.abs())), "values")
    assert not bool(torch.isnan(out).any())
    into = r.clone() if residual else x.clone()
    training.dropout_counter(x if residual else into, into if residual else None, into, p, seed=seed, offset=offset)
    assert torch.equal(into, out)


@pytest.mark.parametrize("V", [(1 << 20) - 1, 1 << 20, 3000017])
def test_embedding_gradient_of_large_vocabularies(V):
    """Keys of 20 bits in two passes of the sort, of more in three."""
    for n, E in ((700, 8), (9000, 8), (140000, 4)):
        gen = _gen(V % 1000 + n)
        ids = torch.randint(-1, V + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
        ids[::7], ids[3::11], ids[5::13] = V - 1, 0, V // 2
        ids[1], ids[2] = 1, V - 2
        g = torch.randn(n, E, generator=gen, device="cuda")
        table = torch.full((V, E), NAN, device="cuda")
        training.embedding_backward(g, ids, table, None, 1, n, V, E)
        want, bound = tu.embedding_backward(g, ids, V, n, 1.0)
        tu.within(table, want[0], bound[0] + 1e-30, "grad_tok")
        old = torch.ones_like(table)
        training.embedding_backward(g, ids, old, None, 1, n, V, E, accumulate=True)
        tu.within(old, want[0] + 1.0, bound[0] + 2 * tu.HALF[F32] * (1.0 + want[0].abs()), "accumulated")
    assert _status() == 0
