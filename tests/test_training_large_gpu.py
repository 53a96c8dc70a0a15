"""The operators at the two ends of a training step where offsets pass 2^31 elements: what lies behind is compared at places."""
import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import training  # noqa: E402
from tests import training_util as tu  # noqa: E402

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _room():
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    yield
    torch.cuda.empty_cache()


def test_dropout_of_more_than_2_to_the_31_values():
    n, p, seed, offset = (1 << 31) + 4099, 0.3, 11, 5
    x = torch.empty(n, dtype=BF16, device="cuda")
    x.uniform_(0.5, 1.5)
    y = torch.full_like(x, float("nan"))
    training.dropout_counter(x, None, y, p, seed=seed, offset=offset)
    for begin in (0, (1 << 31) - 4096, n - 4099 // 8 * 8 - 3):
        begin = begin // 8 * 8
        count = min(4096, n - begin)
        keep, inv = tu.kept(count, p, seed, offset + begin // 8)
        want = torch.where(keep.cuda(), x[begin:begin + count].double() * inv, torch.zeros((), dtype=torch.float64, device="cuda"))
        tu.within(y[begin:begin + count], want, (tu.HALF[BF16] + 2.0 ** -22) * want.abs())
    assert not bool(torch.isnan(y[-1000:]).any())


def test_embedding_of_a_table_of_more_than_2_to_the_31_values():
    V, E, B, S = 35000, 65536, 2, 9
    tok = torch.empty(V, E, dtype=BF16, device="cuda")
    tok.uniform_(-1, 1)
    ids = torch.tensor([0, V - 1, 33000, 12, V - 2, V, -1, 40, V - 1] * B, dtype=torch.int32, device="cuda")
    out = torch.full((B * S, E), float("nan"), dtype=BF16, device="cuda")
    training.embedding_scaled(ids, tok, None, out, B, S, V, E, scale=2.0)
    ok = (ids >= 0) & (ids < V)
    assert torch.equal(out[ok], tok[ids[ok].long()] * 2) and bool((out[~ok] == 0).all())     # (twice a value is exact)
    grad = torch.full((V, E), float("nan"), dtype=BF16, device="cuda")
    g = torch.randn(B * S, E, device="cuda").to(BF16)
    training.embedding_backward(g, ids, grad, None, B, S, V, E)
    rows = torch.tensor([0, 12, 40, 33000, V - 2, V - 1, 34000, 1], device="cuda")
    for v in rows.tolist():
        picked = g[ids == v].double()
        want = picked.sum(0) if len(picked) else torch.zeros(E, dtype=torch.float64, device="cuda")
        tu.within(grad[v], want, (tu.HALF[BF16] + 4 * tu.HALF[torch.float32]) * picked.abs().sum(0) if len(picked) else torch.zeros_like(want))
    assert not bool(torch.isnan(grad[::997]).any())


@pytest.mark.parametrize("by_token", [True, False])
def test_loss_with_weights_of_more_than_2_to_the_31_values(by_token):
    N, E, V = 70, 4160, 520000
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = torch.empty(V, E, dtype=BF16, device="cuda").normal_(0, E ** -0.5, generator=gen)
    x = torch.randn(N, E, generator=gen, device="cuda").to(BF16)
    targets = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
    targets[0], targets[1], targets[2] = V - 1, 0, -1
    z = torch.empty(N, V, dtype=torch.float64, device="cuda")
    for a in range(0, V, 20000):
        z[:, a:a + 20000] = x.double() @ w[a:a + 20000].double().t()
    ok = targets >= 0
    lse64 = torch.logsumexp(z, 1) * ok
    loss64 = (lse64 - z.gather(1, targets.clamp(min=0).long()[:, None])[:, 0]) * ok
    wl = w if by_token else w.t().contiguous()
    loss, lse, g = torch.full((N,), float("nan"), device="cuda"), torch.full((N,), float("nan"), device="cuda"), torch.rand(N, generator=gen, device="cuda")
    training.linear_cross_entropy(x, wl, targets, loss, lse, N, E, V, by_token=by_token)
    # 260 instructions of 16 products, each cut off by a step of the running sum at most (which is about 1); sums of exponentials to 1e-5
    assert float((lse.double() - lse64).abs().max()) <= 260 * 2.0 ** -23 * 8 + 2e-5 and float((loss.double() - loss64).abs().max()) <= 260 * 2.0 ** -23 * 16 + 2e-5
    gx, gw = torch.full_like(x, float("nan")), torch.full_like(wl, float("nan"))
    training.linear_cross_entropy_backward(x, wl, targets, lse, g, gx, gw, N, E, V, by_token=by_token)
    dz = torch.exp(z.sub_(lse.double()[:, None])) * ok[:, None]
    dz[torch.arange(N, device="cuda"), targets.clamp(min=0).long()] -= ok.double()
    dz *= g.double()[:, None]
    dx = torch.zeros(N, E, dtype=torch.float64, device="cuda")
    for a in range(0, V, 20000):
        dx += dz[:, a:a + 20000] @ w[a:a + 20000].double()
    assert float((gx.double() - dx).norm() / dx.norm()) <= 2 * tu.HALF[BF16]
    for v in [0, V - 1, V // 2 + 1, 516300] + targets[3:6].tolist():
        want = dz[:, v] @ x.double()
        got = (gw[v] if by_token else gw[:, v]).double()
        assert float((got - want).norm() / want.norm()) <= 2 * tu.HALF[BF16], v
    assert not bool(torch.isnan(gw.view(-1)[::10007]).any())
