"""The loss and its gradient over the whole range of values: rows that weigh or measure very differently, values next to the type's largest, infinities and NaN
in rows that take part, sums of many terms of one sign."""
import math

import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import training  # noqa: E402
from tests import training_util as tu  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _case(N, E, V, dtype, seed):
    gen = _gen(seed)
    w = torch.randn(V, E, generator=gen, device="cuda") * (1.5 / E ** 0.5)
    targets = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
    x = torch.randn(N, E, generator=gen, device="cuda") + 1.5 * w[targets.long()]
    return x.to(dtype), w.to(dtype), targets


def _nan_like(t):
    return torch.full_like(t, NAN)


def _forward(x, w, targets, by_token):
    N, (V, E) = x.shape[0], w.shape
    wl = w if by_token else w.t().contiguous()
    loss, lse = torch.full((N,), NAN, device="cuda"), torch.full((N,), NAN, device="cuda")
    training.linear_cross_entropy(x, wl, targets, loss, lse, N, E, V, by_token=by_token)
    return loss, lse


def _backward(x, w, targets, lse, g, by_token):
    N, (V, E) = x.shape[0], w.shape
    wl = w if by_token else w.t().contiguous()
    gx, gw = _nan_like(x), _nan_like(wl)
    training.linear_cross_entropy_backward(x, wl, targets, lse, g, gx, gw, N, E, V, by_token=by_token)
    return gx, gw if by_token else gw.t()


class _Fp32:
    """float64 results for fp32 calls and bounds that go row by row.

    An operand is two fp16 numbers, 2^-22 of the value, and the product of the two low ones is left out (2^-22); below 2^-39 of the largest value of
    its row (x) or of the matrix (W) nothing is kept.  TMEM adds up 24 instructions that may each cut off a step (2^-23), then fp32 additions follow, one for
    128 inner indices and one for each of at most 74 pairs that share a tile.  A row's gradient of the logits keeps 2^-29 of its weight at least; a row of x in the
    weights' gradient 2^-38 of the largest |g| max|x| of all rows, made 2^a finer for a row that is a (at most 8) binades and some more below that."""

    def __init__(self, x, w, targets, g, lse):
        x, w, g, lse = x.double(), w.double(), g.double(), lse.double()
        (N, E), V = x.shape, w.shape[0]
        step, half = 2.0 ** -23, 2.0 ** -24
        run = lambda k: 24 * step + (-(-k // 128) + 76) * half  # noqa: E731
        xa, wa, xmax, wmax = x.abs(), w.abs(), x.abs().max(1, keepdim=True).values, w.abs().max()
        z, at = x @ w.t(), targets.long()
        ez = xa @ wa.t() * (3 * 2.0 ** -22 + run(E)) + 2.0 ** -38 * E * xmax * wmax
        rows = torch.arange(N, device=x.device)
        self.lse, self.e_lse = torch.logsumexp(z, 1), ez.max(1).values + (64 + V / 1024 + 40) * half + 2.0 ** -21 + 2.0 ** -22 * torch.logsumexp(z, 1).abs()
        self.loss, self.e_loss = self.lse - z[rows, at], 2 * self.e_lse + half * z[rows, at].abs()
        p = torch.exp(z - lse[:, None])
        dz, ga = p.clone(), g.abs()[:, None]
        dz[rows, at] -= 1
        edz = p * (2 * ez + (z - lse[:, None]).abs() * 2.0 ** -22 + 2.0 ** -21)
        edz[rows, at] += 2.0 ** -23
        edz = (edz + (2.0 ** -22 + 2.0 ** -22) * dz.abs() + 2.0 ** -29) * ga
        dz = dz * g[:, None]
        self.dx, self.dw = dz @ w, dz.t() @ x
        da = dz.abs() + edz
        self.e_dx = edz @ wa + da @ wa * (3 * 2.0 ** -22 + run(V)) + 2.0 ** -39 * wmax * da.sum(1, keepdim=True) + 2 * half * self.dx.abs() + 1e-38
        most = (ga * xmax).max()
        a = torch.log2(most / (ga * xmax).clamp(min=1e-300)).sub(6).floor().clamp(0, 8)
        floor = 2.0 ** -38 * most * 2.0 ** -a / ga.clamp(min=1e-200) * (ga > 0)
        self.e_dw = edz.t() @ xa + da.t() @ xa * (3 * 2.0 ** -22 + run(N)) + da.t() @ floor.expand(N, E) + 2 * half * self.dw.abs() + 1e-38


@pytest.mark.parametrize("by_token", [True, False])
@pytest.mark.parametrize("light", [1.0, 1e-4, 1e-6, 1e-8, 1e-12, 1e-20])
def test_fp32_gradient_of_rows_that_weigh_little(by_token, light):
    """One row of weight 1, the others of `light`: the gradient of every row is as good as if it were alone."""
    N, E, V = 300, 256, 5000
    x, w, targets = _case(N, E, V, F32, 5)
    g = torch.full((N,), light, device="cuda")
    g[17], g[200] = 1.0, -light / 3
    _, lse = _forward(x, w, targets, by_token)
    gx, gw = _backward(x, w, targets, lse, g, by_token)
    ref = _Fp32(x, w, targets, g, lse)
    tu.within(gx, ref.dx, ref.e_dx, "grad_x")
    tu.within(gw, ref.dw, ref.e_dw, "grad_w")


@pytest.mark.parametrize("by_token", [True, False])
@pytest.mark.parametrize("large,small", [(1e8, 1.0), (1.0, 1e-10), (1e30, 1e-30)])
def test_fp32_rows_of_unequal_magnitude(by_token, large, small):
    N, E, V = 200, 128, 1500
    x, w, targets = _case(N, E, V, F32, 6)
    x[::3] *= small
    x[7] *= large
    g = torch.ones(N, device="cuda")
    loss, lse = _forward(x, w, targets, by_token)
    gx, gw = _backward(x, w, targets, lse, g, by_token)
    ref = _Fp32(x, w, targets, g, lse)
    others = torch.arange(N, device="cuda") != 7           # (row 7's own logits are so large that its p is 0 or 1; an lse of 1e30 has no digits for it)
    tu.within(loss[others], ref.loss[others], ref.e_loss[others], "loss")
    tu.within(lse, ref.lse, ref.e_lse, "lse")
    tu.within(gx[others], ref.dx[others], ref.e_dx[others], "grad_x")
    g[7] = 0.0                                             # its gradients left out, the others' show in the weights' too
    gx, gw = _backward(x, w, targets, lse, g, by_token)
    ref = _Fp32(torch.where(others[:, None], x, torch.zeros_like(x)), w, targets, g, torch.where(others, lse, torch.full_like(lse, math.log(V))))
    tu.within(gw, ref.dw, ref.e_dw, "grad_w")
    assert bool((gx[7] == 0).all())


@pytest.mark.parametrize("by_token", [True, False])
def test_fp32_values_next_to_the_largest(by_token):
    """3.3e38 in x or in W: finite values, so finite logits where the other factor is small."""
    N, E, V = 40, 64, 300
    x, w, targets = _case(N, E, V, F32, 7)
    g = torch.ones(N, device="cuda")
    for which in (0, 1):
        xs, ws = (x * 1e33, w * 1e-32) if which == 0 else (x * 1e-32, w * 1e33)
        big = xs if which == 0 else ws
        big[3, 5] = 3.3e38
        loss, lse = _forward(xs, ws, targets, by_token)
        ref = _Fp32(xs, ws, targets, g, lse)
        tu.within(lse, ref.lse, ref.e_lse, "lse")
        tu.within(loss, ref.loss, ref.e_loss, "loss")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by_token", [True, False])
def test_logits_that_are_infinite(dtype, by_token):
    """A logit that overflows to +infinity: log-sum-exp and loss are infinite (a target of +infinity itself: inf - inf).  To -infinity: it counts for nothing.  The other rows are as ever."""
    N, E, V = 70, 64, 700
    x, w, targets = _case(N, E, V, dtype, 8)
    targets[:] = 1
    w[650], w[651] = 0, 0
    x[:, 0], w[:, 0] = 0, 0                                # column 0 meets only these
    want = _forward(x, w, targets, by_token)
    w[650, 0], w[651, 0] = 2.0, -2.0
    x[3, 0], x[68, 0] = 2e38, -2e38                        # one logit of such a row is +infinity, one -infinity
    loss, lse = _forward(x, w, targets, by_token)
    hit = torch.zeros(N, dtype=torch.bool, device="cuda")
    hit[[3, 68]] = True
    assert bool((lse[hit] == INF).all()) and bool((loss[hit] == INF).all()), (lse[hit], loss[hit])
    assert torch.equal(loss[~hit], want[0][~hit]) and torch.equal(lse[~hit], want[1][~hit]) if dtype == BF16 else float((loss[~hit] - want[0][~hit]).abs().max()) < 1e-5
    targets[3] = 650
    loss, lse = _forward(x, w, targets, by_token)
    assert float(lse[3]) == INF and math.isnan(float(loss[3])) and float(loss[68]) == INF
    targets[3], x[68, 0] = 651, 0                          # the target's logit is -infinity
    loss, lse = _forward(x, w, targets, by_token)
    assert float(lse[3]) == INF and float(loss[3]) == INF and math.isfinite(float(loss[68]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by_token", [True, False])
def test_nan_in_a_row_that_takes_part_stays_in_it(dtype, by_token):
    N, E, V = 300, 72, 900
    x, w, targets = _case(N, E, V, dtype, 9)
    g = torch.rand(N, generator=_gen(1), device="cuda") + 0.5
    loss0, lse0 = _forward(x, w, targets, by_token)
    gx0, _ = _backward(x, w, targets, lse0, g, by_token)
    x[5, 3], x[290] = NAN, NAN
    loss, lse = _forward(x, w, targets, by_token)
    bad = torch.zeros(N, dtype=torch.bool, device="cuda")
    bad[[5, 290]] = True
    assert bool(torch.isnan(loss[bad]).all() and torch.isnan(lse[bad]).all())
    assert torch.equal(loss[~bad], loss0[~bad]) and torch.equal(lse[~bad], lse0[~bad])
    gx, gw = _backward(x, w, targets, lse, g, by_token)
    assert torch.equal(gx[~bad], gx0[~bad]) and bool(torch.isnan(gx[bad]).all()) and bool(torch.isnan(gw).all())


def test_bf16_weight_gradient_over_many_rows_of_one_sign():
    """262144 terms of one sign.  The tensor core's sums are cut off, up to 2^-23 of what they come to for each 16 terms and always downwards; a sum of at most 128 stages (512 instructions) stays within
    2^-14 of itself, however many rows there are, and what follows is rounded either way, as are p and the results.  A result is off by up to 2^-8 of itself (evenly spread: 2^-8 / sqrt(3) at one sigma),
    alike in the columns of a row, whose sums are nearly the same; over 1023 rows that leaves 2^-8 / sqrt(3 * 1023) < 2^-13.7 at one sigma.  Four of them, and 2^-14."""
    N, E, V = 262144, 4864, 1024
    gen = _gen(2)
    x = torch.rand(N, E, generator=gen, device="cuda", dtype=BF16).add_(1.0)
    w, targets, g = torch.zeros(V, E, dtype=BF16, device="cuda"), torch.zeros(N, dtype=torch.int32, device="cuda"), torch.ones(N, device="cuda")
    w[:, 0] = (torch.randn(V, generator=gen, device="cuda") * 0.5).to(BF16)
    p = torch.softmax(x[:, :1].double() * w[:, 0].double(), 1)
    lse = -torch.log(p[:, 0] / torch.exp(x[:, 0].double() * w[0, 0].double())).float()
    gw = _nan_like(w)
    training.linear_cross_entropy_backward(x, w, targets, lse, g, None, gw, N, E, V)
    want = torch.zeros(V, E, dtype=torch.float64, device="cuda")
    for a in range(0, N, 16384):
        want += p[a:a + 16384].t() @ x[a:a + 16384].double()
    short = 1.0 - gw[1:].double() / want[1:]               # (row 0 is every row's target)
    assert abs(float(short.mean())) < 2.0 ** -14 + 4 * 2.0 ** -13.7, float(short.mean())


@pytest.mark.parametrize("by_token", [True, False])
def test_bf16_loss_of_wide_rows_of_one_sign(by_token):
    """Logits of 65536 terms of one sign: cut off at most 64 times (16 stages) before they leave the tensor core's sums."""
    N, E, V = 70, 65536, 300
    gen = _gen(4)
    x = (torch.rand(N, E, generator=gen, device="cuda") + 0.5).to(BF16)
    w = ((torch.rand(V, E, generator=gen, device="cuda") + 0.5) * torch.linspace(0, 8, V, device="cuda")[:, None] / E).to(BF16)
    targets = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
    loss, lse = _forward(x, w, targets, by_token)
    z = x.double() @ w.double().t()
    cut = float(z.max()) * (64 * 2.0 ** -23 + (E // 1024 + 2) * 2.0 ** -24)
    want = torch.logsumexp(z, 1)
    assert float((lse.double() - want).abs().max()) < cut + 2.0 ** -20
    assert float((loss.double() - (want - z.gather(1, targets.long()[:, None])[:, 0])).abs().max()) < 2 * cut + 2.0 ** -20


@pytest.mark.parametrize("by_token", [True, False])
def test_bf16_gradient_of_wide_rows(by_token):
    """Logits over 257 stages: their sums are put by on the way, in the backward too."""
    N, E, V = 70, 16400, 300
    x, w, targets = _case(N, E, V, BF16, 11)
    g = torch.rand(N, generator=_gen(12), device="cuda") - 0.3
    ref = tu.Loss(x, w, targets, g, BF16)
    loss, lse = _forward(x, w, targets, by_token)
    tu.within(lse, ref.lse, ref.e_lse, "lse")
    tu.within(loss, ref.loss, ref.e_loss, "loss")
    gx, gw = _backward(x, w, targets, lse, g, by_token)
    (dx, dw), (ex, ew) = ref.gradients(lse)
    tu.within(gx, dx, ex, "grad_x")
    tu.within(gw, dw, ew, "grad_w")


@pytest.mark.parametrize("by_token", [True, False])
@pytest.mark.parametrize("sw,sg", [(1e37, 1e-36), (1e-36, 1e37)])
def test_fp32_scales_that_undo_one_another(by_token, sw, sg):
    """Weights of 1e37 and gradients of 1e-36, or the other way round: grad_x is of ordinary size."""
    N, E, V = 60, 64, 500
    x, w, targets = _case(N, E, V, F32, 13)
    x, w, g = x / sw, w * sw, torch.full((N,), sg, device="cuda")
    _, lse = _forward(x, w, targets, by_token)
    gx, _ = _backward(x, w, targets, lse, g, by_token)     # (grad_w passes the range of fp32 in one of them)
    ref = _Fp32(x, w, targets, g, lse)
    tu.within(gx, ref.dx, ref.e_dx + 2.0 ** -20 * ref.dx.abs().max(), "grad_x")           # (values of 1e-37 are scaled by 2^126 at most)


def test_gradients_of_another_shape_are_refused():
    x, w, t = torch.zeros(4, 8, device="cuda"), torch.zeros(16, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    f = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="grad_w has rows"):
        training.linear_cross_entropy_backward(x, w, t, f, f.clone(), None, torch.zeros(8, 16, device="cuda"), 4, 8, 16)
    with pytest.raises(ValueError, match="grad_pos has rows"):
        training.embedding_backward(x, t, None, torch.zeros(8, 2, device="cuda"), 2, 2, 16, 8)
