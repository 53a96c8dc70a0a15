"""Embedding and its gradient, dropout from a counter, the loss and its gradient against plain float64 forms (tests/training_util.py)."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import _capi, training  # noqa: E402
from tests import training_util as tu  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _ids(gen, n, V, lo=0, hi=None):
    return torch.randint(lo, V if hi is None else hi, (n,), generator=gen, device="cuda", dtype=torch.int32)


def _nan(*shape, dtype=F32):
    return torch.full(shape, float("nan"), device="cuda", dtype=dtype)


def _status():
    st = C.c_int(-1)
    _capi.check(_capi.lib().hipgpt_kernel_status(C.byref(st)))
    return st.value


# ---- embedding --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,S,V,E,pos", [(1, 1, 1, 1, True), (2, 3, 7, 5, True), (3, 5, 50, 64, False), (4, 33, 1000, 256, True), (2, 17, 300, 1000, False), (1, 9, 11, 2050, True)])
def test_embedding(dtype, B, S, V, E, pos):
    gen = _gen(B * 1000 + E)
    tok, table = _normal(gen, V, E, dtype=dtype), _normal(gen, S, E, dtype=dtype) if pos else None
    ids = _ids(gen, B * S, V, -2, V + 2)
    out = _nan(B * S, E, dtype=dtype)
    training.embedding_scaled(ids, tok, table, out, B, S, V, E, scale=3.7)
    scale = float(np.float32(3.7))
    want, mag = tu.embedding(ids, tok, table, S, scale)
    tu.within(out, want, 2 * tu.HALF[F32] * mag + tu.HALF[dtype] * (want.abs() * (1 + 2 ** -20) + 2 ** -22 * mag), "rows")
    assert bool((out[(ids < 0) | (ids >= V)] == 0).all())


BACKWARD_SIZES = [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 5), (5, 13, 40, 64), (4, 256, 5000, 256), (3, 700, 90, 200), (300, 7, 1500, 48), (1, 4500, 3, 33), (9, 2000, 70000, 16), (200, 1, 17, 520),
                  (20, 2000, 300, 1024), (70, 2000, 50000, 8)]         # several rounds of copies a piece; several tiles a block of the sort


@pytest.mark.parametrize("dtype,gt", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("B,S,V,E", BACKWARD_SIZES)
def test_embedding_gradient(dtype, gt, B, S, V, E):
    gen = _gen(B * 77 + V)
    n = B * S
    g = _normal(gen, n, E, dtype=dtype)
    # half of the tokens spread over the vocabulary, some outside it, the others one id
    ids = _ids(gen, n, V, -1, V + 1)
    ids[torch.rand(n, generator=gen, device="cuda") < 0.5] = V // 2
    g[ids < 0] = float("nan")                    # what lies under an id outside is not looked at
    want, bound = tu.embedding_backward(g, ids, V, S, float(np.float32(1.3)))
    h = tu.HALF[gt] if gt == BF16 else 0.0
    for with_tok, with_pos in ((True, True), (True, False), (False, True)):
        tok, pos = _nan(V, E, dtype=gt) if with_tok else None, _nan(S, E, dtype=gt) if with_pos else None
        training.embedding_backward(g, ids, tok, pos, B, S, V, E, scale=1.3)
        if with_tok:
            tu.within(tok, want[0], bound[0] + h * (want[0].abs() + bound[0]) + 1e-30, "grad_tok")
        if with_pos:
            tu.within(pos, want[1], bound[1] + h * (want[1].abs() + bound[1]) + 1e-30, "grad_pos")
    # added to what is there; rows without tokens stay as they are, and twice the same call gives the same bits
    old_t, old_p = _normal(gen, V, E, dtype=gt), _normal(gen, S, E, dtype=gt)
    runs = []
    for _ in range(2):
        tok, pos = old_t.clone(), old_p.clone()
        training.embedding_backward(g, ids, tok, pos, B, S, V, E, scale=1.3, accumulate=True)
        runs.append((tok, pos))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    tok, pos = runs[0]
    for got, old, w, b in ((tok, old_t, want[0], bound[0]), (pos, old_p, want[1], bound[1])):
        full = old.double() + w
        tu.within(got, full, b + (tu.HALF[gt] + 2 * tu.HALF[F32]) * (full.abs() + b) + 1e-30, "accumulated")
    absent = torch.ones(V, dtype=torch.bool, device="cuda")
    absent[ids[(ids >= 0) & (ids < V)].long()] = False
    assert torch.equal(tok[absent], old_t[absent])


def test_embedding_gradient_of_unaligned_tensors_and_of_no_tokens():
    gen = _gen(5)
    B, S, V, E = 3, 20, 31, 64
    buf = _normal(gen, B * S * E + 1)
    g = buf[1:].view(B * S, E)                   # four bytes off a 16-byte boundary
    ids = _ids(gen, B * S, V)
    tok = torch.full((V * E + 3,), 7.0, device="cuda")
    training.embedding_backward(g, ids, tok[1:1 + V * E].view(V, E), None, B, S, V, E)
    want, bound = tu.embedding_backward(g, ids, V, S, 1.0)
    tu.within(tok[1:1 + V * E].view(V, E), want[0], bound[0] + 1e-30)
    assert float(tok[0]) == 7.0 and bool((tok[1 + V * E:] == 7.0).all())
    table = _nan(V, E)
    training.embedding_backward(g[:0], ids[:0], table, None, 0, S, V, E)
    assert bool((table == 0).all())
    table.fill_(2.0)
    training.embedding_backward(g[:0], ids[:0], table, None, 0, S, V, E, accumulate=True)
    assert bool((table == 2.0).all())
    all_outside = torch.full_like(ids, V)
    training.embedding_backward(g, all_outside, table, None, B, S, V, E)
    assert bool((table == 0).all())


# ---- dropout ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2048, 5003])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.99999])
def test_dropout(dtype, n, p):
    gen = _gen(n)
    x, r = _normal(gen, n, dtype=dtype), _normal(gen, n, dtype=dtype)
    seed, offset = 0xF123456789ABCDEF, (1 << 40) + 17
    keep, inv = tu.kept(n, p, seed, offset)
    keep = keep.cuda()
    bad = ~keep
    x[bad] = float("nan")                        # a dropped value is zero whatever it was
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    y = torch.where(keep, x.double() * inv, zero)
    for res in (None, r):
        out = _nan(n, dtype=dtype)
        training.dropout_counter(x, res, out, p, seed=seed, offset=offset)
        want = y if res is None else y + res.double()
        mag = y.abs() + (0 if res is None else res.double().abs())
        tu.within(out, want, (3 * tu.HALF[F32]) * mag + tu.HALF[dtype] * (want.abs() + 2 ** -22 * mag), "values")
    # in place, over the input and over the residual
    a = x.clone()
    training.dropout_counter(a, None, a, p, seed=seed, offset=offset)
    b = r.clone()
    training.dropout_counter(x, b, b, p, seed=seed, offset=offset)
    assert torch.equal(b, out)
    # and from an address that is no multiple of 16 bytes
    big = torch.zeros(n + 1, dtype=dtype, device="cuda")
    big[1:] = x
    c = torch.zeros(n + 1, dtype=dtype, device="cuda")
    training.dropout_counter(big[1:], None, c[1:], p, seed=seed, offset=offset)
    assert torch.equal(c[1:], a) and float(c[0]) == 0.0


def test_dropout_counter_word_moves_the_mask_of_a_captured_call():
    n, p = 4096, 0.3
    x, out = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    word = torch.zeros(1, dtype=torch.int64, device="cuda")
    training.dropout_counter(x, None, out, p, seed=5, counter=word)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        training.dropout_counter(x, None, out, p, seed=5, counter=word)
        word += n // 8
    word.zero_()
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        keep, _ = tu.kept(n, p, 5, step * (n // 8))
        assert torch.equal(out.cpu() != 0, keep)


# ---- the loss ---------------------------------------------------------------------------------------------------------

def _loss_case(N, E, V, dtype, seed, outside=0.0, spread=1.5):
    gen = _gen(seed)
    w = _normal(gen, V, E, scale=spread / E ** 0.5)
    targets = _ids(gen, N, V)
    x = _normal(gen, N, E) + 1.5 * w[targets.long()]
    targets[torch.rand(N, generator=gen, device="cuda") < outside] = -100
    if outside and N > 2:
        targets[1] = V
    g = torch.rand(N, generator=gen, device="cuda") - 0.3
    return x.to(dtype), w.to(dtype), targets, g


def _lay(w, by_token):
    return w if by_token else w.t().contiguous()


LOSS_SIZES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (64, 64, 256), (65, 72, 257), (257, 40, 100), (300, 256, 1000), (130, 200, 5000), (700, 130, 1500), (33, 1000, 129), (600, 512, 777)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by_token", [True, False])
@pytest.mark.parametrize("N,E,V", LOSS_SIZES)
def test_loss_and_gradient(dtype, by_token, N, E, V):
    for outside in (0.0, 0.4):
        x, w, targets, g = _loss_case(N, E, V, dtype, N + E + V, outside)
        ref = tu.Loss(x, w, targets, g, dtype)
        x[~ref.valid] = float("nan")             # rows that take no part: nothing of them is looked at
        g[~ref.valid] = float("inf")
        wl = _lay(w, by_token)
        loss, lse = _nan(N), _nan(N)
        training.linear_cross_entropy(x, wl, targets, loss, lse, N, E, V, by_token=by_token)
        tu.within(lse, ref.lse, ref.e_lse, "lse")
        tu.within(loss, ref.loss, ref.e_loss, "loss")
        assert bool((loss[~ref.valid] == 0).all() and (lse[~ref.valid] == 0).all())
        (dx, dw), (ex, ew) = ref.gradients(lse)
        for with_x, with_w in ((True, True), (True, False), (False, True)):
            gx, gw = _nan(N, E, dtype=dtype) if with_x else None, _nan(*wl.shape, dtype=dtype) if with_w else None
            training.linear_cross_entropy_backward(x, wl, targets, lse, g, gx, gw, N, E, V, by_token=by_token)
            if with_x:
                tu.within(gx, dx, ex, "grad_x")
                assert bool((gx[~ref.valid] == 0).all())
            if with_w:
                tu.within(gw if by_token else gw.t(), dw, ew, "grad_w")
        old = _normal(_gen(3), V, E, dtype=dtype)
        gw = _lay(old, by_token).clone()
        training.linear_cross_entropy_backward(x, wl, targets, lse, g, None, gw, N, E, V, by_token=by_token, accumulate=True)
        full = old.double() + dw
        tu.within(gw if by_token else gw.t(), full, ew + (tu.HALF[dtype] + 2 * tu.HALF[F32]) * (full.abs() + ew), "accumulated grad_w")
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by_token", [True, False])
def test_loss_gradient_over_several_pieces_of_the_vocabulary(dtype, by_token):
    N, E, V = 4500, 72, 26000                    # the logits' gradient would be 240 (bf16) or 480 MB in one piece
    x, w, targets, g = _loss_case(N, E, V, dtype, 1, 0.1)
    ref = tu.Loss(x, w, targets, g, dtype)
    wl = _lay(w, by_token)
    loss, lse, gx, gw = _nan(N), _nan(N), _nan(N, E, dtype=dtype), _nan(*wl.shape, dtype=dtype)
    training.linear_cross_entropy(x, wl, targets, loss, lse, N, E, V, by_token=by_token)
    tu.within(loss, ref.loss, ref.e_loss, "loss")
    (dx, dw), (ex, ew) = ref.gradients(lse)
    for _ in range(2):
        training.linear_cross_entropy_backward(x, wl, targets, lse, g, gx, gw, N, E, V, by_token=by_token)
        tu.within(gx, dx, ex, "grad_x")
        tu.within(gw if by_token else gw.t(), dw, ew, "grad_w")
    assert _status() == 0


@pytest.mark.parametrize("by_token", [True, False])
def test_a_common_weight_of_the_rows_is_not_rounded_into_the_gradient(by_token):
    """All rows weigh the same, by a number that bf16 would round by nearly half a step (2^-8): with p near 1 / V, -g w[t] is nearly all of a row's gradient, and must not come out
    smaller than it is throughout.  The share of the wanted gradient that is missing: p - 1 is rounded by at most p < 2^-10 and the results' own roundings go either way (2^-9 / sqrt(N E) < 2^-15
    of it), so less than 2^-9 with room; g rounded would be 2^-8 - 2^-11."""
    N, E, V = 300, 64, 4096
    x, w, targets, g = _loss_case(N, E, V, BF16, 9)
    x.mul_(2.0 ** -4)                            # (powers of two: still bf16 values)
    w.mul_(0.25)
    g.fill_(1.0 + 2.0 ** -8 - 2.0 ** -11)
    ref = tu.Loss(x, w, targets, g, BF16)
    assert float(ref.z.abs().max()) < 0.69       # p < 4 / V = 2^-10
    wl = _lay(w, by_token)
    loss, lse, gx, gw = _nan(N), _nan(N), _nan(N, E, dtype=BF16), _nan(*wl.shape, dtype=BF16)
    training.linear_cross_entropy(x, wl, targets, loss, lse, N, E, V, by_token=by_token)
    training.linear_cross_entropy_backward(x, wl, targets, lse, g, gx, gw, N, E, V, by_token=by_token)
    (dx, dw), _ = ref.gradients(lse)
    for got, want in ((gx, dx), (gw if by_token else gw.t(), dw)):
        missing = 1.0 - float((got.double() * want).sum() / (want * want).sum())
        assert abs(missing) < 2.0 ** -9


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,E,V", [(1, 8, 2), (300, 72, 1001)])
def test_loss_of_no_row_that_takes_part(dtype, N, E, V):
    x, w, targets, g = _nan(N, E, dtype=dtype), _normal(_gen(1), V, E, dtype=dtype), torch.full((N,), V, dtype=torch.int32, device="cuda"), _nan(N)
    loss, lse, gx, gw = _nan(N), _nan(N), _nan(N, E, dtype=dtype), _nan(V, E, dtype=dtype)
    training.linear_cross_entropy(x, w, targets, loss, lse, N, E, V)
    training.linear_cross_entropy_backward(x, w, targets, lse, g, gx, gw, N, E, V)
    assert all(bool((t == 0).all()) for t in (loss, lse, gx, gw))
    old = _normal(_gen(2), V, E, dtype=dtype)
    gw = old.clone()
    training.linear_cross_entropy_backward(x, w, targets, lse, g, None, gw, N, E, V, accumulate=True)
    assert torch.equal(gw, old) and _status() == 0


def test_the_calls_through_ctypes_give_the_same_bits(monkeypatch):
    from hipgpt_b200 import launchers
    N, E, V = 40, 72, 300
    x, w, targets, g = _loss_case(N, E, V, BF16, 4, 0.2)
    ids = _ids(_gen(6), N, V, -1, V + 1)
    pos = _normal(_gen(7), 8, E, dtype=BF16)

    def calls():
        out, y, loss, lse = _nan(N, E, dtype=BF16), _nan(N, E, dtype=BF16), _nan(N), _nan(N)
        gx, gw, gt, gp = _nan(N, E, dtype=BF16), _nan(V, E, dtype=BF16), _nan(V, E), _nan(8, E)
        training.embedding_scaled(ids, w, pos, out, 5, 8, V, E, scale=2.0)
        training.dropout_counter(x, out, y, 0.3, seed=-5, offset=1 << 40)
        training.linear_cross_entropy(x, w, targets, loss, lse, N, E, V)
        training.linear_cross_entropy_backward(x, w, targets, lse, g, gx, gw, N, E, V)
        training.embedding_backward(gx, ids, gt, gp, 5, 8, V, E)
        return [out, y, loss, lse, gx, gw, gt, gp]

    first = calls()
    monkeypatch.setattr(launchers, "_native", launchers._ThroughCtypes)
    assert all(torch.equal(a, b) for a, b in zip(first, calls()))


# ---- the calls together, captured, side by side -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_step_with_tied_weights(dtype):
    """ids -> embedding -> dropout -> loss and all the way back, both gradients into one table, against float64 with the mask given."""
    B, S, V, E, p, seed = 3, 50, 700, 72, 0.25, 99
    gen, N, scale = _gen(4), B * S, 2.5
    tok, pos = _normal(gen, V, E, dtype=dtype, scale=0.3), _normal(gen, S, E, dtype=dtype, scale=0.3)
    ids, targets = _ids(gen, N, V), _ids(gen, N, V)
    targets[7:20] = -1
    x, y, loss, lse = _nan(N, E, dtype=dtype), _nan(N, E, dtype=dtype), _nan(N), _nan(N)
    g = torch.where(targets >= 0, 1.0 / float((targets >= 0).sum()), 0.0).float()
    gy, gx, gtok, gpos = _nan(N, E, dtype=dtype), _nan(N, E, dtype=dtype), _nan(V, E, dtype=dtype), _nan(S, E, dtype=dtype)
    training.embedding_scaled(ids, tok, pos, x, B, S, V, E, scale=scale)
    training.dropout_counter(x, None, y, p, seed=seed, offset=3)
    training.linear_cross_entropy(y, tok, targets, loss, lse, N, E, V)
    training.linear_cross_entropy_backward(y, tok, targets, lse, g, gy, gtok, N, E, V)
    training.dropout_counter(gy, None, gx, p, seed=seed, offset=3)
    gtok0 = gtok.clone()
    training.embedding_backward(gx, ids, gtok, None, B, S, V, E, scale=scale, accumulate=True)
    training.embedding_backward(gx, ids, None, gpos, B, S, V, E, scale=scale)
    keep, inv = tu.kept(N * E, p, seed, 3)
    mask = keep.cuda().view(N, E).double() * inv
    t64, p64 = tok.double().requires_grad_(), pos.double().requires_grad_()
    h = (t64[ids.long()] * scale + p64.repeat(B, 1)) * mask
    ok = targets >= 0
    l64 = torch.nn.functional.cross_entropy(h @ t64.t(), torch.where(ok, targets, torch.zeros_like(targets)).long(), reduction="none") * ok
    (l64 * g.double()).sum().backward()
    # three roundings of the storage type on the way to a loss, six to the table's gradient, each relative to what is there; halves of them add up at most
    eps = 2 * tu.HALF[dtype] + 2e-6
    assert float((loss.double() - l64.detach()).abs().max()) <= 8 * eps * float(l64.detach().max())
    for got, want in ((gtok, t64.grad), (gpos, p64.grad)):
        assert float((got.double() - want).norm() / want.norm()) <= 8 * eps
    assert not torch.equal(gtok, gtok0) and _status() == 0


def _calls(gen, dtype, B, S, V, E):
    """The five calls on tensors of their own: [(call, outputs)]."""
    N = B * S
    tok, pos, g = _normal(gen, V, E, dtype=dtype), _normal(gen, S, E, dtype=dtype), _normal(gen, N, E, dtype=dtype)
    ids, targets, grad = _ids(gen, N, V, -1), _ids(gen, N, V, -1), torch.rand(N, generator=gen, device="cuda")
    x = _normal(gen, N, E, dtype=dtype, scale=E ** -0.5)
    out, drop, loss, lse = _nan(N, E, dtype=dtype), _nan(N, E, dtype=dtype), _nan(N), _nan(N)
    gt, gp, gx, gw = _nan(V, E, dtype=dtype), _nan(S, E, dtype=dtype), _nan(N, E, dtype=dtype), _nan(V, E, dtype=dtype)
    w = tok
    return (lambda: (training.embedding_scaled(ids, tok, pos, out, B, S, V, E, scale=1.5),
                     training.dropout_counter(x, g, drop, 0.2, seed=1),
                     training.embedding_backward(g, ids, gt, gp, B, S, V, E),
                     training.linear_cross_entropy(x, w, targets, loss, lse, N, E, V),
                     training.linear_cross_entropy_backward(x, w, targets, lse, grad, gx, gw, N, E, V))), [out, drop, gt, gp, loss, lse, gx, gw], [tok, pos, g, x, grad]


def _snapshot(outs):
    torch.cuda.synchronize()
    return [o.clone() for o in outs]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_calls_replay_on_new_inputs_and_graphs_do_not_meet(dtype):
    gen = _gen(8)
    jobs = [_calls(gen, dtype, 2, 130, 900, 136), _calls(gen, dtype, 5, 17, 333, 64)]
    graphs = []
    for call, _, _ in jobs:
        call()                                   # what a first call sets up is no part of a graph
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append(graph)
    for _ in range(2):
        want = []
        for call, outs, ins in jobs:
            for t in ins[:4]:
                t.copy_(_normal(gen, *t.shape, dtype=dtype, scale=0.2))
            call()
            want.append(_snapshot(outs))
            for o in outs:
                o.fill_(float("nan"))
        _capi.lib().hipgpt_release_workspace()   # a graph has buffers of its own
        streams = [torch.cuda.Stream() for _ in jobs]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, outs, _), w in zip(jobs, want):
            for o, e in zip(outs, w):
                assert torch.equal(o, e)
    assert _status() == 0


def test_streams_and_threads_side_by_side_give_the_bits_of_one_alone():
    import threading
    gen = _gen(12)
    jobs = [_calls(gen, F32, 3, 200, 1500, 96), _calls(gen, BF16, 4, 128, 2000, 200), _calls(gen, BF16, 1, 40, 5000, 72), _calls(gen, F32, 7, 9, 50, 33)]
    want = []
    for call, outs, _ in jobs:
        call()
        want.append(_snapshot(outs))
        for o in outs:
            o.fill_(float("nan"))
    torch.cuda.synchronize()
    errors = []

    def work(job):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    job[0]()
        except Exception as e:                   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for (_, outs, _), w in zip(jobs, want):
        for o, e in zip(outs, w):
            assert torch.equal(o, e)
    assert _status() == 0


def test_python_refusals_on_the_gpu():
    x, w, t, f = torch.zeros(4, 8, device="cuda"), torch.zeros(16, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="values"):
        training.linear_cross_entropy(x, w, t, f, f.clone(), 5, 8, 16)
    with pytest.raises(ValueError, match="contiguous"):
        training.linear_cross_entropy(x.t(), w, t, f, f.clone(), 4, 8, 16)
    with pytest.raises(ValueError, match="targets"):
        training.linear_cross_entropy(x, w, t.long(), f, f.clone(), 4, 8, 16)
    with pytest.raises(ValueError, match="w"):
        training.linear_cross_entropy(x, w.bfloat16(), t, f, f.clone(), 4, 8, 16)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        training.dropout_counter(x.half(), None, x.half(), 0.1, seed=1)
    with pytest.raises(_capi.HipGPTError, match="outside"):
        training.dropout_counter(x, None, x.clone(), 1.0, seed=1)
    with pytest.raises(_capi.HipGPTError, match="not summed"):
        training.embedding_backward(x, t, w.bfloat16(), None, 2, 2, 16, 8)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("code,block", [(701, 0), (702, 1), (703, 2), (703, 3), (704, 0)])
def test_an_expired_wait_of_the_loss_stores_no_loss(dtype, code, block):
    """The parts of one block are missing, so no row's loss is stored; the status names the wait; the next call is as ever.  What is waited for may have come before, so
    that nothing has to wait: then once more, in the end with one stage a tile, where the products wait for what becomes of their sums."""
    for E in (520,) * 10 + (64,) * 20:
        N, V = 600, 40000
        x, w, targets, _ = _loss_case(N, E, V, dtype, 3)
        loss, lse = _nan(N), _nan(N)
        run = lambda: training.linear_cross_entropy(x, w, targets, loss, lse, N, E, V)  # noqa: E731, B023
        run()
        want = _snapshot([loss, lse])
        loss.fill_(-7.0)
        _capi.check(_capi.lib().hipgpt_debug_expire_wait(code, block))
        run()
        torch.cuda.synchronize()
        status = _status()
        if status:
            break
    assert status == code and bool((loss == -7.0).all())
    run()
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1]) and _status() == 0
