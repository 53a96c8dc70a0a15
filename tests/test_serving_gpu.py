"""Rotary positions, a cache in pages and attention over it against plain float64 forms (tests/serving_util.py)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from hipgpt_b200 import _capi, serving  # noqa: E402
from tests import serving_util as su  # noqa: E402
from tests.serving_util import BF16, F32, HALF, Batch, within  # noqa: E402

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _status():
    st = C.c_int(-1)
    _capi.check(_capi.lib().hipgpt_kernel_status(C.byref(st)))
    return st.value


# ---- rotary -----------------------------------------------------------------------------------------------------------

def _rotary_bound(want, mag, dtype):
    # two products of rounded factors (2^-22 of a unit in the sine), a rounded sum, the storage type
    return mag * 2.0 ** -21 + HALF[dtype] * (want.abs() + mag * 2.0 ** -20) + 1e-38


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 2, 2), (8, 16, 32, 32), (33, 5, 64, 32), (7, 3, 80, 20), (300, 8, 128, 128), (5, 2, 48, 0), (3, 1, 1000, 998), (64, 40, 128, 64), (2, 3, 10, 6)])
def test_rotary(dtype, interleaved, T, H, D, R):
    gen = _gen(T * 1000 + D)
    x = _normal(gen, T, H, D, dtype=dtype)
    freq = serving.rotary_frequencies(R, base=10000.0)
    words = serving.rotary_words(freq)
    positions = torch.randint(-1000, 1 << 20, (T,), generator=gen, device="cuda", dtype=torch.int32)
    positions[0] = 0
    if T > 1:
        positions[1] = (1 << 31) - 1
    for inverse, magnitude in ((False, 1.0), (True, 1.2079441)):
        out = torch.full_like(x, float("nan"))
        serving.rotary(x, positions, words, out, T, H, D, R, interleaved=interleaved, magnitude=magnitude, inverse=inverse)
        # the frequency's own 64 bits: position * 2^-64 of a turn, and its float64 form the 2^-53 of the angle
        want, mag = su.rotated(x, positions, freq, R, interleaved, magnitude, inverse)
        within(out, want, _rotary_bound(want, mag, dtype) + mag * positions.abs().double()[:, None, None] * 2.0 ** -50, "rotated")
        assert torch.equal(out[..., R:], x[..., R:])
        y = x.clone()
        serving.rotary(y, positions, words, y, T, H, D, R, interleaved=interleaved, magnitude=magnitude, inverse=inverse)
        assert torch.equal(y, out), "in place"


def test_rotary_of_a_part_of_wider_rows_and_unaligned():
    gen = _gen(3)
    T, H, D, R = 50, 4, 64, 64
    words = serving.rotary_words(serving.rotary_frequencies(R))
    positions = torch.arange(T, device="cuda", dtype=torch.int32) + 100000
    for dtype in (F32, BF16):
        packed = _normal(gen, T, 3 * H * D, dtype=dtype)
        before = packed.clone()
        q, k = packed[:, :H * D], packed[:, H * D:2 * H * D]
        want = torch.empty(T, H, D, device="cuda", dtype=dtype)
        serving.rotary(q.contiguous(), positions, words, want, T, H, D, R)
        serving.rotary(q, positions, words, q, T, H, D, R)
        assert torch.equal(q, want.view(T, -1)) and torch.equal(packed[:, H * D:], before[:, H * D:])
        serving.rotary(q, positions, words, k, T, H, D, R, inverse=True)          # one part of a row into the one beside it
        assert torch.equal(packed[:, 2 * H * D:], before[:, 2 * H * D:]) and torch.equal(q, want.view(T, -1))
        wide = torch.full((T, H * D + 3), 7.0, device="cuda", dtype=dtype)
        serving.rotary(before[:, :H * D], positions, words, wide[:, 1:1 + H * D], T, H, D, R)
        assert torch.equal(wide[:, 1:1 + H * D], want.view(T, -1)) and bool((wide[:, 0] == 7).all()) and bool((wide[:, 1 + H * D:] == 7).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_backward_is_the_transpose(interleaved):
    """Against differences: the rotation is linear, so its gradient along any direction is what the inverse call gives."""
    gen = _gen(9)
    T, H, D, R = 20, 3, 48, 32
    words = serving.rotary_words(serving.rotary_frequencies(R, scaling="ramp", factor=8.0, original=4096))
    positions = torch.randint(0, 100000, (T,), generator=gen, device="cuda", dtype=torch.int32)
    x, g, d = (_normal(gen, T, H, D) for _ in range(3))
    outs = [torch.empty_like(x) for _ in range(3)]
    for src, out, inv in ((x + d, outs[0], False), (x - d, outs[1], False), (g, outs[2], True)):
        serving.rotary(src, positions, words, out, T, H, D, R, interleaved=interleaved, magnitude=1.1, inverse=inv)
    along = ((outs[0].double() - outs[1].double()) / 2 * g.double()).sum()
    by_gradient = (outs[2].double() * d.double()).sum()
    scale = (g.double().abs() * d.double().abs()).sum() * 4
    assert abs(float(along - by_gradient)) <= float(scale) * 2.0 ** -20


def test_rotary_frequencies_scaled():
    R = 64
    plain = serving.rotary_frequencies(R, base=10000.0)
    i = torch.arange(R // 2, dtype=torch.float64)
    assert torch.allclose(plain, 10000.0 ** (-2 * i / R), rtol=1e-14)
    assert torch.allclose(serving.rotary_frequencies(R, scaling="linear", factor=4.0), plain / 4, rtol=1e-14)
    raised = serving.rotary_frequencies(R, scaling="base", factor=4.0)
    assert float(raised[0]) == 1.0 and abs(float(raised[-1] / plain[-1]) - 0.25) < 1e-12
    ramp = serving.rotary_frequencies(R, scaling="ramp", factor=8.0, original=4096, low=1.0, high=4.0)
    turns = 4096 * plain / (2 * torch.pi)
    keep = ((turns - 1) / 3).clamp(0, 1)
    assert torch.allclose(ramp, plain * (keep + (1 - keep) / 8), rtol=1e-12)


# ---- the cache --------------------------------------------------------------------------------------------------------

SEQS = [(3, 70), (0, 0), (1, 1), (0, 33), (40, 40), (17, 300), (5, 2), (1, 129), (130, 513)]


def _tokens(batch, heads, D, dtype, seed=5):
    gen = _gen(seed)
    x = _normal(gen, batch.T, heads, D, dtype=dtype) * torch.exp2(torch.randint(-20, 20, (batch.T, heads, 1), generator=gen, device="cuda").float()).to(dtype)
    if batch.T > 8:
        x[1] = 0.0
        x[2, 0] = 448.0 / 127 * torch.arange(D, device="cuda").to(dtype) / D      # beside borders
        x[3, :, 0] = float("nan")
        x[4, :, D - 1] = float("-inf")
        x[5] = (torch.randint(-254, 255, x[5].shape, generator=gen, device="cuda").float() / 2).to(dtype)       # halves: ties
        x[5, :, 0] = 127.0
        x[6] = torch.randn(x[6].shape, generator=gen, device="cuda") * 2.0 ** -130
    return x


@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,D,page", [(1, 16, 16), (8, 128, 64), (3, 48, 16), (2, 80, 128), (5, 64, 1024)])
def test_cache_written_and_read_back(fmt, dtype, heads, D, page):
    batch = Batch(SEQS, page, seed=heads, before=2, behind=3)
    k, v = _tokens(batch, heads, D, dtype), _tokens(batch, heads, D, dtype, seed=6)
    cache = serving.PagedCache(batch.num_pages, page, heads, D, dtype=dtype, format=fmt)
    arrays = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    for t in arrays:
        t.view(torch.uint8).fill_(0x2A)
    before = [t.clone() for t in arrays]
    serving.cache_write(cache, k, v, *batch.args)
    row, at, slot = batch.places()
    other = torch.ones(batch.num_pages, page, dtype=torch.bool, device="cuda")
    other[at, slot] = False
    for t, old in zip(arrays, before):
        t, old = (x.view(torch.int32 if x.dim() == 3 else torch.uint8).transpose(1, 2)[other] for x in (t, old))
        assert torch.equal(t, old), "what is no token's place"
    outs = [torch.full_like(k, float("nan")) for _ in range(2)]
    keep = torch.zeros(batch.T, dtype=torch.bool, device="cuda")
    keep[batch.first[0]:batch.first[-1]] = True
    for o in outs:
        o[~keep] = 5.0
    serving.cache_read(cache, *outs, *batch.args)
    for x, o, held, scale in ((k, outs[0], cache.k, cache.k_scale), (v, outs[1], cache.v, cache.v_scale)):
        want = torch.zeros(batch.T, heads, D, device="cuda", dtype=torch.float64)
        if fmt == "plain":
            want[row] = x[row].double()
        else:
            code, unit = su.quantised(x[row], fmt)
            assert torch.equal(held[at, :, slot].double(), code)
            assert torch.equal(scale[at, :, slot].double().nan_to_num(-1.0), unit.nan_to_num(-1.0))
            want[row] = code * unit[..., None]
        assert torch.equal(o[keep].float().nan_to_num(-7.0, -8.0, -9.0), want[keep].to(dtype).float().nan_to_num(-7.0, -8.0, -9.0))
        assert bool((o[~keep] == 5.0).all()), "rows of no sequence"


def test_cache_of_parts_of_wider_rows_and_unaligned():
    for dtype in (F32, BF16):
        for fmt in ("plain", "e4m3", "int8"):
            heads, D, page = 2, 48, 16
            batch = Batch(SEQS, page, seed=4)
            packed = _normal(_gen(8), batch.T, 3 * heads * D + 1, dtype=dtype)
            caches = [serving.PagedCache(batch.num_pages, page, heads, D, dtype=dtype, format=fmt) for _ in range(3)]
            for c in caches:
                c.k.view(torch.uint8).zero_(), c.v.view(torch.uint8).zero_()
                if c.k_scale is not None:
                    c.k_scale.zero_(), c.v_scale.zero_()
            W = heads * D
            for first, c in ((1, caches[0]), (0, caches[1])):                      # off and on 16-byte boundaries (the stride is odd: one value after the other)
                serving.cache_write(c, packed[:, first:first + W], packed[:, first + W:first + 2 * W], *batch.args)
            serving.cache_write(caches[2], packed[:, 1:1 + W].contiguous(), packed[:, 1 + W:1 + 2 * W].contiguous(), *batch.args)
            for a, b in ((caches[0].k, caches[2].k), (caches[0].v, caches[2].v)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            back = torch.full((batch.T, 2 * W + 1), 3.0, device="cuda", dtype=dtype)
            serving.cache_read(caches[0], back[:, :W], back[:, W:2 * W], *batch.args)
            whole = [torch.empty(batch.T, W, device="cuda", dtype=dtype) for _ in range(2)]
            serving.cache_read(caches[2], *whole, *batch.args)
            assert torch.equal(back[:, :W], whole[0]) and torch.equal(back[:, W:2 * W], whole[1]) and bool((back[:, 2 * W] == 3.0).all())


# ---- attention --------------------------------------------------------------------------------------------------------

def _attend(batch, heads, H, D, dtype, fmt, causal=True, scale=None, seed=2, wild=None, spread=1.0):
    cache, k, v = su.filled_cache(batch, heads, D, dtype, fmt, seed=seed, wild=wild)
    q = _normal(_gen(seed + 50), batch.T, H, D, dtype=dtype, scale=spread)
    out = torch.full_like(q, float("nan"))
    serving.paged_attention(cache, q, out, *batch.args, H, causal=causal, scale=scale)
    want, bound, mine = su.attention(batch, k, v, q, H, causal, float(torch.tensor(D ** -0.5 if scale is None else scale)), dtype, fmt)
    return cache, q, out, want, bound, mine


DECODE = [(1, 1), (1, 16), (1, 17), (1, 300), (0, 5), (1, 0), (1, 1000), (1, 2049)]
CHUNKS = [(100, 100), (1, 40), (0, 0), (64, 500), (7, 3), (33, 1031), (129, 129)]


@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,H,D,page", [(1, 1, 16, 16), (2, 8, 128, 64), (3, 3, 32, 16), (1, 20, 64, 128), (2, 2, 80, 32), (4, 8, 48, 1024)])
@pytest.mark.parametrize("seqs", [DECODE, CHUNKS, [(3, 700), (2, 2)], [(700, 900)], [(300, 8000), (129, 129), (40, 900), (33, 34), (1, 3000)]],
                         ids=["tokens", "chunks", "few", "long", "far"])
def test_attention(fmt, dtype, heads, H, D, page, seqs):
    batch = Batch(seqs, page, seed=D, before=1, behind=2)
    for causal in (True, False):
        _, _, out, want, bound, mine = _attend(batch, heads, H, D, dtype, fmt, causal=causal)
        within(out[mine], want[mine], bound[mine], f"causal={causal}")
        assert bool(torch.isnan(out[~mine]).all()), "rows of no sequence are left as they were"
    assert _status() == 0


@pytest.mark.parametrize("dtype,fmt", [(F32, "plain"), (BF16, "plain"), (BF16, "e4m3"), (F32, "int8")])
def test_attention_peaked_scaled_and_strided(dtype, fmt):
    batch = Batch([(50, 400), (1, 900)], 32, seed=7)
    heads, H, D = 2, 4, 64
    _, _, out, want, bound, _ = _attend(batch, heads, H, D, dtype, fmt, scale=3.0, spread=4.0)
    within(out, want, bound, "scores of hundreds")
    cache, q, out, want, bound, _ = _attend(batch, heads, H, D, dtype, fmt, scale=0.01)
    within(out, want, bound, "flat")
    # a part of wider rows, on odd places, into another
    packed, wide = _normal(_gen(1), batch.T, 3 * H * D + 1, dtype=dtype), torch.full((batch.T, H * D + 5), 2.0, device="cuda", dtype=dtype)
    packed[:, 1:1 + H * D] = q.view(batch.T, -1)
    serving.paged_attention(cache, packed[:, 1:1 + H * D], wide[:, 2:2 + H * D], *batch.args, H, scale=0.01)
    assert torch.equal(wide[:, 2:2 + H * D], out.view(batch.T, -1)) and bool((wide[:, :2] == 2).all()) and bool((wide[:, 2 + H * D:] == 2).all())


@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("seqs", [[(1, 200), (40, 300)], [(4, 60), (3, 200)], [(300, 400)], [(1, 2), (300, 5000)]])
def test_what_a_row_does_not_see_does_not_matter(fmt, dtype, seqs):
    """NaN and infinities in keys and values of the sequence's later tokens: the rows before them are as they were without."""
    batch = Batch(seqs, 16, seed=3)
    heads, H, D = 2, 4, 32
    n, length = batch.seqs[-1]
    p = length - 2                                                  # the last row but one sees it, the one before does not
    page, slot = int(batch.table[-1, p // 16]), p % 16

    def wild(name, x):
        x[page, 1, slot, 3] = float("nan") if name == "k" else float("inf")
    first = batch.first[-2]
    _, _, out, want, bound, _ = _attend(batch, heads, H, D, dtype, fmt, wild=wild)
    clean = torch.ones(batch.T, H, dtype=torch.bool, device="cuda")
    clean[first + n - 2:, H // heads:] = False
    within(out[clean], want[clean], bound[clean], "rows that do not see it")
    assert not bool(torch.isfinite(out[~clean]).all(-1).any()), "rows that do"


@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_numbers_that_are_no_pages(fmt, dtype):
    """Pages outside the cache hold no tokens: not read, not written, not seen; lengths and offsets beyond what there is are cut."""
    batch = Batch([(1, 100), (20, 90), (2, 30), (70, 75)], 16, seed=11)
    heads, H, D = 2, 2, 32
    batch.table[0, 3], batch.table[1, 5], batch.table[2] = 1 << 30, -7, batch.num_pages
    batch.pages.copy_(batch.table)
    _, _, out, want, bound, mine = _attend(batch, heads, H, D, dtype, fmt)
    within(out, want, bound)
    assert bool((out[batch.first[2]:batch.first[3]] == 0).all()), "rows that see nothing"
    cache = serving.PagedCache(batch.num_pages, 16, heads, D, dtype=dtype, format=fmt)
    x = _normal(_gen(1), batch.T, heads, D, dtype=dtype)
    back = [torch.full_like(x, float("nan")) for _ in range(2)]
    serving.cache_write(cache, x, x, *batch.args)
    serving.cache_read(cache, *back, *batch.args)
    row = batch.places()[0]
    nowhere = torch.ones(batch.T, dtype=torch.bool, device="cuda")
    nowhere[row] = False
    assert bool((back[0][nowhere] == 0).all()) and int(nowhere.sum()) >= 2
    if fmt == "plain":
        assert torch.equal(back[0][row], x[row])
    # lengths beyond the table and below zero, offsets beyond the rows and out of order
    lengths, offsets = torch.tensor([1 << 30, -5, 7, (1 << 31) - 1], dtype=torch.int32).cuda(), torch.tensor([-3, 40, 12, 1 << 30, 5], dtype=torch.int32).cuda()
    q, out = _normal(_gen(2), batch.T, H, D, dtype=dtype), torch.zeros(batch.T, H, D, device="cuda", dtype=dtype)
    serving.cache_write(cache, x, x, offsets, lengths, batch.pages, batch.T, batch.B)
    serving.cache_read(cache, *back, offsets, lengths, batch.pages, batch.T, batch.B)
    serving.paged_attention(cache, q, out, offsets, lengths, batch.pages, batch.T, batch.B, H)
    torch.cuda.synchronize()
    assert _status() == 0


def _step(cache, batch, qkv, words, positions, out, H, heads, D):
    q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + heads) * D], qkv[:, (H + heads) * D:]
    turned = qkv[:, :(H + heads) * D]
    serving.rotary(turned, positions, words, turned, batch.T, H + heads, D, D)
    serving.cache_write(cache, k, v, *batch.args)
    serving.paged_attention(cache, q, out, *batch.args, H)


@pytest.mark.parametrize("dtype,fmt", [(F32, "plain"), (F32, "int8"), (BF16, "plain"), (BF16, "e4m3"), (BF16, "int8")])
def test_prompts_and_tokens_one_after_the_other(dtype, fmt):
    """Rotation, cache and attention as a program calls them: prompts in two pieces and then tokens, captured or not, give what one pass over all tokens gives."""
    heads, H, D, page = 2, 4, 64, 16
    lens = [90, 41, 130]
    gen = _gen(77)
    words = serving.rotary_words(serving.rotary_frequencies(D))
    stream = [_normal(gen, n, (H + 2 * heads) * D, dtype=dtype) for n in lens]
    whole = Batch([(n, n) for n in lens], page, seed=1)
    cache = serving.PagedCache(whole.num_pages, page, heads, D, dtype=dtype, format=fmt)

    def feed(pieces, cache, capture=False):
        outs = [torch.empty(n, H, D, device="cuda", dtype=dtype) for n in lens]
        for some in pieces:                                         # [(from, to)] for each sequence
            seqs = [(b - a, b) for a, b in some]
            batch = Batch(seqs, page, seed=1, width=whole.table.shape[1])
            batch.pages.copy_(whole.pages)
            qkv = torch.cat([stream[i][a:b] for i, (a, b) in enumerate(some)])
            positions = torch.cat([torch.arange(a, b) for a, b in some]).int().cuda()
            out = torch.empty(batch.T, H, D, device="cuda", dtype=dtype)
            if capture:
                kept, graph = qkv.clone(), torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    _step(cache, batch, qkv, words, positions, out, H, heads, D)
                qkv.copy_(kept)
                graph.replay()
            else:
                _step(cache, batch, qkv, words, positions, out, H, heads, D)
            for i, (a, b) in enumerate(some):
                outs[i][a:b] = out[batch.first[i]:batch.first[i + 1]]
        return outs
    once = feed([[(0, n) for n in lens]], cache)
    steps = [[(0, 30), (0, 40), (0, 0)], [(30, 89), (40, 40), (0, 129)], [(89, 90), (40, 41), (129, 130)]]
    parts, captured = feed(steps, cache), feed(steps, cache, capture=True)
    kv = [torch.empty(whole.T, heads, D, device="cuda", dtype=dtype) for _ in range(2)]
    serving.cache_read(cache, *kv, *whole.args)
    for i, n in enumerate(lens):
        assert torch.equal(parts[i], captured[i])
        # two ways to sum the same terms: each within the plain form's bound of it
        turned = torch.empty(n, H, D, device="cuda", dtype=dtype)
        serving.rotary(stream[i][:, :H * D], torch.arange(n, device="cuda", dtype=torch.int32), words, turned, n, H, D, D)
        b = Batch([(n, n)], 16, seed=1)
        rows = slice(whole.first[i], whole.first[i + 1])
        vals = [torch.zeros(b.num_pages, heads, 16, D, dtype=torch.float64, device="cuda") for _ in range(2)]
        row, at, slot = b.places()
        for val, x in zip(vals, kv):
            val[at, :, slot] = x[rows][row].double()
        if fmt == "int8" or dtype == F32:
            # what cache_read rounds to the storage type, the attention takes as it is
            for val, held, scale in ((vals[0], cache.k, cache.k_scale), (vals[1], cache.v, cache.v_scale)):
                if scale is not None:
                    p = torch.arange(n)
                    pg, sl = whole.table[i].long()[p // page].cuda(), (p % page).cuda()
                    val[at, :, slot] = held[pg, :, sl].double() * scale[pg, :, sl].double()[..., None]
        want, bound, _ = su.attention(b, vals[0], vals[1], turned, H, True, float(torch.tensor(D ** -0.5)), dtype, fmt)
        within(once[i], want, bound, "one pass")
        within(parts[i], want, bound, "in pieces")


def test_two_streams_and_runs_give_the_same_bits():
    batch = Batch([(1, 3000), (1, 70), (1, 1)], 64, seed=2)
    cache, q, out, want, bound, _ = _attend(batch, 2, 8, 64, BF16, "e4m3")
    within(out, want, bound)
    other = Batch([(64, 900)], 64, seed=2)
    cache2, q2, out2, want2, bound2, _ = _attend(other, 2, 8, 64, BF16, "plain")
    outs = [(torch.empty_like(out), torch.empty_like(out2)) for _ in range(6)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(outs):
        with torch.cuda.stream(streams[i % 3]):
            serving.paged_attention(cache, q, a, *batch.args, 8)
            serving.paged_attention(cache2, q2, b, *other.args, 8)
    torch.cuda.synchronize()
    for a, b in outs:
        assert torch.equal(a, out) and torch.equal(b, out2)


def test_a_captured_call_sees_lengths_of_its_replay():
    batch = Batch([(1, 500), (1, 64)], 16, seed=5)
    heads, H, D = 2, 2, 32
    cache, k, v = su.filled_cache(batch, heads, D, F32, "plain")
    q, out = _normal(_gen(1), 2, H, D), torch.empty(2, H, D, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.paged_attention(cache, q, out, *batch.args, H)
    for lens in ((500, 64), (1, 3), (333, 0)):
        batch.seqs = [(1, n) for n in lens]
        batch.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        serving.paged_attention(serving.PagedCache(400, 64, 1, 32), torch.zeros(1, 1, 32, device="cuda"), torch.empty(1, 1, 32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32).cuda(),
                                torch.tensor([20000], dtype=torch.int32).cuda(), torch.full((1, 400), -1, dtype=torch.int32).cuda(), 1, 1, 1)      # a call in between with a larger buffer
        graph.replay()
        want, bound, _ = su.attention(batch, k, v, q, H, True, float(torch.tensor(D ** -0.5)), F32, "plain")
        within(out, want, bound)


def test_places_beyond_2_31():
    """A cache of more than 2^31 elements: its last pages."""
    heads, D, page = 8, 128, 64
    pages = (1 << 31) // (heads * D * page) + 40
    cache = serving.PagedCache(pages, page, heads, D, dtype=BF16, format="int8")
    n = 100
    batch = Batch([(n, n), (1, 33)], page, seed=1)
    batch.pages.copy_(torch.where(batch.table >= 0, batch.table + pages - batch.num_pages, batch.table))
    gen = _gen(2)
    k, v = _normal(gen, batch.T, heads, D, dtype=BF16), _normal(gen, batch.T, heads, D, dtype=BF16)
    full = Batch([(n, n), (33, 33)], page, seed=1)
    full.pages.copy_(batch.pages)
    k2, v2 = _normal(gen, full.T, heads, D, dtype=BF16), _normal(gen, full.T, heads, D, dtype=BF16)
    serving.cache_write(cache, k2, v2, *full.args)
    back = [torch.empty_like(k2) for _ in range(2)]
    serving.cache_read(cache, *back, *full.args)
    for x, y in ((k2, back[0]), (v2, back[1])):
        code, unit = su.quantised(x, "int8")
        assert torch.equal(y, (code * unit[..., None]).to(BF16))
    q, out = _normal(gen, batch.T, heads, D, dtype=BF16), torch.empty(batch.T, heads, D, device="cuda", dtype=BF16)
    serving.paged_attention(cache, q, out, *batch.args, heads)
    vals = []
    for x in (k2, v2):
        code, unit = su.quantised(x, "int8")
        val = torch.zeros(full.num_pages, heads, page, D, dtype=torch.float64, device="cuda")
        row, at, slot = full.places()
        val[at, :, slot] = (code * unit[..., None])[row]
        vals.append(val)
    want, bound, _ = su.attention(batch, vals[0], vals[1], q, heads, True, float(torch.tensor(D ** -0.5)), BF16, "int8")
    within(out, want, bound)


def test_through_ctypes(monkeypatch):
    """Without the extension the same calls give the same bits."""
    from hipgpt_b200 import launchers
    batch = Batch([(1, 100), (30, 60)], 16, seed=8)
    cache, q, out, want, bound, _ = _attend(batch, 2, 4, 32, F32, "int8")
    words, pos = serving.rotary_words(serving.rotary_frequencies(32)), torch.arange(batch.T, device="cuda", dtype=torch.int32)
    results = []
    for _ in range(2):
        turned, o = torch.empty_like(q), torch.empty_like(q)
        back = [torch.empty(batch.T, 2, 32, device="cuda") for _ in range(2)]
        serving.rotary(q, pos, words, turned, batch.T, 4, 32, 32)
        serving.cache_write(cache, turned[:, :2].contiguous(), q[:, 2:].contiguous(), *batch.args)
        serving.cache_read(cache, *back, *batch.args)
        serving.paged_attention(cache, q, o, *batch.args, 4)
        results.append((turned, *back, o))
        monkeypatch.setattr(launchers, "_native", launchers._ThroughCtypes)
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("fmt", ["plain", "int8"])
@pytest.mark.parametrize("code,block", [(1001, 0), (1002, 3), (1003, 1), (1004, 2), (1005, 0), (1006, 5), (1007, 4), (1008, 1), (1009, 6), (1010, 2)])
def test_an_expired_wait_stores_no_part_of_a_value(fmt, code, block):
    """Every row of the result is as ever, or nothing was stored there; the next call is as ever."""
    batch = Batch([(300, 8000), (129, 129), (40, 900)], 64, seed=3)          # five units of 128 keys a block
    cache, q, out, want, bound, mine = _attend(batch, 2, 8, 128, BF16, fmt)
    within(out, want, bound)
    if code == 1010 and fmt == "plain":
        pytest.skip("plain rows have no ring")
    for _ in range(20):
        got = torch.full_like(out, -7.0)
        _capi.check(_capi.lib().hipgpt_debug_expire_wait(code, block))
        serving.paged_attention(cache, q, got, *batch.args, 8)
        torch.cuda.synchronize()
        status = _status()
        if status:
            break
    assert status == code and _status() == 0
    same, left = (got == out).all(-1), (got == -7.0).all(-1)
    assert bool((same | left).all()) and bool(left.any()) and bool(same.any())
    serving.paged_attention(cache, q, got, *batch.args, 8)
    assert torch.equal(got, out)


@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("n,length", [(1024, 16000), (1, 30000)])
def test_long_calls_give_the_same_bits_every_time(fmt, n, length):
    """Many tiles in flight in every block: what one stage hands to the next is there when it is used, and is used before it goes."""
    batch = Batch([(n, length), (n, length // 2)], 128, seed=4)
    cache, q, out, want, bound, _ = _attend(batch, 4, 16, 128, BF16, fmt)
    within(out, want, bound)
    got = torch.empty_like(out)
    for _ in range(60):
        got.fill_(float("nan"))
        serving.paged_attention(cache, q, got, *batch.args, 16)
        assert torch.equal(got, out)


@pytest.mark.parametrize("fmt", ["plain", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("seqs", [[(300, 900), (70, 80)], [(1, 900), (4, 500)], [(20, 700)]], ids=["many", "tokens", "some"])
def test_rows_of_any_magnitude(fmt, dtype, seqs):
    """Values of zeros, tiny and large ones page beside page, keys and queries far from one: the powers of two that rows and tiles share follow them."""
    batch = Batch(seqs, 64, seed=13)
    heads, H, D = 2, 4, 64

    def wild(name, x):
        if name == "k":
            x *= 2.0 ** -30
        else:
            for page in range(len(x)):
                x[page] *= (0.0, 2.0 ** -20, 1.0, 2.0 ** 10)[page % 4]
    _, _, out, want, bound, _ = _attend(batch, heads, H, D, dtype, fmt, wild=wild, spread=2.0 ** 31)
    within(out, want, bound)

    def tiny(name, x):
        x *= 2.0 ** -100                                            # scores of zero, values near the smallest numbers
    _, _, out, want, bound, _ = _attend(batch, heads, H, D, dtype, fmt, wild=tiny, spread=2.0 ** -100)
    within(out, want, bound)


@pytest.mark.parametrize("fmt", ["plain", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nothing_but_nan(fmt, dtype):
    """Every value NaN: every row that sees one is NaN, and the call comes back."""
    batch = Batch([(600, 20000), (1, 20000), (3, 3)], 64, seed=1)

    def wild(name, x):
        if name == "v":
            x.fill_(float("nan"))
    cache, _, _ = su.filled_cache(batch, 2, 64, dtype, fmt, wild=wild)
    q = _normal(_gen(1), batch.T, 4, 64, dtype=dtype)
    out = torch.zeros_like(q)
    serving.paged_attention(cache, q, out, *batch.args, 4)
    assert bool(torch.isnan(out).all()) and _status() == 0


def test_many_short_sequences():
    """More sequences than a block has threads, some empty, of one token and more."""
    gen = torch.Generator().manual_seed(5)
    seqs = [(int(n), int(n) + int(m)) for n, m in zip(torch.randint(0, 3, (700,), generator=gen), torch.randint(0, 40, (700,), generator=gen))]
    for dtype, fmt in ((F32, "plain"), (BF16, "e4m3")):
        for group in (2, 40):                                       # few rows a sequence, and many
            batch = Batch(seqs, 16, seed=6)
            _, _, out, want, bound, mine = _attend(batch, 1, group, 32, dtype, fmt)
            within(out[mine], want[mine], bound[mine])
    x = _normal(_gen(3), batch.T, 1, 32, dtype=BF16)
    cache = serving.PagedCache(batch.num_pages, 16, 1, 32, dtype=BF16, format="plain")
    back = [torch.full_like(x, float("nan")) for _ in range(2)]
    serving.cache_write(cache, x, x, *batch.args)
    serving.cache_read(cache, *back, *batch.args)
    assert torch.equal(back[0], x) and torch.equal(back[1], x)


# Sequences of many rows: 8-bit rows are widened before the attention
WIDE = [(700, 2100), (0, 0), (900, 900), (1, 5), (1200, 1000)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,H,D,page", [(1, 4, 128, 16), (2, 8, 64, 1024), (1, 8, 48, 128), (2, 8, 80, 64), (1, 3, 16, 32)])
def test_codes_widened_before(fmt, heads, H, D, page):
    batch = Batch(WIDE, page, seed=D, before=1, behind=2)
    assert batch.T * (H // heads) >= 1536 * batch.B
    for causal in (True, False):
        _, _, out, want, bound, mine = _attend(batch, heads, H, D, BF16, fmt, causal=causal)
        within(out[mine], want[mine], bound[mine], f"causal={causal}")
        assert bool(torch.isnan(out[~mine]).all())
    assert _status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_codes_widened_before_of_any_magnitude(fmt):
    batch = Batch([(1000, 1300), (700, 800)], 64, seed=13)

    def wild(name, x):
        if name == "k":
            x *= 2.0 ** -30
        else:
            for page in range(len(x)):
                x[page] *= (0.0, 2.0 ** -20, 1.0, 2.0 ** 10)[page % 4]
    _, _, out, want, bound, _ = _attend(batch, 2, 8, 64, BF16, fmt, wild=wild, spread=2.0 ** 31)
    within(out, want, bound)

    def tiny(name, x):
        x *= 2.0 ** -100
    _, _, out, want, bound, _ = _attend(batch, 2, 8, 64, BF16, fmt, wild=tiny, spread=2.0 ** -100)
    within(out, want, bound)

    def zeros(name, x):
        if name == "v":
            x.zero_()
    _, _, out, want, bound, _ = _attend(batch, 2, 8, 64, BF16, fmt, wild=zeros)
    assert bool((out == 0).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_codes_widened_before_what_is_not_seen_and_no_pages(fmt):
    batch = Batch([(700, 900), (1000, 1200)], 16, seed=3)
    heads, H, D = 2, 8, 32
    p = 1200 - 2
    page, slot = int(batch.table[-1, p // 16]), p % 16

    def wild(name, x):
        x[page, 1, slot, 3] = float("nan") if name == "k" else float("inf")
    _, _, out, want, bound, _ = _attend(batch, heads, H, D, BF16, fmt, wild=wild)
    clean = torch.ones(batch.T, H, dtype=torch.bool, device="cuda")
    clean[700 + 1000 - 2:, H // heads:] = False
    within(out[clean], want[clean], bound[clean], "rows that do not see it")
    assert not bool(torch.isfinite(out[~clean]).all(-1).any()), "rows that do"
    batch.table[0, 3], batch.table[0, 55], batch.table[1, 10:40] = 1 << 30, -7, batch.num_pages
    batch.pages.copy_(batch.table)
    _, _, out, want, bound, mine = _attend(batch, heads, H, D, BF16, fmt)
    within(out, want, bound, "pages that are none")
    q, out = _normal(_gen(2), batch.T, H, D, dtype=BF16), torch.zeros(batch.T, H, D, device="cuda", dtype=BF16)
    cache = su.filled_cache(batch, heads, D, BF16, fmt)[0]
    for offsets, lengths in (([-3, 1500, 1 << 30], [1 << 30, -5]), ([0, 1700, 400], [(1 << 31) - 1, 0]), ([900, 100, 1600], [7, 1200])):
        serving.paged_attention(cache, q, out, torch.tensor(offsets, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), batch.pages, batch.T, batch.B, H)
        torch.cuda.synchronize()
        assert _status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_codes_widened_before_in_graphs_on_streams_and_every_time(fmt):
    batch = Batch([(900, 5000), (900, 901)], 64, seed=6)
    cache, q, out, want, bound, _ = _attend(batch, 2, 8, 128, BF16, fmt)
    within(out, want, bound)
    graphs = [(torch.cuda.CUDAGraph(), torch.empty_like(out)) for _ in range(2)]
    for graph, got in graphs:
        with torch.cuda.graph(graph):
            serving.paged_attention(cache, q, got, *batch.args, 8)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros_like(out) for _ in range(30)]
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        with torch.cuda.stream(streams[i % 3]):
            serving.paged_attention(cache, q, got, *batch.args, 8)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in outs + [got for _, got in graphs]:
        assert torch.equal(got, out)
    batch.seqs = [(900, 3000), (900, 950)]                           # a replay sees what the lengths hold then
    batch.lengths.copy_(torch.tensor([3000, 950], dtype=torch.int32))
    serving.paged_attention(cache, q, out, *batch.args, 8)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    seen_nan = torch.isnan(out)                                      # (the second sequence's keys from 901 on were never written)
    assert torch.equal(torch.isnan(graphs[0][1]), seen_nan) and torch.equal(graphs[0][1].nan_to_num(), out.nan_to_num())
    assert not bool(seen_nan[:900].any()) and bool(seen_nan[-1].all())


@pytest.mark.parametrize("code,block", [(1001, 0), (1002, 3), (1003, 1), (1004, 2), (1005, 0), (1006, 5), (1007, 4), (1008, 1), (1009, 6)])
def test_codes_widened_before_an_expired_wait(code, block):
    batch = Batch([(900, 5000), (900, 901)], 64, seed=6)
    cache, q, out, want, bound, _ = _attend(batch, 2, 8, 128, BF16, "int8")
    within(out, want, bound)
    for _ in range(20):
        got = torch.full_like(out, -7.0)
        _capi.check(_capi.lib().hipgpt_debug_expire_wait(code, block))
        serving.paged_attention(cache, q, got, *batch.args, 8)
        torch.cuda.synchronize()
        status = _status()
        if status:
            break
    assert status == code and _status() == 0
    same, left = (got == out).all(-1), (got == -7.0).all(-1)
    assert bool((same | left).all()) and bool(left.any()) and bool(same.any())
    serving.paged_attention(cache, q, got, *batch.args, 8)
    assert torch.equal(got, out)


@pytest.mark.parametrize("heads,H,D,page", [(1, 4, 128, 16), (2, 4, 64, 1024), (1, 3, 48, 128), (2, 2, 80, 64), (2, 4, 16, 32), (3, 3, 32, 16)])
def test_pieces_cut_before(heads, H, D, page):
    """fp32 rows enough that keys and values are cut into pieces once: sequences that end inside a place, see nothing, have no rows or one."""
    batch = Batch([(300, 700), (0, 0), (500, 500), (1, 5), (400, 333), (97, 1025)], page, seed=D, before=1, behind=2)
    for causal in (True, False):
        _, _, out, want, bound, mine = _attend(batch, heads, H, D, F32, "plain", causal=causal)
        within(out[mine], want[mine], bound[mine], f"causal={causal}")
        assert bool(torch.isnan(out[~mine]).all())
    assert _status() == 0


def test_pieces_cut_before_what_is_not_seen_and_no_pages():
    batch = Batch([(200, 900), (330, 1200)], 16, seed=3)
    heads, H, D = 2, 4, 32
    for p in (1200 - 2, 1200 - 200, 1199):                           # in the places of tiles that do not see them, too
        page, slot = int(batch.table[-1, p // 16]), p % 16

        def wild(name, x):
            x[page, 1, slot, 3] = float("nan") if name == "k" else float("inf")
        _, _, out, want, bound, _ = _attend(batch, heads, H, D, F32, "plain", wild=wild)
        clean = torch.ones(batch.T, H, dtype=torch.bool, device="cuda")
        clean[200 + 330 - (1200 - p):, H // heads:] = False
        within(out[clean], want[clean], bound[clean], "rows that do not see it")
        assert not bool(torch.isfinite(out[~clean]).all(-1).any()), "rows that do"
    batch.table[0, 3], batch.table[0, 55], batch.table[1, 10:40] = 1 << 30, -7, batch.num_pages
    batch.pages.copy_(batch.table)
    _, _, out, want, bound, mine = _attend(batch, heads, H, D, F32, "plain")
    within(out, want, bound, "pages that are none")
    q, out = _normal(_gen(2), batch.T, H, D), torch.zeros(batch.T, H, D, device="cuda")
    cache = su.filled_cache(batch, heads, D, F32, "plain")[0]
    for offsets, lengths in (([-3, 400, 1 << 30], [1 << 30, -5]), ([0, 500, 100], [(1 << 31) - 1, 0]), ([300, 100, 530], [7, 1200])):
        serving.paged_attention(cache, q, out, torch.tensor(offsets, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), batch.pages, batch.T, batch.B, H)
        torch.cuda.synchronize()
        assert _status() == 0


@pytest.mark.parametrize("D", [32, 64, 128])
def test_pieces_cut_before_in_graphs_on_streams_and_every_time(D):
    batch = Batch([(300, 3000), (200, 901)], 64, seed=6)
    cache, q, out, want, bound, _ = _attend(batch, 2, 4, D, F32, "plain")
    within(out, want, bound)
    graphs = [(torch.cuda.CUDAGraph(), torch.empty_like(out)) for _ in range(2)]
    for graph, got in graphs:
        with torch.cuda.graph(graph):
            serving.paged_attention(cache, q, got, *batch.args, 4)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros_like(out) for _ in range(30)]
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        with torch.cuda.stream(streams[i % 3]):
            serving.paged_attention(cache, q, got, *batch.args, 4)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in outs + [got for _, got in graphs]:
        assert torch.equal(got, out)
    batch.lengths.copy_(torch.tensor([2000, 900], dtype=torch.int32))
    serving.paged_attention(cache, q, out, *batch.args, 4)
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[1][1], out)
