"""Plain float64 forms of the operators of hipgpt_b200/serving.py and bounds on how far fp32 arithmetic may be from them."""
import torch

from hipgpt_b200 import serving
from tests.training_util import HALF, within  # noqa: F401

F32, BF16 = torch.float32, torch.bfloat16
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class Batch:
    """Sequences of (new tokens, length with them), their pages dealt in no order; rows in front of the first sequence and behind the last belong to none."""

    def __init__(self, seqs, page, seed=0, spare=2, before=0, behind=0, width=0):
        gen = torch.Generator().manual_seed(seed)
        self.seqs, self.page = seqs, page
        held = [-(-length // page) for _, length in seqs]
        self.num_pages = sum(held) + spare
        deal = torch.randperm(self.num_pages, generator=gen).tolist()
        most = max(held + [width, 1])
        table = torch.full((len(seqs), most), -1, dtype=torch.int32)
        for b, h in enumerate(held):
            table[b, :h] = torch.tensor([deal.pop() for _ in range(h)], dtype=torch.int32)
        first = [before]
        for n, _ in seqs:
            first.append(first[-1] + n)
        self.T, self.B = first[-1] + behind, len(seqs)
        self.first = first
        self.offsets, self.lengths, self.pages = torch.tensor(first, dtype=torch.int32).cuda(), torch.tensor([x for _, x in seqs], dtype=torch.int32).cuda(), table.cuda()
        self.table = table

    @property
    def args(self):
        return self.offsets, self.lengths, self.pages, self.T, self.B

    def places(self):
        """(row of the call, page, slot) of each new token that has a place."""
        out = []
        for b, (n, length) in enumerate(self.seqs):
            for i in range(n):
                p = length - n + i
                if p >= 0 and 0 <= int(self.table[b, p // self.page]) < self.num_pages:
                    out.append((self.first[b] + i, int(self.table[b, p // self.page]), p % self.page))
        return [torch.tensor(x, dtype=torch.long, device="cuda") for x in zip(*out)] if out else [torch.zeros(0, dtype=torch.long, device="cuda")] * 3


def quantised(x, fmt):
    """(codes as float64, scales as float64) of the rows of x, from the formats' definitions."""
    x = x.double()
    fine = torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(fine, x, torch.zeros_like(x))
    most = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        unit = (most / 127.0).float().double().clamp(min=2.0 ** -126)
        code = torch.round(x / unit)
    else:
        unit = torch.full_like(most, 2.0 ** -126)
        while bool((most > 448.0 * unit).any()):
            unit = torch.where(most > 448.0 * unit, unit * 2, unit)
        y = x / unit
        step = torch.full_like(y, 2.0 ** -9)
        for e in range(-5, 9):
            step = torch.where(y.abs() >= 2.0 ** e, torch.full_like(step, 2.0 ** (e - 3)), step)
        code = torch.round(y / step) * step
    return torch.where(fine, code, torch.zeros_like(code)), torch.where(fine, unit, torch.full_like(unit, float("nan")))[..., 0]


def filled_cache(batch, heads, D, dtype, fmt, seed=1, scale=1.0, wild=None):
    """A cache of normal values in the places that the batch's sequences have, and of what must not matter in all others; the values it stands for
    as float64, [pages][heads][page][D]."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (batch.num_pages, heads, batch.page, D)
    used = torch.zeros(batch.num_pages, batch.page, dtype=torch.bool)
    for b, (_, length) in enumerate(batch.seqs):
        for p in range(length):
            page = int(batch.table[b, p // batch.page]) if p // batch.page < batch.table.shape[1] else -1
            if 0 <= page < batch.num_pages:
                used[page, p % batch.page] = True
    used = used.cuda()[:, None, :]
    cache = serving.PagedCache(batch.num_pages, batch.page, heads, D, dtype=dtype, format=fmt)
    values = []
    for name in "kv":
        x = (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)
        if wild is not None:
            wild(name, x)
        if fmt == "plain":
            getattr(cache, name).copy_(torch.where(used[..., None], x, torch.full_like(x, float("nan"))))
            values.append(x.double())
        else:
            code, unit = quantised(x, fmt)
            junk = torch.full_like(code, float("nan") if fmt == "e4m3" else -128.0)
            getattr(cache, name).copy_(torch.where(used[..., None], code, junk).to(CODES[fmt]))
            getattr(cache, name + "_scale").copy_(torch.where(used.expand(shape[:3]), unit, torch.full_like(unit, float("nan"))).float())
            values.append(code * unit[..., None])
    return cache, values[0], values[1]


def rows_of(values, batch, b, h):
    """(rows [length][D] of one head as float64, whether a position has a page)."""
    length = min(batch.seqs[b][1], batch.table.shape[1] * batch.page)
    p = torch.arange(length)
    page = batch.table[b].long()[p // batch.page]
    there = (page >= 0) & (page < batch.num_pages)
    return values[torch.where(there, page, torch.zeros_like(page)).cuda(), h, (p % batch.page).cuda()], there.cuda()


def attention(batch, k, v, q, H, causal, scale, dtype, fmt):
    """(out float64 [T][H][D], bound, rows that are any sequence's)."""
    heads, D = k.shape[1], k.shape[3]
    G = H // heads
    out = torch.zeros(batch.T, H, D, dtype=torch.float64, device="cuda")
    bound, mine = torch.zeros_like(out), torch.zeros(batch.T, dtype=torch.bool, device="cuda")
    step = 2.0 ** -23
    for b, (n, length) in enumerate(batch.seqs):
        f = batch.first[b]
        mine[f:f + n] = True
        if n == 0:
            continue
        for h in range(heads):
            kk, there = rows_of(k, batch, b, h)
            vv, _ = rows_of(v, batch, b, h)
            qq = q[f:f + n, h * G:(h + 1) * G].double()
            seen = there[None].expand(n, -1)
            if causal:
                seen = seen & (torch.arange(len(kk), device="cuda")[None] <= torch.arange(length - n, length, device="cuda")[:, None])
            if not len(kk):
                continue
            # a key with an infinity or NaN matters to the rows that see it alone
            wild = ~(torch.isfinite(kk).all(-1) & torch.isfinite(vv).all(-1))
            vv, kk = (torch.where(wild[:, None], torch.zeros_like(x), x) for x in (vv, kk))
            z = torch.einsum("ngd,kd->ngk", qq, kk) * scale
            z = z.masked_fill(~seen[:, None], float("-inf"))
            top = z.amax(-1, keepdim=True)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            e = torch.exp(z - top)
            p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
            o = torch.einsum("ngk,kd->ngd", p, vv)
            # scores: three bf16 pieces of an fp32 operand (2^-24 each) without the products below 2^-24; D / 16 instructions that cut off; scales and differences rounded
            mag = torch.einsum("ngd,kd->ngk", qq.abs(), kk.abs()) * scale
            zf = torch.where(seen[:, None], z, torch.zeros_like(z))
            ez = mag * (12 * step) + zf.abs() * 2 * step + (zf - top).abs() * step
            rel = ez + 2.0 ** -21                                           # and the exponential
            if dtype == BF16:
                rel = rel + HALF[BF16]                                      # P is rounded (its sum is not)
            keys = len(kk)
            rel = rel + (keys / 16 + 32) * step                             # sums of probabilities and of P V
            pv = torch.einsum("ngk,kd->ngd", p * rel, vv.abs()) + o.abs() * (p * rel).sum(-1, keepdim=True)
            if fmt != "plain":
                # Codes: a probability times its value's scale is held in fp16 pieces, divided by a power of two that brings the largest such product to 2^13 at least.  Below fp16's normal numbers
                # the pieces stop at its smallest step, 2^-24: half of one, 2^-25, of a code, that is 2^-38 of the largest scale times the code, for each key.  A scale times its code is less than
                # twice the largest value of a row (e4m3: the largest is above 224 scales, of 448).
                pv = pv + keys * 2.0 ** -37 * vv.abs().max()
            o = o.masked_fill((seen & wild[None]).any(-1)[:, None, None], float("nan"))
            out[f:f + n, h * G:(h + 1) * G] = o
            bound[f:f + n, h * G:(h + 1) * G] = pv + HALF[dtype] * (o.abs() + pv) + 1e-37
    return out, bound, mine


def rotated(x, positions, freq, R, interleaved, magnitude, inverse):
    """float64 rotation of x [T][H][D], and the magnitude of the two products of each element."""
    x = x.double()
    angle = positions.double()[:, None] * freq.double().to(x.device)
    c, s = torch.cos(angle)[:, None] * magnitude, torch.sin(angle)[:, None] * magnitude
    if inverse:
        s = -s
    even = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    odd = even + 1 if interleaved else even + R // 2
    out, mag = x.clone(), torch.zeros_like(x)
    a, b = x[..., even], x[..., odd]
    out[..., even], out[..., odd] = a * c - b * s, a * s + b * c
    # sines and cosines are off by 2^-22 of a unit at most (the angle's rounding, sincospi, the magnitude's product)
    mag[..., even] = mag[..., odd] = (a.abs() + b.abs()) * abs(magnitude)
    return out, mag


