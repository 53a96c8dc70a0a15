"""Plain float64 forms of the operators of hipgpt_b200/training.py and bounds on how far fp32 arithmetic may be from them.

A rounding is off by at most half a step relative to the value: HALF[dtype].  Sums on the tensor core are cut off, which is up to a whole step
of fp32 (2^-23) for each instruction of 16 products that adds to the running sum; a running sum is at most the sum of the magnitudes."""
import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def philox_bits(blocks, seed):
    """The eight 16-bit words of each 64-bit counter (list of ints), Philox4x32-10, in Python integers."""
    out = []
    for c in blocks:
        w = [c & 0xFFFFFFFF, c >> 32 & 0xFFFFFFFF, 0, 0]
        k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
        for _ in range(10):
            a, b = w[0] * 0xD2511F53, w[2] * 0xCD9E8D57
            w = [b >> 32 ^ w[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ w[3] ^ k[1], a & 0xFFFFFFFF]
            k = [k[0] + 0x9E3779B9 & 0xFFFFFFFF, k[1] + 0xBB67AE85 & 0xFFFFFFFF]
        for x in w:
            out += [x & 0xFFFF, x >> 16]
    return out


def kept(n, p, seed, offset):
    """(mask [n], 1 / the probability of being kept) of dropout_counter."""
    t = min(65535, int(np.floor(float(np.float32(p)) * 65536.0 + 0.5)))
    bits = philox_bits([(offset + b) % (1 << 64) for b in range((n + 7) // 8)], seed)[:n]
    return torch.tensor(bits) >= t, 65536.0 / (65536 - t)


def embedding(ids, tok, pos, S, scale):
    """float64 rows and the sum of the magnitudes that an element is made of."""
    V = tok.shape[0]
    ok = (ids >= 0) & (ids < V)
    rows = tok.double()[ids.long().clamp(0, max(V - 1, 0))] * scale
    p = pos.double().repeat(ids.numel() // S, 1) if pos is not None else torch.zeros_like(rows)
    return torch.where(ok[:, None], rows + p, torch.zeros_like(rows)), rows.abs() + p.abs()


def embedding_backward(g, ids, V, S, scale):
    """float64 (grad_tok, grad_pos) and bounds on the errors of fp32 sums in any order: a sum of k terms is off by less than k half steps of
    the sum of the magnitudes."""
    ok = (ids >= 0) & (ids < V)
    gd = torch.where(ok[:, None], g.double(), torch.zeros((), dtype=torch.float64, device=g.device))
    at = torch.where(ok, ids, torch.zeros_like(ids)).long()
    E = g.shape[1]
    tok = torch.zeros(max(V, 1), E, dtype=torch.float64, device=g.device)
    mag, cnt = tok.clone(), torch.zeros(max(V, 1), dtype=torch.float64, device=g.device)
    tok.index_add_(0, at, gd)
    mag.index_add_(0, at, gd.abs())
    cnt.index_add_(0, at, ok.double())
    pos, pmag = gd.view(-1, S, E).sum(0), gd.abs().view(-1, S, E).sum(0)
    h = 2.0 ** -24
    return (tok[:V] * scale, pos), (((cnt[:V, None] + 2) * h * mag[:V]) * abs(scale), (ids.numel() // S + 2) * h * pmag)


class Loss:
    """float64 losses and gradients for x [N][E], w [V][E] (already by token), and bounds."""

    def __init__(self, x, w, targets, g, dtype):
        V = w.shape[0]
        self.dtype, self.valid = dtype, (targets >= 0) & (targets < V)
        zero = torch.zeros((), dtype=torch.float64, device=x.device)
        self.x, self.w = torch.where(self.valid[:, None], x.double(), zero), w.double()
        self.at = torch.where(self.valid, targets, torch.zeros_like(targets)).long()
        E = x.shape[1]
        step = 2.0 ** -23
        products = 1 if dtype == torch.bfloat16 else 3
        cut = 0.0 if dtype == torch.bfloat16 else 2.0 ** -22                 # an fp32 operand as two fp16 numbers, and lo lo left out
        self.tiny = 0.0 if dtype == torch.bfloat16 else 2.0 ** -39           # of the largest of a matrix: where lo is a subnormal
        self.products, self.cut, self.step = products, cut, step
        z = self.x @ self.w.t()
        mag = self.x.abs() @ self.w.abs().t()
        big = E * (self.x.abs().max() * self.w.abs().max() if self.x.numel() else zero)
        # per logit: the operands, and the running sum of ceil(E / 16) instructions (the last stage of 64 is whole)
        self.ez = mag * (2 * cut + (products * (-(-E // 64) * 4) + 4) * step) + 2 * self.tiny * big
        self.lse = torch.where(self.valid, torch.logsumexp(z, 1), zero)
        zt = z.gather(1, self.at[:, None])[:, 0]
        self.loss = torch.where(self.valid, self.lse - zt, zero)
        # sums of exponentials: 128 columns one after the other, then the parts by eight warps; exponentials of arguments that are rounded to 2^-24 of up to
        # their distance from the maximum times log2 e (weighted by themselves that is below 2^-24 * 4), ex2 to 2^-22; the logarithm to 2^-22 of itself
        parts = -(-V // 128)
        self.e_sum = (64 + 16 + parts / 8 + 16 + 8) * 2.0 ** -24 + 2.0 ** -21
        row = self.ez.max(1).values
        self.e_lse = row + self.e_sum + 2.0 ** -22 * (self.lse.abs() + 20)
        self.e_loss = self.e_lse + row + 2.0 ** -22 * self.lse.abs()
        if g is None:
            return
        self.g = torch.where(self.valid, g.double(), zero)
        self.z = z

    def gradients(self, lse):
        """(dx, dW by token) and their bounds, from the lse (fp32) that the call is given."""
        lse = lse.double()
        p = torch.where(self.valid[:, None], torch.exp(self.z - lse[:, None]), torch.zeros((), dtype=torch.float64, device=self.z.device))
        dz = p.clone()
        dz[torch.arange(len(dz), device=dz.device), self.at] -= self.valid.double()
        dz *= self.g[:, None]
        # p is off by what its logit is off, by the rounding of z - lse, by ex2; p - 1 is rounded; then g; then the storage type
        rel = 2 * self.ez + (self.z - lse[:, None]).abs() * 2.0 ** -22 + 2.0 ** -21
        edz = self.g.abs()[:, None] * (p * rel + 2.0 ** -23 * dz.bool())
        edz = edz + (HALF[torch.bfloat16] if self.dtype == torch.bfloat16 else self.cut + 2.0 ** -22) * (dz.abs() + edz)
        edz = edz + self.tiny * self.g.abs().max()
        N, V = dz.shape
        dx, dw = dz @ self.w, dz.t() @ self.x
        wa, xa, da = self.w.abs() + 0.0, self.x.abs(), dz.abs() + edz
        run = lambda k: 2 * self.cut + (self.products * (-(-k // 64) * 4) + 8) * self.step  # noqa: E731
        ex = edz @ wa + (da @ wa) * run(V) + self.tiny * (da.sum(1, keepdim=True) * wa.max())
        ew = edz.t() @ xa + (da.t() @ xa) * run(N) + self.tiny * (da.sum(0)[:, None] * (xa.max() if xa.numel() else 0.0))
        h = HALF[self.dtype]
        return (dx, dw), (ex * (1 + h) + h * dx.abs() + 1e-38, ew * (1 + h) + h * dw.abs() + 1e-38)


def within(got, want, bound, what=""):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert not torch.isnan(got).any(), what
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, f"{what}: {worst} beyond its bound; error {float((got.double() - want).abs().max())}"
