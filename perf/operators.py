"""The operators at the two ends of a training step, as cases that can be timed and compared.

  embed        out[t] = scale tok[id_t] + pos[t mod S]; an id outside the vocabulary gives a row of zeros
  embed_bwd    gradients of both tables from the gradient of the rows
  dropout      [residual +] x / (1 - p) where an element's 16 random bits let it through; the bits come from Philox4x32-10
  loss         softmax cross entropy of x W^T against target ids: the loss and the log of the sum of exponentials per row
  loss_bwd     gradients of x and W from the gradient of the losses; a target outside the vocabulary takes a row out

Types: "f32", "bf16", and for embed_bwd "bf16_f32" (16-bit gradients summed into fp32 tables).  The weights of the loss lie as [V][E] ("ve",
a token embedding used twice) or as [E][V] ("ev", HipGPT's own output projection).  Token ids and targets are distributed as
words are: id k with a share that falls as 1 / k.
"""
from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # the default model's embedding in generation's batch of prompts: latency of one call
        dict(name="embed_small", kind="embed", B=8, S=16, V=5000, E=256, type="f32", pos=True),
        # a long batch of a wide model with 16-bit tables and scaled rows
        dict(name="embed_large", kind="embed", B=16, S=2048, V=50021, E=1024, type="bf16", pos=False),
        # the default model's training step
        dict(name="embed_bwd_train", kind="embed_bwd", B=32, S=256, V=5000, E=256, type="f32", pos=True),
        # the same long batch: 16-bit gradients summed into fp32 tables
        dict(name="embed_bwd_large", kind="embed_bwd", B=16, S=2048, V=50021, E=1024, type="bf16_f32", pos=False),
        # the tail of a sub-layer in the default model's training step
        dict(name="dropout_train", kind="dropout", n=32 * 256 * 256, type="f32", residual=True, p=0.1),
        # activations of a wide feed-forward layer in 16 bits: the forward pass, and the backward pass on a gradient
        dict(name="dropout_large", kind="dropout", n=16 * 2048 * 2048 - 5, type="bf16", residual=False, p=0.2),
        # the loss of a few rows against the default model's vocabulary: latency of one call
        dict(name="loss_small", kind="loss", N=64, E=256, V=5000, type="f32", layout="ev", ignored=0.0),
        # the default model's training step
        dict(name="loss_train", kind="loss", N=8192, E=256, V=5000, type="f32", layout="ev", ignored=0.0),
        # a large vocabulary, tied weights in 16 bits
        dict(name="loss_large", kind="loss", N=8192, E=1024, V=65536, type="bf16", layout="ve", ignored=0.0),
        # the default model's training step
        dict(name="loss_bwd_train", kind="loss_bwd", N=8192, E=256, V=5000, type="f32", layout="ev", ignored=0.0),
        # a padded batch of ragged sizes, a fifth of whose rows take no part
        dict(name="loss_bwd_ragged", kind="loss_bwd", N=1531, E=776, V=20011, type="bf16", layout="ve", ignored=0.2),
        # a large vocabulary, tied weights in 16 bits: the largest call
        dict(name="loss_bwd_large", kind="loss_bwd", N=8192, E=1024, V=65536, type="bf16", layout="ve", ignored=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths: multiples of 64 as models have them, or any."""
    e = _log_int(rng, lo, hi)
    return max(64, e // 64 * 64) if rng.random() < 0.6 else e


def draw(rng):
    kind = rng.choice(["embed", "embed_bwd", "dropout", "loss", "loss_bwd"])
    if kind in ("embed", "embed_bwd"):
        while True:
            case = dict(kind=kind, B=_log_int(rng, 1, 64), S=_log_int(rng, 1, 2048), V=_log_int(rng, 50, 65536), E=_width(rng, 16, 2048),
                        type=rng.choice(["f32", "bf16"] + ["bf16_f32"] * (kind == "embed_bwd")), pos=rng.random() < 0.5)
            if case["B"] * case["S"] * case["E"] <= 1 << 25 and case["V"] * case["E"] <= 1 << 26:
                return case
    if kind == "dropout":
        return dict(kind=kind, n=_log_int(rng, 1000, 1 << 26), type=rng.choice(["f32", "bf16"]), residual=rng.random() < 0.5, p=round(rng.uniform(0.02, 0.6), 3))
    while True:
        case = dict(kind=kind, N=_log_int(rng, 16, 8192), E=_width(rng, 48, 2048), V=_log_int(rng, 200, 65536), type=rng.choice(["f32", "bf16"]),
                    layout=rng.choice(["ev", "ve"]), ignored=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.7), 2)]))
        # fp32 operands take three products on the tensor pipe
        if case["N"] * case["E"] * case["V"] * (3 if case["type"] == "f32" else 1) <= 8192 * 1024 * 65536:
            return case


def _dtype(case):
    return torch.float32 if case["type"] == "f32" else torch.bfloat16


def _words(n, V, gen):
    """Ids whose shares fall as 1 / rank."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return ((V + 1.0) ** u).long().sub_(1).clamp_(0, V - 1).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, t = case["kind"], _dtype(case)

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = dict(case)
    if kind in ("embed", "embed_bwd"):
        B, S, V, E = (case[k] for k in "BSVE")
        s["ids"] = _words(B * S, V, gen)
        s["scale"] = math.sqrt(E)
        gt = torch.float32 if case["type"] == "bf16_f32" else t
        if kind == "embed":
            s["tok"], s["table"] = normal(V, E, scale=0.02), (normal(S, E, scale=0.02) if case["pos"] else None)
            s["out"] = torch.empty(B * S, E, device="cuda", dtype=t)
        else:
            s["grad"] = normal(B * S, E, scale=1e-3)
            s["grad_tok"] = torch.empty(V, E, device="cuda", dtype=gt)
            s["grad_pos"] = torch.empty(S, E, device="cuda", dtype=gt) if case["pos"] else None
    elif kind == "dropout":
        s["x"] = normal(case["n"])
        s["res"] = normal(case["n"]) if case["residual"] else None
        s["out"] = torch.empty_like(s["x"])
        s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ (seed * 2654435761), (seed % 1000) << 30
    else:
        N, E, V = (case[k] for k in "NEV")
        targets = _words(N, V, gen)
        # logits with a spread of about 1.5, that of the target above the others: a model in the middle of its training
        w = torch.randn(V, E, generator=gen, device="cuda").mul_(1.5 / math.sqrt(E))
        x = torch.randn(N, E, generator=gen, device="cuda").add_(w[targets.long()], alpha=2.0)
        if case["ignored"]:
            targets = torch.where(torch.rand(N, generator=gen, device="cuda") < case["ignored"], torch.full_like(targets, -1), targets)
        s["targets"] = targets
        s["x"] = x.to(t)
        s["w"] = (w.t() if case["layout"] == "ev" else w).to(t).contiguous()
        if kind == "loss":
            s["loss"], s["lse"] = torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
        else:
            wk = s["w"].float() if case["layout"] == "ve" else s["w"].float().t()
            lse = torch.empty(N, device="cuda")
            for a in range(0, N, 2048):
                lse[a:a + 2048] = torch.logsumexp(s["x"][a:a + 2048].float() @ wk.t(), 1)
            valid = targets >= 0
            s["lse"] = torch.where(valid, lse, torch.zeros_like(lse))
            # the mean over the rows that take part
            s["grad_loss"] = torch.where(valid, 1.0 / valid.sum().clamp(min=1), 0.0).float()
            s["grad_x"], s["grad_w"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
    return s


def _philox_bits(blocks, seed):
    """The eight 16-bit words of each counter, as integers [blocks][8]: Philox4x32-10 (Salmon et al., 2011), two halves of each output word, the low one first."""
    low = 0xFFFFFFFF
    c0, c1 = blocks & low, (blocks >> 32) & low
    c2 = c3 = torch.zeros_like(blocks)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57             # (64 bits hold the product; the sign bit is cut off with the mask)
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1, 8)


def _threshold(p):
    return min(65535, int(math.floor(p * 65536.0 + 0.5)))


def _run_own(s):
    from hipgpt_b200 import training

    kind = s["kind"]
    if kind == "embed":
        training.embedding_scaled(s["ids"], s["tok"], s["table"], s["out"], s["B"], s["S"], s["V"], s["E"], scale=s["scale"])
        return s["out"]
    if kind == "embed_bwd":
        training.embedding_backward(s["grad"], s["ids"], s["grad_tok"], s["grad_pos"], s["B"], s["S"], s["V"], s["E"], scale=s["scale"])
        return [s["grad_tok"], s["grad_pos"]]
    if kind == "dropout":
        training.dropout_counter(s["x"], s["res"], s["out"], s["p"], seed=s["seed"], offset=s["offset"])
        return s["out"]
    by_token = s["layout"] == "ve"
    if kind == "loss":
        training.linear_cross_entropy(s["x"], s["w"], s["targets"], s["loss"], s["lse"], s["N"], s["E"], s["V"], by_token=by_token)
        return [s["loss"], s["lse"]]
    training.linear_cross_entropy_backward(s["x"], s["w"], s["targets"], s["lse"], s["grad_loss"], s["grad_x"], s["grad_w"], s["N"], s["E"], s["V"], by_token=by_token)
    return [s["grad_x"], s["grad_w"]]


def run(s):
    if own:
        return _run_own(s)
    kind, t = s["kind"], _dtype(s)
    if kind == "embed":
        V, S = s["V"], s["S"]
        ids = s["ids"].long()
        valid = ((ids >= 0) & (ids < V))[:, None]
        rows = s["tok"][ids.clamp(0, V - 1)].float() * s["scale"]
        if s["table"] is not None:
            rows = rows + s["table"].float().repeat(s["B"], 1)
        return torch.where(valid, rows, torch.zeros_like(rows)).to(t)
    if kind == "embed_bwd":
        V, S, E = s["V"], s["S"], s["E"]
        ids = s["ids"].long()
        valid = (ids >= 0) & (ids < V)
        g = torch.where(valid[:, None], s["grad"].float(), torch.zeros((), device="cuda"))
        tok = torch.zeros(V, E, device="cuda").index_add_(0, torch.where(valid, ids, torch.zeros_like(ids)), g)
        return [(tok * s["scale"]).to(s["grad_tok"].dtype), None if s["grad_pos"] is None else g.view(-1, S, E).sum(0).to(s["grad_pos"].dtype)]
    if kind == "dropout":
        n, thr = s["n"], _threshold(s["p"])
        bits = _philox_bits(torch.arange((n + 7) // 8, device="cuda") + s["offset"], s["seed"]).reshape(-1)[:n]
        y = torch.where(bits >= thr, s["x"].float() * (65536.0 / (65536 - thr)), torch.zeros((), device="cuda"))
        return (y if s["res"] is None else y + s["res"].float()).to(t)
    valid = ((s["targets"] >= 0) & (s["targets"] < s["V"]))[:, None]
    at = torch.where(valid, s["targets"].long()[:, None], torch.zeros((), device="cuda", dtype=torch.long))
    zero = torch.zeros((), device="cuda")
    x = torch.where(valid, s["x"].float(), zero)
    w = s["w"].float() if s["layout"] == "ev" else s["w"].float().t()
    z = x @ w
    if kind == "loss":
        m = z.amax(1, keepdim=True)
        lse = m + torch.exp(z - m).sum(1, keepdim=True).log()
        return [torch.where(valid, lse - z.gather(1, at), zero)[:, 0], torch.where(valid, lse, zero)[:, 0]]
    dz = torch.exp(z - s["lse"][:, None])
    dz = dz.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32)) * torch.where(valid, s["grad_loss"][:, None], zero)
    dw = x.t() @ dz if s["layout"] == "ev" else dz.t() @ x
    return [(dz @ w.t()).to(t), dw.to(t)]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "dropout":
        keep = _keep(case["n"], s["seed"], s["offset"], _threshold(case["p"]))
        y = s["x"].double().masked_fill_(~keep, 0.0).mul_(65536.0 / (65536 - _threshold(case["p"])))
        return y if s["res"] is None else y.add_(s["res"].double())
    if kind == "embed":
        out = torch.nn.functional.embedding(s["ids"].long(), s["tok"].double()).mul_(s["scale"]).view(case["B"], case["S"], case["E"])
        return (out if s["table"] is None else out.add_(s["table"].double())).view(-1, case["E"])
    if kind == "embed_bwd":
        order = torch.argsort(s["ids"].long(), stable=True)
        ids, counts = torch.unique_consecutive(s["ids"].long()[order], return_counts=True)
        sums = torch.segment_reduce(s["grad"].double()[order], "sum", lengths=counts)
        tok = torch.zeros(case["V"], case["E"], device="cuda", dtype=torch.float64)
        tok[ids] = sums * s["scale"]
        return [tok, None if s["grad_pos"] is None else s["grad"].double().view(case["B"], case["S"], -1).sum(0)]
    N, V = case["N"], case["V"]
    x, t = s["x"].double(), s["targets"].long()
    w = s["w"].double() if case["layout"] == "ve" else s["w"].double().t().contiguous()
    loss, lse = torch.zeros(N, device="cuda", dtype=torch.float64), torch.zeros(N, device="cuda", dtype=torch.float64)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for rows in ((t >= 0) & (t < V)).nonzero()[:, 0].split(1024):
        z = torch.einsum("ne,ve->nv", x[rows], w)
        if kind == "loss":
            lse[rows] = torch.logsumexp(z, 1)
            loss[rows] = torch.nn.functional.cross_entropy(z, t[rows], reduction="none")
            continue
        d = z.sub_(s["lse"].double()[rows, None]).exp_()
        d[torch.arange(len(rows), device="cuda"), t[rows]] -= 1
        d *= s["grad_loss"].double()[rows, None]
        dx[rows] = torch.einsum("nv,ve->ne", d, w)
        dw += torch.einsum("nv,ne->ve", d, x[rows])
    if kind == "loss":
        return [loss, lse]
    return [dx, dw if case["layout"] == "ve" else dw.t().contiguous()]


def _keep(n, seed, offset, thr):
    """The elements that dropout lets through, by 32-bit words kept in halves of 16 bits (no product passes 2^34)."""
    import numpy as np

    blocks = np.arange(offset, offset + (n + 7) // 8, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)

    def product(a, m):
        x, y = a * np.uint64(m & 0xFFFF), a * np.uint64(m >> 16)
        lo = x + ((y & np.uint64(0xFFFF)) << np.uint64(16))
        return ((y >> np.uint64(16)) + (lo >> np.uint64(32))) & low, lo & low

    c = [blocks & low, blocks >> np.uint64(32), np.zeros_like(blocks), np.zeros_like(blocks)]
    k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        (h0, l0), (h1, l1) = product(c[0], 0xD2511F53), product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ np.uint64(k[0]), l1, h0 ^ c[3] ^ np.uint64(k[1]), l0]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    keep = np.empty((len(blocks), 8), dtype=bool)
    for j in range(4):
        keep[:, 2 * j] = (c[j] & np.uint64(0xFFFF)) >= thr
        keep[:, 2 * j + 1] = (c[j] >> np.uint64(16)) >= thr
    return torch.from_numpy(keep.reshape(-1)[:n]).cuda()


def _distinct(n, V):
    """How many different ids n words have, on the average."""
    k = torch.arange(1, V + 1, dtype=torch.float64)
    share = torch.log((k + 1) / k) / math.log(V + 1)
    return float((1 - (1 - share) ** n).sum())


def work(case):
    es = 4 if case["type"] == "f32" else 2
    kind = case["kind"]
    if kind == "dropout":
        return {"bytes": case["n"] * es * (3 if case["residual"] else 2), "flops": 2.0 * case["n"]}
    if kind in ("embed", "embed_bwd"):
        n, E = case["B"] * case["S"], case["E"]
        pos = case["S"] * E if case["pos"] else 0
        if kind == "embed":
            return {"bytes": 4 * n + es * (n * E + _distinct(n, case["V"]) * E + pos), "flops": 2.0 * n * E}
        gs = 2 if case["type"] == "bf16" else 4
        return {"bytes": 4 * n + es * n * E + gs * (case["V"] * E + pos), "flops": (2.0 if case["pos"] else 1.0) * n * E}
    n, E, V = case["N"] * (1 - case["ignored"]), case["E"], case["V"]
    if kind == "loss":
        return {"bytes": es * (n + V) * E + 12 * case["N"], "flops": 2.0 * n * E * V}
    return {"bytes": 2 * es * (n + V) * E + 12 * case["N"], "flops": 6.0 * n * E * V}
