"""The operators of serving a ragged batch from a cache in pages, as cases that can be timed and compared.

  rotary       y = m R(position) x on a part of each head, its pairs interleaved or in halves; backward: the inverse rotation
  cache        new rows of K and V are written to the pages of their sequences, in the cache's format, and read back
  attend       attention of each sequence's new tokens, the last of its length, over the pages of its keys and values

A cache's format: "plain" (values of the activations' type), "e4m3" (the smallest power of two as scale that brings a row of a head to at
most 448) or "int8" (scale max / 127, codes to the nearest, ties to even); one fp32 scale per token and head.  A batch: offsets [B + 1] of the
sequences' new tokens, lengths [B] with them, page numbers [B][most pages].  Pages are dealt to the sequences in no order.
"""
from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # queries and keys of the default model's heads, one token of each sequence of generation's batch: latency of one call
        dict(name="rotary_token", kind="rotary", T=8, H=16, D=32, R=32, type="f32", interleaved=False, backward=False, far=256, factor=1.0),
        # a long prompt's queries and keys in 16 bits, frequencies slowed down for far positions
        dict(name="rotary_long", kind="rotary", T=32768, H=40, D=128, R=128, type="bf16", interleaved=False, backward=False, far=1000000, factor=8.0),
        # the gradient of a training batch, half of each head turned, neighbours as pairs
        dict(name="rotary_train", kind="rotary", T=16 * 2048, H=16, D=64, R=32, type="f32", interleaved=True, backward=True, far=2048, factor=1.0),
        # one token of each sequence of a batch in generation: latency of the two calls
        dict(name="cache_token", kind="cache", B=64, n=1, ctx=8192, heads=8, D=128, page=64, type="bf16", format="e4m3"),
        # ragged prompts of a wide model
        dict(name="cache_prompts", kind="cache", B=12, n=4096, ctx=6000, heads=8, D=128, page=128, type="bf16", format="int8"),
        # the default model's prompts, and a head width between the powers of two
        dict(name="cache_odd", kind="cache", B=37, n=256, ctx=777, heads=8, D=48, page=16, type="f32", format="e4m3"),
        # the default model's generation: eight sequences, one token each: latency of one call
        dict(name="attend_token", kind="attend", B=8, n=1, ctx=77, H=8, heads=8, D=32, page=16, type="f32", format="plain"),
        # generation with long contexts from a cache of 8 bits, four query heads a head of it
        dict(name="attend_token_long", kind="attend", B=32, n=1, ctx=32768, H=32, heads=8, D=128, page=64, type="bf16", format="e4m3"),
        # generation of many sequences, a head of the cache for each query head
        dict(name="attend_token_many", kind="attend", B=100, n=1, ctx=2048, H=16, heads=16, D=64, page=32, type="bf16", format="plain"),
        # the default model's prompts in fp32, ragged, behind what is cached already
        dict(name="attend_prompts", kind="attend", B=32, n=256, ctx=512, H=8, heads=8, D=32, page=16, type="f32", format="plain"),
        # pieces of ragged prompts in 16 bits
        dict(name="attend_chunk", kind="attend", B=5, n=1100, ctx=8000, H=32, heads=8, D=128, page=64, type="bf16", format="plain"),
        # a long prompt's last piece over a cache of 8 bits: the largest call
        dict(name="attend_chunk_long", kind="attend", B=1, n=4096, ctx=32768, H=32, heads=8, D=128, page=128, type="bf16", format="int8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _seconds(case):
    """A rough floor, to bound what a drawn case costs: fp32 operands take several products on the tensor pipe."""
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] * (6 if case["type"] == "f32" else 1) / 1.5e15


def draw(rng):
    kind = rng.choice(["rotary", "cache", "attend", "attend"])
    if kind == "rotary":
        while True:
            D = rng.choice([32, 48, 64, 80, 128])
            case = dict(kind=kind, T=_log_int(rng, 1, 32768), H=_log_int(rng, 1, 48), D=D, R=rng.choice([D, D, D // 2, D // 4]), type=rng.choice(["f32", "bf16"]),
                        interleaved=rng.random() < 0.5, backward=rng.random() < 0.4, far=_log_int(rng, 100, 1000000), factor=rng.choice([1.0, 4.0, 8.0]))
            if case["T"] * case["H"] * case["D"] <= 32768 * 40 * 128:
                return case
    while True:
        D, heads, group, page = rng.choice([32, 48, 64, 80, 128]), rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 64, 128])
        ctx = _log_int(rng, 16, 32768)
        n = 1 if rng.random() < 0.5 else min(ctx, _log_int(rng, 2, 4096))
        case = dict(kind=kind, B=_log_int(rng, 1, 128), n=n, ctx=ctx, heads=heads, D=D, page=page, type=rng.choice(["f32", "bf16"]), format=rng.choice(["plain", "e4m3", "int8"]))
        if kind == "attend":
            case["H"] = heads * group
        largest = listed()[4 if kind == "cache" else 11]
        if case["B"] * ctx * heads * D <= 1 << 30 and _seconds(case) <= _seconds(largest):
            return case


def _dtype(case):
    return torch.float32 if case["type"] == "f32" else torch.bfloat16


def _batch(case):
    """(new tokens, length with them) of each sequence: spread over the upper three quarters of the range, the first at its end."""
    out = []
    for b in range(case["B"]):
        part = 1.0 if b == 0 else 0.25 + 0.75 * (b * 0.6180339887498949 % 1.0)
        n = max(1, round(case["n"] * part))
        out.append((n, max(n, round(case["ctx"] * part))))
    return out


def _frequencies(R, factor, base=10000.0, original=4096, low=1.0, high=4.0):
    """Radians per position, float64: where a turn is longer than original / low positions, slowed down by the factor; shorter than original / high: as it
    is; a straight line in between."""
    f = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if factor == 1.0:
        return f
    keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
    return f * (keep + (1 - keep) / factor)


def _quantise(x, fmt):
    """(codes, scales) of the rows of x, fp32: whole codes by quotients in 64 bits."""
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        scale = (amax / 127.0).clamp(min=2.0 ** -126)
        return torch.round(x.double() / scale.double()).to(torch.int8), scale[..., 0]
    _, e = torch.frexp(amax / 448.0)
    s = torch.ldexp(torch.ones_like(amax), e - 1)
    s = torch.where(amax > s * 448.0, s * 2.0, s)                      # (a power of two itself has the exponent above its own)
    s = torch.where(amax > 0, s, torch.ones_like(s)).clamp(min=2.0 ** -126)
    return (x / s).to(torch.float8_e4m3fn), s[..., 0]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = _dtype(case)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(t)

    s = dict(case)
    if case["kind"] == "rotary":
        T, H, D, R = (case[k] for k in "THDR")
        s["x"], s["out"] = normal(T, H, D), torch.empty(T, H, D, device="cuda", dtype=t)
        first = torch.randint(0, max(1, case["far"] - T), (1,), generator=gen, device="cuda", dtype=torch.int32)
        s["positions"] = first + torch.arange(T, device="cuda", dtype=torch.int32) % case["far"]
        s["magnitude"] = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
        s["freq"] = _frequencies(R, case["factor"])
        if own:
            from hipgpt_b200 import serving
            s["words"] = serving.rotary_words(s["freq"])
        return s
    heads, D, page = case["heads"], case["D"], case["page"]
    s["batch"] = _batch(case)
    counts = [n for n, _ in s["batch"]]
    lens = [length for _, length in s["batch"]]
    held = [-(-length // page) for length in lens]
    s["T"], s["num_pages"] = sum(counts), sum(held) + 3
    s["offsets"] = torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    deal = torch.randperm(s["num_pages"], generator=gen, device="cuda").int()
    s["pages"] = torch.zeros(len(lens), max(held), dtype=torch.int32, device="cuda")
    for b, h in enumerate(held):
        s["pages"][b, :h] = deal[sum(held[:b]):sum(held[:b]) + h]
    # keys have a few wide channels, as those of trained models do
    gain = torch.ones(heads, 1, D, device="cuda")
    gain[:, :, torch.randperm(D, generator=gen, device="cuda")[:max(1, D // 32)]] = 4.0
    shape = (s["num_pages"], heads, page, D)
    if case["kind"] == "cache":
        s["k"] = (torch.randn(s["T"], heads, D, generator=gen, device="cuda") * gain[:, 0]).to(t)
        s["v"] = normal(s["T"], heads, D)
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        codes = {"plain": t, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[case["format"]]
        s["k_cache"], s["v_cache"] = torch.zeros(shape, device="cuda", dtype=codes), torch.zeros(shape, device="cuda", dtype=codes)
        s["k_scale"], s["v_scale"] = torch.zeros(shape[:3], device="cuda"), torch.zeros(shape[:3], device="cuda")
    else:
        for name, wide in (("k", gain), ("v", torch.ones_like(gain))):
            if case["format"] == "plain":
                s[name + "_cache"], s[name + "_scale"] = (torch.randn(shape, generator=gen, device="cuda") * wide).to(t), None
            else:
                parts = [_quantise((torch.randn(p, *shape[1:], generator=gen, device="cuda") * wide).to(t).float(), case["format"]) for p in _pieces(shape)]
                s[name + "_cache"], s[name + "_scale"] = torch.cat([c for c, _ in parts]), torch.cat([z for _, z in parts]).contiguous()
        s["q"] = normal(s["T"], case["H"], D)
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["cache"] = _handle(s)
    return s


def _pieces(shape):
    """Pages at a time, so that what a step holds in 64 bits stays below a gigabyte."""
    per = max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))
    return [min(per, shape[0] - a) for a in range(0, shape[0], per)]


def _handle(s):
    from hipgpt_b200 import serving

    plain = s["format"] == "plain"
    return serving.PagedCache(s["num_pages"], s["page"], s["heads"], s["D"], dtype=_dtype(s), format=s["format"], k=s["k_cache"], v=s["v_cache"],
                              k_scale=None if plain else s["k_scale"], v_scale=None if plain else s["v_scale"])


def _run_own(s):
    from hipgpt_b200 import serving

    if s["kind"] == "rotary":
        serving.rotary(s["x"], s["positions"], s["words"], s["out"], s["T"], s["H"], s["D"], s["R"], interleaved=s["interleaved"], magnitude=s["magnitude"], inverse=s["backward"])
        return s["out"]
    batch = s["offsets"], s["lengths"], s["pages"], s["T"], s["B"]
    if s["kind"] == "cache":
        serving.cache_write(s["cache"], s["k"], s["v"], *batch)
        serving.cache_read(s["cache"], s["k_out"], s["v_out"], *batch)
        return [s["k_out"], s["v_out"]]
    serving.paged_attention(s["cache"], s["q"], s["out"], *batch, s["H"])
    return s["out"]


def _places(s):
    """(page, slot) of each new token."""
    pages, slots = [], []
    for b, (n, length) in enumerate(s["batch"]):
        at = torch.arange(length - n, length, device="cuda")
        pages.append(s["pages"][b].long()[at // s["page"]])
        slots.append(at % s["page"])
    return torch.cat(pages), torch.cat(slots)


def run(s):
    if own:
        return _run_own(s)
    t = _dtype(s)
    if s["kind"] == "rotary":
        R, x = s["R"], s["x"].float()
        angle = s["positions"].double()[:, None] * s["freq"].cuda()        # far positions lose theirs in 32 bits
        c, sn = (torch.cos(angle) * s["magnitude"]).float()[:, None], (torch.sin(angle) * s["magnitude"]).float()[:, None]
        if s["backward"]:
            sn = -sn
        a, b = (x[..., 0:R:2], x[..., 1:R:2]) if s["interleaved"] else (x[..., :R // 2], x[..., R // 2:R])
        y = torch.stack([a * c - b * sn, a * sn + b * c], -1 if s["interleaved"] else -2).flatten(-2)
        return torch.cat([y, x[..., R:]], -1).to(t)
    if s["kind"] == "cache":
        page, slot = _places(s)
        out = []
        for name in "kv":
            x, cache = s[name], s[name + "_cache"]
            if s["format"] == "plain":
                cache[page, :, slot] = x
                out.append(cache[page, :, slot])
                continue
            codes, scale = _quantise(x.float(), s["format"])
            cache.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
            s[name + "_scale"][page, :, slot] = scale
            back = cache.view(torch.uint8)[page, :, slot].view(cache.dtype)
            out.append((back.float() * s[name + "_scale"][page, :, slot][..., None]).to(t))
        return out
    H, heads, D = s["H"], s["heads"], s["D"]
    out, first = torch.empty_like(s["q"]), 0
    for b, (n, length) in enumerate(s["batch"]):
        at = s["pages"][b, :-(-length // s["page"])].long()
        q = s["q"][first:first + n].float().view(n, heads, H // heads, D)
        seen = torch.arange(length, device="cuda")[None] <= torch.arange(length - n, length, device="cuda")[:, None]
        hidden = torch.zeros(n, 1, length, device="cuda").masked_fill_(~seen[:, None], float("-inf"))
        step = max(1, min(heads, (1 << 29) // (n * (H // heads) * length)))          # heads at a time: at most 2 GB of scores
        for h in range(0, heads, step):
            k, v = (_rows(s, name, at, slice(h, min(heads, h + step)))[:, :length] for name in "kv")
            z = q[:, h:h + step].transpose(0, 1).reshape(len(k), -1, D) @ k.transpose(1, 2)
            z = z.view(len(k), n, -1, length) * (1.0 / math.sqrt(D)) + hidden
            p = torch.exp(z - z.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = (p.view(len(k), -1, length) @ v).view(len(k), n, -1, D)
            out[first:first + n].view(n, heads, -1, D)[:, h:h + step] = o.transpose(0, 1).to(t)
        first += n
    return out


def _rows(s, name, at, some):
    """The rows of a sequence's pages as the values that they stand for, for some heads: [heads][tokens][D]."""
    x = s[name + "_cache"][:, some]
    x = x[at] if s["format"] != "e4m3" else x.view(torch.uint8)[at].view(x.dtype)
    x = x.float()
    if s["format"] != "plain":
        x = x * s[name + "_scale"][:, some][at][..., None]
    return x.transpose(0, 1).reshape(x.shape[1], -1, s["D"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        R, x = case["R"], s["x"].double()
        turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["freq"].cuda())[:, None]
        if case["backward"]:
            turn = turn.conj()
        pairs = x[..., :R].unflatten(-1, (R // 2, 2) if case["interleaved"] else (2, R // 2))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        x[..., :R] = (y if case["interleaved"] else y.transpose(-1, -2)).flatten(-2)
        return x
    if case["kind"] == "cache":
        out = []
        for x in (s["k"].double(), s["v"].double()):
            most = x.abs().amax(-1, keepdim=True)
            if case["format"] == "int8":
                unit = (most / 127.0).float().double()
                x = torch.round(x / unit.clamp(min=2.0 ** -126)) * unit
            elif case["format"] == "e4m3":
                unit = torch.exp2(torch.ceil(torch.log2((most / 448.0).clamp(min=2.0 ** -126))))
                y = x / unit
                # four significant bits down to 2^-6, steps of 2^-9 below
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                x = torch.round(y / step) * step * unit
            out.append(x)
        return out
    H, heads, D, page = case["H"], case["heads"], case["D"], case["page"]
    if work(case)["flops"] > 4e12:
        return None
    out, first = torch.empty(s["T"], H, D, dtype=torch.float64, device="cuda"), 0
    for b, (n, length) in enumerate(_batch(case)):
        token = torch.arange(length, device="cuda")
        at, slot = s["pages"][b].long()[token // page], token % page
        for h in range(heads):
            k, v = (_exact_rows(s[name + "_cache"], s[name + "_scale"], at, slot, h) for name in "kv")
            mine = slice(h * (H // heads), (h + 1) * (H // heads))
            step = max(1, (1 << 26) // (length * (H // heads)))
            for a in range(0, n, step):
                rows = torch.arange(a, min(n, a + step), device="cuda")
                z = torch.einsum("ngd,kd->ngk", s["q"][first + rows][:, mine].double(), k) / math.sqrt(D)
                z.masked_fill_((token[None] > (length - n + rows)[:, None])[:, None], float("-inf"))
                out[first + rows, mine] = torch.einsum("ngk,kd->ngd", torch.softmax(z, -1), v)
        first += n
    return out


def _exact_rows(cache, scale, at, slot, h):
    raw = cache[:, h].view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache[:, h]
    rows = raw[at, slot].contiguous()
    rows = rows.view(cache.dtype).double() if cache.dtype == torch.float8_e4m3fn else rows.double()
    return rows if scale is None else rows * scale[:, h][at, slot].double()[:, None]


def work(case):
    es = 4 if case["type"] == "f32" else 2
    if case["kind"] == "rotary":
        n = case["T"] * case["H"]
        return {"bytes": 2 * n * case["D"] * es + 4 * case["T"] + 4 * case["R"], "flops": 3.0 * n * case["R"]}
    heads, D = case["heads"], case["D"]
    row = D * es if case["format"] == "plain" else D + 4                 # a row of a head in the cache
    batch = _batch(case)
    T = sum(n for n, _ in batch)
    if case["kind"] == "cache":
        return {"bytes": 4 * T * heads * (D * es + row), "flops": 6.0 * T * heads * D}
    seen = sum(n * length - n * (n - 1) // 2 for n, length in batch)
    return {"bytes": 2 * T * case["H"] * D * es + 2 * heads * row * sum(length for _, length in batch), "flops": 4.0 * D * case["H"] * seen}
