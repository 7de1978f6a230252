"""Operators of a vision-language request's path, as cases that can be timed: the norms around a sub-layer, rotary positions with
several axes, pages of the key-value cache on the move, log probabilities from logits and straight from hidden rows.

Each case is one call. Where ``own`` is false it is computed in its plain form, in elementary torch operations; where it is true
the framework's kernels are called. Sizes come from the presets and tests of this repository or are generic.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 16                       # tokens of a page of the key-value cache
EPS = 1e-6
NEG = float("-inf")
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(rows, dim, dtype="bf16", post=True, layer=False, gate=False, scale=1.0, w_bias=0.0):
    return dict(op="norm", rows=rows, dim=dim, dtype=dtype, post=post, layer=layer, gate=gate, scale=scale, w_bias=w_bias)


def _mrope(tokens, hq, hkv, dim=128, rot=128, layout="chunks", norm=False, kv=16, pads=0, far=0):
    return dict(op="mrope", tokens=tokens, hq=hq, hkv=hkv, dim=dim, rot=rot, layout=layout, norm=norm, kv=kv, pads=pads, far=far)


def _axial(rows, heads, dim):
    return dict(op="axial", rows=rows, heads=heads, dim=dim)


def _pages(job, moved, pool, layers, hkv, dim=128, kv=16):
    return dict(op="pages", job=job, moved=moved, pool=pool, layers=layers, hkv=hkv, dim=dim, kv=kv)


def _scores(rows, vocab, dtype="fp32", top=0, masked=0.0, empty=0):
    return dict(op="scores", rows=rows, vocab=vocab, dtype=dtype, top=top, masked=masked, empty=empty)


def _head(rows, width, vocab, softcap=0.0, scale=1.0, bias=False):
    return dict(op="head", rows=rows, width=width, vocab=vocab, softcap=softcap, scale=scale, bias=bias)


def listed():
    cases = {
        # One decode row of a model with norms before and after each sub-layer: the launch is all there is.
        "norm one row": _norm(1, 2560, w_bias=1.0),
        # The engine's largest step (8192 prompt tokens) of such a model at the widest preset's hidden size.
        "norm 8192 rows": _norm(8192, 5120),
        # A vision tower's block with a per-channel branch scale and layer norms: 37 x 37 patches and a class token, fp32.
        "norm tower fp32": _norm(1370, 1024, dtype="fp32", post=False, layer=True, gate=True),
        # A prompt of 8191 tokens, most of them of images, far into a long document: per-head q/k norms, interleaved sections.
        "mrope 8191 tokens": _mrope(8191, 64, 8, layout="interleaved", norm=True, far=120000),
        # An ordinary prompt with one image; half of each head turns, in pairs of neighbours.
        "mrope 1031 tokens": _mrope(1031, 32, 2, rot=64, layout="pairs", pads=9),
        # A step with a small image over a cache of 8-bit values.
        "mrope 203 tokens 8-bit": _mrope(203, 28, 4, kv=8),
        # A vision tower over a few images: 16 heads of 80.
        "axial 5476 patches": _axial(5476, 16, 80),
        # Copy on write of three pages in all layers of the 8 billion preset.
        "pages copy 3": _pages("copy", 3, 48, 32, 8),
        # A prompt of 4800 tokens leaves for the host tier of the prompt cache.
        "pages gather 301": _pages("gather", 301, 512, 32, 8),
        # A token's log probability with the 20 most likely ones, as an answer with log probabilities asks for at every step.
        "scores one row top 20": _scores(1, 151936, top=20),
        # A batch of rows under structured output: most tokens are masked, one row has nothing left.
        "scores 509 rows top 5": _scores(509, 128256, dtype="bf16", top=5, masked=0.7, empty=1),
        # Perplexity: a window of 2048 tokens is scored at the 8 billion preset's width and vocabulary.
        "head 2047 rows": _head(2047, 4096, 128256),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def draw(rng):
    def log(lo, hi):
        return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))

    kind = rng.choice(["norm", "norm", "mrope", "mrope", "axial", "pages", "pages", "scores", "scores", "head", "head"])
    if kind == "norm":
        layer = rng.random() < 0.3
        return _norm(log(1, 8192), log(64, 5120), dtype=rng.choice(["bf16", "bf16", "fp32"]) if layer else "bf16", post=not layer,
                     layer=layer, gate=layer and rng.random() < 0.7, scale=rng.choice([1.0, 1.0, 0.22]), w_bias=rng.choice([0.0, 1.0]))
    if kind == "mrope":
        hkv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 128, 128])
        layout = rng.choice(["chunks", "interleaved", "pairs"])
        return _mrope(log(1, 8191), hkv * rng.choice([1, 4, 7, 8]), hkv, dim, dim // 2 if layout == "pairs" else dim, layout,
                      rng.random() < 0.4, rng.choice([16, 16, 8]) if dim % 64 == 0 else 16, rng.choice([0, 0, 5]), rng.choice([0, 1000, 120000]))
    if kind == "axial":
        return _axial(log(4, 5476), rng.choice([12, 16]), rng.choice([64, 72, 80]))
    if kind == "pages":
        moved = log(1, 301)
        return _pages(rng.choice(["copy", "copy", "gather", "scatter"]), moved, 2 * moved + rng.randint(1, 40), log(2, 32), rng.choice([1, 2, 8]),
                      rng.choice([64, 128]), rng.choice([16, 16, 8]))
    if kind == "scores":
        return _scores(log(1, 512), log(1000, 151936), rng.choice(["fp32", "bf16"]), rng.choice([0, 1, 5, 20, 50]), rng.choice([0.0, 0.0, 0.9]),
                       rng.choice([0, 0, 1]))
    return _head(log(1, 2047), 8 * log(16, 512), log(500, 128256), rng.choice([0.0, 0.0, 30.0]), rng.choice([1.0, 0.125]), rng.random() < 0.3)


# ----------------------------------------------------------------------------- inputs
def _axes(case):
    """(frequencies of the half, the axis each turns with): sections in proportion 2 : 3 : 3, in chunks or taking turns."""
    half = case["rot"] // 2
    i = torch.arange(half)
    t, h = half // 4, (half - half // 4) // 2
    if case["layout"] == "interleaved":
        axis = torch.where((i % 3 == 1) & (i < 3 * h), 1, torch.where((i % 3 == 2) & (i < 3 * h), 2, 0))
    else:
        axis = (i >= t).int() + (i >= t + h).int()
    theta = 1e6 if case["far"] else 1e4
    return (1.0 / theta ** (2.0 * i.double() / case["rot"])).float(), axis.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def rn(*shape, scale=1.0, dtype=torch.bfloat16, shift=0.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale + shift).to(dtype)

    s = dict(case=case)
    if case["op"] == "norm":
        t, n, d = TYPES[case["dtype"]], case["rows"], case["dim"]
        s.update(x=rn(n, d, scale=3.0, dtype=t), res=rn(n, d, scale=8.0, dtype=t), pre_w=rn(d, scale=0.3, shift=1.0 - case["w_bias"], dtype=t))
        s["post_w"] = rn(d, scale=0.3, shift=1.0 - case["w_bias"], dtype=t) if case["post"] else None
        s["gate"] = rn(d, scale=0.2, shift=0.3, dtype=t) if case["gate"] else None
        s["pre_b"] = rn(d, scale=0.2, dtype=t) if case["layer"] else None
    elif case["op"] == "mrope":
        T, hq, hkv, D, kv = case["tokens"], case["hq"], case["hkv"], case["dim"], case["kv"]
        pages = (T + BLOCK - 1) // BLOCK + 7
        s["qkv"] = rn(T, (hq + 2 * hkv) * D)
        pos = case["far"] + torch.arange(T, device=dev)
        grid = torch.randint(0, 96, (2, T), generator=g, device=dev)
        image = torch.rand(T, generator=g, device=dev) < 0.8         # rows of images share a time and differ in row and column
        s["pos"] = torch.stack([torch.where(image, pos - pos % 64, pos), torch.where(image, pos - pos % 64 + grid[0], pos),
                                torch.where(image, pos - pos % 64 + grid[1], pos)]).int()
        table = torch.randperm(pages, generator=g, device=dev)
        at = torch.arange(T, device=dev)
        slots = table[at // BLOCK] * BLOCK + at % BLOCK
        s["slots"] = torch.where(at >= T - case["pads"], -1, slots).int()
        s["live"] = at[:max(0, T - case["pads"])]
        inv, axis = _axes(case)
        s.update(inv=inv.to(dev), axis=axis.to(dev), q_w=None, k_w=None)
        if case["norm"]:
            s.update(q_w=rn(D, scale=0.3, shift=1.0), k_w=rn(D, scale=0.3, shift=1.0))
        if kv == 16:
            s.update(k=rn(pages, hkv, BLOCK, D), v=rn(pages, hkv, BLOCK, D))
        else:
            z = dict(device=dev)
            s.update(k=torch.zeros(pages, hkv, BLOCK, D, dtype=torch.uint8, **z), v=torch.zeros(pages, hkv, BLOCK, D, dtype=torch.uint8, **z),
                     km=torch.zeros(pages, hkv, BLOCK, D // 64, 2, dtype=torch.bfloat16, **z),
                     vm=torch.zeros(pages, hkv, BLOCK, D // 64, 2, dtype=torch.bfloat16, **z))
    elif case["op"] == "axial":
        R, H, D = case["rows"], case["heads"], case["dim"]
        side = max(1, math.isqrt(R))
        at = torch.arange(R, device=dev)
        inv = 1.0 / 1e4 ** (torch.arange(0, D // 2, 2).double() / (D // 2))
        s.update(qkv=rn(R, 3 * H * D), pos=torch.stack([at // side, at % side]).int(), inv=torch.cat([inv, inv]).float().to(dev),
                 axis=(torch.arange(D // 2) >= D // 4).int().to(dev))
    elif case["op"] == "pages":
        L, P, n, D = 2 * case["layers"], case["pool"], case["moved"], case["dim"]
        ids = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
        s.update(src=ids[:n], dst=ids[n:2 * n])
        if case["kv"] == 16:
            s["slabs"] = [rn(L, P, case["hkv"], BLOCK, D)]
        else:
            s["slabs"] = [torch.randint(0, 256, (L, P, case["hkv"], BLOCK, D), generator=g, device=dev, dtype=torch.uint8),
                          rn(L, P, case["hkv"], BLOCK, D // 64, 2)]
        if case["job"] == "scatter":
            s["data"] = torch.cat([x[:, s["src"]].reshape(-1).view(torch.uint8) for x in s["slabs"]])
        if own:                  # the pool of a serving program keeps this list of its slabs
            from mlxcel_b200.ops import pages
            s["handle"] = pages.PageSlabs([layer for x in s["slabs"] for layer in x])
    elif case["op"] == "scores":
        R, V = case["rows"], case["vocab"]
        x = torch.randn(R, V, generator=g, device=dev) * 2.5
        x[torch.arange(R, device=dev), torch.randint(0, V, (R,), generator=g, device=dev)] += 9.0
        if case["masked"]:
            x.masked_fill_(torch.rand(R, V, generator=g, device=dev) < case["masked"], NEG)
        if case["empty"]:
            x[R // 2] = NEG
        s.update(logits=x.to(TYPES[case["dtype"]]), ids=torch.randint(0, V, (R,), generator=g, device=dev))
    else:
        R, K, V = case["rows"], case["width"], case["vocab"]
        s.update(x=rn(R, K), w=rn(V, K, scale=2.5 / math.sqrt(K)), ids=torch.randint(0, V, (R,), generator=g, device=dev),
                 bias=rn(V, scale=0.5) if case["bias"] else None)
    return s


# ----------------------------------------------------------------------------- one pass
def run(s):
    return {"norm": _run_norm, "mrope": _run_mrope, "axial": _run_axial, "pages": _run_pages, "scores": _run_scores, "head": _run_head}[s["case"]["op"]](s)


def _run_norm(s):
    c = s["case"]
    if own:
        from mlxcel_b200.ops import norms
        y, h = norms.branch_norm(s["x"], s["res"], post_w=s["post_w"], gate=s["gate"], scale=c["scale"], pre_w=s["pre_w"], pre_b=s["pre_b"],
                                 layer_norm=c["layer"], eps=EPS, w_bias=c["w_bias"])
        return dict(y=y, h=h)
    b = s["x"].float()
    if s["post_w"] is not None:
        b = b * torch.rsqrt((b * b).mean(-1, keepdim=True) + EPS) * (s["post_w"].float() + c["w_bias"])
    if s["gate"] is not None:
        b = b * s["gate"].float()
    h = s["res"].float() + c["scale"] * b
    z = h - h.mean(-1, keepdim=True) if c["layer"] else h
    y = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * (s["pre_w"].float() + c["w_bias"])
    if s["pre_b"] is not None:
        y = y + s["pre_b"].float()
    return dict(y=y.to(s["x"].dtype), h=h.to(s["x"].dtype))


def _turn(x, cos, sin, rot, pairs):
    """Rotates the first ``rot`` columns of x [T, H, D] by the angles of cos / sin [T, rot / 2]."""
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _codes(x):
    """8-bit codes of groups of 64 with a bf16 (scale, offset) pair."""
    z = x.unflatten(-1, (-1, 64))
    low, high = z.amin(-1, keepdim=True), z.amax(-1, keepdim=True)
    scale, low = ((high - low) / 255.0).bfloat16().float(), low.bfloat16().float()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round((z - low) / scale).clamp(0, 255).to(torch.uint8).flatten(-2), torch.cat([scale, low], -1).bfloat16()


def _values(s, name, at):
    """What the codes of the written rows stand for."""
    codes, meta = s[name][at[0], :, at[1]], s[name + "m"][at[0], :, at[1]].float()
    return (codes.float().unflatten(-1, (-1, 64)) * meta[..., 0:1] + meta[..., 1:2]).flatten(-2).bfloat16()


def _run_mrope(s):
    c = s["case"]
    T, hq, hkv, D, kv = c["tokens"], c["hq"], c["hkv"], c["dim"], c["kv"]
    slots = s["slots"][s["live"]].long() if kv != 16 or not own else None
    at = (slots // BLOCK, slots % BLOCK) if slots is not None else None
    if own:
        from mlxcel_b200.ops import KVLayer, rotary
        layer = KVLayer(s["k"], s["v"], s.get("km"), s.get("vm"), BLOCK, kv)
        q = rotary.mrope_append(s["qkv"], s["pos"], s["slots"], s["inv"], s["axis"], layer, Hq=hq, Hkv=hkv, D=D, rot_dim=c["rot"],
                                traditional=c["layout"] == "pairs", q_norm_w=s["q_w"], k_norm_w=s["k_w"], norm_eps=EPS)
    else:
        x = s["qkv"].view(T, hq + 2 * hkv, D).float()
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        if c["norm"]:
            q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["q_w"].float()
            k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["k_w"].float()
        # (angles of far positions keep their digits in 64 bits)
        angle = s["pos"].double().t()[:, s["axis"].long()] * s["inv"].double()
        cos, sin = angle.cos().float(), angle.sin().float()
        q = _turn(q, cos, sin, c["rot"], c["layout"] == "pairs").bfloat16().view(T, hq * D)
        k, v = _turn(k, cos, sin, c["rot"], c["layout"] == "pairs")[s["live"]], v[s["live"]]
        if kv == 16:
            s["k"][at[0], :, at[1]], s["v"][at[0], :, at[1]] = k.bfloat16(), v.bfloat16()
        else:
            (s["k"][at[0], :, at[1]], s["km"][at[0], :, at[1]]), (s["v"][at[0], :, at[1]], s["vm"][at[0], :, at[1]]) = _codes(k), _codes(v)
    return dict(q=q, k=s["k"], v=s["v"]) if kv == 16 else dict(q=q, k=_values(s, "k", at), v=_values(s, "v", at))


def _run_axial(s):
    c = s["case"]
    if own:
        from mlxcel_b200.ops import rotary
        q, k, v = rotary.axial_rope(s["qkv"], s["pos"], s["inv"], s["axis"], heads=c["heads"], D=c["dim"])
        return dict(q=q, k=k, v=v)
    x = s["qkv"].view(c["rows"], 3, c["heads"], c["dim"]).float()
    angle = s["pos"].double().t()[:, s["axis"].long()] * s["inv"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    q, k = (_turn(x[:, i], cos, sin, c["dim"], False) for i in (0, 1))
    return dict(q=q.transpose(0, 1).contiguous(), k=k.transpose(0, 1).contiguous(), v=x[:, 2].transpose(0, 1).contiguous())


def _run_pages(s):
    job = s["case"]["job"]
    if own:
        if job == "copy":
            s["handle"].copy(s["src"], s["dst"])
        elif job == "gather":
            return dict(data=s["handle"].gather(s["src"]))
        else:
            s["handle"].scatter(s["dst"], s["data"])
        return dict(enumerate(s["slabs"]))
    dev = s["slabs"][0].device
    src, dst = torch.tensor(s["src"], device=dev), torch.tensor(s["dst"], device=dev)
    if job == "gather":
        parts = [x[:, src].reshape(-1).view(torch.uint8) for x in s["slabs"]]
        return dict(data=parts[0] if len(parts) == 1 else torch.cat(parts))
    first = 0
    for x in s["slabs"]:
        if job == "copy":
            x[:, dst] = x[:, src]
        else:
            size = x[:, 0].numel() * x.element_size() * len(s["dst"])
            x[:, dst] = s["data"][first:first + size].view(x.dtype).view(x.shape[0], len(s["dst"]), *x.shape[2:])
            first += size
    return dict(enumerate(s["slabs"]))


def _measure(x, ids):
    """Log probability of ids, entropy and log normaliser of fp32 rows; a row with nothing left has probability 0 everywhere."""
    top = x.amax(-1, keepdim=True)
    base = torch.where(top == NEG, torch.zeros_like(top), top)
    e = torch.exp(x - base)
    total = e.sum(-1)
    lse = base[:, 0] + torch.log(total)
    gone = total == 0
    got = x.gather(1, ids[:, None])[:, 0]
    logprob = torch.where(got == NEG, got, got - lse)
    mean = torch.where(e > 0, e * (x - base), torch.zeros_like(x)).sum(-1) / total
    return logprob, torch.where(gone, torch.zeros_like(total), torch.log(total) - mean), lse


def _run_scores(s):
    top = s["case"]["top"]
    if own:
        from mlxcel_b200.ops import logprobs
        r = logprobs.token_logprobs(s["logits"], s["ids"], top=top)
        out = dict(logprob=r.logprob, entropy=r.entropy, lse=r.lse)
        return dict(out, top_ids=r.top_ids, top_logprobs=r.top_logprobs) if top else out
    x = s["logits"].float()
    logprob, entropy, lse = _measure(x, s["ids"])
    out = dict(logprob=logprob, entropy=entropy, lse=lse)
    if top:
        v, i = torch.sort(x, dim=-1, descending=True, stable=True)           # ties to the lowest index
        v = v[:, :top]
        out.update(top_ids=i[:, :top].int(), top_logprobs=torch.where(v == NEG, v, v - lse[:, None]))
    return out


def _run_head(s):
    c = s["case"]
    if own:
        from mlxcel_b200.ops import logprobs
        r = logprobs.head_logprobs(s["x"], s["w"], s["ids"], bias=s["bias"], scale=c["scale"], softcap=c["softcap"])
        return dict(logprob=r.logprob, entropy=r.entropy, lse=r.lse)
    x = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        x = x + s["bias"].float()
    x = x * c["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    logprob, entropy, lse = _measure(x, s["ids"])
    return dict(logprob=logprob, entropy=entropy, lse=lse)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "norm":
        n, d, size = case["rows"], case["dim"], 4 if case["dtype"] == "fp32" else 2
        vectors = 1 + case["post"] + case["gate"] + case["layer"]
        return dict(bytes=size * d * (4 * n + vectors), flops=n * d * (8 + 4 * case["post"] + case["gate"] + 2 * case["layer"]))
    if case["op"] == "mrope":
        T, heads, D = case["tokens"], case["hq"] + 2 * case["hkv"], case["dim"]
        kept = T - min(T, case["pads"])
        row = 2 * D if case["kv"] == 16 else D + D // 64 * 4
        return dict(bytes=T * heads * D * 2 + T * case["hq"] * D * 2 + kept * 2 * case["hkv"] * row + T * 16,
                    flops=T * (case["hq"] + case["hkv"]) * (3 * case["rot"] + (4 * D if case["norm"] else 0)))
    if case["op"] == "axial":
        n = case["rows"] * case["heads"] * case["dim"]
        return dict(bytes=3 * n * (2 + 4) + case["rows"] * 8, flops=2 * n * 3)
    if case["op"] == "pages":
        row = case["dim"] * 2 if case["kv"] == 16 else case["dim"] + case["dim"] // 64 * 4
        return dict(bytes=2 * case["moved"] * 2 * case["layers"] * case["hkv"] * BLOCK * row, flops=0)
    if case["op"] == "scores":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * (20 + 8 * case["top"]), flops=5 * n)
    R, K, V = case["rows"], case["width"], case["vocab"]
    return dict(bytes=2 * K * (R + V) + R * 20 + (2 * V if case["bias"] else 0), flops=2 * R * K * V + 6 * R * V)


# ----------------------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "norm":
        def rms(t, w):
            return t / torch.sqrt(torch.mean(t.pow(2), 1, True) + EPS) * (w.to(f) + case["w_bias"])
        branch = rms(s["x"].to(f), s["post_w"]) if case["post"] else s["x"].to(f)
        h = s["res"].to(f) + case["scale"] * (branch * s["gate"].to(f) if case["gate"] else branch)
        if not case["layer"]:
            return dict(y=rms(h, s["pre_w"]), h=h)
        var, mean = torch.var_mean(h, 1, correction=0, keepdim=True)
        return dict(y=(h - mean) / torch.sqrt(var + EPS) * (s["pre_w"].to(f) + case["w_bias"]) + s["pre_b"].to(f), h=h)
    if case["op"] in ("mrope", "axial"):
        rot = case["rot"] if case["op"] == "mrope" else case["dim"]
        D, half = case["dim"], rot // 2
        # as complex numbers: pair i of a head, times e^(i angle)
        angle = torch.stack([s["pos"][a].to(f) * s["inv"][i].to(f) for i, a in enumerate(s["axis"].tolist())], 1)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        first = torch.arange(half, device="cuda") * (2 if case.get("layout") == "pairs" else 1)
        second = first + (1 if case.get("layout") == "pairs" else half)

        def rotated(t):
            z = torch.complex(t[..., first], t[..., second]) * turn
            t = t.clone()
            t[..., first], t[..., second] = z.real, z.imag
            return t
        if case["op"] == "axial":
            q, k, v = s["qkv"].to(f).view(case["rows"], 3, case["heads"], D).unbind(1)
            return dict(q=rotated(q).transpose(0, 1), k=rotated(k).transpose(0, 1), v=v.transpose(0, 1))
        q, k, v = s["qkv"].to(f).view(case["tokens"], -1, D).split([case["hq"], case["hkv"], case["hkv"]], 1)
        if case["norm"]:
            q = q / torch.sqrt(q.pow(2).mean(2, True) + EPS) * s["q_w"].to(f)
            k = k / torch.sqrt(k.pow(2).mean(2, True) + EPS) * s["k_w"].to(f)
        q = rotated(q).reshape(case["tokens"], -1)
        if case["kv"] != 16:
            return dict(q=q, k=None, v=None)
        k, out = rotated(k), {}
        for name, new in (("k", k), ("v", v)):
            flat = s[name].to(f).transpose(1, 2).reshape(-1, case["hkv"], D)            # [slot, head, D]
            flat[s["slots"][s["live"]].long()] = new[s["live"]]
            out[name] = flat.view(-1, BLOCK, case["hkv"], D).transpose(1, 2)
        return dict(q=q, **out)
    if case["op"] == "pages":
        return None                                       # bytes are moved, nothing is computed
    if case["op"] == "scores":
        top = case["top"]
        lp, en, ls, ti, tp = [], [], [], [], []
        for r0 in range(0, case["rows"], 64):
            x = s["logits"][r0:r0 + 64].to(f)
            ls.append(torch.logsumexp(x, 1))
            p = torch.where(torch.isinf(ls[-1])[:, None], torch.zeros_like(x), torch.exp(x - ls[-1][:, None]))
            en.append(-torch.special.xlogy(p, p).sum(1))
            pick = x.gather(1, s["ids"][r0:r0 + 64, None])
            lp.append(torch.where(torch.isinf(pick), pick, pick - ls[-1][:, None])[:, 0])
            if top:
                order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :top]
                best = x.gather(1, order)
                ti.append(order.int())
                tp.append(torch.where(torch.isinf(best), best, best - ls[-1][:, None]))
        out = dict(logprob=torch.cat(lp), entropy=torch.cat(en), lse=torch.cat(ls))
        return dict(out, top_ids=torch.cat(ti), top_logprobs=torch.cat(tp)) if top else out
    # head: parts of the vocabulary, joined through logaddexp; the entropy is lse - sum p z
    x = s["x"].to(f)
    parts = []
    for v0 in range(0, case["vocab"], 8192):
        z = x @ s["w"][v0:v0 + 8192].to(f).T
        if case["bias"]:
            z += s["bias"][v0:v0 + 8192].to(f)
        z *= case["scale"]
        if case["softcap"]:
            z = torch.tanh(z / case["softcap"]) * case["softcap"]
        part = torch.logsumexp(z, 1)
        here = (s["ids"] >= v0) & (s["ids"] < v0 + 8192)
        pick = z.gather(1, (s["ids"] - v0).clamp(0, z.shape[1] - 1)[:, None])[:, 0]
        parts.append((part, (torch.exp(z - part[:, None]) * z).sum(1), torch.where(here, pick, torch.zeros_like(pick))))
    lse = torch.logsumexp(torch.stack([p[0] for p in parts]), 0)
    mean = sum(torch.exp(p[0] - lse) * p[1] for p in parts)
    return dict(logprob=sum(p[2] for p in parts) - lse, entropy=lse - mean, lse=lse)
