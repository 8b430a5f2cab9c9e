"""More of a decoder layer's operators, as measurable cases: the norms between
its parts, rotary positions of one or several axes, the gated feed-forward's
two projections with their activation and product, each with its gradients,
and differential attention over the paged 8-bit cache.

  own                False: the plain forms in torch; True: the package's kernels
  listed()           the named cases
  draw(rng)          one more case of the same ranges
  prepare(case, s)   what a program holds before the call, from seed s
  run(state)         one pass; returns its outputs whole
  work(case)         bytes and operations a pass cannot do without
  exact(case, s)     run's outputs from the definitions, in 64 bits

The cache holds codes 1..255 for -127..127 and one f32 scale per block of
tokens and head; keys are [block][head][token][dim], values
[block][head][dim][token].
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

_held = {}


def context():
    """One context per program, as the package asks for (one per host thread)."""
    if "ctx" not in _held:
        import haagenti_amd as H
        _held["ctx"] = H.HipContext(0)
    return _held["ctx"]


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # the norm before a layer's projections in a step of eight requests, Llama-3-8B's width: latency
        dict(name="norm_step", kind="norm", rows=8, n=4096, dtype="bf16", norm="rms", weight="same", bias=False, back=False,
             add=False, pad=0),
        # layer norm of a long prompt's hidden states, parameters kept in f32
        dict(name="norm_prompt", kind="norm", rows=8192, n=4096, dtype="bf16", norm="layer", weight="f32", bias=True,
             back=False, add=False, pad=0),
        # its gradients over a training step's tokens, the residual path's gradient added on the way
        dict(name="norm_train", kind="norm", rows=8192, n=4096, dtype="bf16", norm="layer", weight="f32", bias=True,
             back=True, add=True, pad=0),
        # gradients of an odd width in rows of a wider buffer
        dict(name="norm_odd", kind="norm", rows=1003, n=1001, dtype="f16", norm="layer", weight="same", bias=True, back=True,
             add=False, pad=5),
        # one new token's queries and keys for each of 16 requests, deep into their texts: latency
        dict(name="rotary_step", kind="rotary", tokens=16, q_heads=32, heads=8, dim=128, rot=128, sections="64", far=131072,
             dtype="bf16", interleaved=False, inverse=False),
        # the queries and keys of a video's patches in time, height and width
        dict(name="rotary_video", kind="rotary", tokens=16200, q_heads=16, heads=4, dim=128, rot=128, sections="16 24 24",
             far=4000, dtype="bf16", interleaved=False, inverse=False),
        # Llama-3-8B's gate and up projections for a single token: weight bytes
        dict(name="gated_token", kind="gated", m=1, n=14336, k=4096, dtype="bf16", weight="same", act="silu", bias=False,
             back=False, pad=0),
        # the same for sixteen requests' tokens straight from INT4
        dict(name="gated_int4", kind="gated", m=16, n=14336, k=4096, dtype="bf16", weight="int4", act="silu", bias=False,
             back=False, pad=0),
        # a training step's 2048 tokens through them: the projections kept for the backward pass, then all gradients
        dict(name="gated_train", kind="gated", m=2048, n=14336, k=4096, dtype="bf16", weight="same", act="silu", bias=False,
             back=True, pad=0),
        # a small odd block with biases, rows of a wider buffer
        dict(name="gated_odd", kind="gated", m=77, n=1003, k=1001, dtype="f16", weight="same", act="gelu", bias=True,
             back=True, pad=5),
        # a running batch of 32 requests of ragged lengths, a new token each
        dict(name="diff_step", kind="diff", requests=32, lo=100, hi=8000, new_lo=1, new_hi=1, q_heads=16, heads=4, dim=128,
             block=32, dtype="bf16", norm=True),
        # two prompts' chunks of about 1500 tokens over what is cached of them
        dict(name="diff_prompts", kind="diff", requests=2, lo=1500, hi=2500, new_lo=1400, new_hi=1536, q_heads=16, heads=4,
             dim=128, block=64, dtype="bf16", norm=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _side(rng, lo, hi):
    """A matrix side: mostly a multiple of 64, as weights have, else any number."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.7 else n


def draw(rng):
    """A case that moves no more bytes and does no more operations than the listed ones."""
    most = [work(c) for c in listed()]
    while True:
        case = _drawn(rng)
        if all(work(case)[m] <= max(w[m] for w in most) for m in ("bytes", "flops")):
            return case


def _drawn(rng):
    kind = rng.choice(["norm", "norm", "rotary", "gated", "gated", "gated", "diff", "diff"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "norm":
        dtype = rng.choice([dtype, dtype, "f32"])
        norm, back = rng.choice(["layer", "layer", "rms"]), rng.random() < 0.5
        weight = rng.choice(["same", "f32", "none"])
        return dict(kind=kind, rows=_log(rng, 1, 8192), n=_side(rng, 64, 16384), dtype=dtype, norm=norm, weight=weight,
                    bias=weight != "none" and norm == "layer", back=back, add=back and rng.random() < 0.5,
                    pad=rng.choice([0, 0, 0, 8, 3]))
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        rot = rng.choice([dim, dim, dim // 2])
        axes, pairs = rng.choice([1, 1, 2, 3, 3]), rot // 2
        cut = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = " ".join(str(b - a) for a, b in zip([0] + cut, cut + [pairs]))
        heads = rng.choice([1, 2, 4, 8])
        return dict(kind=kind, tokens=_log(rng, 1, 16384), q_heads=heads * rng.choice([1, 2, 4, 8]), heads=heads, dim=dim,
                    rot=rot, sections=sections, far=_log(rng, 64, 1000000), dtype=rng.choice([dtype, dtype, "f32"]),
                    interleaved=rng.random() < 0.4, inverse=rng.random() < 0.4)
    if kind == "gated":
        back = rng.random() < 0.5
        return dict(kind=kind, m=_log(rng, 1, 2048), n=_side(rng, 64, 14336), k=_side(rng, 64, 8192), dtype=dtype,
                    weight="same" if back else rng.choice(["same", "int4"]),
                    act=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", "none"]), bias=rng.random() < 0.3, back=back,
                    pad=rng.choice([0, 0, 0, 8, 3]))
    heads = rng.choice([1, 2, 4, 8])
    new = 1 if rng.random() < 0.55 else _log(rng, 2, 768)
    requests = _log(rng, 1, 48 if new == 1 else max(1, min(16, 2048 // new)))
    hi = _log(rng, 16, 131072 // requests if new == 1 else 4000)
    return dict(kind=kind, requests=requests, lo=min(hi, rng.choice([0, 1, hi // 4, hi // 2])), hi=hi,
                new_lo=max(1, new - rng.randint(0, new // 3)), new_hi=new, q_heads=heads * rng.choice([1, 2, 3, 4, 4, 8]),
                heads=heads, dim=rng.choice([64, 128, 128, 128, 96, 192, 256]), block=rng.choice([16, 32, 64, 128]),
                dtype=dtype, norm=rng.random() < 0.7)


def _spread(lo, hi, n, at):
    """n whole numbers of lo..hi that look unordered; the largest is hi."""
    v = [lo + int((hi - lo + 1) * (((i + 1) * 0.6180339887 + at) % 1.0)) for i in range(n)]
    v[n // 2] = hi
    return v


def _requests(case):
    """(tokens cached before, new tokens) of each request."""
    n = case["requests"]
    return _spread(case["lo"], case["hi"], n, 0.11), _spread(case["new_lo"], case["new_hi"], n, 0.37)


def _sections(case):
    """Pairs of dimensions that each axis turns."""
    return [int(x) for x in case["sections"].split()]


def _cdiv(a, b):
    return (a + b - 1) // b


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _int4(w):
    """The INT4 buffer of a matrix: a truncated f16 scale per 32 values in row order, then the nibbles, low first."""
    n = w.numel()
    g = _cdiv(n, 32)
    p = torch.zeros(g * 32, device="cuda")
    p[:n] = w.reshape(-1)
    p = p.view(g, 32)
    mx = p.abs().amax(1)
    scale = torch.where(mx > 1e-10, mx / 7.0, torch.ones_like(mx))
    h = scale.half()
    h = torch.where(h.float() > scale, (h.view(torch.int16) - 1).view(torch.half), h)
    q = (torch.round(p / scale[:, None]).clamp(-8, 7) + 8).to(torch.uint8).view(-1)
    q[n:] = 0
    q = q[:_cdiv(n, 2) * 2]
    return torch.cat([h.view(torch.uint8), q[0::2] | (q[1::2] << 4)])


def _pages(lens, case, gen, width):
    """Block tables (unordered blocks, no block twice) for requests of these lengths, and the number of blocks."""
    counts = [_cdiv(x, case["block"]) for x in lens]
    blocks = sum(counts) + 7
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    c = _ints(counts)
    first = torch.cumsum(c, 0) - c
    at = torch.arange(width, device="cuda")[None, :]
    held = at < c[:, None]
    table[held] = order[(first[:, None] + at)[held].long()]
    return table, blocks


def _codes(shape, gen):
    """Codes as rows of about normal values leave them."""
    return (torch.randn(shape, generator=gen, device="cuda") * 36 + 128).round().clamp(1, 255).to(torch.uint8)


def _scales(shape, gen):
    """f32 scales of 8 significant bits."""
    s = (torch.rand(shape, generator=gen, device="cuda") + 2.5) / 127
    return ((s.view(torch.int32) + 0xffff) & -0x10000).view(torch.float32)


def _positions(case, gen):
    """A token's place on each axis: far into a text, or frames of a picture's rows and columns after one."""
    t, axes = case["tokens"], len(_sections(case))
    base = case["far"] - torch.randint(0, max(1, case["far"] // 2), (1,), generator=gen, device="cuda")
    if axes == 1:
        return (base - torch.randint(0, case["far"] // 2, (1, t), generator=gen, device="cuda")).to(torch.int32)
    side = max(1, int(math.sqrt(t / 18)))
    at = torch.arange(t, device="cuda")
    grid = [at // (side * side), at // side % side, at % side]
    return (torch.stack(grid[3 - axes:]) + base).to(torch.int32)


def prepare(case, seed):
    kind, gen, dt = case["kind"], _gen(seed), DTYPES[case["dtype"]]
    s = dict(case=case)
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        # hidden states: some channels far larger than the others, rows off their mean
        x = torch.randn((rows, n + case["pad"]), generator=gen, device="cuda")
        x *= 1 + 7 * (torch.rand((n + case["pad"],), generator=gen, device="cuda") > 0.99)
        s["x"] = (x + torch.randn((rows, 1), generator=gen, device="cuda") * 0.5).to(dt)[:, :n]
        wt = dt if case["weight"] == "same" else torch.float32
        s["weight"] = None if case["weight"] == "none" else (1 + 0.2 * torch.randn((n,), generator=gen, device="cuda")).to(wt)
        s["bias"] = _randn((n,), gen, wt, 0.2) if case["bias"] else None
        if case["back"]:
            s["dy"] = _randn((rows, n), gen, dt, 0.1)
            s["add"] = _randn((rows, n), gen, dt, 0.1) if case["add"] else None
        return s
    if kind == "rotary":
        h = case["q_heads"] + case["heads"]
        # queries and keys are parts of the rows of a joint projection
        qkv = _randn((case["tokens"], h + case["heads"], case["dim"]), gen, dt)
        pairs = case["rot"] // 2
        s["x"] = qkv[:, :h]
        s["positions"] = _positions(case, gen)
        s["inv_freq"] = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)).float()
        return s
    if kind == "gated":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _randn((m, k + case["pad"]), gen, dt)[:, :k]
        for name in ("gate", "up"):
            w = torch.randn((n, k), generator=gen, device="cuda") * 0.02
            s[name] = _int4(w) if case["weight"] == "int4" else w.to(dt)
            s[name + "_bias"] = _randn((n,), gen, dt, 0.3) if case["bias"] else None
        if case["back"]:
            s["dy"] = _randn((m, n), gen, dt, 0.05)
        return s
    lens, new = _requests(case)
    total = [a + b for a, b in zip(lens, new)]
    h, b, d = case["heads"], case["block"], case["dim"]
    table, blocks = _pages(total, case, gen, _cdiv(max(total), b) + 1)
    s.update(table=table, k=_codes((blocks, h, b, d), gen), v=_codes((blocks, h, d, b), gen),
             k_scale=_scales((blocks, h), gen), v_scale=_scales((blocks, h), gen))
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    s.update(q=_randn((start[-1], case["q_heads"], d), gen, dt, 1.5), start=_ints(start), kv_len=_ints(total),
             max_q=max(new), max_kv=max(total), scale=(d // 2) ** -0.5,
             lam=0.2 + 0.6 * torch.rand((case["q_heads"],), generator=gen, device="cuda"),
             norm_weight=1 + 0.2 * torch.randn((d,), generator=gen, device="cuda") if case["norm"] else None)
    return s


# ------------------------------------------------------------------ plain forms

EPS, GAIN = 1e-5, 0.8


def _norm(s):
    case, x = s["case"], s["x"].float()
    w = 1.0 if s["weight"] is None else s["weight"].float()
    if case["norm"] == "layer":
        x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    x = x * r
    dt = DTYPES[case["dtype"]]
    if not case["back"]:
        y = x * w
        return (y if s["bias"] is None else y + s["bias"].float()).to(dt)
    dy = s["dy"].float()
    g = dy * w
    dx = g - x * (g * x).mean(1, keepdim=True)
    if case["norm"] == "layer":
        dx = dx - g.mean(1, keepdim=True)
    dx = dx * r
    if s["add"] is not None:
        dx = dx + s["add"].float()
    return dict(dx=dx.to(dt), dweight=None if s["weight"] is None else (dy * x).sum(0),
                dbias=dy.sum(0) if case["bias"] else None)


def _axis_of(case, device):
    return torch.repeat_interleave(torch.arange(len(_sections(case)), device=device),
                                   torch.tensor(_sections(case), device=device))


def _rotary(s):
    case, x = s["case"], s["x"].float()
    pos = s["positions"][_axis_of(case, x.device)].t().double()             # token, pair
    angle = pos * s["inv_freq"].double()
    c, n = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    n = -n if case["inverse"] else n
    pairs, rot = case["rot"] // 2, case["rot"]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"] else (x[..., :pairs], x[..., pairs:rot])
    a, b = a * c - b * n, b * c + a * n
    turned = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1).to(DTYPES[case["dtype"]])


def _act(x, act):
    """act(x) and its derivative."""
    one = torch.ones_like(x)
    if act == "relu":
        on = (x > 0).float()
        return x * on, on
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)
    if act == "silu":
        p = 1 / (1 + torch.exp(-x))
        return x * p, p * (1 + x * (1 - p))
    return x, one


def _int4_values(buf, n, k):
    g = _cdiv(n * k, 32)
    scale = buf[:2 * g].view(torch.half).float()
    b = buf[2 * g:]
    q = torch.stack([b & 15, b >> 4], 1).reshape(-1)[:n * k].float() - 8
    return (q * scale.repeat_interleave(32)[:n * k]).view(n, k)


def _gated(s):
    case, x = s["case"], s["x"].float()
    dt = DTYPES[case["dtype"]]
    w = [_int4_values(s[i], case["n"], case["k"]) if case["weight"] == "int4" else s[i].float() for i in ("gate", "up")]
    g, u = x @ w[0].t(), x @ w[1].t()
    if case["bias"]:
        g, u = g + s["gate_bias"].float(), u + s["up_bias"].float()
    a, slope = _act(g, case["act"])
    y = a * u
    if not case["back"]:
        return y.to(dt)
    dy = s["dy"].float()
    du, dg = dy * a, dy * u * slope
    return dict(y=y.to(dt), dx=(dg @ w[0] + du @ w[1]).to(dt), dgate=(dg.t() @ x).to(dt), dup=(du.t() @ x).to(dt),
                dgate_bias=dg.sum(0) if case["bias"] else None, dup_bias=du.sum(0) if case["bias"] else None)


def _diff(s):
    case = s["case"]
    h, d, b = case["heads"], case["dim"], case["block"]
    g, r, nq = case["q_heads"] // h, case["requests"], s["max_q"]
    n = _cdiv(s["max_kv"], b)
    t = s["table"][:, :n].clamp(min=0).long()
    start, kv_len = s["start"].long(), s["kv_len"].long()
    k = (s["k"][t].float() - 128) * s["k_scale"][t][..., None, None]
    k = k.transpose(1, 2).reshape(r, h, n * b, d)
    v = (s["v"][t].float() - 128) * s["v_scale"][t][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(r, h, n * b, d)
    i = torch.arange(nq, device=k.device)
    rows = start[1:] - start[:-1]
    q = s["q"][(start[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)].float()
    q = q.view(r, nq, h, g, d).permute(0, 2, 1, 3, 4).reshape(r, h, nq * g, d)
    last = (kv_len - rows)[:, None] + i[None, :]
    hidden = (torch.arange(n * b, device=k.device)[None, None, :] > last[:, :, None])[:, None, :, None, :]
    maps = []
    for j in range(2):
        half = slice(j * d // 2, (j + 1) * d // 2)
        p = (q[..., half] @ k[..., half].transpose(2, 3).contiguous()).mul_(s["scale"]).view(r, h, nq, g, n * b)
        p.masked_fill_(hidden, -math.inf)
        top = p.amax(-1, keepdim=True)
        p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total = p.sum(-1, keepdim=True)
        p = p.div_(torch.where(total > 0, total, 1.0))
        maps.append(p.view(r, h, nq * g, n * b) @ v)
    lam = s["lam"].view(1, h, 1, g, 1)
    o = maps[0].view(r, h, nq, g, d) - lam * maps[1].view(r, h, nq, g, d)
    if s["norm_weight"] is not None:
        o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_weight"] * GAIN
    at = torch.arange(s["q"].shape[0], device=k.device)
    of = torch.searchsorted(start, at, right=True) - 1
    return o[of, :, at - start[of]].reshape(-1, h * g, d).to(s["q"].dtype)


def _package(s):
    """The calls that a user of the package makes."""
    import haagenti_amd.compute as K
    case, kind, ctx = s["case"], s["case"]["kind"], context()
    if kind == "norm":
        if not case["back"]:
            return K.norm(ctx, s["x"], s["weight"], s["bias"], kind=case["norm"], eps=EPS)
        dx, dweight, dbias = K.norm_backward(ctx, s["dy"], s["x"], s["weight"], bias=case["bias"], kind=case["norm"], eps=EPS,
                                             add=s["add"])
        return dict(dx=dx, dweight=dweight, dbias=dbias)
    if kind == "rotary":
        return K.rotary(ctx, s["x"], s["positions"], s["inv_freq"], sections=_sections(case),
                        interleaved=case["interleaved"], inverse=case["inverse"])
    if kind == "gated":
        w = [K.Int4Weight(s[i], case["n"], case["k"]) if case["weight"] == "int4" else s[i] for i in ("gate", "up")]
        if not case["back"]:
            return K.gated_linear(ctx, s["x"], *w, gate_bias=s["gate_bias"], up_bias=s["up_bias"], act=case["act"])
        y, saved = K.gated_linear(ctx, s["x"], *w, gate_bias=s["gate_bias"], up_bias=s["up_bias"], act=case["act"], save=True)
        d = K.gated_linear_backward(ctx, s["dy"], s["x"], *w, saved, act=case["act"], bias=case["bias"])
        return dict(y=y, dx=d.dx, dgate=d.dgate, dup=d.dup, dgate_bias=d.dgate_bias, dup_bias=d.dup_bias)
    if "cache" not in s:        # the handle that such a program keeps
        s["cache"] = K.KvCache(ctx, s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s["cache"].diff_attention(s["q"], s["lam"], s["table"], s["start"], s["kv_len"], max_q=s["max_q"],
                                     max_kv=s["max_kv"], scale=s["scale"], norm_weight=s["norm_weight"], eps=EPS,
                                     gain=GAIN if case["norm"] else 1.0)


def run(state):
    if own:
        return _package(state)
    return {"norm": _norm, "rotary": _rotary, "gated": _gated, "diff": _diff}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        wt = 0 if case["weight"] == "none" else size if case["weight"] == "same" else 4
        grads = 4 * n * ((wt > 0) + case["bias"]) if case["back"] else 0
        tensors = 3 + case["add"] if case["back"] else 2
        weights = n * wt * (1 + (case["bias"] and not case["back"]))
        return {"bytes": tensors * rows * n * size + weights + grads, "flops": 0}
    if kind == "rotary":
        x = case["tokens"] * (case["q_heads"] + case["heads"]) * case["dim"] * size
        return {"bytes": 2 * x + 4 * case["tokens"] * len(_sections(case)) + 2 * case["rot"], "flops": 0}
    if kind == "gated":
        m, n, k = case["m"], case["n"], case["k"]
        w = _cdiv(n * k, 32) * 2 + _cdiv(n * k, 2) if case["weight"] == "int4" else 2 * n * k
        moved = 2 * m * k + 2 * w + 4 * n * case["bias"] + 2 * m * n
        if not case["back"]:
            return {"bytes": moved, "flops": 4 * m * n * k}
        # the output's gradient in; those of x, both weights and the biases out
        moved += 2 * m * n + 2 * m * k + 4 * n * k + 8 * n * case["bias"]
        return {"bytes": moved, "flops": 12 * m * n * k}
    lens, new = _requests(case)
    h, d = case["heads"], case["dim"]
    pairs = sum(c * a + c * (c + 1) // 2 for a, c in zip(lens, new))
    cached = sum(a + c for a, c in zip(lens, new))
    # two maps over half the dimensions each, both over all of V
    return {"bytes": 2 * h * d * cached + 4 * sum(new) * case["q_heads"] * d, "flops": 6 * case["q_heads"] * d * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_norm(s):
    case, n = s["case"], s["case"]["n"]
    x = s["x"].double().requires_grad_(case["back"])
    w = None if s["weight"] is None else s["weight"].double().requires_grad_(case["back"])
    b = None if s["bias"] is None else s["bias"].double().requires_grad_(case["back"])
    if case["norm"] == "layer":
        y = torch.nn.functional.layer_norm(x, (n,), w, b, EPS)
    else:
        y = x / torch.sqrt(x.square().sum(1, keepdim=True) / n + EPS)
        y = y if w is None else y * w
    if not case["back"]:
        return y
    y.backward(s["dy"].double())
    dx = x.grad if s["add"] is None else x.grad + s["add"].double()
    return dict(dx=dx, dweight=None if w is None else w.grad, dbias=None if b is None else b.grad)


def _exact_rotary(s):
    """Pairs as complex numbers, section by section."""
    case, x = s["case"], s["x"].double()
    out, j = x.clone(), 0
    pairs = case["rot"] // 2
    for axis, count in enumerate(_sections(case)):
        at = torch.arange(j, j + count, device=x.device)
        first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + pairs)
        angle = s["positions"][axis].double()[:, None] * s["inv_freq"][at].double()[None, :]
        turn = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle)[:, None]
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        out[..., first], out[..., second] = z.real, z.imag
        j += count
    return out


def _exact_gated(s):
    case = s["case"]
    n, k, back = case["n"], case["k"], case["back"]
    w = []
    for name in ("gate", "up"):
        if case["weight"] == "int4":
            g = _cdiv(n * k, 32)
            nibbles = s[name][2 * g:]
            q = torch.zeros(2 * nibbles.numel(), dtype=torch.float64, device="cuda")
            q[0::2], q[1::2] = (nibbles % 16).double() - 8, (nibbles // 16).double() - 8
            at = torch.arange(n * k, device="cuda") // 32
            w.append((q[:n * k] * s[name][:2 * g].view(torch.half).double()[at]).view(n, k))
        else:
            w.append(s[name].double().requires_grad_(back))
    x = s["x"].double().requires_grad_(back)
    b = [None if s[i] is None else s[i].double().requires_grad_(back) for i in ("gate_bias", "up_bias")]
    z, u = torch.nn.functional.linear(x, w[0], b[0]), torch.nn.functional.linear(x, w[1], b[1])
    F = torch.nn.functional
    y = u * {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
             "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[case["act"]](z)
    if not back:
        return y
    y.backward(s["dy"].double())
    return dict(y=y.detach(), dx=x.grad, dgate=w[0].grad, dup=w[1].grad, dgate_bias=None if b[0] is None else b[0].grad,
                dup_bias=None if b[1] is None else b[1].grad)


def _exact_diff(s):
    case = s["case"]
    h, d, b, g = case["heads"], case["dim"], case["block"], case["q_heads"] // case["heads"]
    lens, new = _requests(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    t0 = 0
    for r, (a, c) in enumerate(zip(lens, new)):
        n = a + c
        blocks = s["table"][r, :_cdiv(n, b)].long()
        for j in range(h):
            k = ((s["k"][blocks, j].double() - 128) * s["k_scale"][blocks, j].double()[:, None, None]).reshape(-1, d)[:n]
            v = (s["v"][blocks, j].double() - 128) * s["v_scale"][blocks, j].double()[:, None, None]
            v = v.transpose(1, 2).reshape(-1, d)[:n]
            lam = s["lam"][j * g:(j + 1) * g].double()[None, :, None]
            for q0 in range(0, c, 512):
                m = min(512, c - q0)
                q = s["q"][t0 + q0:t0 + q0 + m, j * g:(j + 1) * g].double().reshape(m * g, d)
                seen = torch.arange(n, device="cuda")[None, :] <= (a + q0 + torch.arange(m, device="cuda"))[:, None]
                p = []
                for e in (0, d // 2):
                    z = (q[:, e:e + d // 2].contiguous() @ k[:, e:e + d // 2].t().contiguous()).view(m, g, n) * s["scale"]
                    p.append(torch.softmax(z.masked_fill(~seen[:, None, :], -math.inf), -1))
                o = ((p[0] - lam * p[1]).view(m * g, n) @ v).view(m, g, d)
                if s["norm_weight"] is not None:
                    o = o / torch.sqrt(o.square().sum(-1, keepdim=True) / d + EPS) * s["norm_weight"].double() * GAIN
                out[t0 + q0:t0 + q0 + m, j * g:(j + 1) * g] = o
        t0 += c
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "gated": _exact_gated, "diff": _exact_diff}[case["kind"]](s)
