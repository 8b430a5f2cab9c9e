"""A decoder layer's work on decoded weights, as measurable cases: matrix
products with their epilogue (16-bit weights as the decoder writes them, or
the package's INT4 buffers), and a paged 8-bit key / value cache: its plan
(block tables and slots from request lengths), appending to it and reading it
back, and attention over it.

  own                False: the plain forms in torch; True: the package's kernels
  listed()           the named cases
  draw(rng)          one more case of the same ranges
  prepare(case, s)   what a program holds before the call, from seed s
  run(state)         one pass; returns its outputs whole
  work(case)         bytes and operations a pass cannot do without
  exact(case, s)     run's outputs from the definitions, in 64 bits

The cache holds codes 1..255 for -127..127 and one f32 scale per block of
tokens and head (never finer than 8 significant bits, rounded up).  Keys are
[block][head][token][dim], values [block][head][dim][token].
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

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
        # the output projection of a Llama-3-8B layer for a single token, with the residual: latency and weight bytes
        dict(name="linear_token", kind="linear", m=1, n=4096, k=4096, dtype="bf16", weight="same", act="none", bias=False,
             mul=False, res=True, out="same", pad=0),
        # that layer's gate for eight requests' tokens straight from INT4, times the up projection
        dict(name="linear_int4_8", kind="linear", m=8, n=14336, k=4096, dtype="bf16", weight="int4", act="silu", bias=False,
             mul=True, res=False, out="same", pad=0),
        # the same gate over a prompt's 2048 tokens with decoded weights
        dict(name="linear_prompt", kind="linear", m=2048, n=14336, k=4096, dtype="bf16", weight="same", act="silu",
             bias=False, mul=True, res=False, out="same", pad=0),
        # an odd classifier head over some rows of a wider buffer: no side a multiple of anything, f32 out
        dict(name="linear_odd", kind="linear", m=77, n=1003, k=1001, dtype="f16", weight="same", act="gelu", bias=True,
             mul=False, res=False, out="f32", pad=5),
        # one step of eight running requests, one new token each: launch latency
        dict(name="plan_step", kind="plan", requests=8, lo=1, hi=4000, new_lo=1, new_hi=1, done=0, block=16, width=512),
        # a busy server's step: prompts arriving beside running requests, some that end
        dict(name="plan_mixed", kind="plan", requests=1024, lo=0, hi=30000, new_lo=1, new_hi=127, done=24, block=32,
             width=1024),
        # a step of 64 requests appending a token each, most into blocks begun before
        dict(name="append_step", kind="append", requests=64, lo=1, hi=2000, new_lo=1, new_hi=1, pad=3, heads=8, dim=128,
             block=16, dtype="bf16", read="bf16"),
        # prompts of about a thousand tokens each
        dict(name="append_prompts", kind="append", requests=8, lo=0, hi=700, new_lo=900, new_hi=1150, pad=0, heads=8,
             dim=128, block=64, dtype="bf16", read="bf16"),
        # three short requests in f16, small heads: latency
        dict(name="attn_short", kind="attention", requests=3, lo=1, hi=290, new_lo=1, new_hi=1, q_heads=16, heads=4,
             dim=64, block=16, dtype="f16"),
        # a running batch of 48 requests of ragged lengths, Llama-3-8B heads
        dict(name="attn_step", kind="attention", requests=48, lo=100, hi=8000, new_lo=1, new_hi=1, q_heads=32, heads=8,
             dim=128, block=32, dtype="bf16"),
        # one request deep into a long document, Llama-70B heads (64 on 8): a single new token
        dict(name="attn_long", kind="attention", requests=1, lo=131001, hi=131001, new_lo=1, new_hi=1, q_heads=64, heads=8,
             dim=128, block=64, dtype="bf16"),
        # two prompts' chunks of about 2000 tokens over what is cached of them
        dict(name="attn_prompts", kind="attention", requests=2, lo=3000, hi=4100, new_lo=1900, new_hi=2048, q_heads=32,
             heads=8, dim=128, block=64, dtype="bf16"),
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
    kind = rng.choice(["linear", "linear", "linear", "plan", "append", "append", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "linear":
        n, k = _side(rng, 64, 14336), _side(rng, 64, 14336)
        return dict(kind=kind, m=_log(rng, 1, 2048), n=n, k=k, dtype=dtype, weight=rng.choice(["same", "same", "int4"]),
                    act=rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.4,
                    mul=rng.random() < 0.3, res=rng.random() < 0.4, out=rng.choice(["same", "same", "f32"]),
                    pad=rng.choice([0, 0, 0, 8, 3]))
    block = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        requests = _log(rng, 1, 1024)
        hi = _log(rng, 8, 30000)
        return dict(kind=kind, requests=requests, lo=rng.choice([0, 0, 1]), hi=hi, new_lo=rng.randint(0, 1),
                    new_hi=_log(rng, 1, 256), done=rng.randint(0, requests // 16), block=block,
                    width=(hi + 256) // block + 1)
    dim = rng.choice([64, 128, 128, 128, 96, 192, 256])
    heads = rng.choice([1, 2, 4, 8, 8])
    if kind == "append":
        new = _log(rng, 1, 2048)
        return dict(kind=kind, requests=_log(rng, 1, max(1, min(128, 8192 // new))), lo=0, hi=_log(rng, 2, 2000),
                    new_lo=max(1, new - rng.randint(0, new // 4)), new_hi=new, pad=rng.choice([0, 0, 5]), heads=heads,
                    dim=dim, block=block, dtype=dtype, read=rng.choice([dtype, "f32"]))
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    new = 1 if rng.random() < 0.55 else _log(rng, 2, 1024)
    requests = _log(rng, 1, 48 if new == 1 else max(1, min(16, 2048 // new)))
    hi = _log(rng, 16, 131072 // requests if new == 1 else 6000)
    return dict(kind=kind, requests=requests, lo=min(hi, rng.choice([0, 1, hi // 4, hi // 2])), hi=hi,
                new_lo=max(1, new - rng.randint(0, new // 3)), new_hi=new, q_heads=heads * group, heads=heads, dim=dim,
                block=block, dtype=dtype)


def _spread(lo, hi, n, at):
    """n whole numbers of lo..hi that look unordered; the largest is hi."""
    v = [lo + int((hi - lo + 1) * (((i + 1) * 0.6180339887 + at) % 1.0)) for i in range(n)]
    v[n // 2] = hi
    return v


def _requests(case):
    """(tokens cached before, new tokens) of each request."""
    n = case["requests"]
    return _spread(case["lo"], case["hi"], n, 0.11), _spread(case["new_lo"], case["new_hi"], n, 0.37)


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
    total = sum(counts)
    blocks = total + 7
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    c = _ints(counts)
    first = torch.cumsum(c, 0) - c
    at = torch.arange(width, device="cuda")[None, :]
    held = at < c[:, None]
    table[held] = order[(first[:, None] + at)[held].long()]
    return table, blocks


def _up_bf16(x):
    """Positive f32 rounded up to 8 significant bits."""
    return ((x.view(torch.int32) + 0xffff) & -0x10000).view(torch.float32)


def _codes(shape, gen):
    """Codes as rows of about normal values leave them."""
    return (torch.randn(shape, generator=gen, device="cuda") * 36 + 128).round().clamp(1, 255).to(torch.uint8)


def _cache(case, blocks, gen):
    h, b, d = case["heads"], case["block"], case["dim"]
    def scales():
        return _up_bf16((torch.rand((blocks, h), generator=gen, device="cuda") + 2.5) / 127)
    return dict(k=_codes((blocks, h, b, d), gen), v=_codes((blocks, h, d, b), gen), k_scale=scales(), v_scale=scales())


def prepare(case, seed):
    kind, gen = case["kind"], _gen(seed)
    s = dict(case=case)
    if kind == "linear":
        m, n, k, dt = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        wide = _randn((m, k + case["pad"]), gen, dt)
        s["x"] = wide[:, :k]
        w = torch.randn((n, k), generator=gen, device="cuda") * 0.02
        s["w"] = _int4(w) if case["weight"] == "int4" else w.to(dt)
        s["bias"] = _randn((n,), gen, dt, 0.5) if case["bias"] else None
        s["mul"] = _randn((m, n), gen, dt) if case["mul"] else None
        s["res"] = _randn((m, n), gen, dt) if case["res"] else None
        return s
    lens, new = _requests(case)
    if kind == "plan":
        for i in range(case["done"]):
            new[(i * 37 + 5) % case["requests"]] = -1
        table, blocks = _pages(lens, case, gen, case["width"])
        need = sum(_cdiv(a + b, case["block"]) - _cdiv(a, case["block"]) for a, b in zip(lens, new) if b > 0)
        spare = need + need // 8 + 2
        cap = blocks + spare
        ring = torch.full((cap,), -1, dtype=torch.int32, device="cuda")
        head = cap - max(1, spare // 2)          # the free blocks wrap around the ring's end
        at = (head + torch.arange(spare, device="cuda")) % cap
        ring[at] = (torch.randperm(spare, generator=gen, device="cuda") + blocks).to(torch.int32)
        s.update(lens=_ints(lens), new=_ints(new), table=table, ring=ring, state=_ints([head, spare]),
                 tokens=sum(x for x in new if x > 0) + 5)
        return s
    total = [a + b for a, b in zip(lens, new)]
    width = _cdiv(max(total), case["block"]) + 1
    table, blocks = _pages(total, case, gen, width)
    s.update(_cache(case, blocks, gen), table=table)
    h, d, dt = case["heads"], case["dim"], DTYPES[case["dtype"]]
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    if kind == "append":
        t, slots, touched = start[-1] + case["pad"], [], []
        rows = table.cpu().tolist()
        for r, (a, c) in enumerate(zip(lens, new)):
            slots += [rows[r][p // case["block"]] * case["block"] + p % case["block"] for p in range(a, a + c)]
            touched += rows[r][a // case["block"]:_cdiv(a + c, case["block"])]
        # k and v are parts of the rows of a joint projection
        qkv = _randn((t, 3 * h * d), gen, torch.float32)
        qkv *= 1 + 3 * (torch.rand((3 * h * d,), generator=gen, device="cuda") > 0.97)
        qkv = qkv.to(dt)
        s.update(rows_k=qkv[:, h * d:2 * h * d].view(t, h, d), rows_v=qkv[:, 2 * h * d:].view(t, h, d),
                 slots=_ints(slots + [-1] * case["pad"]), blocks=_ints(touched))
        return s
    s.update(q=_randn((start[-1], case["q_heads"], d), gen, dt, 1.5), start=_ints(start), kv_len=_ints(total),
             max_q=max(new), max_kv=max(total), scale=1 / math.sqrt(d))
    return s


# ------------------------------------------------------------------ plain forms

def _act(x, act):
    if act == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "silu":
        return x / (1 + torch.exp(-x))
    return x


def _int4_values(buf, n, k):
    g = _cdiv(n * k, 32)
    scale = buf[:2 * g].view(torch.half).float()
    b = buf[2 * g:]
    q = torch.stack([b & 15, b >> 4], 1).reshape(-1)[:n * k].float() - 8
    return (q * scale.repeat_interleave(32)[:n * k]).view(n, k)


def _linear(s):
    case = s["case"]
    w = _int4_values(s["w"], case["n"], case["k"]) if case["weight"] == "int4" else s["w"].float()
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _act(y, case["act"])
    if s["mul"] is not None:
        y = y * s["mul"].float()
    if s["res"] is not None:
        y = y + s["res"].float()
    return y


def _plan(s):
    b, cap, dev = s["case"]["block"], s["ring"].numel(), s["lens"].device
    lens, new, table = s["lens"].long(), s["new"].long(), s["table"]
    r, width = table.shape
    head, count = s["state"][0].long(), s["state"][1].long()
    have, end = (lens + b - 1) // b, lens + new.clamp(min=0)
    want = (end + b - 1) // b - have
    done, wide = new < 0, (new >= 0) & ((end + b - 1) // b > width)
    want = torch.where(done | wide, 0, want)
    through = torch.cumsum(want, 0)
    short = ~done & ~wide & (through > count) & (want > 0)
    served = ~done & ~wide & ~short
    take = torch.where(served, want, 0)
    first = torch.cumsum(take, 0) - take
    rows = new.clamp(min=0)
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), torch.cumsum(rows, 0)])
    kv_len = torch.where(served, end, 0)
    status = torch.where(wide, 2, torch.where(short, 8, 0))
    # blocks taken from the ring's head go to the tables
    col = torch.arange(width, device=dev)[None, :]
    fresh = (col >= have[:, None]) & (col < (have + take)[:, None])
    ids = s["ring"][(head + first[:, None] + col - have[:, None]) % cap]
    table.copy_(torch.where(fresh, ids, table))
    # slots of the new rows
    at = torch.arange(s["tokens"], device=dev)
    q = torch.searchsorted(start, at, right=True) - 1
    live = (at < start[-1])
    q = q.clamp(max=r - 1)
    pos = lens[q] + at - start[q]
    slot = table[q, (pos // b).clamp(max=width - 1)].long() * b + pos % b
    slots = torch.where(live & served[q], slot, -1)
    # finished requests' blocks go to the ring's tail
    give = torch.where(done, have, 0)
    back = torch.cumsum(give, 0) - give
    tail = (head + count + back[:, None] + col) % cap
    given = done[:, None] & (col < have[:, None])
    wide_ring = torch.cat([s["ring"], s["ring"][:1]])
    wide_ring[torch.where(given, tail, cap)] = table
    s["ring"].copy_(wide_ring[:cap])
    taken = take.sum()
    state = torch.stack([(head + taken) % cap, count - taken + give.sum()])
    i32 = torch.int32
    return dict(start=start.to(i32), kv_len=kv_len.to(i32), slots=slots.to(i32), status=status.to(i32), table=table,
                ring=s["ring"], state=state.to(i32))


def _store(codes, scale, x, s, heads_last):
    """Rows x into the blocks s["blocks"] of codes [block][head][token][dim] (in place); heads_last: [..][dim][token]."""
    b, blocks, slots = s["case"]["block"], s["blocks"].long(), s["slots"].long()
    n = blocks.numel()
    x = x.float()
    where = torch.full((scale.shape[0] + 1,), n, dtype=torch.int64, device=x.device)
    where[blocks] = torch.arange(n, device=x.device)
    row = where[torch.where(slots >= 0, slots // b, scale.shape[0])]
    off = slots % b
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(2)
    amax = torch.zeros((n + 1, x.shape[1]), device=x.device).scatter_reduce(0, row[:, None].expand_as(top), top, "amax")
    first = torch.full((n + 1,), b, dtype=torch.int64, device=x.device).scatter_reduce(0, row, off, "amin")[:n]
    old = torch.where(first[:, None] > 0, scale[blocks], 0.0)
    now = torch.maximum(old, _up_bf16(amax[:n] / 127))
    div = torch.where(now > 0, now, 1.0)
    held = codes[blocks]
    held = held.transpose(2, 3) if heads_last else held
    again = torch.round((held.float() - 128) * old[:, :, None, None] / div[:, :, None, None]) + 128
    before = torch.arange(b, device=x.device)[None, None, :, None] < first[:, None, None, None]
    held = torch.where(before, again.to(torch.uint8), held)
    div = torch.cat([div, torch.ones_like(div[:1])])
    code = torch.nan_to_num(x / div[row][:, :, None], nan=0.0, posinf=127.0, neginf=-127.0)
    code = torch.round(code).clamp(-127, 127) + 128
    held = torch.cat([held, torch.zeros_like(held[:1])])
    held[row, :, off] = code.to(torch.uint8)
    held = held[:n]
    codes[blocks] = held.transpose(2, 3) if heads_last else held
    scale[blocks] = now
    return ((held.float() - 128) * now[:, :, None, None]).transpose(1, 2)


def _append(s):
    dt = DTYPES[s["case"]["read"]]
    k = _store(s["k"], s["k_scale"], s["rows_k"], s, False).to(dt)
    v = _store(s["v"], s["v_scale"], s["rows_v"], s, True).to(dt)
    return dict(k=k, v=v, k_scale=s["k_scale"], v_scale=s["v_scale"])


def _attention(s):
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
    p = (q @ k.transpose(2, 3).contiguous()).mul_(s["scale"]).view(r, h, nq, g, n * b)
    last = (kv_len - rows)[:, None] + i[None, :]
    hidden = torch.arange(n * b, device=k.device)[None, None, :] > last[:, :, None]
    p.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(r, h, nq * g, n * b) @ v
    o = o.view(r, h, nq, g, d) / torch.where(total > 0, total, 1.0)
    at = torch.arange(s["q"].shape[0], device=k.device)
    of = torch.searchsorted(start, at, right=True) - 1
    return o[of, :, at - start[of]].reshape(-1, h * g, d).to(s["q"].dtype)


def _package(s):
    """The calls that a user of the package makes."""
    import haagenti_amd.compute as K
    case, kind = s["case"], s["case"]["kind"]
    if kind == "linear":
        w = K.Int4Weight(s["w"], case["n"], case["k"]) if case["weight"] == "int4" else s["w"]
        return K.linear(context(), s["x"], w, bias=s["bias"], act=case["act"], mul=s["mul"], residual=s["res"],
                        out_dtype=torch.float32 if case["out"] == "f32" else None)
    if kind == "plan":
        p = K.kv_plan(context(), s["lens"], s["new"], s["table"], s["ring"], s["state"], case["block"], s["tokens"])
        return dict(start=p.start, kv_len=p.kv_len, slots=p.slots, status=p.status, table=s["table"], ring=s["ring"],
                    state=p.state)
    if "cache" not in s:        # the handle that such a program keeps
        s["cache"] = K.KvCache(context(), s["k"], s["v"], s["k_scale"], s["v_scale"])
    if kind == "append":
        s["cache"].append(s["rows_k"], s["rows_v"], s["slots"])
        k, v = s["cache"].read(s["blocks"], dtype=DTYPES[case["read"]])
        return dict(k=k, v=v, k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s["cache"].attention(s["q"], s["table"], s["start"], s["kv_len"], max_q=s["max_q"], max_kv=s["max_kv"],
                                scale=s["scale"])


def run(state):
    if own:
        return _package(state)
    case = state["case"]
    if case["kind"] == "linear":
        return _linear(state).to(torch.float32 if case["out"] == "f32" else DTYPES[case["dtype"]])
    return {"plan": _plan, "append": _append, "attention": _attention}[case["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        w = _cdiv(n * k, 32) * 2 + _cdiv(n * k, 2) if case["weight"] == "int4" else 2 * n * k
        extra = 2 * n * case["bias"] + 2 * m * n * (case["mul"] + case["res"])
        return {"bytes": 2 * m * k + w + extra + m * n * (4 if case["out"] == "f32" else 2), "flops": 2 * m * n * k}
    lens, new = _requests(case)
    if kind == "plan":
        # lengths in, starts, lengths and statuses out, a slot per row, a block id read and written per block taken
        need = sum(_cdiv(a + c, case["block"]) - _cdiv(a, case["block"]) for a, c in zip(lens, new))
        return {"bytes": 4 * (5 * case["requests"] + sum(new) + 2 * need), "flops": 0}
    h, d = case["heads"], case["dim"]
    if kind == "append":
        t = sum(new)
        blocks = sum(_cdiv(a + c, case["block"]) - a // case["block"] for a, c in zip(lens, new))
        size = 4 if case["read"] == "f32" else 2
        # rows in, codes out; the touched blocks' codes in and their values out
        return {"bytes": 2 * h * d * (3 * t + blocks * case["block"] * (1 + size)) + 16 * blocks * h, "flops": 0}
    pairs = sum(c * a + c * (c + 1) // 2 for a, c in zip(lens, new))
    cached = sum(a + c for a, c in zip(lens, new))
    return {"bytes": 2 * h * d * cached + 4 * sum(new) * case["q_heads"] * d,
            "flops": 4 * case["q_heads"] * d * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_linear(s):
    case = s["case"]
    n, k = case["n"], case["k"]
    x = s["x"].double()
    if case["weight"] == "int4":
        g = _cdiv(n * k, 32)
        nibbles = s["w"][2 * g:]
        w = torch.zeros(2 * nibbles.numel(), dtype=torch.float64, device="cuda")
        w[0::2], w[1::2] = (nibbles % 16).double() - 8, (nibbles // 16).double() - 8
        at = torch.arange(n * k, device="cuda") // 32
        w = (w[:n * k] * s["w"][:2 * g].view(torch.half).double()[at]).view(n, k)
    else:
        w = s["w"].double()
    z = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
    z = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]](z)
    z = z if s["mul"] is None else z * s["mul"].double()
    return z if s["res"] is None else z + s["res"].double()


def _up8(x):
    """x >= 0 rounded up to 8 significant bits."""
    f, e = torch.frexp(x)
    return torch.ldexp(torch.ceil(f * 256) / 256, e)


def _exact_store(codes, scale, x, s, values):
    """Request by request, block by block, as the rows arrive; returns the touched blocks' values and the scales."""
    case = s["case"]
    b = case["block"]
    codes, scale, x = codes.double() - 128, scale.double().clone(), x.double()
    codes = codes.transpose(2, 3).contiguous() if values else codes
    lens, new = _requests(case)
    rows, t0 = s["table"].cpu().tolist(), 0
    for r, (a, c) in enumerate(zip(lens, new)):
        p = a
        while p < a + c:
            n = min(b - p % b, a + c - p)
            k, o = rows[r][p // b], p % b
            part = x[t0:t0 + n].transpose(0, 1)                   # head, token, dim
            was = scale[k] if o else torch.zeros_like(scale[k])
            now = torch.maximum(was, _up8(part.abs().amax((1, 2)) / 127))
            codes[k, :, :o] = torch.round(codes[k, :, :o] * (was / now)[:, None, None])
            codes[k, :, o:o + n] = torch.round(part / now[:, None, None]).clamp(-127, 127)
            scale[k] = now
            p, t0 = p + n, t0 + n
    blocks = s["blocks"].long()
    return (codes[blocks] * scale[blocks][:, :, None, None]).transpose(1, 2), scale


def _exact_attention(s):
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
            for q0 in range(0, c, 512):
                m = min(512, c - q0)
                q = s["q"][t0 + q0:t0 + q0 + m, j * g:(j + 1) * g].double().reshape(m * g, d)
                z = (q @ k.t().contiguous()).view(m, g, n) * s["scale"]
                seen = torch.arange(n, device="cuda")[None, :] <= (a + q0 + torch.arange(m, device="cuda"))[:, None]
                z = z.masked_fill(~seen[:, None, :], -math.inf)
                out[t0 + q0:t0 + q0 + m, j * g:(j + 1) * g] = (torch.softmax(z, -1).view(m * g, n) @ v).view(m, g, d)
        t0 += c
    return out


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _exact_linear(s)
    if case["kind"] == "append":
        k, ks = _exact_store(s["k"], s["k_scale"], s["rows_k"], s, False)
        v, vs = _exact_store(s["v"], s["v_scale"], s["rows_v"], s, True)
        return dict(k=k, v=v, k_scale=ks, v_scale=vs)
    return _exact_attention(s)
