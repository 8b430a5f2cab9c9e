"""Plain 64-bit forms of the decoder-layer operators (numpy), for the tests."""
import math

import numpy as np


def act(z, name):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "gelu":
        return 0.5 * z * (1 + np.vectorize(math.erf)(z / math.sqrt(2.0)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        with np.errstate(over="ignore"):
            return z / (1 + np.exp(-z))
    return z


def int4_parts(buf, n, k):
    """(integers -8..7, scales) of an INT4 buffer, both n x k."""
    g = (n * k + 31) // 32
    s = np.frombuffer(buf[:2 * g].tobytes(), np.float16).astype(np.float64)
    b = buf[2 * g:].astype(np.int64)
    q = np.stack([b & 15, b >> 4], 1).reshape(-1)[:n * k] - 8
    return q.reshape(n, k).astype(np.float64), np.repeat(s, 32)[:n * k].reshape(n, k)


def half_ulp(y, dtype):
    """Half a unit in the last place of the 16- or 32-bit type at |y|."""
    bits, least = {"f16": (10, -24), "bf16": (7, -133), "f32": (23, -149)}[dtype]
    e = np.floor(np.log2(np.maximum(np.abs(y), 1e-300)))
    return np.ldexp(0.5, np.maximum(e - bits, least).astype(np.int64))


def up8(x):
    """x >= 0 rounded up to 8 significant bits."""
    f, e = np.frexp(x)
    return np.ldexp(np.ceil(f * 256) / 256, e)


def append(codes, scale, rows, slots, bs):
    """Appends rows (tokens, heads, dim; f64) at slots to codes (blocks,
    heads, tokens, dim; integers -127..127 or what is there) and scales."""
    codes, scale = codes.astype(np.float64), scale.astype(np.float64)
    t, n = 0, len(slots)
    while t < n:
        s = int(slots[t])
        if s < 0 or s >= codes.shape[0] * bs:
            t += 1
            continue
        b, o, m = s // bs, s % bs, 1
        while t + m < n and o + m < bs and int(slots[t + m]) == s + m:
            m += 1
        x = np.swapaxes(rows[t:t + m], 0, 1)
        amax = np.max(np.where(np.isfinite(x), np.abs(x), 0.0), axis=(1, 2))
        old = scale[b] if o else np.zeros_like(scale[b])
        now = np.maximum(old, up8(amax / 127))
        div = np.where(now > 0, now, 1.0)[:, None, None]
        if o:
            grown = (now > old)[:, None, None]
            again = np.clip(np.rint(codes[b, :, :o] * old[:, None, None] / div), -127, 127)
            codes[b, :, :o] = np.where(grown, again, codes[b, :, :o])
        with np.errstate(invalid="ignore"):
            q = np.clip(np.rint(x / div), -127, 127)
        codes[b, :, o:o + m] = np.where(np.isnan(x), 0.0, q)
        scale[b] = now
        t += m
    return codes, scale


def attention(q, k, v, kv_len, scale):
    """One request: q (rows, heads, dim), k and v (tokens, kv heads, dim),
    f64; returns the output and sum p |v| (what rounding p costs scales with),
    and the largest sum |q k| scale."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    out, mass, size = np.zeros_like(q), np.zeros_like(q), 0.0
    for i in range(rows):
        n = min(max(kv_len - rows + i + 1, 0), k.shape[0])
        if n == 0:
            continue
        for h in range(heads):
            kk, vv = k[:n, h // group], v[:n, h // group]
            z = kk @ q[i, h] * scale
            size = max(size, float(np.max(np.abs(kk) @ np.abs(q[i, h]) * scale)))
            p = np.exp(z - z.max())
            p /= p.sum()
            out[i, h], mass[i, h] = p @ vv, p @ np.abs(vv)
    return out, mass, size


def plan(lens, new, table, ring, state, bs, tokens):
    """hh_kv_plan by its rules, request by request."""
    table, ring = table.copy(), ring.copy()
    cap, (head, count) = len(ring), (int(state[0]), int(state[1]))
    width = table.shape[1]
    start, kv_len, status, slots = [0], [], [], np.full(tokens, -1, np.int64)
    taken, wanted, freed = 0, 0, []
    for r, (n, a) in enumerate(zip(lens, new)):
        n, a, s0 = int(n), int(a), start[-1]
        rows = max(a, 0)
        code, held = 0, 0
        have, need = (max(n, 0) + bs - 1) // bs, (max(n, 0) + rows + bs - 1) // bs
        if n < 0:
            code = 7
        elif a < 0:
            freed += [int(x) for x in table[r, :min(have, width)]]
        elif need > width or (rows and s0 + rows > tokens):
            code = 2
        else:
            wanted += need - have
            if need > have and wanted > count:
                code = 8
            else:
                for b in range(have, need):
                    table[r, b] = ring[(head + taken) % cap]
                    taken += 1
                for i in range(rows):
                    slots[s0 + i] = table[r, (n + i) // bs] * bs + (n + i) % bs
                held = n + rows
        kv_len.append(held)
        status.append(code)
        start.append(min(s0 + rows, tokens))
    for j, b in enumerate(freed):
        if count + j < cap:
            ring[(head + count + j) % cap] = b
    after = [(head + taken) % cap if cap else 0, min(count - taken + len(freed), cap)]
    return dict(start=start, kv_len=kv_len, status=status, slots=slots, table=table, ring=ring, state=after)
