"""The operators of a decoder layer together, as a program uses them: the
example's layer with positions, prompts and then single tokens, and a layer's
feed-forward half trained for a step, against the same in 64 bits."""
import importlib.util
import os

import numpy as np
import pytest

import norm_ref
import test_gpu_compute as G

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    return ex


def plain(w, ins, prompts, heads, kv_heads, theta):
    """The layer over whole sequences in float64, without a cache."""
    w = {n: t.double().cpu().numpy() for n, t in w.items()}
    ins = [x.double().cpu().numpy() for x in ins]
    hidden = ins[0].shape[1]
    d, group = hidden // heads, heads // kv_heads
    norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)  # noqa: E731
    freq = theta ** (-np.arange(d // 2) / (d // 2))
    start, outs = np.concatenate([[0], np.cumsum(prompts)]), []
    for r in range(len(prompts)):
        x = np.concatenate([ins[0][start[r]:start[r + 1]]] + [y[r:r + 1] for y in ins[1:]])
        qkv = (norm(x) @ w["qkv"].T).reshape(len(x), heads + 2 * kv_heads, d)
        turned = norm_ref.rotary(qkv[:, :heads + kv_heads], np.arange(len(x))[None], freq, [d // 2], False, False)[0]
        o = np.zeros((len(x), heads, d))
        for h in range(heads):
            z = turned[:, h] @ turned[:, heads + h // group].T * d ** -0.5
            z[np.triu(np.ones(z.shape, bool), 1)] = -np.inf
            p = np.exp(z - z.max(1, keepdims=True))
            o[:, h] = p / p.sum(1, keepdims=True) @ qkv[:, heads + kv_heads + h // group]
        x = x + o.reshape(len(x), -1) @ w["o"].T
        g, u = norm(x) @ w["gate"].T, norm(x) @ w["up"].T
        outs.append(x + (g / (1 + np.exp(-g)) * u) @ w["down"].T)
    return outs


def test_layer_with_positions():
    prompts, steps, theta = [70, 3, 1, 129], 5, 10000.0
    w, ins, outs, _ = example().run(256, 4, 2, 512, prompts, steps, theta=theta)
    want = plain(w, ins, prompts, 4, 2, theta)
    start = np.concatenate([[0], np.cumsum(prompts)])
    for r in range(len(prompts)):
        got = np.concatenate([outs[0][start[r]:start[r + 1]].double().cpu().numpy()]
                             + [y[r:r + 1].double().cpu().numpy() for y in outs[1:]])
        # a bf16 rounding (2^-9 of each value) at each of about 12 places that feed the output, and keys and values
        # in steps of 1 / 127 of their block's largest (at most 4 times their rms: 0.5 * 4 / 127 / sqrt(3) of it each)
        rel = np.linalg.norm(got - want[r]) / np.linalg.norm(want[r])
        assert rel <= 12 * 2.0 ** -9 + 2 * 0.5 * 4 / 127, (r, rel)


def step(c, K, x, w, b, gate, up, down, dout):
    """Forward and backward of x + down(gated(norm(x))): the output and every gradient."""
    h = K.norm(c, x, w, b)
    y, saved = K.gated_linear(c, h, gate, up, save=True)
    out = K.linear(c, y, down, residual=x)
    dy = K.linear(c, dout, down.t().contiguous())
    g = K.gated_linear_backward(c, dy, h, gate, up, saved)
    dx, dw, db = K.norm_backward(c, g.dx, x, w, bias=True, add=dout)
    return dict(out=out, dx=dx, dw=dw, db=db, dgate=g.dgate, dup=g.dup)


def tensors(rows, hidden, ffn, seed):
    t = G.T()
    g = t.Generator("cuda").manual_seed(seed)
    r = lambda scale, *s: (t.randn(*s, generator=g, device="cuda") * scale).bfloat16()  # noqa: E731
    return [r(1, rows, hidden), 1 + r(0.2, hidden).float(), r(0.2, hidden).float(), r(hidden ** -0.5, ffn, hidden),
            r(hidden ** -0.5, ffn, hidden), r(ffn ** -0.5, hidden, ffn), r(1, rows, hidden)]


@pytest.mark.parametrize("rows,hidden,ffn", [(200, 256, 704), (65, 130, 333), (1, 64, 64)])
def test_a_training_step(rows, hidden, ffn):
    t, K = G.T(), G.K()
    args = tensors(rows, hidden, ffn, rows)
    got = step(G.ctx(), K, *args)
    x, w, b, gate, up, down, dout = [a.double().requires_grad_() for a in args]
    h = t.nn.functional.layer_norm(x, (hidden,), w, b, 1e-5)
    out = x + (t.nn.functional.silu(h @ gate.t()) * (h @ up.t())) @ down.t()
    out.backward(dout.detach())
    want = dict(out=out.detach(), dx=x.grad, dw=w.grad, db=b.grad, dgate=gate.grad, dup=up.grad)
    for name, y in want.items():
        # bf16 roundings (2^-9 of each value) on the way to a gradient: the norm's output, y, dy, dg and du, the products'
        # outputs: at most 6 of them after another, each of errors that don't depend on each other
        rel = float((got[name].double() - y).norm() / y.norm())
        assert rel <= 6 * 2.0 ** -9, (name, rel)


def test_a_training_step_captured():
    t, K, c = G.T(), G.K(), G.ctx()
    sets = [tensors(200, 256, 704, seed) for seed in (1, 2)]
    want = [{n: y.clone() for n, y in step(c, K, *s).items()} for s in sets]
    held = [a.clone() for a in sets[0]]
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        outs = step(c, K, *held)
    for i in range(5):
        for a, b in zip(held, sets[i % 2]):
            a.copy_(b)
        step(c, K, *tensors(300, 256, 1000, 3))      # other sizes meanwhile
        graph.replay()
        t.cuda.synchronize()
        for n, y in want[i % 2].items():
            assert t.equal(outs[n], y), (i, n)
