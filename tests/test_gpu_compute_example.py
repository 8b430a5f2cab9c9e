"""examples/decoder_layer.py: a layer decoded from LZ4 blocks of tiles, then a
prompt and single tokens through the operators, against the same layer in 64
bits on the decoded weights."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def plain(w, ins, prompts, heads, kv_heads):
    """The layer over whole sequences in float64, without a cache."""
    w = {n: t.double().cpu().numpy() for n, t in w.items()}
    ins = [x.double().cpu().numpy() for x in ins]
    hidden = ins[0].shape[1]
    d, group = hidden // heads, heads // kv_heads
    norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)  # noqa: E731
    start = np.concatenate([[0], np.cumsum(prompts)])
    outs = []
    for r, n in enumerate(prompts):
        x = np.concatenate([ins[0][start[r]:start[r + 1]]] + [y[r:r + 1] for y in ins[1:]])
        qkv = (norm(x) @ w["qkv"].T).reshape(len(x), heads + 2 * kv_heads, d)
        o = np.zeros((len(x), heads, d))
        for h in range(heads):
            k, v = qkv[:, heads + h // group], qkv[:, heads + kv_heads + h // group]
            z = qkv[:, h] @ k.T * d ** -0.5
            z[np.triu(np.ones(z.shape, bool), 1)] = -np.inf
            p = np.exp(z - z.max(1, keepdims=True))
            o[:, h] = p / p.sum(1, keepdims=True) @ v
        x = x + o.reshape(len(x), -1) @ w["o"].T
        y = norm(x)
        g = y @ w["gate"].T
        outs.append(x + (g / (1 + np.exp(-g)) * (y @ w["up"].T)) @ w["down"].T)
    return outs


def test_layer_from_compressed_weights_to_hidden_states():
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    prompts, steps = [70, 3, 1, 129], 5
    w, ins, outs, _ = ex.run(256, 4, 2, 512, prompts, steps)
    want = plain(w, ins, prompts, 4, 2)
    start = np.concatenate([[0], np.cumsum(prompts)])
    for r, n in enumerate(prompts):
        got = np.concatenate([outs[0][start[r]:start[r + 1]].double().cpu().numpy()]
                             + [y[r:r + 1].double().cpu().numpy() for y in outs[1:]])
        # a bf16 rounding (2^-9 of each value) at each of about 12 places that feed the output, and keys and values
        # in steps of 1 / 127 of their block's largest (at most 4 times their rms: 0.5 * 4 / 127 / sqrt(3) of it each)
        rel = np.linalg.norm(got - want[r]) / np.linalg.norm(want[r])
        assert rel <= 12 * 2.0 ** -9 + 2 * 0.5 * 4 / 127, (r, rel)
