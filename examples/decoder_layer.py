"""A decoder layer from its compressed weights to hidden states: the layer's
LZ4 blocks of HCT-T tiles are decoded on the GPU in one launch, and requests
of several lengths run through it with the operators of haagenti_amd.compute
-- a prompt first, then one token at a time -- over a paged 8-bit cache.

    python examples/decoder_layer.py [--hidden 4096 --heads 32 --kv-heads 8 --ffn 14336 --theta 500000]

Weights are random (there is no checkpoint to load); norms have no weight, and
positions are left out without --theta."""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import haagenti_amd as H  # noqa: E402
import haagenti_amd.compute as K  # noqa: E402


def shapes(hidden, heads, kv_heads, ffn):
    dim = hidden // heads
    return dict(qkv=((heads + 2 * kv_heads) * dim, hidden), o=(hidden, hidden), gate=(ffn, hidden), up=(ffn, hidden),
                down=(hidden, ffn))


def encode(weights, retention):
    """LZ4 blocks of whole tiles, tensor after tensor: (bytes, block lengths, [(rows, cols, k, tiles per block)])."""
    k = H.hctt_retain_count(retention)
    per = H.FUSED_BLOCK_BYTES // H.hctt_tile_bytes(k)
    lz4, blocks, tensors = H.Lz4Compressor(), [], []
    for w in weights.values():
        tiles = H.hctt_encode(w, k).tobytes()
        step = per * H.hctt_tile_bytes(k)
        blocks += [lz4.compress(tiles[a:a + step]) for a in range(0, len(tiles), step)]
        tensors.append((w.shape[0], w.shape[1], k, per))
    return b"".join(blocks), [len(b) for b in blocks], tensors


def decode(ctx, names, blob, lens, tensors):
    """The layer's weights in bf16, in one launch."""
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a).view(t)).cuda()  # noqa: E731
    offs = np.concatenate([[0], np.cumsum(lens)[:-1]]).astype(np.uint64)
    outs = {n: torch.empty(r, c, dtype=torch.bfloat16, device="cuda") for n, (r, c, _, _) in zip(names, tensors)}
    status = torch.zeros(len(lens) * 32, dtype=torch.uint8, device="cuda")
    rc = ctx.hctt_decode_lz4_fused(
        dev(np.frombuffer(blob, np.uint8).copy(), np.uint8), len(blob), dev(offs, np.int64),
        dev(np.asarray(lens, np.uint32), np.int32), len(lens), status,
        [(r, c, k, outs[n]) for n, (r, c, k, _) in zip(names, tensors)], [t[3] for t in tensors], dtype=H.BF16,
        stream=torch.cuda.current_stream().cuda_stream)
    if rc != H.OK or status.cpu().numpy().view(np.int32)[0::8].any():
        raise RuntimeError(f"layer decode failed: {rc}")
    return outs


class Layer:
    def __init__(self, ctx, weights, heads, kv_heads, blocks, block_size=64, requests=4, width=64, theta=None):
        self.ctx, self.w, self.heads, self.kv_heads = ctx, weights, heads, kv_heads
        self.dim = weights["o"].shape[0] // heads
        self.cache = K.KvCache.create(ctx, blocks, block_size, kv_heads, self.dim)
        self.ring, self.state = K.free_ring(blocks)
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        pairs = self.dim // 2
        self.inv_freq = None if theta is None else float(theta) ** (-torch.arange(pairs, device="cuda") / pairs)

    def step(self, x, new, max_q, max_kv):
        """Hidden states x of the requests' new tokens (new per request) through the layer."""
        ctx, w, h, kv, d = self.ctx, self.w, self.heads, self.kv_heads, self.dim
        plan = K.kv_plan(ctx, self.lens, new, self.table, self.ring, self.state, self.cache.block_size, x.shape[0])
        qkv = K.linear(ctx, K.norm(ctx, x, kind="rms"), w["qkv"]).view(-1, h + 2 * kv, d)
        if self.inv_freq is not None:       # queries and keys turn by their place in their request
            first = torch.repeat_interleave(self.lens - plan.start[:-1], new, output_size=x.shape[0])
            at = first + torch.arange(x.shape[0], dtype=torch.int32, device="cuda")
            K.rotary(ctx, qkv[:, :h + kv], at, self.inv_freq, out=qkv[:, :h + kv])
        self.cache.append(qkv[:, h:h + kv], qkv[:, h + kv:], plan.slots)
        o = self.cache.attention(qkv[:, :h], self.table, plan.start, plan.kv_len, max_q=max_q, max_kv=max_kv)
        x = K.linear(ctx, o.view(-1, h * d), w["o"], residual=x)
        y = K.gated_linear(ctx, K.norm(ctx, x, kind="rms"), w["gate"], w["up"], act="silu")
        self.lens, self.state = plan.kv_len, plan.state
        return K.linear(ctx, y, w["down"], residual=x)


def run(hidden, heads, kv_heads, ffn, prompts, steps, retention=0.3, seed=0, theta=None):
    """Prompts of these lengths, then `steps` tokens each; returns (the weights decoded, the inputs of every step, the
    outputs of every step, milliseconds per single-token step)."""
    rng = np.random.default_rng(seed)
    ctx = H.HipContext(0)
    sh = shapes(hidden, heads, kv_heads, ffn)
    host = {n: rng.normal(0, 0.02, s).astype(np.float32) for n, s in sh.items()}
    weights = decode(ctx, list(sh), *encode(host, retention))
    longest = max(prompts) + steps
    blocks = sum((p + steps + 63) // 64 for p in prompts)
    layer = Layer(ctx, weights, heads, kv_heads, blocks, 64, len(prompts), (longest + 63) // 64, theta)
    ins, outs, t0 = [], [], 0.0
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for i in range(steps + 1):
        new = prompts if i == 0 else [1] * len(prompts)
        x = torch.randn(sum(new), hidden, generator=gen, device="cuda").to(torch.bfloat16)
        new = torch.tensor(new, dtype=torch.int32, device="cuda")
        if i == 1:
            torch.cuda.synchronize()
            t0 = time.perf_counter()
        ins.append(x)
        outs.append(layer.step(x, new, max(prompts) if i == 0 else 1, longest))
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t0) / max(steps, 1) * 1e3 if steps else 0.0
    return weights, ins, outs, ms


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("hidden", 1024), ("heads", 8), ("kv-heads", 2), ("ffn", 3584), ("steps", 32)):
        p.add_argument("--" + name, type=int, default=value)
    p.add_argument("--prompts", type=int, nargs="+", default=[200, 31, 1, 500])
    p.add_argument("--theta", type=float, default=None)
    a = p.parse_args()
    _, _, outs, ms = run(a.hidden, a.heads, a.kv_heads, a.ffn, a.prompts, a.steps, theta=a.theta)
    print(f"{len(a.prompts)} prompts of {a.prompts} tokens and {a.steps} steps: {ms:.3f} ms a step, "
          f"hidden states of rms {float(outs[-1].float().square().mean().sqrt()):.3f}")


if __name__ == "__main__":
    main()
