"""A small decoder stack served end to end: the split FFN next to attention on the 8-bit paged cache.

    python examples/decoder_layers.py [--layers 4] [--prompt 200] [--samples 3] [--steps 16]

Two prompts are prefilled as one ragged batch, each is forked into samples that share its pages, the
samples are decoded token by token (one CUDA-graph-free step = reserve, then per layer norm, q/k/v,
append, attend, output product, norm, split FFN), half of them are then dropped, the pool is
compacted and decoding goes on. Weights are random; the next token of each sample is drawn from
a seeded table of embeddings.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

if str(Path(__file__).resolve().parents[1]) not in sys.path:
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch

from ffn_residual_mesh_b200 import synth
from ffn_residual_mesh_b200.engine import LayerSpec, ResidualMesh
from ffn_residual_mesh_b200.kvcache import PagedKvCache, RotaryTable


def norm(x):
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).half()


def quantise(x):
    """Groupwise int8 activations on the device (formats.quantize_groupwise_q8's rule)."""
    g = x.float().view(x.shape[0], -1, 32)
    s = torch.maximum(g.abs().amax(-1) / torch.tensor(127.0, device=x.device), torch.tensor(1e-12, device=x.device))
    return (g / s[..., None]).round().clamp(-128, 127).to(torch.int8).view(x.shape), s.contiguous()


class Decoder:
    """``layers`` decoder layers of d_model ``heads * head_dim``."""

    def __init__(self, layers=4, heads=8, kv_heads=2, head_dim=64, d_ff=256, max_tokens=512, pages=256, page_tokens=16, seed=0):
        self.layers, self.heads, self.kv_heads, self.head_dim = layers, heads, kv_heads, head_dim
        d = heads * head_dim
        self.ffn = ResidualMesh(d, d_ff, 2, layers, max_tokens, base_tile_rows=64)
        self.unsplit = torch.ones(-(-d_ff // 64), dtype=torch.uint8, device="cuda")  # every row tile flagged
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.qkv, self.out = [], []
        for i in range(layers):
            w = synth.make_layer(seed + i, d_ff, d)
            self.ffn.load_layer(i, LayerSpec(w.gate_codes, w.up_codes, w.gate_alpha, w.up_alpha, w.down, w.gate_beta, w.up_beta,
                                             keep_fallback=True))
            self.qkv.append((torch.randn(d, (heads + 2 * kv_heads) * head_dim, device="cuda", generator=g) * d ** -0.5).half())
            self.out.append((torch.randn(d, d, device="cuda", generator=g) * d ** -0.5).half())
        self.cache = PagedKvCache(layers, pages, kv_heads, head_dim, page_tokens=page_tokens, max_seqs=64)
        self.rope = RotaryTable(head_dim, pages * page_tokens)
        self.embed = torch.randn(1000, d, device="cuda", generator=g).half()

    def ffn_layer(self, i, x):
        """The split FFN with its base sums in HBM: unsplit projection minus residual."""
        z, s = quantise(x)
        full, low = ([torch.empty(x.shape[0], self.ffn.d_ff, device="cuda") for _ in range(2)] for _ in range(2))
        self.ffn.residual(i, z, s, *full, fallback_tiles=self.unsplit)
        self.ffn.residual(i, z, s, *low)
        y = torch.empty_like(x)
        self.ffn.forward(i, z, s, full[0] - low[0], full[1] - low[1], y16=y)
        return y

    def step(self, tokens, tables, lengths, starts=None):
        """Hidden states of the step's tokens (ids, one row each) after all layers."""
        x = self.embed[tokens]
        H, K = self.heads, self.kv_heads
        for i in range(self.layers):
            qkv = (norm(x) @ self.qkv[i]).view(len(tokens), H + 2 * K, self.head_dim)
            q = self.cache.append(i, qkv[:, H:H + K], qkv[:, H + K:], tables, lengths, starts=starts, rope=self.rope, q=qkv[:, :H])
            a = self.cache.attend(i, q, tables, lengths, starts=starts)
            x = x + a.view(len(tokens), -1) @ self.out[i]
            x = x + self.ffn_layer(i, norm(x))
        return x


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run(layers=4, prompt=200, samples=3, steps=16, seed=0, **kw):
    """Returns the last hidden states, tables, lengths and page counts."""
    model = Decoder(layers, seed=seed, **kw)
    cache, g = model.cache, torch.Generator(device="cuda").manual_seed(seed + 1)
    lens = [prompt, max(1, prompt // 3)]
    # two empty sequences with room for the prompts
    width = -(-(prompt + 2 * steps) // cache.page_tokens)
    tables, lengths = torch.full((2, width), -1, dtype=torch.int32, device="cuda"), ints([0, 0])
    tables, lengths, _ = cache.fork(tables, lengths, ints([-1, -1]), ints(lens))
    x = model.step(torch.randint(0, 1000, (sum(lens),), device="cuda", generator=g), tables, lengths, ints([0, lens[0], sum(lens)]))
    parents = [0] * samples + [1] * samples  # samples of each prompt share its pages
    for t in range(2 * steps):
        if t == steps:  # keep the first sample of each prompt, hand the other pages back, close the gaps
            parents = [0, samples]
        tables, lengths, info = cache.fork(tables, lengths, ints(parents), ints([1] * len(parents)))
        if t == steps:
            tables, info = cache.compact(tables, lengths)
        ids = torch.randint(0, 1000, (2,), device="cuda", generator=g).repeat_interleave(len(parents) // 2)
        x = model.step(ids, tables, lengths)
        parents = list(range(len(parents)))
        if t == steps - 1:
            before = x
    cache.check()
    model.ffn.check_device_error()
    return {"samples": before, "last": x, "tables": tables, "lengths": lengths, "info": info}


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 4), ("prompt", 200), ("samples", 3), ("steps", 16)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    start = time.perf_counter()
    r = run(a.layers, a.prompt, a.samples, a.steps)
    torch.cuda.synchronize()
    print(f"{a.layers} layers, two prompts, {2 * a.samples} samples, {2 * a.steps} steps in {time.perf_counter() - start:.2f} s; "
          f"sequences hold {r['lengths'].tolist()} tokens in pages {r['tables'].max().item() + 1} of the pool at most")


if __name__ == "__main__":
    main()
