"""A transformer layer with MXFP4 weights and an 8-bit key/value cache: a prompt, then tokens one at a time.

    python examples/mx_layer.py

Weights are quantized once and used by ``matmul_mxfp4``; with ``quantized_mlp`` the MLP's inputs are
quantized too (``matmul_mxfp4_mxfp4``).  Keys and values go to pages with ``kv8_append`` and are read by
``kv8_attention``, the same calls for prompts (``cu_seqlens``) and for single tokens.
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import metalops_amd as mo  # noqa: E402


def rms_norm(x, weight, eps=1e-5):
    f = x.float()
    return (f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + eps) * weight).to(x.dtype)


class MxLayer:
    """x + attention(norm(x)), then x + mlp(norm(x)); weights [out, in] as a checkpoint holds them."""

    def __init__(self, weights, heads, kv_heads, quantized_mlp=False):
        self.heads, self.kv_heads, self.quantized_mlp = heads, kv_heads, quantized_mlp
        self.norms = [w.float() for w in (weights["norm1"], weights["norm2"])]
        self.packed = {n: mo.quantize_mxfp4(weights[n]) for n in ("qkv", "o", "gate_up", "down")}

    def linear(self, name, x):
        if self.quantized_mlp and name in ("gate_up", "down"):
            return mo.matmul_mxfp4_mxfp4(*mo.quantize_mxfp4(x), *self.packed[name], x.dtype)
        return mo.matmul_mxfp4(x, *self.packed[name])

    def __call__(self, x, cache, table, before, after, cu_seqlens=None, max_context=0):
        """x [T, hidden]: new tokens of table's sequences, which hold ``before`` tokens and then ``after``."""
        D = cache.head_dim
        qkv = self.linear("qkv", rms_norm(x, self.norms[0])).view(len(x), -1, D)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)
        mo.kv8_append(cache, k, v, table, before, cu_seqlens)
        y = mo.kv8_attention(q, cache, table, after, cu_seqlens, max_context=max_context)
        x = x + self.linear("o", y.flatten(1))
        gate, up = self.linear("gate_up", rms_norm(x, self.norms[1])).chunk(2, -1)
        return x + self.linear("down", torch.nn.functional.silu(gate) * up)


def make_weights(hidden, heads, kv_heads, head_dim, inner, device, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device).manual_seed(seed)

    def w(n, k):
        return (torch.randn(n, k, generator=g, device=device) / k ** 0.5).to(dtype)
    return {"qkv": w((heads + 2 * kv_heads) * head_dim, hidden), "o": w(hidden, heads * head_dim), "gate_up": w(2 * inner, hidden),
            "down": w(hidden, inner), "norm1": torch.ones(hidden, device=device), "norm2": torch.ones(hidden, device=device)}


def make_cache(lengths, kv_heads, head_dim, page, device):
    """A cache for sequences of up to ``lengths`` tokens, their pages dealt out in turn, and the block table."""
    width, free = max(-(-n // page) for n in lengths), 0
    table = torch.zeros(len(lengths), width, dtype=torch.int32)
    for j in range(width):
        for b, n in enumerate(lengths):
            if j * page < n:
                table[b, j] = free
                free += 1
    return mo.KV8Cache.empty(free, kv_heads, head_dim, page, device), table.to(device)


def generate(layer, prompts, steps, cache, table):
    """The layer's outputs for the prompts (a list of [n, hidden]) and for ``steps`` tokens after each: a
    token's output is the next one's input."""
    device = table.device
    n = torch.tensor([len(p) for p in prompts], dtype=torch.int32)
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), n.cumsum(0, dtype=torch.int32)]).to(device)
    lens, longest = n.to(device), int(n.max())
    first = layer(torch.cat(prompts), cache, table, torch.zeros_like(lens), lens, cu, longest)
    x, tokens = first[(cu[1:] - 1).long()], []
    for i in range(steps):
        x = layer(x, cache, table, lens, lens + 1, None, longest + i + 1)
        lens = lens + 1
        tokens.append(x)
    return first, tokens


def main():
    device, hidden, heads, kv_heads, D, inner, page = "cuda", 4096, 32, 8, 128, 14336, 64
    lengths, steps = (2000, 700, 1, 1333), 64
    weights = make_weights(hidden, heads, kv_heads, D, inner, device)
    for quantized_mlp in (False, True):
        layer = MxLayer(weights, heads, kv_heads, quantized_mlp)
        prompts = [torch.randn(n, hidden, device=device).bfloat16() for n in lengths]
        for timed in (False, True):
            cache, table = make_cache([n + steps for n in lengths], kv_heads, D, page, device)
            torch.cuda.synchronize()
            t = time.perf_counter()
            generate(layer, prompts, steps, cache, table)
            torch.cuda.synchronize()
        t = time.perf_counter() - t
        print("%s activations in the MLP: %d prompt tokens and %d x %d tokens through a layer in %.1f ms; cache %.1f MB"
              % ("4-bit" if quantized_mlp else "bf16", sum(lengths), steps, len(lengths), 1e3 * t,
                 sum(x.numel() for x in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)) / 1e6), flush=True)


if __name__ == "__main__":
    main()
