"""The example that runs the MXFP4 products, the 8-bit cache and its attention together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "mx_layer.py")
    spec = importlib.util.spec_from_file_location("mx_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(ex, layer, x, cache, table, ctx, n_new):
    """The layer in 64 bits for one sequence's last n_new tokens, with the packed weights' and the cache's own values."""
    import metalops_amd as mo
    W = {n: mo.dequantize_mxfp4(*p, torch.float32).double() for n, p in layer.packed.items()}
    K, V = (t[0, :ctx].double() for t in mo.kv8_read(cache, table, torch.tensor([ctx], dtype=torch.int32, device="cuda"), torch.float32))
    D, G = cache.head_dim, layer.heads // layer.kv_heads

    def norm(a, w):
        return a * torch.rsqrt(a.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double()
    x = x.double()
    q = (norm(x, layer.norms[0]) @ W["qkv"].T)[:, : layer.heads * D].view(-1, layer.heads, D)
    out = torch.empty_like(q)
    pos = ctx - n_new + torch.arange(n_new, device=x.device)
    for h in range(layer.heads):
        s = q[:, h] @ K[:, h // G].T.contiguous() / D ** 0.5
        s = s.masked_fill(torch.arange(ctx, device=x.device)[None] > pos[:, None], float("-inf"))
        out[:, h] = torch.softmax(s, -1) @ V[:, h // G]
    x = x + out.flatten(1) @ W["o"].T
    gate, up = (norm(x, layer.norms[1]) @ W["gate_up"].T).chunk(2, -1)
    return x + (torch.nn.functional.silu(gate) * up) @ W["down"].T


# Roundings to bf16 on the way to the output, each at most 2^-8 of its tensor's norm: norm, qkv, attention, o, sum, norm,
# gate_up, silu, product, down, sum; the scores' (2^-8 of q, at scores of a few units) count for four more.
TOL = 15 * 2.0 ** -8


@pytest.mark.parametrize("heads,kv_heads,D,page", [(8, 2, 64, 16), (4, 4, 128, 64)])
def test_layer(ex, heads, kv_heads, D, page):
    hidden, inner, steps, lengths = 512, 1056, 5, (77, 1, 130)
    layer = ex.MxLayer(ex.make_weights(hidden, heads, kv_heads, D, inner, "cuda"), heads, kv_heads)
    g = torch.Generator("cuda").manual_seed(1)
    prompts = [torch.randn(n, hidden, generator=g, device="cuda").bfloat16() for n in lengths]
    cache, table = ex.make_cache([n + steps for n in lengths], kv_heads, D, page, "cuda")
    first, _ = ex.generate(layer, prompts, 0, cache, table)
    at = 0
    for b, n in enumerate(lengths):
        want = plain(ex, layer, prompts[b], cache, table[b:b + 1], n, n)
        assert (first[at:at + n].double() - want).norm() <= TOL * want.norm()
        at += n
    # Tokens: the same prompts again, and the last token's output from the one before.
    cache, table = ex.make_cache([n + steps for n in lengths], kv_heads, D, page, "cuda")
    first2, tokens = ex.generate(layer, prompts, steps, cache, table)
    assert torch.equal(first, first2)
    for b, n in enumerate(lengths):
        want = plain(ex, layer, tokens[-2][b:b + 1], cache, table[b:b + 1], n + steps, 1)
        assert (tokens[-1][b:b + 1].double() - want).norm() <= TOL * want.norm()


def test_quantized_mlp(ex):
    """Inputs of the MLP in 4 bits: an element is off by 2^-2 of itself or of its block's scale, at most; two layers of that."""
    hidden, heads, D = 512, 4, 64
    weights = ex.make_weights(hidden, heads, heads, D, 1056, "cuda")
    x, outs = [torch.randn(40, hidden, device="cuda").bfloat16()], []
    for quantized in (False, True):
        cache, table = ex.make_cache([40], heads, D, 32, "cuda")
        outs.append(ex.generate(ex.MxLayer(weights, heads, heads, quantized), x, 0, cache, table)[0].float())
    assert (outs[0] - outs[1]).norm() <= 0.5 * outs[0].norm() and not torch.equal(*outs)
