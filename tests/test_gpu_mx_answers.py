"""The example in which answers share a prompt: products with epilogues, rotary positions, the pool and shared attention together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "mx_layer.py")
    spec = importlib.util.spec_from_file_location("mx_layer_answers", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(layer, x, cache, table, ctx):
    """The layer in 64 bits for the token at the end of one row of the table, with the packed weights' and the cache's own values."""
    import metalops_amd as mo
    W = {n: mo.dequantize_mxfp4(*p, torch.float32).double() for n, p in layer.packed.items()}
    K, V = (t[0, :ctx].double() for t in mo.kv8_read(cache, table, torch.tensor([ctx], dtype=torch.int32, device="cuda"), torch.float32))
    D, G = cache.head_dim, layer.heads // layer.kv_heads

    def norm(a, w, eps):
        return a * torch.rsqrt(a.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    x = x.double()
    q = (norm(x, layer.norms[0], 1e-5) @ W["qkv"].T)[:, : layer.heads * D].view(layer.heads, D)
    q = norm(q, layer.head_norms[0], 1e-6)
    turn = (ctx - 1) * layer.inv_freq.double()
    a, b = q.chunk(2, -1)
    q = torch.cat((a * turn.cos() - b * turn.sin(), b * turn.cos() + a * turn.sin()), -1)
    out = torch.stack([torch.softmax(q[h] @ K[:, h // G].T.contiguous() / D ** 0.5, -1) @ V[:, h // G] for h in range(layer.heads)])
    x = x + out.flatten()[None] @ W["o"].T
    y = norm(x, layer.norms[1], 1e-5)
    return x + (torch.nn.functional.silu(y @ W["gate"].T) * (y @ W["up"].T)) @ W["down"].T


# Roundings to bf16, each at most 2^-8 of its tensor's norm: norm, qkv, rotation, attention, o with its sum, norm, up, gated
# product, down with its sum; those of q before the scores count for six more at scores of a few units.
TOL = 15 * 2.0 ** -8


@pytest.mark.parametrize("heads,kv_heads,D,page,prompt", [(8, 2, 64, 16, 77), (4, 4, 128, 64, 130), (8, 4, 128, 16, 64), (4, 2, 64, 32, 5)])
def test_answers(ex, heads, kv_heads, D, page, prompt):
    import metalops_amd as mo
    hidden, inner, steps = 512, 1056, 20
    layer = ex.AnswersLayer(ex.make_weights(hidden, heads, kv_heads, D, inner, "cuda"), heads, kv_heads, D)
    g = torch.Generator("cuda").manual_seed(2)
    text, first = (torch.randn(n, hidden, generator=g, device="cuda").bfloat16() for n in (prompt, 5))
    pool = mo.KV8Pool.empty(1, 40, kv_heads, D, page)
    outs, table, lens = ex.answers(layer, text, first, steps, pool, {7: [3, 3, 0, 4], 13: [1, -1, 3, 1]})
    assert [len(x) for x in outs] == [5] * 7 + [4] * 6 + [3] * 7 and lens.tolist() == [prompt + steps] * 3
    for b in range(3):
        want = plain(layer, outs[-2][b:b + 1], pool.caches[0], table[b:b + 1], prompt + steps)
        assert (outs[-1][b:b + 1].double() - want).norm() <= TOL * want.norm()
    # Two answers with one parent remain alike; refs are how many entries of the table name each page.
    assert torch.equal(outs[-1][0], outs[-1][2])
    named = torch.bincount(table[table >= 0].long(), minlength=40).int()
    assert torch.equal(named, pool.refs) and int((pool.refs > 0).sum()) >= -(-(prompt + steps) // page)
    assert int(mo.kv8_resize(pool, table, lens, torch.zeros_like(lens))) == 0 and not pool.refs.any() and (table == -1).all()


def test_answers_are_those_of_copies(ex):
    """Answers of a shared prompt against the same ones with kv8_attention, whose parts have another order: the last token's
    output differs by roundings only."""
    import metalops_amd as mo
    hidden, heads, kv_heads, D, page, prompt, steps = 512, 8, 2, 64, 16, 100, 3
    layer = ex.AnswersLayer(ex.make_weights(hidden, heads, kv_heads, D, 1056, "cuda"), heads, kv_heads, D)
    g = torch.Generator("cuda").manual_seed(3)
    text, first = (torch.randn(n, hidden, generator=g, device="cuda").bfloat16() for n in (prompt, 6))
    outs, _, _ = ex.answers(layer, text, first, steps, mo.KV8Pool.empty(1, 32, kv_heads, D, page))
    for b in (0, 5):
        alone, _, _ = ex.answers(layer, text, first[b:b + 1], steps, mo.KV8Pool.empty(1, 32, kv_heads, D, page))
        for i in range(steps):
            assert (outs[i][b].float() - alone[i][0].float()).norm() <= 2 * (i + 1) * TOL * alone[i][0].float().norm()


def test_captured_step(ex):
    """A step captured into a graph: pages, rotation, append, attention and products, replayed as often as there are tokens."""
    import metalops_amd as mo
    hidden, heads, kv_heads, D, page, prompt, steps, n = 512, 8, 2, 64, 16, 70, 24, 6
    layer = ex.AnswersLayer(ex.make_weights(hidden, heads, kv_heads, D, 1056, "cuda"), heads, kv_heads, D)
    g = torch.Generator("cuda").manual_seed(4)
    text, first = (torch.randn(k, hidden, generator=g, device="cuda").bfloat16() for k in (prompt, n))
    results = []
    for captured in (False, True):
        pool = mo.KV8Pool.empty(1, 32, kv_heads, D, page)
        table = pool.table(1, -(-(prompt + steps) // page))
        lens, none = (torch.full((1,), k, dtype=torch.int32, device="cuda") for k in (prompt, 0))
        mo.kv8_resize(pool, table, none, lens)
        layer(text, pool.caches[0], table, none, lens, None, prompt, torch.arange(prompt, dtype=torch.int32, device="cuda"))
        table, lens = mo.kv8_fork(pool, table, lens, torch.zeros(n, dtype=torch.int32, device="cuda"), release=True)
        x, lacking = first.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")

        def step():
            more = lens + 1
            lacking.add_(mo.kv8_resize(pool, table, lens, more))
            x.copy_(layer(x, pool.caches[0], table, lens, more, None, prompt + steps, lens, prompt // page))
            lens.copy_(more)
        outs = []
        if captured:
            held = [t.clone() for t in (table, lens, x, pool.refs)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            for t, h in zip((table, lens, x, pool.refs), held):
                t.copy_(h)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        for i in range(steps):
            graph.replay() if captured else step()
            outs.append(x.clone())
            if i % 5 == 0:
                torch.cuda.synchronize()
                ex.rms_norm(x, layer.norms[0])
        assert lacking.item() == 0 and lens.tolist() == [prompt + steps] * n
        results.append((torch.stack(outs), table.clone(), pool.refs.clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)
