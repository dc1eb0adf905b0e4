"""Performance cases of the microscaled operators: 4-bit weights and activations, 8-bit key/value cache.

The listed cases are the steps of serving a model whose linear layers hold 4-bit
microscaled weights (MXFP4: blocks of 32 e2m1 values with a power-of-two scale) and
whose attention reads a paged cache of e4m3 values with a power-of-two scale for each
page and head: weights converted at load time, products of decode and prefill, tokens
appended to the cache, attention of single tokens and of prompts.  ``draw`` gives
further cases of the same ranges.

``run`` has two forms.  Where ``own`` is false it computes in elementary torch
operations, in fp32; where it is true it makes a user's calls of metalops_amd.
``exact`` computes the definition in 64 bits, with code of its own.
"""
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_ES = {"f16": 2, "bf16": 2, "f32": 4}
_DEV = "cuda"
# No drawn case does more than the largest listed one of its kind.
_MOST_FLOPS = 2 * 2048 * 4096 * 14336
_MOST_FLOPS_F32 = _MOST_FLOPS // 16
_MOST_WEIGHTS = 4096 * 14336
_MOST_NEW = 2048 * 3 * 8 * 128            # elements of K that one append adds
_MOST_CONTEXT = 131072 * 8 * 128          # elements of K that one attention reads


def _text(values):
    """One number for each sequence, as a case holds them."""
    return " ".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split()]


def listed():
    return [
        # Loading a model: a bf16 nn.Linear weight converted, and expanded again for a layer that stays dense.
        {"name": "load_linear", "op": "load", "x": "bf16", "out": "bf16", "layout": "nk", "N": 14336, "K": 4096},
        # An fp32 weight held [K, N], as the q4_0 functions take it, of an odd width.
        {"name": "load_kn_odd", "op": "load", "x": "f32", "out": "f16", "layout": "kn", "N": 1001, "K": 4096},
        # The smallest product: one attention output projection of a decode step.
        {"name": "w4_o_m1", "op": "w4", "x": "f16", "M": 1, "K": 4096, "N": 4096},
        # Batched decode, long K: the down projection of 16 sequences.
        {"name": "w4_down_m16", "op": "w4", "x": "bf16", "M": 16, "K": 14336, "N": 4096},
        # Prefill of a long prompt: the largest product.
        {"name": "w4_up_m2048", "op": "w4", "x": "f16", "M": 2048, "K": 4096, "N": 14336},
        # The same prefill with the activations microscaled too: converted, then multiplied in 4 bits.
        {"name": "w4a4_up_m2048", "op": "w4a4", "x": "bf16", "M": 2048, "K": 4096, "N": 14336},
        # A short prompt with sizes that are whole tiles of nothing.
        {"name": "w4a4_ragged_m77", "op": "w4a4", "x": "f16", "M": 77, "K": 4128, "N": 1001},
        # Prompts of three sequences written to an empty cache.
        {"name": "append_prompts", "op": "append", "x": "bf16", "new": "2048 2048 1025", "start": "0 0 0",
         "heads": 8, "D": 128, "page": 64},
        # A decode step of 64 sequences: one token each, into pages that hold some already.
        {"name": "append_token_b64", "op": "append", "x": "f16", "new": _text([1] * 64),
         "start": _text((i * 37) % 1000 for i in range(64)), "heads": 8, "D": 128, "page": 64},
        # One user's decode step behind a long context.
        {"name": "attend_b1_32k", "op": "attend", "x": "bf16", "new": "1", "context": "32768", "heads": 8, "group": 4,
         "D": 128, "page": 64, "window": 0},
        # A decode step of a batch with contexts of every length.
        {"name": "attend_b32_ragged", "op": "attend", "x": "f16", "new": _text([1] * 32),
         "context": _text(1 + (i * 2477) % 8192 for i in range(32)), "heads": 8, "group": 4, "D": 128, "page": 64,
         "window": 0},
        # Prompts: a fresh one, and one that continues a context already in the cache.
        {"name": "attend_prompts", "op": "attend", "x": "bf16", "new": "2048 1500", "context": "4096 1500",
         "heads": 8, "group": 4, "D": 128, "page": 64, "window": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Column counts: whole tiles, multiples of 8, and odd ones."""
    r = rng.random()
    if r < 0.5:
        return 128 * _log(rng, max(1, lo // 128), hi // 128)
    return 8 * _log(rng, lo // 8, hi // 8) if r < 0.75 else _log(rng, lo, hi)


def draw(rng):
    op = rng.choice(["load", "w4", "w4", "w4", "w4a4", "w4a4", "append", "attend", "attend", "attend"])
    x = rng.choice(["f16", "bf16"])
    if op in ("load", "w4", "w4a4"):
        K = 128 * _log(rng, 4, 112) if rng.random() < 0.6 else 32 * _log(rng, 16, 448)
        N = _width(rng, 512, 14336)
        if op == "load":
            x, out = rng.choice(["f32", "f16", "bf16"]), rng.choice(["f32", "f16", "bf16"])
            N = max(1, min(N, _MOST_WEIGHTS * 4 // (K * (_ES[x] + _ES[out]))))
            return {"op": op, "x": x, "out": out, "layout": rng.choice(["nk", "nk", "kn"]), "N": N, "K": K}
        if op == "w4" and rng.random() < 0.2:
            x = "f32"
        most = _MOST_FLOPS_F32 if x == "f32" else _MOST_FLOPS
        return {"op": op, "x": x, "M": max(1, min(_log(rng, 1, 2048), most // (2 * K * N))), "K": K, "N": N}
    D, page = rng.choice([64, 80, 96, 128, 128, 128, 256]), rng.choice([16, 32, 64, 64, 128])
    heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    if op == "append":
        B = _log(rng, 1, 64)
        longest = 1 if rng.random() < 0.5 else max(1, min(_log(rng, 2, 2048), _MOST_NEW // (B * heads * D)))
        new = [rng.randint(1, longest) for _ in range(B)]
        start = [0 if rng.random() < 0.3 else rng.randint(1, 2000) for _ in range(B)]
        return {"op": op, "x": rng.choice(["f32", "f16", "bf16", "bf16"]), "new": _text(new), "start": _text(start), "heads": heads,
                "D": D, "page": page}
    group = rng.choice([1, 2, 4, 4, 7, 8, 16])
    while heads * group > 64:
        group //= 2
    window = 0 if rng.random() < 0.75 else _log(rng, 16, 4096)
    if rng.random() < 0.65:                  # decode, sometimes with a few drafted tokens
        B = _log(rng, 1, 64)
        longest = max(1, min(_log(rng, 64, 32768), _MOST_CONTEXT // (B * heads * D)))
        n = 1 if rng.random() < 0.7 else rng.randint(2, 8)
        # A slot that serves nobody has a context of zero.
        context = [0 if rng.random() < 0.05 else max(n, rng.randint(1, longest)) for _ in range(B)]
        new = [n] * B
    else:
        B = _log(rng, 1, 4)
        longest = _log(rng, 16, 2048)
        new = [rng.randint(1, longest) for _ in range(B)]
        context = [n + (0 if rng.random() < 0.5 else rng.randint(0, 2048)) for n in new]
        scale = sum(n * c for n, c in zip(new, context)) * 4 * heads * group * D / (_MOST_FLOPS / 2)
        if scale > 1:
            new = [max(1, int(n / scale)) for n in new]
            context = [n + max(0, c - n) for n, c in zip(new, context)]
    return {"op": op, "x": x, "new": _text(new), "context": _text(context), "heads": heads, "group": group, "D": D,
            "page": page, "window": window}


# ---- the formats, in plain torch -----------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(byte):
    """2^(byte - 127) in fp32 of a tensor of whole numbers 0..254; NaN for 255."""
    byte = byte.to(torch.int32)
    f = torch.where(byte == 0, torch.full_like(byte, 0x00400000), byte << 23)
    return torch.where(byte == 255, torch.full_like(byte, 0x7FC00000), f).view(torch.float32)


def _biased_exponent(amax):
    return (amax.float().view(torch.int32) >> 23) & 255


def _mx_quantize(x):
    """[..., K] -> e2m1 codes 0..15 [..., K] and scale bytes [..., K/32]."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    byte = (_biased_exponent(b.abs().amax(-1)) - 2).clamp(0, 254)
    v = b * _pow2(254 - byte)[..., None]
    a = v.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    # Halfway values go to the even code.
    for i, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a >= t) if i % 2 else (a > t)
    code |= (v < 0).to(torch.uint8) << 3
    return code.reshape(x.shape), byte.to(torch.uint8)


def _mx_pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _mx_values(code, byte):
    """Codes and scale bytes to the fp32 values they stand for."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=code.device)
    v = table[code.long()].reshape(*code.shape[:-1], -1, 32)
    return (v * _pow2(byte)[..., None]).reshape(code.shape)


def _mx_unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)


def _kv_byte(amax):
    """The smallest scale that leaves nothing above e4m3's 448."""
    bits = amax.float().view(torch.int32)
    return (((bits >> 23) & 255) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 247)


def _e4m3(x):
    return x.to(torch.float8_e4m3fn)


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=_DEV) * std).to(dtype)


def _activations(g, *shape, dtype=torch.float32):
    """Normal values with a few channels that are several times larger, as hidden states have them."""
    x = torch.randn(*shape, generator=g, device=_DEV)
    big = 1 + 7 * (torch.rand(shape[-1], generator=g, device=_DEV) < 0.02)
    return (x * big).to(dtype)


def _pages(g, B, width, spare=3):
    """A block table [B, width] of pages in no order, and how many pages there are."""
    P = B * width + spare
    return torch.randperm(P, generator=g, device=_DEV)[:B * width].reshape(B, width).to(torch.int32), P


def _filled(g, P, heads, page, D):
    """Cache tensors whose pages hold keys or values of ordinary sizes."""
    codes = torch.empty(P, heads, page, D, dtype=torch.uint8, device=_DEV)
    byte = torch.empty(P, heads, dtype=torch.uint8, device=_DEV)
    step = max(1, (1 << 26) // (heads * page * D))
    for i in range(0, P, step):
        x = _activations(g, min(step, P - i), heads, page, D)
        b = _kv_byte(x.abs().amax((-1, -2)))
        codes[i:i + step] = _e4m3(x * _pow2(254 - b)[..., None, None]).view(torch.uint8)
        byte[i:i + step] = b.to(torch.uint8)
    return codes, byte


def _lens(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _cumulative(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return _lens(out)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    st = {"case": case}
    if op == "load":
        shape = (case["N"], case["K"]) if case["layout"] == "nk" else (case["K"], case["N"])
        st["weight"] = _randn(g, *shape, dtype=_DT[case["x"]], std=0.02)
        return st
    if op in ("w4", "w4a4"):
        st["x"] = _activations(g, case["M"], case["K"], dtype=_DT[case["x"]])
        code, st["scales"] = _mx_quantize(_randn(g, case["N"], case["K"], std=0.02))
        st["packed"] = _mx_pack(code)
        return st
    heads, D, page, new = case["heads"], case["D"], case["page"], _ints(case["new"])
    B = len(new)
    start = _ints(case["start"]) if op == "append" else None
    context = _ints(case["context"]) if op == "attend" else [s + n for s, n in zip(start, new)]
    st["table"], P = _pages(g, B, max(1, -(-max(context) // page)))
    kc, kb = _filled(g, P, heads, page, D)
    vc, vb = _filled(g, P, heads, page, D)
    # Keys are held token by token, values channel by channel.
    st["cache"] = (kc, vc.transpose(2, 3).contiguous(), kb, vb)
    st["context"] = _lens(context)
    # Sequences that add equally many tokens need no offsets.
    st["cu"] = None if len(set(new)) == 1 else _cumulative(new)
    T = sum(new)
    if op == "attend":
        st["q"] = _randn(g, T, heads * case["group"], D, dtype=_DT[case["x"]], std=1.5)
        st["max_context"] = max(context)
        st["lens"] = list(zip(new, context))
    else:
        st["k"] = _activations(g, T, heads, D, dtype=_DT[case["x"]])
        st["v"] = _randn(g, T, heads, D, dtype=_DT[case["x"]])
        st["start"] = _lens(start)
        # The pages that the new tokens fall into, and how far those are filled afterwards.
        first = [s // page for s in start]
        width = max(-(-c // page) - f for c, f in zip(context, first))
        cols = (torch.tensor(first, device=_DEV)[:, None] + torch.arange(width, device=_DEV)).clamp(max=st["table"].shape[1] - 1)
        st["tail"] = st["table"].gather(1, cols)
        st["tail_lens"] = _lens([c - f * page for c, f in zip(context, first)])
    if own:
        import metalops_amd as mo
        st["cache"] = mo.KV8Cache(*st["cache"])
    return st


# ---- one pass ------------------------------------------------------------------------------------

def _run_own(st):
    import metalops_amd as mo
    case = st["case"]
    op = case["op"]
    if op == "load":
        w = st["weight"] if case["layout"] == "nk" else st["weight"].t()
        return mo.dequantize_mxfp4(*mo.quantize_mxfp4(w), _DT[case["out"]])
    if op == "w4":
        return mo.matmul_mxfp4(st["x"], st["packed"], st["scales"])
    if op == "w4a4":
        return mo.matmul_mxfp4_mxfp4(*mo.quantize_mxfp4(st["x"]), st["packed"], st["scales"], dtype=_DT[case["x"]])
    if op == "append":
        mo.kv8_append(st["cache"], st["k"], st["v"], st["table"], st["start"], cu_seqlens=st["cu"])
        return mo.kv8_read(st["cache"], st["tail"], st["tail_lens"], dtype=torch.bfloat16)
    return mo.kv8_attention(st["q"], st["cache"], st["table"], st["context"], cu_seqlens=st["cu"],
                            window=case["window"], max_context=st["max_context"])


def _token_rows(st):
    """For each new token its sequence, and where it stands among that sequence's new ones."""
    B = st["table"].shape[0]
    T = (st["k"] if "k" in st else st["q"]).shape[0]
    at = torch.arange(T, device=_DEV)
    if st["cu"] is None:
        return at // (T // B), at % (T // B)
    seq = torch.repeat_interleave(torch.arange(B, device=_DEV), st["cu"].diff().long())
    return seq, at - st["cu"][:-1].long()[seq]


def _plain_append(st, x, codes, byte, by_channel):
    """Tokens x [T, heads, D] into pages: codes [P, heads, page, D] (or [P, heads, D, page]) and scales, in place."""
    page = st["case"]["page"]
    seq, nth = _token_rows(st)
    pos = st["start"].long()[seq] + nth
    ids, inv = torch.unique(st["table"].long()[seq, pos // page], return_inverse=True)
    amax = torch.zeros(len(ids), x.shape[1], device=_DEV)
    amax.scatter_reduce_(0, inv[:, None].expand(-1, x.shape[1]), x.float().abs().amax(-1), "amax")
    older = torch.zeros(len(ids), dtype=torch.bool, device=_DEV)
    older[inv] = pos // page * page < st["start"].long()[seq]
    was = byte[ids].int()
    now = _kv_byte(amax)
    now = torch.where(older[:, None], torch.maximum(was, now), now)
    shrink = torch.where(older[:, None], _pow2(127 + was - now), torch.ones_like(amax))
    pages = codes[ids].transpose(2, 3) if by_channel else codes[ids]
    pages = _e4m3(pages.contiguous().view(torch.float8_e4m3fn).float() * shrink[..., None, None])
    pages = pages.view(torch.uint8)
    pages[inv, :, pos % page] = _e4m3(x.float() * _pow2(254 - now)[inv][..., None]).view(torch.uint8)
    codes[ids] = pages.transpose(2, 3) if by_channel else pages
    byte[ids] = now.to(torch.uint8)


def _plain_read(codes, byte, table, by_channel):
    """The values of the table's pages, fp32 [B, width*page, heads, D]."""
    t = table.long()
    c = codes[t]
    c = c.transpose(3, 4) if by_channel else c
    v = c.contiguous().view(torch.float8_e4m3fn).float() * _pow2(byte[t])[..., None, None]
    B, W, H, page, D = v.shape
    return v.permute(0, 1, 3, 2, 4).reshape(B, W * page, H, D)


def _plain_attend(st):
    case = st["case"]
    kc, vc, kb, vb = st["cache"]
    q, G, H, D, page = st["q"], case["group"], case["heads"], case["D"], case["page"]
    out = torch.empty_like(q)
    at = 0
    for b, (n, L) in enumerate(st["lens"]):
        rows = slice(at, at + n)
        at += n
        if L == 0:
            out[rows] = 0
            continue
        t = st["table"][b:b + 1, :-(-L // page)]
        k = _plain_read(kc, kb, t, False)[0, :L].permute(1, 2, 0).contiguous()
        v = _plain_read(vc, vb, t, True)[0, :L].permute(1, 0, 2).contiguous()
        qq = q[rows].float().reshape(n, H, G, D).permute(1, 0, 2, 3).reshape(H, n * G, D)
        s = (qq @ k).reshape(H, n, G, L) * D ** -0.5
        last = L - n + torch.arange(n, device=_DEV)
        key = torch.arange(L, device=_DEV)
        keep = key[None] <= last[:, None]
        if case["window"]:
            keep &= key[None] > last[:, None] - case["window"]
        s = s.masked_fill(~keep[None, :, None], float("-inf"))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
        o = p.reshape(H, n * G, L) @ v
        den = p.sum(-1).reshape(H, n * G, 1)
        o = torch.where(den > 0, o / den, torch.zeros_like(o))
        out[rows] = o.reshape(H, n, G, D).permute(1, 0, 2, 3).reshape(n, H * G, D).to(q.dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    op = case["op"]
    if op == "load":
        w = state["weight"] if case["layout"] == "nk" else state["weight"].t()
        code, byte = _mx_quantize(w)
        return _mx_values(_mx_unpack(_mx_pack(code)), byte).to(_DT[case["out"]])
    if op in ("w4", "w4a4"):
        x = state["x"].float() if op == "w4" else _mx_values(*_mx_quantize(state["x"]))
        return (x @ _mx_values(_mx_unpack(state["packed"]), state["scales"]).t()).to(_DT[case["x"]])
    if op == "append":
        kc, vc, kb, vb = state["cache"]
        _plain_append(state, state["k"], kc, kb, False)
        _plain_append(state, state["v"], vc, vb, True)
        k, v = _plain_read(kc, kb, state["tail"], False), _plain_read(vc, vb, state["tail"], True)
        keep = torch.arange(k.shape[1], device=_DEV)[None] < state["tail_lens"][:, None]
        return [torch.where(keep[..., None, None], t, torch.zeros_like(t)).to(torch.bfloat16) for t in (k, v)]
    return _plain_attend(state)


# ---- what a pass cannot do without -----------------------------------------------------------------

def _pairs(n, L, window):
    """Query and key pairs of one sequence under the causal rule."""
    total = 0
    if n > L:
        n = L
    if not window:
        return n * L - n * (n - 1) // 2
    for i in range(n):
        total += min(window, L - n + i + 1)
    return total


def work(case):
    op = case["op"]
    if op in ("load", "w4", "w4a4"):
        K, N = case["K"], case["N"]
        packed = N * K // 2 + N * (K // 32)
        if op == "load":
            return {"bytes": K * N * (_ES[case["x"]] + _ES[case["out"]]) + 2 * packed, "flops": 0}
        M = case["M"]
        byt = packed + _ES[case["x"]] * M * (K + N)
        return {"bytes": byt, "flops": 2 * M * K * N}
    H, D, page = case["heads"], case["D"], case["page"]
    T = sum(_ints(case["new"]))
    if op == "append":
        read = sum(s + n - s // page * page for s, n in zip(_ints(case["start"]), _ints(case["new"])))
        # New K and V in, their codes out, and the touched pages' codes in and values out (bf16).
        return {"bytes": 2 * H * D * (T * (_ES[case["x"]] + 1) + read * (1 + 2)), "flops": 0}
    byt = 2 * _ES[case["x"]] * T * H * case["group"] * D
    flops = 0
    for n, L in zip(_ints(case["new"]), _ints(case["context"])):
        seen = min(L, case["window"] + n - 1) if case["window"] else L
        byt += 2 * H * seen * D
        flops += 4 * H * case["group"] * D * _pairs(n, L, case["window"])
    return {"bytes": byt, "flops": flops}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def _ldexp(v, e):
    """v * 2^e in fp64, the power made from its bits (torch.ldexp's is rounded on the GPU)."""
    return v * ((e.long() + 1023) << 52).view(torch.float64)


def _exact_mx(x):
    """The nearest e2m1 multiple of each block's scale 2^(floor(log2(amax)) - 2), fp64."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 1 - 2, torch.full_like(amax, -127).int()).clamp(-127, 127)
    v = _ldexp(b, -e)
    # Spacing 1/2 below 2, 1 below 4, 2 below 6, which is the largest; round() takes halves to the even multiple.
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).double()
    v = (torch.round(v / step) * step).clamp(-6, 6)
    return _ldexp(v, e).reshape(x.shape)


def _exact_weight(st):
    p = st["packed"]
    nib = torch.empty(p.shape[0], p.shape[1], 2, dtype=torch.int64, device=p.device)
    nib[..., 0], nib[..., 1] = p % 16, p // 16
    mag = nib % 8
    # Exponent field (2 bits) and mantissa bit: subnormal 0.5, else (1 + m/2) * 2^(exp - 1).
    ex, m = mag // 2, (mag % 2).double()
    v = torch.where(ex == 0, m / 2, _ldexp(1 + m / 2, (ex - 1).clamp(min=0)))
    v = torch.where(nib >= 8, -v, v).reshape(p.shape[0], -1, 32)
    return _ldexp(v, st["scales"].long()[..., None] - 127).reshape(p.shape[0], -1)


def _exact_e4m3(v):
    """fp64 to the nearest multiple of e4m3's spacing, halves to even; no value is above 448."""
    ex = (torch.frexp(v)[1] - 1).clamp(min=-6)
    return _ldexp(torch.round(_ldexp(v, 3 - ex)), ex - 3)


def _exact_codes(codes, byte):
    """uint8 e4m3 codes and scale bytes to fp64, from the bit fields."""
    c = codes.long()
    ex, m = c // 8 % 16, (c % 8).double()
    v = torch.where(ex == 0, _ldexp(m, torch.full_like(ex, -9)), _ldexp(8 + m, ex - 10))
    v = torch.where(c >= 128, -v, v)
    return _ldexp(v, byte.long().reshape(*byte.shape, *[1] * (v.dim() - byte.dim())) - 127)


def _exact_append(case, st, x, codes, byte):
    """codes [P, heads, page, D] -> values [B, width*page, heads, D] of the touched pages."""
    page, H, D = case["page"], case["heads"], case["D"]
    B, width = st["tail"].shape
    out = torch.zeros(B, width * page, H, D, dtype=torch.float64, device=_DEV)
    at = 0
    for b, (s, n) in enumerate(zip(_ints(case["start"]), _ints(case["new"]))):
        xs, first = x[at:at + n].double(), s // page * page
        at += n
        for p0 in range(first, s + n, page):
            lo, hi = max(s, p0), min(s + n, p0 + page)
            tok = xs[lo - s:hi - s].permute(1, 0, 2)                      # [heads, tokens, D]
            amax = tok.abs().amax((1, 2))
            e = torch.frexp(amax)[1] - 1 - 8
            e = torch.where(_ldexp(amax, -e) > 448, e + 1, e)
            e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(min=-126)
            j = (p0 - first) // page
            pid = int(st["tail"][b, j])
            if p0 < s:
                old_e = byte[pid].int() - 127
                e = torch.maximum(e, old_e)
                old = _exact_codes(codes[pid, :, :s - p0], byte[pid])
                old = _ldexp(_exact_e4m3(_ldexp(old, -e[:, None, None])), e[:, None, None])
                out[b, p0 - first:s - first] = old.permute(1, 0, 2)
            new = _ldexp(_exact_e4m3(_ldexp(tok, -e[:, None, None])), e[:, None, None])
            out[b, lo - first:hi - first] = new.permute(1, 0, 2)
    return out


def _raw_cache(st):
    c = st["cache"]
    return c if isinstance(c, tuple) else (c.k_codes, c.v_codes, c.k_scales, c.v_scales)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "load":
        return _exact_mx(st["weight"] if case["layout"] == "nk" else st["weight"].t())
    if op == "w4":
        return st["x"].double() @ _exact_weight(st).t()
    if op == "w4a4":
        return _exact_mx(st["x"]) @ _exact_weight(st).t()
    kc, vc, kb, vb = _raw_cache(st)
    if op == "append":
        return [_exact_append(case, st, st["k"], kc, kb), _exact_append(case, st, st["v"], vc.transpose(2, 3), vb)]
    G, H, D, page = case["group"], case["heads"], case["D"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=_DEV)
    at = 0
    for b, (n, L) in enumerate(st["lens"]):
        rows, at = slice(at, at + n), at + n
        if L == 0:
            continue
        ids = st["table"][b, :-(-L // page)].long()
        key = torch.arange(L, device=_DEV)
        last = L - n + torch.arange(n, device=_DEV)[:, None]
        drop = key > last
        if case["window"]:
            drop = drop | (key <= last - case["window"])
        for h in range(H):
            k = _exact_codes(kc[ids, h], kb[ids, h]).reshape(-1, D)[:L]
            v = _exact_codes(vc[ids, h], vb[ids, h]).transpose(1, 2).reshape(-1, D)[:L]
            for i in range(h * G, h * G + G):
                s = st["q"][rows, i].double() @ k.t() / math.sqrt(D)
                s[drop] = -math.inf
                w = torch.softmax(s, -1).nan_to_num(0.0)
                out[rows, i] = w @ v
    return out
