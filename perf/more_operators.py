"""Performance cases of what stands around the microscaled products and the 8-bit key/value cache.

The listed cases are the steps of serving a model whose linear layers hold MXFP4 weights
and whose attention reads the paged 8-bit cache, where several answers grow from one prompt:
linear layers with bias, activation, gate and residual; norms and rotary positions of queries
and keys ahead of the cache; attention of sequences that share a prefix; pages dealt out,
shared, copied and moved together.  ``draw`` gives further cases of the same ranges.

``run`` has two forms.  Where ``own`` is false it computes in elementary torch operations, in
fp32 (angles in fp64); where it is true it makes a user's calls of metalops_amd.  ``exact``
computes the definition in 64 bits, with code of its own.
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
_MOST_ROTATED = 8192 * 40 * 128           # elements of q and k
_MOST_PREFIX = 4 * 64 * 32 * 128 * 16384  # operations of the attention over prefixes
_MOST_SHARED = 32768 * 8 * 128            # codes of K in all prefixes, and of the sequences' own tokens
_MOST_PAGES = 2048 * 4 * 8 * 64 * 128     # codes of K that a pool holds


def _text(values):
    """One number for each sequence, as a case holds them."""
    return " ".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split()]


def listed():
    return [
        # The smallest product: the attention's output projection of one decoded token, added to the residual stream.
        {"name": "linear_o_m1", "op": "linear", "x": "f16", "M": 1, "K": 4096, "N": 4096, "bias": "", "act": "", "mul": False, "res": True},
        # A short prompt through a layer of odd sizes: bias (kept in fp32), gelu and a residual.
        {"name": "linear_odd_m77", "op": "linear", "x": "bf16", "M": 77, "K": 4128, "N": 1001, "bias": "f32", "act": "gelu", "mul": False,
         "res": True},
        # Prefill of a long prompt: the gate of an MLP, multiplied by the up projection's result.
        {"name": "linear_gate_m2048", "op": "linear", "x": "bf16", "M": 2048, "K": 4096, "N": 14336, "bias": "", "act": "silu", "mul": True,
         "res": False},
        # A decode step of four sequences: norms of the heads of q and k, and their rotation.
        {"name": "rope_tokens", "op": "rope", "x": "bf16", "T": 4, "heads": 32, "kv_heads": 8, "D": 128, "rotary": 128, "axes": "",
         "norm": "bf16", "pairs": False, "far": 30000},
        # An image's patches among text: three axes of positions, no norms, a head that is no power of two.
        {"name": "rope_image", "op": "rope", "x": "f16", "T": 2501, "heads": 16, "kv_heads": 16, "D": 80, "rotary": 80, "axes": "8 16 16",
         "norm": "", "pairs": False, "far": 2000},
        # A long prompt at the end of a long context.
        {"name": "rope_prompt", "op": "rope", "x": "bf16", "T": 8192, "heads": 32, "kv_heads": 8, "D": 128, "rotary": 128, "axes": "",
         "norm": "f32", "pairs": False, "far": 131072},
        # Eight answers to one short prompt, a token each.
        {"name": "shared_b8_2k", "op": "shared", "x": "f16", "prefix": "2048", "members": "8", "n": 1, "own": _text(1 + 23 * i for i in range(8)),
         "heads": 8, "group": 4, "D": 128, "page": 64},
        # A batch of users behind four system prompts of every length, three drafted tokens each.
        {"name": "shared_prompts", "op": "shared", "x": "bf16", "prefix": "32768 5000 64 901", "members": "9 17 5 9", "n": 3,
         "own": _text(3 + (i * 131) % 1500 for i in range(40)), "heads": 8, "group": 4, "D": 128, "page": 64},
        # 64 users behind one system prompt: the largest.
        {"name": "shared_b64_16k", "op": "shared", "x": "bf16", "prefix": "16384", "members": "64", "n": 1,
         "own": _text(1 + (i * 97) % 1024 for i in range(64)), "heads": 8, "group": 4, "D": 128, "page": 64},
        # A beam step of a small model: four beams take over from their parents and grow by a token.
        {"name": "pages_beams", "op": "pages", "do": "beams", "layers": 4, "heads": 4, "D": 64, "page": 16, "pages": 256,
         "lens": "100 100 100 100", "parents": "0 0 2 1", "grow": 1},
        # Four prompts, sixteen answers to each: rows forked, grown by a token (which copies the page they share), freed.
        {"name": "pages_answers", "op": "pages", "do": "answers", "layers": 8, "heads": 8, "D": 128, "page": 64, "pages": 512,
         "lens": "1000 1333 1999 70", "parents": _text(i // 16 for i in range(64)), "grow": 1},
        # A pool that a long run has left full of holes, moved together: the largest.
        {"name": "pages_compact", "op": "pages", "do": "compact", "layers": 4, "heads": 8, "D": 128, "page": 64, "pages": 2048,
         "lens": _text(64 + (i * 571) % 1900 for i in range(56)), "parents": "", "grow": 0},
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
    op = rng.choice(["linear", "linear", "linear", "rope", "rope", "shared", "shared", "shared", "pages", "pages"])
    if op == "linear":
        x = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
        K = 128 * _log(rng, 4, 112) if rng.random() < 0.6 else 32 * _log(rng, 16, 448)
        N = _width(rng, 512, 14336)
        most = _MOST_FLOPS_F32 if x == "f32" else _MOST_FLOPS
        return {"op": op, "x": x, "M": max(1, min(_log(rng, 1, 2048), most // (2 * K * N))), "K": K, "N": N,
                "bias": rng.choice(["", x, "f32"]), "act": rng.choice(["", "relu", "silu", "gelu", "gelu_tanh"]),
                "mul": rng.random() < 0.4, "res": rng.random() < 0.6}
    if op == "rope":
        D = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
        kv = rng.choice([1, 2, 4, 8, 8, 16])
        heads = kv * rng.choice([1, 2, 4, 4, 7, 8])
        rotary = D if rng.random() < 0.7 else 8 * rng.randint(2, D // 8)
        axes = rng.choice([1, 1, 2, 3, 4])
        cuts = sorted(rng.sample(range(1, rotary // 2), axes - 1))
        axes = _text(b - a for a, b in zip([0] + cuts, cuts + [rotary // 2])) if cuts else ""
        return {"op": op, "x": rng.choice(["f32", "f16", "bf16", "bf16"]), "T": max(1, min(_log(rng, 1, 8192), _MOST_ROTATED // ((heads + kv) * D) // 2)),
                "heads": heads, "kv_heads": kv, "D": D, "rotary": rotary, "axes": axes, "norm": rng.choice(["", "f32", "f16", "bf16"]),
                "pairs": rng.random() < 0.3, "far": _log(rng, 100, 1000000)}
    D, page = rng.choice([64, 80, 96, 128, 128, 128, 256]), rng.choice([16, 32, 64, 64, 128])
    heads = rng.choice([1, 2, 4, 8, 8, 16])
    if op == "shared":
        group = rng.choice([1, 2, 4, 4, 7, 8])
        while heads * group > 64:
            group //= 2
        S = rng.choice([1, 1, 1, 2, 3, 5])
        members = [_log(rng, 1, 64 // S) for _ in range(S)]
        n = 1 if rng.random() < 0.7 else rng.randint(2, 8)
        longest = max(16, min(16384, _MOST_PREFIX // (4 * sum(members) * n * heads * group * D), _MOST_SHARED // (heads * D * S)))
        prefix = [_log(rng, 1, longest) for _ in range(S)]
        most = _log(rng, n, max(n, min(1500, _MOST_SHARED // (heads * D * sum(members)))))
        # A slot that serves nobody has no context of its own.
        own_lens = [0 if rng.random() < 0.05 else rng.randint(n, max(n, most)) for _ in range(sum(members))]
        return {"op": op, "x": rng.choice(["f16", "bf16"]), "prefix": _text(prefix), "members": _text(members), "n": n, "own": _text(own_lens),
                "heads": heads, "group": group, "D": D, "page": page}
    layers = _log(rng, 1, 8)
    do = rng.choice(["beams", "answers", "compact"])
    most = max(24, min(2048, _MOST_PAGES // (layers * heads * page * D)))
    pages = _log(rng, 24, most)
    B = rng.randint(1, max(1, min(48, pages // 8)))
    longest = max(1, pages // 2 // B)                       # pages of a sequence
    lens = [rng.randint(0 if rng.random() < 0.1 else 1, longest * page) for _ in range(B)]
    grow = 1 if rng.random() < 0.7 else rng.randint(2, page)
    rows = B if do == "beams" else max(1, min(64, pages // 4, _log(rng, 1, 64)))
    parents = [rng.randrange(B) if rng.random() < 0.95 else -1 for _ in range(rows)]
    return {"op": op, "do": do, "layers": layers, "heads": heads, "D": D, "page": page, "pages": pages, "lens": _text(lens),
            "parents": "" if do == "compact" else _text(parents), "grow": 0 if do == "compact" else grow}


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
    """[..., K] -> packed e2m1 codes [..., K/2] and scale bytes [..., K/32]."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    byte = (_biased_exponent(b.abs().amax(-1)) - 2).clamp(0, 254)
    v = b * _pow2(254 - byte)[..., None]
    a = v.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a >= t) if i % 2 else (a > t)
    code = (code | ((v < 0).to(torch.uint8) << 3)).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _mx_values(packed, byte):
    """Codes and scale bytes to the fp32 values they stand for."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=packed.device)
    code = torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)
    v = table[code.long()].reshape(*code.shape[:-1], -1, 32)
    return (v * _pow2(byte)[..., None]).reshape(code.shape)


def _kv_byte(amax):
    """The smallest scale that leaves nothing above e4m3's 448."""
    bits = amax.float().view(torch.int32)
    return (((bits >> 23) & 255) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 247)


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 7919 + 31)
    return g


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=_DEV) * std).to(dtype)


def _activations(g, *shape, dtype=torch.float32):
    """Normal values with a few channels that are several times larger, as hidden states have them."""
    x = torch.randn(*shape, generator=g, device=_DEV)
    big = 1 + 7 * (torch.rand(shape[-1], generator=g, device=_DEV) < 0.02)
    return (x * big).to(dtype)


def _filled(g, P, heads, page, D):
    """Cache tensors whose pages hold keys or values of ordinary sizes."""
    codes = torch.empty(P, heads, page, D, dtype=torch.uint8, device=_DEV)
    byte = torch.empty(P, heads, dtype=torch.uint8, device=_DEV)
    step = max(1, (1 << 26) // (heads * page * D))
    for i in range(0, P, step):
        x = _activations(g, min(step, P - i), heads, page, D)
        b = _kv_byte(x.abs().amax((-1, -2)))
        codes[i:i + step] = (x * _pow2(254 - b)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        byte[i:i + step] = b.to(torch.uint8)
    return codes, byte


def _lens(values):
    return torch.tensor(list(values), dtype=torch.int32, device=_DEV)


def _cumulative(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _used(n, page):
    return -(-n // page)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    st = {"case": case}
    if op == "linear":
        M, K, N, dt = case["M"], case["K"], case["N"], _DT[case["x"]]
        st["x"] = _activations(g, M, K, dtype=dt)
        st["packed"], st["scales"] = _mx_quantize(_randn(g, N, K, std=0.02))
        st["bias"] = _randn(g, N, dtype=_DT[case["bias"]], std=0.5) if case["bias"] else None
        st["mul"] = _activations(g, M, N, dtype=dt) if case["mul"] else None
        st["res"] = _activations(g, M, N, dtype=dt) if case["res"] else None
        return st
    if op == "rope":
        T, H, Hk, D, R, dt = case["T"], case["heads"], case["kv_heads"], case["D"], case["rotary"], _DT[case["x"]]
        # q and k are parts of the qkv projection's result.
        qkv = _activations(g, T, (H + 2 * Hk) * D, dtype=dt).view(T, H + 2 * Hk, D)
        st["q"], st["k"] = qkv[:, :H], qkv[:, H:H + Hk]
        A = max(1, len(case["axes"].split()))
        first = torch.randint(0, max(1, case["far"] - T), (A, 1), generator=g, device=_DEV)
        at = first + (torch.arange(T, device=_DEV) if A == 1 else torch.randint(0, 64, (A, T), generator=g, device=_DEV))
        st["positions"] = at.to(torch.int32).reshape(T) if A == 1 else at.to(torch.int32)
        # The bases' logarithm differs from seed to seed a little, as models' do.
        base = 10000.0 * (1 + 49 * float(torch.rand((), generator=g, device=_DEV)))
        st["inv_freq"] = (base ** (-torch.arange(0, R, 2, dtype=torch.float64, device=_DEV) / R)).float()
        st["sections"] = tuple(_ints(case["axes"])) or None
        w = [(1 + _randn(g, D, std=0.2)).to(_DT[case["norm"]]) if case["norm"] else None for _ in range(2)]
        st["q_weight"], st["k_weight"] = w
        return st
    heads, D, page = case["heads"], case["D"], case["page"]
    if op == "shared":
        prefix, members, own_lens, n = _ints(case["prefix"]), _ints(case["members"]), _ints(case["own"]), case["n"]
        S, B, G = len(prefix), len(own_lens), case["group"]
        Wp, W = max(1, _used(max(prefix), page)), max(1, _used(max(own_lens), page))
        P = sum(_used(v, page) for v in prefix + own_lens) + 3
        order = iter(torch.randperm(P, generator=g, device=_DEV).tolist())
        rows = [[next(order) if j < _used(v, page) else -1 for j in range(w)] for w, vs in ((Wp, prefix), (W, own_lens)) for v in vs]
        st["prefix_table"], st["table"] = _lens(sum(rows[:S], [])).view(S, Wp), _lens(sum(rows[S:], [])).view(B, W)
        kc, kb = _filled(g, P, heads, page, D)
        vc, vb = _filled(g, P, heads, page, D)
        # Keys are held token by token, values channel by channel.
        st["cache"] = (kc, vc.transpose(2, 3).contiguous(), kb, vb)
        st["prefix_lens"], st["context"] = _lens(prefix), _lens(own_lens)
        st["groups"] = None if S == 1 else _lens(_cumulative(members))
        st["q"] = _randn(g, B * n, heads * G, D, dtype=_DT[case["x"]], std=1.5)
        st["max_prefix"], st["max_context"] = max(prefix), max(own_lens)
        # What the host knows of the batch: every prefix's members, filled up with -1.
        most, at = max(members), _cumulative(members)
        st["members"] = torch.tensor([[at[s] + i if i < m else -1 for i in range(most)] for s, m in enumerate(members)], device=_DEV)
        if own:
            import metalops_amd as mo
            st["cache"] = mo.KV8Cache(*st["cache"])
        return st
    lens, L, P = _ints(case["lens"]), case["layers"], case["pages"]
    B, W = len(lens), max(1, max(_used(v + case["grow"], page) for v in lens))
    used = [_used(v, page) for v in lens]
    order = iter(torch.randperm(P, generator=g, device=_DEV).tolist())
    st["table"] = _lens(next(order) if j < u else -1 for u in used for j in range(W)).view(B, W)
    if case["do"] == "beams" and B > 1:
        # Beams of one prompt share its first pages, and the last of them only now and then.
        share = min(used) - 1
        st["table"][1:, :max(0, share)] = st["table"][0, :max(0, share)]
    st["refs"] = torch.bincount(st["table"][st["table"] >= 0].long(), minlength=P).to(torch.int32)
    st["lens"], st["page"] = _lens(lens), page
    if case["parents"]:
        parents = _ints(case["parents"])
        st["parents"] = _lens(parents)
        st["grown"] = _lens((lens[p] if p >= 0 else 0) + (case["grow"] if p >= 0 else 0) for p in parents)
        st["none"] = torch.zeros_like(st["grown"])
    u8 = dict(generator=g, device=_DEV, dtype=torch.uint8)
    # Codes below NaN's.
    st["k"] = torch.randint(0, 126, (L, P, heads, page, D), **u8)
    st["v"] = torch.randint(0, 126, (L, P, heads, D, page), **u8)
    st["ks"] = torch.randint(110, 130, (L, P, heads), **u8)
    st["vs"] = torch.randint(110, 130, (L, P, heads), **u8)
    if own:
        import metalops_amd as mo
        st["pool"] = mo.KV8Pool([mo.KV8Cache(*(st[n][i] for n in ("k", "v", "ks", "vs"))) for i in range(L)])
    return st


# ---- one pass ------------------------------------------------------------------------------------

def _codes(st):
    return [st["k"].view(torch.float8_e4m3fn), st["v"].view(torch.float8_e4m3fn), st["ks"], st["vs"]]


def _run_own(st):
    import metalops_amd as mo
    case = st["case"]
    op = case["op"]
    if op == "linear":
        return mo.linear_mxfp4(st["x"], st["packed"], st["scales"], bias=st["bias"], activation=case["act"] or None, multiply=st["mul"],
                               residual=st["res"])
    if op == "rope":
        return mo.qk_norm_rope(st["q"], st["k"], st["positions"], st["inv_freq"], st["q_weight"], st["k_weight"], eps=1e-6,
                               sections=st["sections"], interleaved=case["pairs"])
    if op == "shared":
        return mo.kv8_shared_attention(st["q"], st["cache"], st["prefix_table"], st["prefix_lens"], st["table"], st["context"],
                                       groups=st["groups"], max_prefix=st["max_prefix"], max_context=st["max_context"])
    pool = st["pool"]
    pool.refs.copy_(st["refs"])             # back to where the pass began
    if case["do"] == "compact":
        table = st["table"].clone()
        live = mo.kv8_compact(pool, table)
        return [table, pool.refs, live] + _codes(st)
    answers = case["do"] == "answers"
    table, lens = mo.kv8_fork(pool, st["table"], st["lens"], st["parents"], release=not answers)
    missing = mo.kv8_resize(pool, table, lens, st["grown"])
    out = [missing, lens] + _codes(st)
    if answers:
        out += [table.clone(), pool.refs.clone()]
        mo.kv8_resize(pool, table, st["grown"], st["none"])
    return out + [table, pool.refs]


def _plain_linear(st):
    case = st["case"]
    y = st["x"].float() @ _mx_values(st["packed"], st["scales"]).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if case["act"] == "relu":
        y = torch.maximum(y, torch.zeros_like(y))
    elif case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    elif case["act"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))
    if st["mul"] is not None:
        y = y * st["mul"].float()
    if st["res"] is not None:
        y = y + st["res"].float()
    return y.to(_DT[case["x"]])


def _plain_rope(st):
    case = st["case"]
    R, pos = case["rotary"], st["positions"]
    if st["sections"] is None:
        pos = pos[:, None]
    else:
        axis = torch.repeat_interleave(torch.arange(len(st["sections"]), device=_DEV), torch.tensor(st["sections"], device=_DEV))
        pos = pos[axis].t()
    angle = pos.double() * st["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        f = x.float()
        if w is not None:
            f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * w.float()
        r, rest = f[..., :R], f[..., R:]
        if case["pairs"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = r[..., :R // 2], r[..., R // 2:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([r, rest], -1).to(x.dtype))
    return out


def _plain_read(codes, byte, table, by_channel):
    """The values of the table's pages, fp32 [rows, H, tokens, D]."""
    t = table.long().clamp(min=0)
    c = codes[t]
    c = c.transpose(3, 4) if by_channel else c
    v = c.contiguous().view(torch.float8_e4m3fn).float() * _pow2(byte[t])[..., None, None]
    R, W, H, page, D = v.shape
    return v.transpose(1, 2).reshape(R, H, W * page, D)


def _plain_shared(st):
    case = st["case"]
    kc, vc, kb, vb = st["cache"]
    H, G, D, n = case["heads"], case["group"], case["D"], case["n"]
    B = st["table"].shape[0]
    q = st["q"].float().view(B, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D) * D ** -0.5
    neg = float("-inf")
    # Of the prefixes: the members' rows stand one after another.
    S, most = st["members"].shape
    k, v = _plain_read(kc, kb, st["prefix_table"], False), _plain_read(vc, vb, st["prefix_table"], True)
    at = st["members"].clamp(min=0)
    rows = q[at].permute(0, 2, 1, 3, 4).reshape(S, H, most * n * G, D)
    s1 = rows @ k.transpose(2, 3).contiguous()
    s1 = s1.masked_fill((torch.arange(k.shape[2], device=_DEV) >= st["prefix_lens"][:, None])[:, None, None], neg)
    m1 = s1.amax(-1, keepdim=True)
    m1 = torch.where(m1 == neg, torch.zeros_like(m1), m1)
    p1 = torch.exp(s1 - m1)
    parts = [m1, p1.sum(-1, keepdim=True), p1 @ v]
    here = (st["members"] >= 0).flatten().nonzero()[:, 0]
    seq = at.flatten()[here]
    spread = []
    for t in parts:
        t = t.reshape(S, H, most, n * G, -1).transpose(1, 2).reshape(S * most, H, n * G, -1)
        full = torch.zeros(B, *t.shape[1:], device=_DEV)
        full[seq] = t[here]
        spread.append(full)
    m1, l1, o1 = spread
    # Of the sequences' own tokens.
    k, v = _plain_read(kc, kb, st["table"], False), _plain_read(vc, vb, st["table"], True)
    s2 = q @ k.transpose(2, 3).contiguous()
    pos = st["context"][:, None] - n + torch.arange(n, device=_DEV)
    pos = pos[:, None, :, None].expand(B, 1, n, G).reshape(B, 1, n * G, 1)
    s2 = s2.masked_fill(torch.arange(k.shape[2], device=_DEV) > pos, neg)
    m2 = s2.amax(-1, keepdim=True)
    m = torch.maximum(torch.where(l1 > 0, m1, torch.full_like(m1, neg)), m2)
    m = torch.where(m == neg, torch.zeros_like(m), m)
    p2, w1 = torch.exp(s2 - m), torch.exp(m1 - m)
    o = (o1 * w1 + p2 @ v) / (l1 * w1 + p2.sum(-1, keepdim=True))
    # A token that stands before its own context sees nothing.
    o = torch.where(pos < 0, torch.zeros_like(o), o)
    return o.view(B, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(B * n, H * G, D).to(st["q"].dtype)


def _count(refs, ids, mask, by):
    refs.index_add_(0, ids.clamp(min=0).flatten().long(), (mask.int() * by).flatten().to(refs.dtype))


def _plain_move(st, src, dst):
    for name in ("k", "v", "ks", "vs"):
        st[name][:, dst] = st[name][:, src]


def _plain_fork(st, refs, release):
    table, lens, parents, page = st["table"], st["lens"], st["parents"].long(), st["page"]
    B, W = table.shape
    cols = torch.arange(W, device=_DEV)
    used = (lens + page - 1) // page
    ok = (parents >= 0) & (parents < B)
    at = parents.clamp(0, B - 1)
    new = torch.where(ok[:, None] & (cols < used[at][:, None]), table[at], -1)
    _count(refs, new, new >= 0, 1)
    if release:
        _count(refs, table, (cols < used[:, None]) & (table >= 0), -1)
    return new, torch.where(ok, lens[at], torch.zeros_like(lens[at]))


def _plain_resize(st, refs, table, lens, new_lens):
    """In place on refs and table; the number of pages that are missing."""
    page, cols = st["page"], torch.arange(table.shape[1], device=_DEV)
    old, new = (lens + page - 1) // page, (new_lens + page - 1) // page
    gone = (cols >= new[:, None]) & (cols < old[:, None]) & (table >= 0)
    _count(refs, table, gone, -1)
    table.masked_fill_(gone, -1)
    need = (cols >= old[:, None]) & (cols < new[:, None])
    # The last page of a sequence that grows, if it is not full and others hold it too.
    last = (cols == old[:, None] - 1) & ((new_lens > lens) & (lens % page != 0))[:, None] & (table >= 0)
    last = last & (refs[table.clamp(min=0).long()] > 1)
    need = need | last
    free = torch.argsort((refs > 0).int(), stable=True)
    missing = (need.sum() - (refs == 0).sum()).clamp(min=0).to(torch.int32).reshape(1)
    rank = (need.flatten().int().cumsum(0).view_as(need) - 1).clamp(0, len(free) - 1)
    need, last = need & (missing == 0), last & (missing == 0)
    given = free[rank].to(torch.int32)
    _plain_move(st, table[last].long(), given[last].long())
    _count(refs, table, last, -1)
    _count(refs, given, need, 1)
    table.copy_(torch.where(need, given, table))
    return missing


def _plain_compact(st, refs, table):
    live = refs > 0
    n = live.sum()
    ids = torch.arange(len(refs), device=_DEV)
    src, dst = ids[live & (ids >= n)], ids[~live & (ids < n)]
    new = ids.to(torch.int32)
    new[src] = dst.to(torch.int32)
    _plain_move(st, src, dst)
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()], table))
    return n.to(torch.int32).reshape(1)


def _plain_pages(st):
    case = st["case"]
    refs = st["refs"].clone()
    if case["do"] == "compact":
        table = st["table"].clone()
        live = _plain_compact(st, refs, table)
        return [table, refs, live] + _codes(st)
    answers = case["do"] == "answers"
    table, lens = _plain_fork(st, refs, not answers)
    missing = _plain_resize(st, refs, table, lens, st["grown"])
    out = [missing, lens] + _codes(st)
    if answers:
        out += [table.clone(), refs.clone()]
        _plain_resize(st, refs, table, st["grown"], st["none"])
    return out + [table, refs]


def run(state):
    if own:
        return _run_own(state)
    return {"linear": _plain_linear, "rope": _plain_rope, "shared": _plain_shared, "pages": _plain_pages}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "linear":
        M, K, N, es = case["M"], case["K"], case["N"], _ES[case["x"]]
        byt = N * K // 2 + N * (K // 32) + es * M * (K + N * (1 + case["mul"] + case["res"])) + (N * _ES[case["bias"]] if case["bias"] else 0)
        return {"bytes": byt, "flops": 2 * M * K * N}
    if op == "rope":
        n = case["T"] * (case["heads"] + case["kv_heads"]) * case["D"]
        return {"bytes": 2 * _ES[case["x"]] * n, "flops": 0}
    H, D, page = case["heads"], case["D"], case["page"]
    if op == "shared":
        G, n, own_lens = case["group"], case["n"], _ints(case["own"])
        byt = 2 * H * D * (sum(_ints(case["prefix"])) + sum(own_lens)) + 2 * _ES[case["x"]] * len(own_lens) * n * H * G * D
        pairs = n * sum(m * p for m, p in zip(_ints(case["members"]), _ints(case["prefix"])))
        pairs += sum(n * v - n * (n - 1) // 2 for v in own_lens if v >= n)
        return {"bytes": byt, "flops": 4 * H * G * D * pairs}
    lens, parents = _ints(case["lens"]), _ints(case["parents"])
    used = [_used(v, page) for v in lens]
    if case["do"] == "compact":
        live = sum(used)
        moved = live * (case["pages"] - live) / case["pages"]        # as many as lie behind the first `live`, on average
    elif case["do"] == "answers":
        moved = sum(1 for p in parents if p >= 0 and lens[p] % page)
    else:
        moved = sum(1 for p in parents if p >= 0 and lens[p] % page and parents.count(p) > 1)
    ints = 4 * (2 * case["pages"] + 2 * sum(used) + 2 * sum(used[p] for p in parents if p >= 0))
    return {"bytes": 2 * moved * case["layers"] * H * (2 * page * D + 2) + ints, "flops": 0}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def _ldexp(v, e):
    """v * 2^e in fp64, the power made from its bits (torch.ldexp's is rounded on the GPU)."""
    return v * ((e.long() + 1023) << 52).view(torch.float64)


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


def _exact_codes(codes, byte):
    """uint8 e4m3 codes and scale bytes to fp64, from the bit fields."""
    c = codes.long()
    ex, m = c // 8 % 16, (c % 8).double()
    v = torch.where(ex == 0, _ldexp(m, torch.full_like(ex, -9)), _ldexp(8 + m, ex - 10))
    v = torch.where(c >= 128, -v, v)
    return _ldexp(v, byte.long().reshape(*byte.shape, *[1] * (v.dim() - byte.dim())) - 127)


def _exact_linear(st):
    case = st["case"]
    y = torch.matmul(st["x"].double(), _exact_weight(st).t())
    if case["bias"]:
        y += st["bias"].double()
    if case["act"] == "relu":
        y.clamp_(min=0)
    elif case["act"] == "silu":
        y *= torch.sigmoid(y)
    elif case["act"] == "gelu":
        y *= torch.special.ndtr(y)
    elif case["act"] == "gelu_tanh":
        y *= torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    if case["mul"]:
        y *= st["mul"].double()
    if case["res"]:
        y += st["res"].double()
    return y


def _exact_rope(st):
    case = st["case"]
    half, sections = case["rotary"] // 2, _ints(case["axes"]) or [case["rotary"] // 2]
    pos = st["positions"].reshape(len(sections), -1).double()
    freq = st["inv_freq"].double()
    turn = torch.empty(pos.shape[1], 1, half, dtype=torch.complex128, device=_DEV)
    i = 0
    for a, width in enumerate(sections):
        for j in range(i, i + width):
            angle = pos[a] * freq[j]
            turn[:, 0, j] = torch.complex(angle.cos(), angle.sin())
        i += width
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        y = x.double().clone()
        if w is not None:
            y /= (y.square().sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt()
            y *= w.double()
        first = slice(0, 2 * half, 2) if case["pairs"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["pairs"] else slice(half, 2 * half)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return out


def _exact_shared(st):
    case = st["case"]
    c = st["cache"]
    kc, vc, kb, vb = c if isinstance(c, tuple) else (c.k_codes, c.v_codes, c.k_scales, c.v_scales)
    H, G, D, n, page = case["heads"], case["group"], case["D"], case["n"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=_DEV)

    def values(ids, count, h):
        k = _exact_codes(kc[ids, h], kb[ids, h]).reshape(-1, D)[:count]
        v = _exact_codes(vc[ids, h], vb[ids, h]).transpose(1, 2).reshape(-1, D)[:count]
        return k, v

    b = 0
    for s, (length, members) in enumerate(zip(_ints(case["prefix"]), _ints(case["members"]))):
        ids = st["prefix_table"][s, :_used(length, page)].long()
        before = [values(ids, length, h) for h in range(H)]
        for b in range(b, b + members):
            L = _ints(case["own"])[b]
            mine = st["table"][b, :_used(L, page)].long()
            pos = L - n + torch.arange(n, device=_DEV)
            hidden = torch.arange(L, device=_DEV)[None] > pos[:, None]
            rows = slice(b * n, b * n + n)
            for h in range(H):
                k, v = values(mine, L, h)
                k, v = torch.cat([before[h][0], k]), torch.cat([before[h][1], v])
                q = st["q"][rows, h * G:h * G + G].double()
                score = torch.matmul(q.reshape(n * G, D), k.t()).reshape(n, G, -1) / math.sqrt(D)
                score[..., length:].masked_fill_(hidden[:, None], -math.inf)
                weight = torch.softmax(score, -1)
                o = torch.matmul(weight.reshape(n * G, -1), v).reshape(n, G, D)
                out[rows, h * G:h * G + G] = torch.where((pos < 0)[:, None, None], torch.zeros_like(o), o)
        b += 1
    return out


def exact(case, seed):
    if case["op"] == "pages":
        return None                          # whole numbers, and codes as they were
    st = prepare(case, seed)
    return {"linear": _exact_linear, "rope": _exact_rope, "shared": _exact_shared}[case["op"]](st)
