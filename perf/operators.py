"""The sequence operators of the folding model, as cases to measure: attention over packed
sequences, the norm and rotation of queries and keys, and the linear layer with 8-bit operands
and a scale for each block of 128.

``run`` computes a case in plain torch (``own`` false) or with this package's operators (``own``
true) on what ``prepare`` made; ``exact`` gives the operator's definition in 64 bits.
"""

import math

import torch

own = False

F8_MAX = 448.0
F32_TINY = 2.0 ** -126


def _dtype(case):
    return {"fp16": torch.float16, "bf16": torch.bfloat16}[case["dtype"]]


def listed():
    return [
        # one 76-residue fold in the diffusion head's token transformer: pair bias, 48-wide heads
        {"name": "attn_fold76_bias", "op": "attention", "dtype": "fp16", "lens": "76", "hq": 16, "hkv": 16, "d": 48,
         "causal": False, "bias": "shared", "pad": 0},
        # four diffusion samples of one 384-residue fold that share the fold's pair bias, 9 padded keys
        {"name": "attn_fold384_bias", "op": "attention", "dtype": "fp16", "lens": "384,384,384,384", "hq": 16,
         "hkv": 16, "d": 48, "causal": False, "bias": "shared", "pad": 9},
        # a batch of proteins of many lengths packed for the language model, every token sees its own protein
        {"name": "attn_packed_lm", "op": "attention", "dtype": "bf16",
         "lens": "76,146,238,384,1022,511,33,640,129,857,300,1,417,96,733,255,128,590,1000,64,201,345,902,16,"
                 "476,77,812,160,279,1021,450,59", "hq": 20, "hkv": 20, "d": 64, "causal": False, "bias": "none",
         "pad": 0},
        # one complex of 2048 residues
        {"name": "attn_long2048", "op": "attention", "dtype": "fp16", "lens": "2048", "hq": 40, "hkv": 40, "d": 64,
         "causal": False, "bias": "none", "pad": 0},
        # prompts of a generative model: causal, four query heads to a key head
        {"name": "attn_causal_grouped", "op": "attention", "dtype": "bf16", "lens": "8192,4099,2048,1,777", "hq": 32,
         "hkv": 8, "d": 128, "causal": True, "bias": "none", "pad": 0},
        # one token of a 40-head model
        {"name": "rope_token", "op": "rope", "dtype": "fp16", "t": 1, "hq": 40, "hkv": 40, "d": 64, "rot": 64,
         "layout": "half", "norm": "layer", "scaling": "none", "maxpos": 2048},
        # a packed batch of the same model
        {"name": "rope_packed", "op": "rope", "dtype": "bf16", "t": 16384, "hq": 40, "hkv": 40, "d": 64, "rot": 64,
         "layout": "half", "norm": "layer", "scaling": "none", "maxpos": 2048},
        # grouped heads, half of each head rotated in pairs, far positions of a stretched context
        {"name": "rope_partial", "op": "rope", "dtype": "fp16", "t": 5003, "hq": 32, "hkv": 8, "d": 128, "rot": 64,
         "layout": "interleaved", "norm": "rms", "scaling": "yarn", "maxpos": 1000000},
        # query, key and value projection of one token
        {"name": "linear_token", "op": "linear", "dtype": "fp16", "m": 1, "n": 7680, "k": 2560, "bias": False},
        # the first feed-forward layer of one 238-residue protein
        {"name": "linear_fold238", "op": "linear", "dtype": "bf16", "m": 238, "n": 10240, "k": 2560, "bias": False},
        # widths that no block size divides
        {"name": "linear_ragged", "op": "linear", "dtype": "fp16", "m": 1283, "n": 1000, "k": 1360, "bias": True},
        # the second feed-forward layer of a large packed batch
        {"name": "linear_batch", "op": "linear", "dtype": "bf16", "m": 16384, "n": 2560, "k": 10240, "bias": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rope", "linear", "linear"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "attention":
        bias = rng.choice(["none", "none", "shared", "each"])
        causal = rng.random() < 0.5
        hkv = rng.choice([1, 2, 3, 5, 8, 16, 20])
        hq = hkv * rng.choice([1, 1, 2, 4])
        d = rng.choice([16, 32, 40, 48, 64, 64, 72, 96, 128, 128])
        longest = 700 if bias != "none" else 4096
        lens = [_log_int(rng, 1, longest) for _ in range(rng.randint(1, 5 if bias != "none" else 12))]
        while len(lens) > 1 and 4 * hq * d * sum(n * n for n in lens) > 7e11:
            lens.pop()
        return {"op": op, "dtype": dtype, "lens": ",".join(map(str, lens)), "hq": hq, "hkv": hkv, "d": d,
                "causal": causal, "bias": bias, "pad": 0 if bias == "none" else rng.choice([0, 3])}
    if op == "rope":
        d = rng.choice([16, 32, 48, 64, 96, 128, 256])
        return {"op": op, "dtype": dtype, "t": _log_int(rng, 1, 8192), "hq": rng.choice([1, 7, 16, 32]),
                "hkv": rng.choice([1, 4, 8]), "d": d, "rot": rng.choice([16, d // 32 * 16 or 16, d]),
                "layout": rng.choice(["half", "interleaved"]), "norm": rng.choice(["none", "rms", "layer"]),
                "scaling": rng.choice(["none", "linear", "yarn"]), "maxpos": rng.choice([512, 1000000])}
    m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 8, 10240), 16 * _log_int(rng, 2, 640)
    while 2 * m * n * k > 8e11:
        m //= 2
    return {"op": op, "dtype": dtype, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5}


# ---- inputs ---------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(case)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    st = {"case": case}
    if case["op"] == "attention":
        lens = [int(x) for x in case["lens"].split(",")]
        t, d = sum(lens), case["d"]
        # one fused projection, as a layer makes it; queries and keys as a norm leaves them
        qkv = randn(t, case["hq"] + 2 * case["hkv"], d)
        qkv[:, :case["hq"]] *= 1.5
        st["qkv"] = qkv.to(dt)
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        st["lens"] = lens
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        if case["bias"] != "none":
            n = max(lens)
            b = 2.0 * randn(1 if case["bias"] == "shared" else len(lens), case["hq"], n, n)
            if case["pad"]:
                hide = min(case["pad"], min(lens) - 1)  # the padded tokens at a fold's end are no keys
                if hide:
                    b[..., min(lens) - hide:min(lens)] = float("-inf")
            if case["causal"]:  # every row keeps its own key
                b.diagonal(dim1=-2, dim2=-1).clamp_(min=0.0)
            st["bias"] = b.to(dt)
        else:
            st["bias"] = None
    elif case["op"] == "rope":
        t, d = case["t"], case["d"]
        st["qkv"] = (3.0 * randn(t, case["hq"] + 2 * case["hkv"], d)).to(dt)
        st["pos"] = torch.randint(0, case["maxpos"], (t,), generator=g, device="cuda", dtype=torch.int32)
        for name in ("q", "k"):
            st[name + "_w"] = None if case["norm"] == "none" else 1.0 + 0.2 * randn(d)
            st[name + "_b"] = 0.1 * randn(d) if case["norm"] == "layer" else None
        if own:
            from esmfold2_mlx_b200 import attention as ops
            scaling = {"none": None, "linear": {"type": "linear", "factor": 4.0},
                       "yarn": {"type": "yarn", "factor": 16.0, "original_length": 4096}}[case["scaling"]]
            st["rotary"] = ops.Rotary(case["rot"], layout=case["layout"], scaling=scaling, device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        x = randn(m, k)
        x[:, :: max(1, k // 7)] *= 20.0  # a few channels far above the others
        st["x"] = x.to(dt)
        w = randn(n, k) / math.sqrt(k)
        nb, kb = -(-n // 128), -(-k // 128)
        pad = torch.zeros(nb * 128, kb * 128, device="cuda")
        pad[:n, :k] = w
        blocks = pad.view(nb, 128, kb, 128)
        ws = torch.clamp(blocks.abs().amax(dim=(1, 3)) / F8_MAX, min=F32_TINY)
        w8 = (blocks / ws[:, None, :, None]).view(nb * 128, kb * 128)[:n, :k].to(torch.float8_e4m3fn).contiguous()
        st["w8"], st["ws"] = w8, ws
        st["bias"] = randn(n) if case["bias"] else None
        if own:
            from esmfold2_mlx_b200 import fp8
            st["weight"] = fp8.BlockWeight(w8, ws)
    return st


def _split(st):
    c = st["case"]
    qkv = st["qkv"]
    return (qkv[:, :c["hq"]], qkv[:, c["hq"]:c["hq"] + c["hkv"]], qkv[:, c["hq"] + c["hkv"]:])


# ---- one pass -------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "rope": _own_rope, "linear": _own_linear}[op](state)
    return {"attention": _plain_attention, "rope": _plain_rope, "linear": _plain_linear}[op](state)


def _own_attention(st):
    from esmfold2_mlx_b200 import attention as ops
    q, k, v = _split(st)
    return ops.attention(q, k, v, st["cu"], causal=st["case"]["causal"], bias=st["bias"])


def _own_rope(st):
    from esmfold2_mlx_b200 import attention as ops
    q, k, _ = _split(st)
    c = st["case"]
    return ops.qk_norm_rope(q, k, st["pos"], st["rotary"], norm=None if c["norm"] == "none" else c["norm"],
                            q_weight=st["q_w"], k_weight=st["k_w"], q_bias=st["q_b"], k_bias=st["k_b"], eps=1e-5)


def _own_linear(st):
    from esmfold2_mlx_b200 import fp8
    return fp8.linear(st["x"], st["weight"], bias=st["bias"])


def _plain_attention(st):
    c = st["case"]
    q, k, v = _split(st)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    group = c["hq"] // c["hkv"]
    beg = 0
    for s, n in enumerate(st["lens"]):
        rows = slice(beg, beg + n)
        beg += n
        step = max(1, int(2 ** 28 // max(1, group * n * n)))  # key heads at a time: 1 GB of scores
        allowed = torch.ones(n, n, dtype=torch.bool, device=q.device).tril() if c["causal"] else None
        for h in range(0, c["hkv"], step):
            e = min(c["hkv"], h + step)
            kk = k[rows, h:e].float().permute(1, 0, 2).repeat_interleave(group, 0)
            vv = v[rows, h:e].float().permute(1, 0, 2).repeat_interleave(group, 0)
            qq = q[rows, h * group:e * group].float().permute(1, 0, 2)
            sc = (qq @ kk.transpose(1, 2)) * (1.0 / math.sqrt(c["d"]))
            if st["bias"] is not None:
                b = st["bias"][s if c["bias"] == "each" else 0]
                sc = sc + b[h * group:e * group, :n, :n].float()
            if allowed is not None:
                sc = sc.masked_fill(~allowed, float("-inf"))
            p = (sc - sc.amax(-1, keepdim=True)).exp()
            o = (p @ vv) / p.sum(-1, keepdim=True)
            out[rows, h * group:e * group] = o.permute(1, 0, 2).to(q.dtype)
    return out


def _frequencies(case, device):
    """Radians a position in 64 bits, and the factor of the rotated part."""
    half = case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64, device=device)
    freq = 10000.0 ** (-i / half)
    if case["scaling"] == "linear":
        return freq / 4.0, 1.0
    if case["scaling"] == "yarn":
        # turns over the trained length: above 32 unchanged, below 1 stretched, a ramp over the pair index between
        length, factor = 4096.0, 16.0

        def pair_at(turns):
            return half * math.log(length / (turns * 2.0 * math.pi)) / math.log(10000.0)

        lo = max(math.floor(pair_at(32.0)), 0)
        hi = min(math.ceil(pair_at(1.0)), case["rot"] - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return freq * (1.0 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _plain_rope(st):
    c = st["case"]
    q, k, _ = _split(st)
    freq, gain = _frequencies(c, q.device)
    ang = st["pos"].double()[:, None] * freq
    cos, sin = (ang.cos() * gain).float()[:, None], (ang.sin() * gain).float()[:, None]
    outs = []
    for x, w, b in ((q, st["q_w"], st["q_b"]), (k, st["k_w"], st["k_b"])):
        y = x.float()
        if c["norm"] == "layer":
            y = y - y.mean(-1, keepdim=True)
        if c["norm"] != "none":
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w
        if b is not None:
            y = y + b
        r, half = c["rot"], c["rot"] // 2
        if c["layout"] == "half":
            y1, y2 = y[..., :half], y[..., half:r]
            rot = torch.cat([y1 * cos - y2 * sin, y2 * cos + y1 * sin], -1)
        else:
            y1, y2 = y[..., 0:r:2], y[..., 1:r:2]
            rot = torch.stack([y1 * cos - y2 * sin, y2 * cos + y1 * sin], -1).flatten(-2)
        outs.append(torch.cat([rot, y[..., r:]], -1).to(x.dtype))
    return tuple(outs)


def _plain_linear(st):
    c = st["case"]
    x = st["x"].float()
    m, k = x.shape
    kb = -(-k // 128)
    pad = torch.zeros(m, kb * 128, device=x.device)
    pad[:, :k] = x
    blocks = pad.view(m, kb, 128)
    # a quotient of tensors: by a number torch multiplies with the rounded inverse
    xs = torch.clamp(blocks.abs().amax(-1) / torch.full((), F8_MAX, device=x.device), min=F32_TINY)
    xq = ((blocks / xs[..., None]).to(torch.float8_e4m3fn).float() * xs[..., None]).view(m, kb * 128)[:, :k]
    wscale = st["ws"].repeat_interleave(128, 0)[:c["n"]].repeat_interleave(128, 1)[:, :k]
    out = xq @ (st["w8"].float() * wscale).t()
    if st["bias"] is not None:
        out = out + st["bias"]
    return out.to(st["x"].dtype)


# ---- bytes and operations that a pass cannot do without -------------------------------------

def work(case):
    if case["op"] == "attention":
        lens = [int(x) for x in case["lens"].split(",")]
        t = sum(lens)
        pairs = [n * (n + 1) // 2 if case["causal"] else n * n for n in lens]
        nbytes = 2 * t * case["d"] * (2 * case["hq"] + 2 * case["hkv"])
        if case["bias"] != "none":
            nbytes += 2 * case["hq"] * (max(pairs) if case["bias"] == "shared" else sum(pairs))
        return {"bytes": nbytes, "flops": 4 * case["hq"] * case["d"] * sum(pairs)}
    if case["op"] == "rope":
        n = case["t"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 4 * n + 4 * case["t"], "flops": 10 * n}
    m, n, k = case["m"], case["n"], case["k"]
    kb, nb = -(-k // 128), -(-n // 128)
    return {"bytes": 2 * m * k + n * k + 4 * nb * kb + 2 * m * n, "flops": 2 * m * n * k}


# ---- the definitions in 64 bits -------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, st)
    if case["op"] == "rope":
        return _exact_rope(case, st)
    return _exact_linear(case, st)


def _exact_attention(case, st):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = st["qkv"].double()
    out = torch.zeros(x.shape[0], hq, d, dtype=torch.float64, device=x.device)
    beg = 0
    for s, n in enumerate(st["lens"]):
        pos = torch.arange(n, device=x.device)
        for h in range(hq):
            kv = h // (hq // hkv)
            keys, vals = x[beg:beg + n, hq + kv], x[beg:beg + n, hq + hkv + kv]
            for r0 in range(0, n, 4096):
                r1 = min(n, r0 + 4096)
                score = torch.einsum("id,jd->ij", x[beg + r0:beg + r1, h], keys) / d ** 0.5
                if case["bias"] == "shared":
                    score += st["bias"][0, h, r0:r1, :n].double()
                elif case["bias"] == "each":
                    score += st["bias"][s, h, r0:r1, :n].double()
                if case["causal"]:
                    score[pos[None, :] > pos[r0:r1, None]] = -math.inf
                prob = torch.softmax(score, -1)
                out[beg + r0:beg + r1, h] = torch.einsum("ij,jd->id", prob, vals)
        beg += n
    return out


def _exact_rope(case, st):
    x = st["qkv"].double()
    hq, hkv, r = case["hq"], case["hkv"], case["rot"]
    freq, gain = _frequencies(case, x.device)
    turn = torch.polar(torch.full_like(freq, gain)[None, :].expand(case["t"], -1).contiguous(),
                       st["pos"].double()[:, None] * freq)[:, None]
    outs = []
    for part, w, b in ((x[:, :hq], st["q_w"], st["q_b"]), (x[:, hq:hq + hkv], st["k_w"], st["k_b"])):
        if case["norm"] == "layer":
            part = (part - part.mean(-1, keepdim=True)) * torch.rsqrt(part.var(-1, unbiased=False, keepdim=True) + 1e-5)
        elif case["norm"] == "rms":
            part = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + 1e-5)
        if w is not None:
            part = part * w.double()
        if b is not None:
            part = part + b.double()
        if case["layout"] == "half":
            z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:r].contiguous()) * turn
            rot = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(part[..., :r].reshape(*part.shape[:2], r // 2, 2).contiguous()) * turn
            rot = torch.view_as_real(z).reshape(*part.shape[:2], r)
        outs.append(torch.cat([rot, part[..., r:]], -1))
    return tuple(outs)


def _round_e4m3(v):
    """The nearest e4m3 value, ties to the even one: 3 mantissa bits, exponents down to -6."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(v / step) * step, -F8_MAX, F8_MAX)


def _exact_linear(case, st):
    m, n, k = case["m"], case["n"], case["k"]
    out = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    wrows = torch.arange(n, device="cuda") // 128
    for b, k0 in enumerate(range(0, k, 128)):
        x = st["x"][:, k0:k0 + 128].double()
        # the scale is a stored 32-bit number, and the quotient that is rounded to 8 bits a 32-bit one
        scale = (x.abs().amax(-1) / F8_MAX).float().clamp(min=F32_TINY).double()
        part = _round_e4m3((x / scale[:, None]).float().double()) @ st["w8"][:, k0:k0 + 128].double().t()
        out += part * scale[:, None] * st["ws"][wrows, b].double()
    return out if st["bias"] is None else out + st["bias"].double()
