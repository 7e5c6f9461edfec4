"""Operators over microscaled 4-bit floating point, as cases that can be timed and checked.

A 4-bit tensor holds E2M1 codes, two to a byte (the lower half is the even column), and one E8M0 scale for every 32 columns.  The cases quantise
activations and weights, multiply activations with 4-bit weights, multiply two 4-bit operands, and run mixture-of-experts layers whose
experts are kept in 4 bits.  Shapes are those of the presets (2048 or 5120 columns; feed-forwards of 10944 or 12288, experts of 1408 or
1536), weights and activations are random; some columns of the activations are large, as the activations of language models are.
"""
import math

import torch

own = False

BLOCK = 32
LITE = dict(width=2048, experts=64, hidden=1408, chosen=6, shared=2, groups=1, kept=1, scale=1.0)
WIDE = dict(width=5120, experts=160, hidden=1536, chosen=6, shared=2, groups=8, kept=3, scale=16.0)
EXACT_LIMIT = 4e12          # multiply-adds in 64 bits that are still quick


# ---- the cases -----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the activations of one token on their way into a 4-bit product: latency alone
        dict(name="quantise_token", kind="quantise", rows=1, cols=2048, dtype="bf16"),
        # the activations of a prompt of two steps' tokens
        dict(name="quantise_prompt", kind="quantise", rows=4096, cols=5120, dtype="bf16"),
        # a checkpoint's fp32 matrix at load time
        dict(name="quantise_weights", kind="quantise", rows=10944, cols=2048, dtype="fp32"),
        # one decoding user: the down projection of the dense feed-forward, residual added
        dict(name="linear_token", kind="linear", tokens=1, rows=2048, cols=10944, residual=True),
        # eight decoding users, the wider model
        dict(name="linear_batch_8", kind="linear", tokens=8, rows=12288, cols=5120, residual=False),
        # a prompt portion of odd length through the gate and up projections of the dense feed-forward
        dict(name="gateup_prompt", kind="gateup", tokens=1531, rows=10944, cols=2048),
        # a short question, both operands in 4 bits
        dict(name="matmul_short", kind="matmul", tokens=77, rows=10944, cols=2048),
        # a whole prompt portion, both operands in 4 bits
        dict(name="matmul_prompt", kind="matmul", tokens=2048, rows=12288, cols=5120),
        # one decoding user, a whole layer: router, experts, shared experts, residual
        dict(name="moe_token", kind="moe", tokens=1, **LITE),
        # eight users, the headline's concurrency
        dict(name="moe_batch_8", kind="moe", tokens=8, **LITE),
        # a few users of the wide model, experts in groups
        dict(name="moe_wide_3", kind="moe", tokens=3, **WIDE),
        # a prompt portion
        dict(name="moe_prompt", kind="moe", tokens=515, **LITE),
    ]


def draw(rng):
    """Tokens over their logarithm, widths of whole blocks, every operator alike; no dearer than the largest listed case."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def blocks(lo, hi):
        return BLOCK * max(1, spread(lo, hi) // BLOCK)
    most = max(work(c)["flops"] for c in listed())
    kind = rng.choice(["quantise", "linear", "gateup", "matmul", "moe", "moe"])
    while True:
        if kind == "quantise":
            case = dict(kind=kind, rows=spread(1, 11000), cols=blocks(256, 6000), dtype=rng.choice(["bf16", "fp16", "fp32"]))
            if case["rows"] * case["cols"] <= 4096 * 5120 * 1.1:
                return case
            continue
        if kind == "moe":
            groups = rng.choice([1, 1, 4, 8])
            case = dict(kind=kind, tokens=spread(1, 600), width=blocks(256, 5120), experts=8 * spread(2, 20), hidden=blocks(128, 1536),
                        chosen=rng.randint(1, 8), shared=rng.randint(0, 2), groups=groups, kept=(groups + 1) // 2, scale=rng.choice([1.0, 2.5]))
        else:
            case = dict(kind=kind, tokens=spread(1, 2048), rows=spread(512, 12288), cols=blocks(512, 11000))
            if kind == "linear":
                case["residual"] = rng.random() < 0.5
            if kind == "gateup":
                case["rows"] = case["rows"] // 8 * 8
        if work(case)["flops"] <= most:
            return case


def _sizes(case):
    return tuple(case[n] for n in ("width", "experts", "hidden", "chosen", "shared", "groups", "kept", "scale"))


def work(case):
    """Every input read once, every output written once; of a layer's experts those that its tokens can be expected to choose."""
    packed = 0.5 + 1 / BLOCK
    if case["kind"] == "quantise":
        n = case["rows"] * case["cols"]
        el = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * (2 * el + 2 * packed), "flops": 4 * n}           # there and back
    if case["kind"] == "moe":
        d, e, f, k, shared = _sizes(case)[:5]
        t = case["tokens"]
        hit = e * (1 - (1 - k / e) ** t) + shared
        return {"bytes": hit * 3 * f * d * packed + 4 * e * d + 6 * t * d, "flops": 6 * t * (k + shared) * f * d + 2 * t * e * d}
    t, n, k = case["tokens"], case["rows"], case["cols"]
    mats = 2 if case["kind"] == "gateup" else 1
    return {"bytes": t * k * 2 + mats * n * k * packed + t * n * 2 * (2 if case.get("residual") else 1), "flops": 2 * mats * t * n * k}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(rows, cols, gen):
    """Normal values; one column in 64 is twenty times as large."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 1 / 64
    return torch.where(loud, x * 20, x)


def _weights(gen, *shape):
    """Codes and scales of normal matrices: what a 4-bit checkpoint holds."""
    codes = torch.empty(*shape[:-1], shape[-1] // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(*shape[:-1], shape[-1] // BLOCK, dtype=torch.uint8, device="cuda")
    flat_c, flat_s = codes.view(-1, codes.shape[-1]), scales.view(-1, scales.shape[-1])
    step = max(1, (1 << 26) // shape[-1])
    for r in range(0, flat_c.shape[0], step):
        part = torch.randn(min(step, flat_c.shape[0] - r), shape[-1], generator=gen, device="cuda") * 0.02
        flat_c[r:r + step], flat_s[r:r + step] = _encode(part)
    return codes, scales


def _plan(case, seed):
    """The inputs of a case as plain tensors."""
    gen = _generator(seed)
    s = {"case": case}
    if case["kind"] == "quantise":
        dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
        x = _activations(case["rows"], case["cols"], gen)
        s["x"] = (x if dtype != torch.float32 else x * 0.02).to(dtype)
    elif case["kind"] == "moe":
        d, e, f, k, shared = _sizes(case)[:5]
        t = case["tokens"]
        s["x"] = torch.randn(t, d, generator=gen, device="cuda").bfloat16()
        s["residual"] = torch.randn(t, d, generator=gen, device="cuda").bfloat16()
        s["router"] = torch.randn(e, d, generator=gen, device="cuda") / math.sqrt(d)
        s["gate"], s["up"] = _weights(gen, e + shared, f, d), _weights(gen, e + shared, f, d)
        s["down"] = _weights(gen, e + shared, d, f)
    else:
        t, n, k = case["tokens"], case["rows"], case["cols"]
        s["x"] = _activations(t, k, gen).bfloat16()
        for name in ("gate", "up") if case["kind"] == "gateup" else ("w",):
            s[name] = _weights(gen, n, k)
        if case.get("residual"):
            s["residual"] = torch.randn(t, n, generator=gen, device="cuda").bfloat16()
    return s


def prepare(case, seed):
    s = _plan(case, seed)
    if own:                  # a program lays its weights out once, when it loads them
        from jittorinfer_b200 import ops
        pair = ("gate", "up")
        if case["kind"] in ("moe", "gateup"):
            s["own_gu"] = ops.mx4_weight(*(ops.Mx4Tensor(*s[n]) for n in pair))
        if case["kind"] == "moe":
            s["own_d"] = ops.mx4_weight(ops.Mx4Tensor(*s["down"]))
        if case["kind"] == "linear":
            s["own_w"] = ops.mx4_weight(ops.Mx4Tensor(*s["w"]))
        if case["kind"] == "matmul":
            s["own_w"] = ops.Mx4Tensor(*s["w"])
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------------------------
def _encode(x):
    """Codes [rows, cols / 2] and scale bytes [rows, cols / 32] of fp32 rows."""
    r, k = x.shape
    b = x.view(r, k // BLOCK, BLOCK)
    top = b.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32)).clamp(-127, 127)
    y = torch.ldexp(b, -e[..., None])
    a = y.abs()
    a = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) * 2, torch.round(a / 2) * 4)).clamp(max=12)    # twice the value
    code = torch.where(a <= 4, a, torch.where(a == 6, 5.0, torch.where(a == 8, 6.0, 7.0))).to(torch.uint8)
    code = (code + torch.signbit(y).to(torch.uint8) * 8).view(r, k // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


def _decode(codes, scales):
    """fp32 values of codes [..., cols / 2]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).view(*codes.shape[:-1], -1, BLOCK)
    return torch.ldexp(v, scales[..., None].int() - 127).view(*codes.shape[:-1], -1)


def _silu(z):
    return z / (1 + torch.exp(-z))


def _choose(x, router, e, k, groups, kept, scale):
    """Chosen experts and their weights: softmax over all experts, the best ``kept`` groups by their best expert, the best k in them."""
    p = torch.softmax(x.double() @ router.double().T, -1)
    sel = p
    if groups > 1:
        g = p.view(-1, groups, e // groups)
        order = torch.sort(g.amax(-1), dim=-1, descending=True, stable=True).indices[:, :kept]
        keep = torch.zeros(p.shape[0], groups, dtype=torch.bool, device=p.device).scatter_(1, order, True)
        sel = torch.where(keep[:, :, None], g, torch.full_like(g, -1.0)).view(p.shape)
    ids = torch.sort(sel, dim=-1, descending=True, stable=True).indices[:, :k]
    return ids, (p.gather(1, ids) * scale).float()


def _moe_plain(s):
    case = s["case"]
    d, e, f, k, shared, groups, kept, scale = _sizes(case)
    ids, w = _choose(s["x"], s["router"], e, k, groups, kept, scale)
    t = case["tokens"]
    ids = torch.cat([ids, torch.arange(e, e + shared, device=ids.device)[None].expand(t, -1)], 1)
    w = torch.cat([w, torch.ones(t, shared, device=w.device)], 1)
    x, out = s["x"].float(), s["residual"].float()

    def expert(rows, pick):
        gate, up, down = (_decode(*(pick(a) for a in s[n])) for n in ("gate", "up", "down"))
        return (_silu(rows @ gate.T) * (rows @ up.T)) @ down.T
    if t * (k + shared) <= e + shared:                       # few pairs: each one's own matrices
        for i in range(t):
            for j in range(k + shared):
                at = ids[i, j:j + 1]
                out[i] += w[i, j] * expert(x[i:i + 1], lambda a: a.index_select(0, at)[0])[0]
        return out.bfloat16()
    share = torch.zeros(t, e + shared, device=w.device).scatter_(1, ids, w)
    for i in range(e + shared):
        out += share[:, i:i + 1] * expert(x, lambda a: a[i])
    return out.bfloat16()


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "quantise":
        return _decode(*_encode(s["x"].float())).to(s["x"].dtype)
    if kind == "linear":
        y = s["x"].float() @ _decode(*s["w"]).T
        return (y + s["residual"].float() if "residual" in s else y).bfloat16()
    if kind == "gateup":
        x = s["x"].float()
        return (_silu(x @ _decode(*s["gate"]).T) * (x @ _decode(*s["up"]).T)).bfloat16()
    if kind == "matmul":
        return (_decode(*_encode(s["x"].float())) @ _decode(*s["w"]).T).bfloat16()
    return _moe_plain(s)


def _run_own(s):
    from jittorinfer_b200 import ops
    case = s["case"]
    if case["kind"] == "quantise":
        return ops.mx4_dequantize(ops.mx4_quantize(s["x"]), s["x"].dtype)
    if case["kind"] == "linear":
        return ops.mx4_linear(s["x"], s["own_w"], residual=s.get("residual"))
    if case["kind"] == "gateup":
        return ops.mx4_gateup(s["x"], s["own_gu"], "silu")
    if case["kind"] == "matmul":
        return ops.mx4_matmul(ops.mx4_quantize(s["x"]), s["own_w"])
    k, shared, groups, kept, scale = _sizes(case)[3:]
    return ops.mx4_moe_layer(s["x"], s["router"], None, k, groups, kept, scale, False, False, s["own_gu"], s["own_d"],
                             n_shared=shared, residual=s["residual"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------
def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.to(torch.int32))


def _value64(codes, scales):
    """sign * (1 or 0).m * 2^(e - 1 or 0), times the block's power of two."""
    c = torch.stack((codes % 16, torch.div(codes, 16, rounding_mode="floor")), -1).flatten(-2).to(torch.int64)
    e, m = (c // 2) % 4, (c % 2).double()
    v = torch.where(e > 0, (1 + m / 2) * _pow2(e - 1), m / 2) * (1 - 2 * (c // 8)).double()
    return v * _pow2(scales.int() - 127).repeat_interleave(BLOCK, -1)


def _nearest64(x):
    """The 4-bit values of rows: the nearest of the 15 by distance, ties to the code that is even."""
    r, k = x.shape
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    out = torch.empty(r, k, dtype=torch.float64, device=x.device)
    step = max(1, (1 << 25) // k)
    for i in range(0, r, step):
        b = x[i:i + step].double().view(-1, k // BLOCK, BLOCK)
        top = b.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(torch.clamp(top, min=2.0 ** -140)))
        e += (_pow2(e + 1) <= top).double() - (_pow2(e) > top).double() * (top > 0)       # the logarithm is rounded: a power of two may fall short
        unit = _pow2(torch.clamp(e - 2, -127, 127))
        y = (b.abs() / unit).clamp(max=6)
        near, dist = torch.zeros_like(y), y.clone()
        for j in range(1, 8):
            dj = (y - grid[j]).abs()
            better = (dj < dist) if j % 2 else (dj <= dist)
            near, dist = torch.where(better, grid[j], near), torch.where(better, dj, dist)
        out[i:i + step] = (torch.sign(b) * near * unit).view(-1, k)
    return out


def exact(case, seed):
    if work(case)["flops"] > 2 * EXACT_LIMIT:
        return None
    s = _plan(case, seed)
    kind = case["kind"]
    if kind == "quantise":
        return _nearest64(s["x"])
    if kind != "moe":
        x = _nearest64(s["x"]) if kind == "matmul" else s["x"].double()
        if kind == "gateup":
            z, u = x @ _value64(*s["gate"]).T, x @ _value64(*s["up"]).T
            return z * torch.sigmoid(z) * u
        y = x @ _value64(*s["w"]).T
        return y + s["residual"].double() if "residual" in s else y
    d, e, f, k, shared, groups, kept, scale = _sizes(case)
    x, out = s["x"].double(), s["residual"].double()
    logits = x @ s["router"].double().T
    p = torch.exp(logits - logits.logsumexp(-1, keepdim=True))
    per_group = e // groups
    chosen = {}
    for t, row in enumerate(p.tolist()):
        best = sorted(range(groups), key=lambda g: (-max(row[g * per_group:(g + 1) * per_group]), g))[:kept]
        open_ = [i for g in best for i in range(g * per_group, (g + 1) * per_group)]
        for i in sorted(open_, key=lambda i: (-row[i], i))[:k]:
            chosen.setdefault(i, []).append((t, row[i] * scale))
        for i in range(e, e + shared):
            chosen.setdefault(i, []).append((t, 1.0))
    for i, pairs in chosen.items():
        rows = torch.tensor([t for t, _ in pairs], device=x.device)
        w = torch.tensor([v for _, v in pairs], dtype=torch.float64, device=x.device)
        gate, up, down = (_value64(s[n][0][i], s[n][1][i]) for n in ("gate", "up", "down"))
        z = x[rows] @ gate.T
        out[rows] += w[:, None] * ((z * torch.sigmoid(z) * (x[rows] @ up.T)) @ down.T)
    return out
