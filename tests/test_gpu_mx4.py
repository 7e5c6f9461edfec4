"""Kernels over microscaled 4-bit tensors against the definition in 64 bits.

Limits.  Quantising is exact.  A product's fp32 sum of K terms is off by at most K 2^-23 times the sum of magnitudes (the tensor cores may cut a
sum where fp32 would round it: a whole step of 2^-23 a term); a result in bf16 by half a step, 2^-8 of its value, more.
"""
import pytest
import torch

from jittorinfer_b200 import ops
from jittorinfer_b200.ops import mx4

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def weights(*shape, seed=0, scale=0.02):
    """A 4-bit tensor and its values in 64 bits."""
    q = ops.mx4_quantize(randn(*shape, seed=seed, scale=scale))
    return q, mx4._dequantize(q, torch.float64)


def within(got, want, lim):
    err = (got.double() - want).abs()
    bad = ~(err <= lim)
    assert not bool(bad.any()), f"{float((err / lim)[bad].max()):.3g} of the limit at {torch.nonzero(bad)[0].tolist()}, {int(bad.sum())} of {bad.numel()}"


def product_limit(x, w, want, dtype):
    return x.shape[1] * 2.0 ** -23 * (x.double().abs() @ w.abs().T) + HALF[dtype] * want.abs() + 1e-30


# ---- quantising -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (7, 2048), (513, 1440), (2, 10944)])
def test_quantize(nat, dtype, rows, cols):
    x = randn(rows, cols, seed=rows, scale=3.0).to(dtype)
    x[0, :32] = 0
    x[-1, -32:] = (torch.arange(-16, 16, device=DEV) / 4).to(dtype)           # every tie
    if dtype != torch.float16 and cols > 64:
        x[0, 32:64] *= 2.0 ** -126          # below the normal numbers
        x[-1, 32:64] *= 2.0 ** 100
    if rows > 2:
        x[1, 7], x[2, cols - 1] = float("nan"), float("inf")
    q = ops.mx4_quantize(x)
    want = mx4._quantize(x.cpu())
    assert torch.equal(q.codes.cpu(), want.codes) and torch.equal(q.scales.cpu(), want.scales)
    for out in (torch.bfloat16, torch.float16, torch.float32):
        assert torch.equal(ops.mx4_dequantize(q, out).cpu().nan_to_num(77.0), mx4._dequantize(want, out).nan_to_num(77.0))


@pytest.mark.parametrize("ld,off", [(100, 0), (104, 3), (200, 1), (64, 0)])
def test_quantize_strided_rows(nat, ld, off):
    x = randn(9, ld + 8, seed=ld, dtype=torch.bfloat16)[:, off:off + 64]
    want = mx4._quantize(x.cpu())
    q = ops.mx4_quantize(x)
    assert torch.equal(q.codes.cpu(), want.codes) and torch.equal(q.scales.cpu(), want.scales)
    q = ops.mx4_quantize(x[:, :32].T.contiguous().T)          # columns are not contiguous
    assert torch.equal(q.codes.cpu(), want.codes[:, :16])
    q = ops.mx4_quantize(x[:1].expand(9, 64))                 # the same row again and again
    assert torch.equal(q.codes.cpu(), want.codes[:1].expand(9, 32))
    assert ops.mx4_quantize(x[:0]).codes.shape == (0, 32)
    assert torch.equal(ops.mx4_quantize(x.contiguous().view(3, 3, 64)).codes.view(9, 32).cpu(), want.codes)


def test_every_code_and_scale(nat):
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)[:, None].repeat(1, 16)
    q = ops.Mx4Tensor(codes.repeat(256, 1), torch.arange(256, dtype=torch.uint8, device=DEV).repeat_interleave(256)[:, None])
    for out in (torch.bfloat16, torch.float16, torch.float32):
        assert torch.equal(ops.mx4_dequantize(q, out).nan_to_num(77.0), mx4._dequantize(q, out).nan_to_num(77.0))


# ---- weights ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(16, 128), (17, 32), (1, 160), (130, 416), (3, 40, 224), (2, 16, 64)])
def test_packed_weights_hold_the_values(nat, shape):
    q, want = weights(*shape, seed=len(shape))
    up, want_up = weights(*shape, seed=9, scale=50.0)              # scales above 2
    assert torch.equal(ops.mx4_weight(q).values(torch.float64)[0], want.float().double())
    pair = ops.mx4_weight(q, up).values(torch.float64)
    assert torch.equal(pair[0], want) and torch.equal(pair[1], want_up)


def scaled(q, add):
    return ops.Mx4Tensor(q.codes, (q.scales.int() + add).clamp(0, 254).to(torch.uint8))


# ---- products with bf16 and fp32 activations --------------------------------------------------------------------------------------
TOKENS = [1, 2, 7, 8, 9, 16, 17, 40, 129, 300]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("N,K", [(16, 32), (1, 128), (33, 160), (200, 2048), (1000, 416)])
def test_linear(nat, dtype, T, N, K):
    q, w = weights(N, K, seed=N + K)
    x = randn(T, K, seed=T, dtype=dtype)
    want = x.double() @ w.T
    pw = ops.mx4_weight(q)
    within(ops.mx4_linear(x, pw), want, product_limit(x, w, want, dtype))
    res = randn(T, N, seed=3, dtype=dtype)
    both = want + res.double()
    lim = product_limit(x, w, both, torch.float32) + 2.0 ** -24 * want.abs()
    within(ops.mx4_linear(x, pw, residual=res, out_dtype=torch.float32), both, lim)
    bias = randn(1, N, seed=4).expand(T, N)
    within(ops.mx4_linear(x, pw, residual=bias), want + bias.double(), product_limit(x, w, want + bias.double(), dtype))


def gated_limit(x, g, u, z, v, want, act, dtype):
    dz, dv = (x.shape[1] * 2.0 ** -23 * (x.double().abs() @ m.abs().T) for m in (g, u))
    # |d act / d z| <= 1.13; exponential, division and product: a few steps of 2^-23 of the result
    return 1.13 * dz * (v.abs() + dv) + want.abs() / v.abs().clamp(min=1e-30) * dv + (2.0 ** -20 + HALF[dtype]) * want.abs() + 1e-30


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("N,K", [(16, 64), (41, 160), (328, 2048)])
def test_gateup(nat, act, dtype, T, N, K):
    (qg, g), (qu, u) = weights(N, K, seed=1, scale=0.05), weights(N, K, seed=2, scale=0.05)
    x = randn(T, K, seed=T, dtype=dtype)
    z, v = x.double() @ g.T, x.double() @ u.T
    want = mx4._act(z, act) * v
    got = ops.mx4_gateup(x, ops.mx4_weight(qg, qu), act)
    within(got, want, gated_limit(x, g, u, z, v, want, act, dtype))


@pytest.mark.parametrize("T", [1, 9, 40, 150])
def test_linear_strided_rows(nat, T):
    q, w = weights(48, 192, seed=5)
    pw = ops.mx4_weight(q)
    wide = randn(T, 400, seed=6, dtype=torch.bfloat16)
    for x in (wide[:, 8:200], wide[:, 3:195], wide[:1, :192].expand(T, 192), wide[:, :384:2]):
        want = x.double() @ w.T
        within(ops.mx4_linear(x, pw), want, product_limit(x, w, want, torch.bfloat16))


@pytest.mark.parametrize("T", [1, 12, 70])
@pytest.mark.parametrize("add", [-100, 10, 120])
def test_linear_scales_far_from_one(nat, T, add):
    q, _ = weights(40, 256, seed=7)
    q = scaled(q, add)
    w = mx4._dequantize(q, torch.float64)
    x = randn(T, 256, seed=8, dtype=torch.bfloat16)
    want = x.double() @ w.T
    within(ops.mx4_linear(x, ops.mx4_weight(q), out_dtype=torch.float32), want, product_limit(x, w, want, torch.float32))


@pytest.mark.parametrize("T", [1, 12, 70])
def test_what_is_not_a_number_stays_in_its_row(nat, T):
    q, w = weights(40, 256, seed=9)
    s = q.scales.clone()
    s[5, 3] = 255
    x = randn(T, 256, seed=10, dtype=torch.bfloat16)
    want = x.double() @ w.T
    got = ops.mx4_linear(x, ops.mx4_weight(ops.Mx4Tensor(q.codes, s)))
    assert bool(got[:, 5].isnan().all())
    keep = [i for i in range(40) if i != 5]
    within(got[:, keep], want[:, keep], product_limit(x, w, want, torch.bfloat16)[:, keep])
    if T > 1:
        x[1, 200] = float("inf")
        got = ops.mx4_linear(x, ops.mx4_weight(q))
        rows = [i for i in range(T) if i != 1]
        within(got[rows], want[rows], product_limit(x, w, want, torch.bfloat16)[rows])
        assert not bool(got[1].isfinite().any() & (w[:, 200] != 0).all())


# ---- both operands in 4 bits ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,N,K", [(1, 1, 32), (1, 300, 2048), (5, 17, 96), (128, 128, 256), (129, 255, 288), (200, 513, 608), (300, 1000, 4096), (77, 64, 10944)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_matmul(nat, T, N, K, out):
    (a, av), (b, bv) = weights(T, K, seed=T, scale=1.0), weights(N, K, seed=N)
    want = av @ bv.T
    within(ops.mx4_matmul(a, b, out), want, product_limit(av, bv, want, out))


@pytest.mark.parametrize("add_a,add_b", [(60, -60), (-90, 20), (100, 10)])
def test_matmul_scales_far_from_one(nat, add_a, add_b):
    a, b = scaled(weights(40, 320, seed=1, scale=1.0)[0], add_a), scaled(weights(72, 320, seed=2)[0], add_b)
    av, bv = (mx4._dequantize(t, torch.float64) for t in (a, b))
    want = av @ bv.T
    within(ops.mx4_matmul(a, b, torch.float32), want, product_limit(av, bv, want, torch.float32))


def test_matmul_block_that_is_not_a_number(nat):
    (a, av), (b, bv) = weights(40, 320, seed=1, scale=1.0), weights(72, 320, seed=2)
    s = b.scales.clone()
    s[70, 9] = 255
    got = ops.mx4_matmul(a, ops.Mx4Tensor(b.codes, s))
    assert bool(got[:, 70].isnan().all()) and bool(got[:, :70].isfinite().all()) and bool(got[:, 71].isfinite().all())


# ---- mixture of experts -----------------------------------------------------------------------------------------------------------
def experts(E, d, F, seed=0):
    (g, gv), (u, uv), (dn, dv) = weights(E, F, d, seed=seed, scale=0.05), weights(E, F, d, seed=seed + 1, scale=0.05), weights(E, d, F, seed=seed + 2, scale=0.05)
    return ops.mx4_weight(g, u), ops.mx4_weight(dn), gv, uv, dv


def moe_want(x, residual, ids, wts, gv, uv, dv, act="silu"):
    """The layer in 64 bits and how far the kernels may be from it: hidden units and an expert's result are rounded to the activations' type."""
    T, k = ids.shape
    half = HALF[x.dtype]
    out = torch.zeros(x.shape, dtype=torch.float64, device=DEV) if residual is None else residual.double()
    lim = torch.zeros_like(out)
    for t in range(T):
        for j in range(k):
            e, w = int(ids[t, j]), float(wts[t, j])
            if not 0 <= e < gv.shape[0]:
                continue
            xr = x[t:t + 1]
            z, v = xr.double() @ gv[e].T, xr.double() @ uv[e].T
            h = mx4._act(z, act) * v
            dh = gated_limit(xr, gv[e], uv[e], z, v, h, act, x.dtype)
            y = h @ dv[e].T
            out[t] += w * y[0]
            lim[t] += abs(w) * (dh @ dv[e].abs().T + h.shape[1] * 2.0 ** -23 * ((h.abs() + dh) @ dv[e].abs().T) + half * y.abs())[0]
    lim = lim * (1 + half) + (half + (k + 1) * 2.0 ** -23) * out.abs() + 1e-30
    return out, lim


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("E,d,F,k", [(4, 64, 32, 2), (8, 160, 96, 8), (66, 256, 160, 6), (5, 2048, 416, 1)])
def test_moe_ffn(nat, dtype, T, E, d, F, k):
    wgu, wd, gv, uv, dv = experts(E, d, F, seed=E)
    x, res = randn(T, d, seed=T, dtype=dtype), randn(T, d, seed=T + 1, dtype=dtype)
    ids = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(31 * t + k))[:k] for t in range(T)]).int().to(DEV)
    wts = torch.rand(T, k, generator=gen(T + 2), device=DEV)
    act = "silu" if T % 2 else "gelu_tanh"
    want, lim = moe_want(x, res, ids, wts, gv, uv, dv, act)
    for _ in range(2):
        within(ops.mx4_moe_ffn(x, res, ids, wts, wgu, wd, act), want, lim)
    want, lim = moe_want(x, None, ids, wts, gv, uv, dv, act)
    within(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd, act), want, lim)


@pytest.mark.parametrize("T", [3, 20])
def test_moe_ffn_choices_outside_and_twice(nat, T):
    wgu, wd, gv, uv, dv = experts(6, 128, 64)
    x = randn(T, 128, seed=1, dtype=torch.bfloat16)
    ids = torch.randint(-2, 8, (T, 7), generator=gen(5), device=DEV, dtype=torch.int32)       # seven of six: some twice, some nowhere
    ids[1] = -1
    wts = randn(T, 7, seed=2)
    want, lim = moe_want(x, None, ids, wts, gv, uv, dv)
    within(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd), want, lim)
    assert not bool(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd)[1].any())


@pytest.mark.parametrize("T", [1, 5, 16, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", [dict(), dict(n_group=4, topk_group=2, norm=True, bias=1), dict(sigmoid=True, norm=True, n_group=2, group_top2=True, scale=2.5), dict(n_shared=2)])
def test_moe_layer(nat, T, dtype, gate):
    E, d, F, k = 16, 256, 96, 3
    gate = {**dict(n_group=1, topk_group=1, scale=1.0, norm=False, sigmoid=False, n_shared=0, group_top2=False, bias=None), **gate}
    wgu, wd, gv, uv, dv = experts(E + gate["n_shared"], d, F)
    x, res, router = randn(T, d, seed=T, dtype=dtype), randn(T, d, seed=2, dtype=dtype), randn(E, d, seed=3, scale=0.0625)
    if gate["bias"] is not None:
        gate["bias"] = randn(E, seed=4, scale=0.02)
    args = (router, gate["bias"], k, gate["n_group"], gate["topk_group"], gate["scale"], gate["norm"], gate["sigmoid"])
    ids, wts = ops.ref.moe_gate(x, *args, gate["n_shared"], gate["group_top2"])
    want, lim = moe_want(x, res, ids, wts, gv, uv, dv)
    # a weight in fp32 from logits that are off by d 2^-23 of their terms
    lim = lim + 2.0 ** -12 * (want - res.double()).abs()
    got = ops.mx4_moe_layer(x, *args, wgu, wd, n_shared=gate["n_shared"], group_top2=gate["group_top2"], residual=res)
    within(got, want, lim)


def test_no_tokens(nat):
    wgu, wd, *_ = experts(4, 64, 32)
    x = randn(0, 64, dtype=torch.bfloat16)
    assert ops.mx4_moe_ffn(x, None, torch.zeros(0, 2, dtype=torch.int32, device=DEV), torch.zeros(0, 2, device=DEV), wgu, wd).shape == (0, 64)
    assert ops.mx4_linear(x, ops.mx4_weight(weights(8, 64)[0])).shape == (0, 8)
    assert ops.mx4_matmul(ops.mx4_quantize(x), weights(8, 64)[0]).shape == (0, 8)
