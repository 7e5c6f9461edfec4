"""4-bit operators where their inputs end: choices without an expert, rows of one token, memory that nobody wrote, scales far apart, strides and
addresses of views.  Limits as in the tests of the single operators."""
import os
import subprocess
import sys

import pytest
import torch

from jittorinfer_b200 import build, ops
from jittorinfer_b200.ops import mx4
from test_gpu_mx4 import DEV, experts, gen, moe_want, product_limit, randn, weights, within

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


def unwritten_memory_is_nan(megabytes=512):
    """What is allocated next finds NaN in it."""
    torch.cuda.empty_cache()
    junk = [torch.full((n, 1 << 18), float("nan"), device=DEV) for n in [1] * 8 + [megabytes]]
    junk += [torch.full((1 << 10,), float("nan"), device=DEV) for _ in range(256)]
    torch.cuda.synchronize()
    del junk


# ---- choices that are no expert ---------------------------------------------------------------------------------------------------
@BOTH
@pytest.mark.parametrize("T", [1, 8, 9, 60])
def test_no_choice_is_an_expert(nat, dtype, T):
    wgu, wd, *_ = experts(4, 2048, 1024)
    x, res = randn(T, 2048, seed=1, dtype=dtype), randn(T, 2048, seed=2, dtype=dtype)
    ids = torch.full((T, 3), -1, dtype=torch.int32, device=DEV)
    ids[:, 1] = 4
    wts = torch.rand(T, 3, generator=gen(3), device=DEV)
    wts[0, 2] = float("nan")
    unwritten_memory_is_nan()
    assert torch.equal(ops.mx4_moe_ffn(x, res, ids, wts, wgu, wd), res)
    unwritten_memory_is_nan()
    assert not bool(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd).any())


@BOTH
@pytest.mark.parametrize("T", [3, 20])
def test_choices_outside_beside_what_is_not_a_number(nat, dtype, T):
    """Some choices are experts, some twice, some not; token 0 and the first expert that it chose are not numbers, and a weight beside a choice that is no
    expert neither."""
    wgu, wd, gv, uv, dv = experts(6, 128, 64)
    x = randn(T, 128, seed=1, dtype=dtype)
    ids = torch.randint(-2, 8, (T, 7), generator=gen(5), device=DEV, dtype=torch.int32)
    ids[ids == 0] = 1
    ids[0, 0], ids[1] = 0, -1
    wts = randn(T, 7, seed=2)
    want, lim = moe_want(x, None, ids, wts, gv, uv, dv)
    q = ops.mx4_quantize(randn(6, 128, 64, seed=2, scale=0.05))              # experts() packs these matrices
    q.scales[0] = 255
    x[0, 3] = float("nan")
    wts[1, 4] = float("nan")
    wts[torch.nonzero((ids < 0) | (ids > 5))[-1].tolist()[0], torch.nonzero((ids < 0) | (ids > 5))[-1].tolist()[1]] = float("inf")
    got = ops.mx4_moe_ffn(x, None, ids, wts, wgu, ops.mx4_weight(q))
    assert bool(got[0].isnan().all()) and not bool(got[1].any())
    within(got[1:], want[1:], lim[1:])


# ---- scales far apart in a row ----------------------------------------------------------------------------------------------------
@BOTH
@pytest.mark.parametrize("T", [1, 3, 8, 20])
def test_blocks_of_zeros_with_a_large_scale(nat, dtype, T):
    """A block without a value says nothing of its row, whatever its scale."""
    E, d, F, k = 4, 128, 96, 2
    q = [ops.mx4_quantize(randn(*s, seed=i, scale=0.05)) for i, s in enumerate(((E, F, d), (E, F, d), (E, d, F)))]
    for t, at in zip(q, (0, 3, 1)):
        t.codes[..., 16 * at:16 * at + 16] = torch.tensor([0x80, 0x08, 0x00, 0x88], dtype=torch.uint8, device=DEV).repeat(4)
        t.scales[..., at] = 254
    gv, uv, dv = (mx4._dequantize(t, torch.float64) for t in q)
    wgu, wd = ops.mx4_weight(q[0], q[1]), ops.mx4_weight(q[2])
    assert all(torch.equal(a, b) for a, b in zip((*wgu.values(torch.float64), *wd.values(torch.float64)), (gv, uv, dv)))
    x = randn(T, d, seed=7, dtype=dtype)
    ids = torch.rand(T, E, generator=gen(T), device=DEV).argsort(-1)[:, :k].int()
    wts = torch.rand(T, k, generator=gen(8), device=DEV)
    want, lim = moe_want(x, None, ids, wts, gv, uv, dv)
    within(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd), want, lim)


def rescaled(q, add):
    return ops.Mx4Tensor(q.codes, (q.scales.int() + add).to(torch.uint8))


@BOTH
@pytest.mark.parametrize("T", [1, 8, 9])
@pytest.mark.parametrize("apart", [20, 60])
def test_blocks_far_below_the_largest_of_their_row(nat, dtype, T, apart):
    """The large blocks meet zeros, in x and in the hidden units: what is left are the small ones."""
    E, d, F, k = 4, 160, 96, 2
    qs = [ops.mx4_quantize(randn(*s, seed=i, scale=0.05)) for i, s in enumerate(((E, F, d), (E, F, d), (E, d, F)))]
    adds = [torch.tensor([0] * 5, device=DEV), torch.tensor([apart] + [0] * 4, device=DEV), torch.tensor([apart, 0, 0], device=DEV)]
    qs = [rescaled(q, a) for q, a in zip(qs, adds)]
    gv, uv, dv = (mx4._dequantize(q, torch.float64) for q in qs)
    x = randn(T, d, seed=7, dtype=dtype)
    x[:, :32] = 0                                    # up: the large block
    qs[0].codes[:, :32] = 0                          # gate: no hidden units where the down matrix is large
    gv[:, :32] = 0
    wgu, wd = ops.mx4_weight(qs[0], qs[1]), ops.mx4_weight(qs[2])
    ids = torch.rand(T, E, generator=gen(T), device=DEV).argsort(-1)[:, :k].int()
    wts = torch.rand(T, k, generator=gen(8), device=DEV)
    want, lim = moe_want(x, None, ids, wts, gv, uv, dv)
    got = ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd)
    assert float(want.abs().min()) > 0 and float(lim.max()) < 0.05 * float(want.abs().max())
    within(got, want, lim)


def test_weights_laid_out_while_capturing(nat):
    E, d, F, T = 4, 128, 96, 3
    q = [ops.mx4_quantize(randn(*s, seed=i, scale=0.05)) for i, s in enumerate(((E, F, d), (E, F, d), (E, d, F)))]
    x, ids, wts = randn(T, d, seed=7, dtype=torch.bfloat16), torch.tensor([[0, 1], [3, 1], [2, 2]], dtype=torch.int32, device=DEV), torch.rand(T, 2, generator=gen(8), device=DEV)
    want, lim = moe_want(x, None, ids, wts, *(mx4._dequantize(t, torch.float64) for t in q))
    ops.mx4_moe_ffn(x, None, ids, wts, ops.mx4_weight(q[0], q[1]), ops.mx4_weight(q[2]))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.mx4_moe_ffn(x, None, ids, wts, ops.mx4_weight(q[0], q[1]), ops.mx4_weight(q[2]))
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    within(got, want, lim)
    del g


@BOTH
@pytest.mark.parametrize("T", [1, 8, 9])
@pytest.mark.parametrize("first,second", [(-50, 120), (30, -110)])
def test_large_down_weights_of_small_hidden_units(nat, dtype, T, first, second):
    """Results of ordinary size whose factors are near the ends of fp32: no step in between may leave it."""
    E, d, F, k = 4, 128, 96, 2
    q = [ops.mx4_quantize(randn(*s, seed=i, scale=0.05)) for i, s in enumerate(((E, F, d), (E, F, d), (E, d, F)))]
    q = [rescaled(t, a) for t, a in zip(q, (first, first, second))]
    q[0].codes &= 0x77                               # positive: a large z passes as it is
    gv, uv, dv = (mx4._dequantize(t, torch.float64) for t in q)
    x = randn(T, d, seed=7, dtype=dtype).abs()
    ids = torch.rand(T, E, generator=gen(T), device=DEV).argsort(-1)[:, :k].int()
    wts = torch.rand(T, k, generator=gen(8), device=DEV)
    want, lim = moe_want(x, None, ids, wts, gv, uv, dv)
    # the hidden units' limit has 1e-30 for fp32's smallest numbers, which here would be all of it: from 2^-100 on they are 2^49 steps of 2^-149 and more
    lim = lim - sum(wts[:, j, None].double() * 1e-30 * dv[ids[:, j].long()].abs().sum(-1) for j in range(k)) * (1 + 2.0 ** -8 * (dtype == torch.bfloat16))
    assert float((lim / want.abs()).median()) < 0.2
    got = ops.mx4_moe_ffn(x, None, ids, wts, ops.mx4_weight(q[0], q[1]), ops.mx4_weight(q[2]))
    within(got, want, lim.clamp(min=0) + 2.0 ** -20 * want.abs())


# ---- rows, strides and sizes ------------------------------------------------------------------------------------------------------
@BOTH
@pytest.mark.parametrize("T", [1, 2])
def test_a_row_of_a_wider_tensor(nat, dtype, T):
    """One token's stride is any: PyTorch calls its row contiguous."""
    E, d, F = 8, 128, 64
    wgu, wd, *_ = experts(E, d, F)
    x, res = randn(T, 3 * d, seed=1, dtype=dtype), randn(T, 2 * d, seed=2, dtype=dtype)
    router = randn(E, d, seed=3, scale=0.1)
    args = (router, None, 2, 1, 1, 1.0, True, False, wgu, wd)
    want = ops.mx4_moe_layer(x[:, d:2 * d].clone(), *args, residual=res[:, d:].clone())
    got = ops.mx4_moe_layer(x[:, d:2 * d], *args, residual=res[:, d:])
    assert torch.equal(got, want)
    ids, wts = torch.zeros(T, 1, dtype=torch.int32, device=DEV), torch.ones(T, 1, device=DEV)
    assert torch.equal(ops.mx4_moe_ffn(x[:, d:2 * d], res[:, d:], ids, wts, wgu, wd), ops.mx4_moe_ffn(x[:, d:2 * d].clone(), res[:, d:].clone(), ids, wts, wgu, wd))


def behind(t, elements):
    """A contiguous copy that begins so many elements behind an aligned address."""
    at = torch.zeros(t.numel() + 8, dtype=t.dtype, device=t.device)[elements:elements + t.numel()].view(t.shape)
    return at.copy_(t)


@BOTH
@pytest.mark.parametrize("T", [1, 3, 20])
def test_a_router_at_an_odd_address(nat, dtype, T):
    E, d, F = 8, 128, 64
    wgu, wd, *_ = experts(E, d, F)
    x, router = randn(T, d, seed=1, dtype=dtype), randn(E, d, seed=3, scale=0.1)
    args = (None, 2, 1, 1, 1.0, True, False, wgu, wd)
    assert torch.equal(ops.mx4_moe_layer(behind(x, 1), behind(router, 1), *args), ops.mx4_moe_layer(x, router, *args))


@BOTH
@pytest.mark.parametrize("T", [1, 3, 9, 20])
def test_a_residual_at_an_odd_address(nat, dtype, T):
    E, d, F = 8, 128, 64
    wgu, wd, *_ = experts(E, d, F)
    x, res, router = randn(T, d, seed=1, dtype=dtype), randn(T, d, seed=2, dtype=dtype), randn(E, d, seed=3, scale=0.1)
    ids, wts = torch.randint(0, E, (T, 2), generator=gen(3), device=DEV, dtype=torch.int32), torch.rand(T, 2, generator=gen(4), device=DEV)
    args = (router, None, 2, 1, 1, 1.0, True, False, wgu, wd)
    for at in (1, 4):
        assert torch.equal(ops.mx4_moe_layer(x, *args, residual=behind(res, at)), ops.mx4_moe_layer(x, *args, residual=res))
        assert torch.equal(ops.mx4_moe_ffn(x, behind(res, at), behind(ids, 1), behind(wts, 1), wgu, wd), ops.mx4_moe_ffn(x, res, ids, wts, wgu, wd))


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 66, 8), (3, 5, 2), (8, 256, 8)])
@pytest.mark.parametrize("F", [32, 64, 96, 448])
def test_few_units_over_many_groups(nat, T, E, k, F):
    """Where the units of gate and up end within a group's first draws, again and again: every run gives every unit's part."""
    d = 64
    wgu, wd, gv, uv, dv = experts(E, d, F, seed=F)
    x = randn(T, d, seed=T, dtype=torch.bfloat16)
    ids = torch.rand(T, E, generator=gen(T), device=DEV).argsort(-1)[:, :k].int()
    wts = torch.rand(T, k, generator=gen(8), device=DEV)
    want, lim = moe_want(x, None, ids, wts, gv, uv, dv)
    first = ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd)
    within(first, want, lim)
    assert all(torch.equal(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd), first) for _ in range(30))
    nat.check_status()


@BOTH
@pytest.mark.parametrize("T", [3, 20])
def test_no_choices(nat, dtype, T):
    wgu, wd, *_ = experts(4, 128, 64)
    x, res = randn(T, 128, seed=1, dtype=dtype), randn(T, 128, seed=2, dtype=dtype)
    none = torch.zeros(T, 0, dtype=torch.int32, device=DEV), torch.zeros(T, 0, device=DEV)
    got = ops.mx4_moe_ffn(x, res, *none, wgu, wd)
    assert torch.equal(got, res) and got.data_ptr() != res.data_ptr()
    assert not bool(ops.mx4_moe_ffn(x, None, *none, wgu, wd).any())


def test_more_fp32_rows_than_a_grid_is_high(nat):
    T = 8 * 65535 + 77
    q, w = weights(16, 32, seed=1)
    x = randn(T, 32, seed=2)
    want = x.double() @ w.T
    within(ops.mx4_linear(x, ops.mx4_weight(q)), want, product_limit(x, w, want, torch.float32))
    wgu, wd, *_ = experts(2, 32, 32)
    x = x[:T // 2 + 50]                              # two choices each
    ids = torch.randint(0, 2, (x.shape[0], 2), generator=gen(3), device=DEV, dtype=torch.int32)
    wts = torch.rand(x.shape[0], 2, generator=gen(4), device=DEV)
    got = ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd)
    assert torch.equal(got[:999], ops.mx4_moe_ffn(x[:999], None, ids[:999], wts[:999], wgu, wd))
    assert torch.equal(got[-999:], ops.mx4_moe_ffn(x[-999:], None, ids[-999:], wts[-999:], wgu, wd))


@pytest.mark.parametrize("T", [1, 12, 70])
def test_no_value_of_an_infinite_row_is_finite(nat, T):
    """On the tensor cores the block of an infinity is NaN, and so is NaN times a weight of 0."""
    (q, w), (u, _) = weights(40, 256, seed=9), weights(40, 256, seed=10)
    x = randn(T, 256, seed=10, dtype=torch.bfloat16)
    clean = ops.mx4_linear(x, ops.mx4_weight(q)), ops.mx4_gateup(x, ops.mx4_weight(q, u))
    for bad in ("inf", "-inf", "nan"):
        x[0, 200] = float(bad)
        for got, was in zip((ops.mx4_linear(x, ops.mx4_weight(q)), ops.mx4_gateup(x, ops.mx4_weight(q, u))), clean):
            assert not bool(got[0].isfinite().any()) and torch.equal(got[1:], was[1:])


def test_padded_rows_are_within_the_bounds_of_the_checking_build(nat):
    """The build that checks indexes counts the rows that there are, not the choices: an expert's rows are padded."""
    checked = build.KERNELS_SO.replace(".so", "_bc.so")
    if not os.path.exists(checked):
        pytest.skip("the checking build is not there")
    code = """
import torch
from jittorinfer_b200 import ops
from jittorinfer_b200.ops import native
assert native.load().jib_bounds_check_enabled() == 1
w = ops.mx4_quantize(torch.randn(8, 64, 64, device="cuda"))
x = torch.randn(20, 64, device="cuda").bfloat16()
ids = torch.arange(40, device="cuda", dtype=torch.int32).view(20, 2) % 8
out = ops.mx4_moe_ffn(x, None, ids, torch.ones(20, 2, device="cuda"), ops.mx4_weight(w, w), ops.mx4_weight(w))
native.check_status()
"""
    env = dict(os.environ, JITTORINFER_KERNELS_SO=checked, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ---- activations with loud columns ------------------------------------------------------------------------------------------------
def planes_loss(x):
    """What two planes of 8 bits may lose of bf16 activations: nothing down to 2^-11 of a block's largest, below at most 2^-21 of it (the second plane's
    smallest step, rounded) or the value."""
    b = x.double().abs().reshape(x.shape[0], -1, 32)
    top = b.amax(-1, keepdim=True)
    return torch.where(b < 2.0 ** -11 * top, torch.minimum(b, 2.0 ** -21 * top), 0.0).reshape(x.shape)


def loud(T, K, by, dtype=torch.bfloat16):
    x = randn(T, K, seed=T)
    x[:, ::37] *= by
    return x.to(dtype)


@pytest.mark.parametrize("T", [1, 9, 40, 150])
@pytest.mark.parametrize("by", [2.0 ** 4, 2.0 ** 9, 2.0 ** 14, 2.0 ** 24])
def test_products_of_loud_columns(nat, T, by):
    N, K = 200, 416
    (q, w), (u, v) = weights(N, K, seed=1, scale=0.05), weights(N, K, seed=2, scale=0.05)
    x = loud(T, K, by)
    want = x.double() @ w.T
    within(ops.mx4_linear(x, ops.mx4_weight(q), out_dtype=torch.float32), want, product_limit(x, w, want, torch.float32) + planes_loss(x) @ w.abs().T)
    z, y = want, x.double() @ v.T
    want = mx4._act(z, "silu") * y
    lost, half = planes_loss(x), 2.0 ** -8
    dz, dy = (K * 2.0 ** -23 * (x.double().abs() @ m.abs().T) + lost @ m.abs().T for m in (w, v))
    within(ops.mx4_gateup(x, ops.mx4_weight(q, u)), want, (1.13 * dz * (y.abs() + dy) + mx4._act(z, "silu").abs() * dy) + (2.0 ** -20 + half) * want.abs() + 1e-30)


@pytest.mark.parametrize("T", [1, 8, 9, 60])
@pytest.mark.parametrize("by", [2.0 ** 4, 2.0 ** 9, 2.0 ** 14])
def test_layers_of_loud_columns(nat, T, by):
    """The few-token form keeps x to 2^-39 of a row's largest and hidden units in fp16; the tiled one has two planes of both."""
    E, d, F, k = 6, 160, 96, 2
    wgu, wd, gv, uv, dv = experts(E, d, F, seed=5)
    x = loud(T, d, by)
    ids = torch.rand(T, E, generator=gen(T), device=DEV).argsort(-1)[:, :k].int()
    wts = torch.rand(T, k, generator=gen(8), device=DEV)
    half = 2.0 ** -8
    lost = torch.maximum(planes_loss(x), 2.0 ** -39 * x.double().abs().amax(-1, keepdim=True))
    want, lim = torch.zeros(T, d, dtype=torch.float64, device=DEV), torch.zeros(T, d, dtype=torch.float64, device=DEV)
    for e in range(E):
        share = (wts.double() * (ids == e)).sum(-1, keepdim=True)
        z, y = x.double() @ gv[e].T, x.double() @ uv[e].T
        dz, dy = (d * 2.0 ** -23 * (x.double().abs() @ m[e].abs().T) + lost @ m[e].abs().T for m in (gv, uv))
        h = mx4._act(z, "silu") * y
        dh = (1.13 * dz * (y.abs() + dy) + mx4._act(z, "silu").abs() * dy) + (2.0 ** -20 + half) * h.abs() + 1e-30
        dh = dh + torch.maximum(planes_loss(h * (1 + half)), 2.0 ** -25 * h.abs().amax(-1, keepdim=True))          # (fp16: half a step of 2^-24 of the largest)
        r = h @ dv[e].T
        want += share * r
        lim += share * (dh @ dv[e].abs().T + F * 2.0 ** -23 * ((h.abs() + dh) @ dv[e].abs().T) + half * r.abs())
    lim = lim * (1 + half) + (half + (k + 1) * 2.0 ** -23) * want.abs() + 1e-30
    within(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd), want, lim)


def test_only_experts_have_factors(nat):
    q = ops.mx4_quantize(randn(3, 40, 224, seed=1))
    one, batch = ops.mx4_weight(ops.Mx4Tensor(q.codes[1], q.scales[1])), ops.mx4_weight(q)
    assert one.factors is None and one.exps is None and batch.factors is not None and not batch.far
    assert one.nbytes() == 2 * 64 * (64 + 4) and batch.nbytes() == 3 * 64 * (2 * (64 + 4 + 4) + 4)         # two chunks of 64 laid-out rows
    assert torch.equal(one.values()[0], batch.values()[0][1])
