"""4-bit operators as they are used: many rows, runs of them in graphs and on streams, what is not a number in another token's expert, sizes past 32 bits.

Limits as in the tests of the single operators."""
import pytest
import torch

from jittorinfer_b200 import ops
from jittorinfer_b200.ops import mx4
from test_gpu_mx4 import DEV, HALF, experts, gated_limit, gen, product_limit, randn, weights, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [33, 64, 65, 97, 129, 193, 385, 700])
@pytest.mark.parametrize("N,K", [(300, 224), (1100, 1504)])
def test_products_of_many_rows(nat, T, N, K):
    (qg, g), (qu, u) = weights(N, K, seed=1, scale=0.05), weights(N, K, seed=2, scale=0.05)
    x = randn(T, K, seed=T, dtype=torch.bfloat16)
    z, v = x.double() @ g.T, x.double() @ u.T
    within(ops.mx4_linear(x, ops.mx4_weight(qg), out_dtype=torch.float32), z, product_limit(x, g, z, torch.float32))
    want = mx4._act(z, "silu") * v
    within(ops.mx4_gateup(x, ops.mx4_weight(qg, qu)), want, gated_limit(x, g, u, z, v, want, "silu", torch.bfloat16))


def layer_want(x, ids, wts, gv, uv, dv):
    """The layer without residual in 64 bits, expert by expert, and how far the kernels may be from it (see the single operator's test)."""
    half = HALF[x.dtype]
    out = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    lim = torch.zeros_like(out)
    for e in range(gv.shape[0]):
        share = (wts.double() * (ids == e)).sum(-1, keepdim=True)
        z, v = x.double() @ gv[e].T, x.double() @ uv[e].T
        h = mx4._act(z, "silu") * v
        dh = gated_limit(x, gv[e], uv[e], z, v, h, "silu", x.dtype)
        y = h @ dv[e].T
        out += share * y
        lim += (wts.double().abs() * (ids == e)).sum(-1, keepdim=True) * (dh @ dv[e].abs().T + h.shape[1] * 2.0 ** -23 * ((h.abs() + dh) @ dv[e].abs().T) + half * y.abs())
    return out, lim * (1 + half) + (half + (ids.shape[1] + 1) * 2.0 ** -23) * out.abs() + 1e-30


@pytest.mark.parametrize("T,E,k", [(70, 3, 2), (300, 4, 2), (515, 40, 6), (1000, 2, 1), (130, 256, 8)])
@pytest.mark.parametrize("choice", ["even", "one", "none"])
def test_layers_of_many_rows(nat, T, E, k, choice):
    d, F = 160, 96
    wgu, wd, gv, uv, dv = experts(E, d, F, seed=E)
    x = randn(T, d, seed=T, dtype=torch.bfloat16)
    ids = torch.rand(T, E, generator=gen(T), device=DEV).argsort(-1)[:, :k].int()
    if choice == "one":
        ids[:, 0] = E - 1                       # all rows at one expert, and some more (twice where a token chose it anyway)
    if choice == "none":
        ids[::2] = -1
    wts = torch.rand(T, k, generator=gen(T + 2), device=DEV)
    want, lim = layer_want(x, ids, wts, gv, uv, dv)
    within(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd), want, lim)
    assert torch.equal(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd), ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd))


@pytest.mark.parametrize("T", [1, 8, 9, 300])
def test_choices_that_are_no_expert_leave_the_residual(nat, T):
    wgu, wd, *_ = experts(4, 160, 96)
    x, res = randn(T, 160, seed=1, dtype=torch.bfloat16), randn(T, 160, seed=2, dtype=torch.bfloat16)
    ids = torch.full((T, 3), -1, dtype=torch.int32, device=DEV)
    ids[:, 1] = 4
    wts = torch.rand(T, 3, generator=gen(3), device=DEV)
    assert torch.equal(ops.mx4_moe_ffn(x, res, ids, wts, wgu, wd), res)
    assert not bool(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd).any())


@pytest.mark.parametrize("F", [32, 64, 96, 160, 256, 288])
def test_hidden_units_of_every_width_between_the_products(nat, F):
    """Widths at which a tile of weights ends inside, at and behind a chunk of hidden units."""
    T, E, k, d = 40, 5, 2, 96
    wgu, wd, gv, uv, dv = experts(E, d, F, seed=F)
    x = randn(T, d, seed=F, dtype=torch.bfloat16)
    ids = torch.rand(T, E, generator=gen(F), device=DEV).argsort(-1)[:, :k].int()
    wts = torch.rand(T, k, generator=gen(F + 2), device=DEV)
    want, lim = layer_want(x, ids, wts, gv, uv, dv)
    within(ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd), want, lim)


@pytest.mark.parametrize("T", [3, 20])
def test_an_expert_that_is_not_a_number_touches_only_those_who_chose_it(nat, T):
    wgu, wd, *_ = experts(4, 128, 64)
    x = randn(T, 128, seed=1, dtype=torch.bfloat16)
    ids = torch.tensor([[0, 2], [2, 3]], dtype=torch.int32, device=DEV)[torch.arange(T, device=DEV).clamp(max=1)].contiguous()
    wts = torch.rand(T, 2, generator=gen(2), device=DEV)
    clean = ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd)
    q = ops.mx4_quantize(randn(4, 128, 64, seed=2, scale=0.05))              # experts() packs these matrices
    q.scales[0] = 255
    got = ops.mx4_moe_ffn(x, None, ids, wts, wgu, ops.mx4_weight(q))
    assert bool(got[0].isnan().all()) and torch.equal(got[1:], clean[1:])
    x[0, 5] = float("inf")
    got = ops.mx4_moe_ffn(x, None, ids, wts, wgu, wd)
    assert not bool(got[0].isfinite().any()) and torch.equal(got[1:], clean[1:])


@pytest.mark.parametrize("T", [3, 20])
@pytest.mark.parametrize("gate", [(2, 1, 1, 1.0, False, False), (2, 4, 2, 1.0, True, True)])
def test_a_row_that_is_not_a_number_in_a_layer(nat, T, gate):
    wgu, wd, *_ = experts(8, 128, 64)
    x, router = randn(T, 128, seed=1, dtype=torch.bfloat16), randn(8, 128, seed=3, scale=0.1)
    clean = ops.mx4_moe_layer(x, router, None, *gate, wgu, wd)
    x[1, 7] = float("nan")
    got = ops.mx4_moe_layer(x, router, None, *gate, wgu, wd)
    others = torch.arange(T, device=DEV) != 1
    assert torch.equal(got[others], clean[others]) and bool(got[1].isnan().all())


@pytest.mark.parametrize("T", [3, 20])
def test_router_and_rows_with_strides(nat, T):
    E, d, F = 8, 128, 64
    wgu, wd, *_ = experts(E, d, F)
    x, res = randn(T, 3 * d, seed=1, dtype=torch.bfloat16), randn(T, 2 * d, seed=2, dtype=torch.bfloat16)
    router, bias = randn(d, E, seed=3, scale=0.1), randn(E, 2, seed=4)
    args = (2, 1, 1, 1.0, True, False, wgu, wd)
    want = ops.mx4_moe_layer(x[:, d:2 * d].contiguous(), router.T.contiguous(), bias[:, 1].contiguous(), *args, residual=res[:, d:].contiguous())
    assert torch.equal(ops.mx4_moe_layer(x[:, d:2 * d], router.T, bias[:, 1], *args, residual=res[:, d:]), want)


def block(x, w):
    """A dense block and an expert layer behind it, and their result quantised and multiplied in 4 bits."""
    y = ops.mx4_linear(ops.mx4_gateup(x, w["gu"]), w["d"], residual=x)
    y = ops.mx4_moe_layer(y, w["router"], None, 2, 1, 1, 1.0, False, False, w["egu"], w["ed"], n_shared=1, residual=y)
    return ops.mx4_matmul(ops.mx4_quantize(y), w["head"])


def block_weights(seed):
    d, F, E = 256, 160, 9
    egu, ed, *_ = experts(E, d, F, seed=seed)
    q = [weights(*s, seed=seed + i, scale=0.05)[0] for i, s in enumerate(((416, d), (416, d), (d, 416), (100, d)))]
    return dict(gu=ops.mx4_weight(q[0], q[1]), d=ops.mx4_weight(q[2]), router=randn(E - 1, d, seed=seed, scale=0.1), egu=egu, ed=ed, head=q[3])


@pytest.mark.parametrize("T", [1, 8, 9, 40])
def test_a_run_captured_and_replayed(nat, T):
    """Replays with new inputs, two graphs at a time on two streams and an eager run beside them: each as the eager run of its inputs."""
    w = block_weights(1)
    xs = [randn(T, 256, seed=i, dtype=torch.bfloat16) for i in range(6)]
    want = [block(x, w) for x in xs]
    ref = ops.mx4_dequantize(w["head"], torch.float32)
    assert want[0].shape == (T, 100) and bool(want[0].isfinite().all()) and ref.shape == (100, 256)
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, ins, outs = [], [], []
    torch.cuda.synchronize()
    for s in streams:
        ins.append(xs[0].clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(block(ins[-1], w))
        graphs.append(g)
    for a in range(0, 6, 2):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                ins[i].copy_(xs[a + i])
                for _ in range(5):
                    graphs[i].replay()
        eager = [block(x, w) for x in xs]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[a]) and torch.equal(outs[1], want[a + 1])
        assert all(torch.equal(e, v) for e, v in zip(eager, want))
    ops.nat().check_status()
    del graphs


@pytest.mark.parametrize("T", [1, 9])
def test_a_run_on_another_stream_than_the_first(nat, T):
    w = block_weights(3)
    x = randn(T, 256, seed=1, dtype=torch.bfloat16)
    want = block(x, w)
    side = torch.cuda.Stream()
    late = torch.zeros_like(x)
    big = torch.ones(1 << 26, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):
            big.mul_(1.0)                        # the rows are written behind a queue of work on this stream
        late.copy_(x)
        got = block(late, w)
    side.synchronize()
    assert torch.equal(got, want)


def test_quantise_past_32_bits(nat):
    rows, cols = 70000, 32768                    # 2.3 thousand million values
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[:-3] = 1.0
    x[-3:] = randn(3, cols, seed=1, dtype=torch.bfloat16)
    q = ops.mx4_quantize(x)
    want = mx4._quantize(x[-3:].cpu())
    assert torch.equal(q.codes[-3:].cpu(), want.codes) and torch.equal(q.scales[-3:].cpu(), want.scales)
    assert torch.equal(q.codes[7], q.codes[-4])
    del x
    assert torch.equal(ops.mx4_dequantize(q)[-3:].cpu(), mx4._dequantize(want, torch.bfloat16))


def test_product_past_32_bits(nat):
    T, N, K = 70000, 32768, 32
    q, _ = weights(N, K, seed=1)
    x = randn(T, K, seed=2, dtype=torch.bfloat16)
    w = ops.mx4_weight(q)
    out = ops.mx4_linear(x, w)
    tail = ops.mx4_linear(x[-200:].contiguous(), w)
    assert torch.equal(out[-200:], tail)
    del out
    out = ops.mx4_matmul(ops.mx4_quantize(x), q)
    assert torch.equal(out[-200:], ops.mx4_matmul(ops.mx4_quantize(x[-200:]), q))
