"""Microscaled 4-bit tensors on the CPU: the format, the operators' definitions and what they refuse."""
import math

import pytest
import torch

from jittorinfer_b200 import ops

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def tensor(rows, cols, seed=0, scale=1.0):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)) * scale


def nearest(row):
    """One block by the definition, value by value."""
    top = max(abs(v) for v in row)
    e = max(-127, math.frexp(top)[1] - 3) if top else -127
    out = []
    for v in row:
        y = abs(v) / 2.0 ** e
        best = min(range(8), key=lambda i: (abs(GRID[i] - min(y, 6.0)), i % 2))
        out.append(math.copysign(GRID[best] * 2.0 ** e, v))
    return out, e + 127


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1.0, 1e-30, 1e-39, 1e30])
def test_quantize_is_the_definition(dtype, scale):
    if dtype == torch.float16 and scale != 1.0:
        scale = {1e-30: 1e-6, 1e-39: 6e-8, 1e30: 1e3}[scale]
    x = tensor(3, 96, 1, scale).to(dtype)
    x[0, :32] = 0
    x[1, 32:64] = torch.arange(-16, 16).to(dtype) / 4 * min(scale, 1.0)            # every tie
    q = ops.mx4_quantize(x)
    v = ops.mx4_dequantize(q, torch.float32).double()
    for r in range(3):
        for b in range(3):
            want, byte = nearest(x[r, 32 * b:32 * b + 32].double().tolist())
            assert v[r, 32 * b:32 * b + 32].tolist() == want and int(q.scales[r, b]) == byte


def test_blocks_that_are_not_numbers():
    x = tensor(2, 64, 2)
    x[0, 5], x[1, 40] = float("nan"), float("-inf")
    q = ops.mx4_quantize(x)
    v = ops.mx4_dequantize(q, torch.float32)
    assert int(q.scales[0, 0]) == 255 and int(q.scales[1, 1]) == 255 and bool(v[0, :32].isnan().all()) and bool(v[1, 32:].isnan().all())
    assert bool(v[0, 32:].isfinite().all()) and bool(v[1, :32].isfinite().all())


def test_values_survive_a_second_round():
    q = ops.mx4_quantize(tensor(5, 128, 3))
    v = ops.mx4_dequantize(q, torch.bfloat16)
    again = ops.mx4_dequantize(ops.mx4_quantize(v), torch.bfloat16)
    assert torch.equal(v, again)


def test_products_are_those_of_the_values():
    x, w, u = tensor(3, 64, 4), ops.mx4_quantize(tensor(17, 64, 5)), ops.mx4_quantize(tensor(17, 64, 6))
    wv, uv = ops.mx4_dequantize(w, torch.float32), ops.mx4_dequantize(u, torch.float32)
    res = tensor(1, 17, 7).expand(3, 17)
    assert torch.allclose(ops.mx4_linear(x, ops.mx4_weight(w), residual=res), x @ wv.T + res, atol=1e-5)
    assert torch.allclose(ops.mx4_gateup(x, ops.mx4_weight(w, u)), torch.nn.functional.silu(x @ wv.T) * (x @ uv.T), atol=1e-5)
    xq = ops.mx4_quantize(x)
    assert torch.allclose(ops.mx4_matmul(xq, w, torch.float32), ops.mx4_dequantize(xq, torch.float32) @ wv.T, atol=1e-5)
    assert ops.mx4_linear(x.bfloat16(), ops.mx4_weight(w)).dtype == torch.bfloat16
    assert ops.mx4_linear(x[:0], ops.mx4_weight(w)).shape == (0, 17)


def experts(E, d, F, seed=0):
    g, u, dn = (ops.mx4_quantize(tensor(E * n, m, seed + i).view(E, n, m)) for i, (n, m) in enumerate([(F, d), (F, d), (d, F)]))
    return ops.mx4_weight(g, u), ops.mx4_weight(dn), [ops.mx4_dequantize(t, torch.float32) for t in (g, u, dn)]


def test_layer_is_gate_and_experts():
    E, shared, d, F, T, k = 8, 1, 64, 32, 5, 3
    wgu, wd, (g, u, dn) = experts(E + shared, d, F)
    x, res, router = tensor(T, d, 20), tensor(T, d, 21), tensor(E, d, 22)
    ids, wts = ops.moe_gate(x, router, None, k, 4, 2, 2.5, True, False, shared)
    want = ops.moe_ffn(x, res, ids, wts, g, u, dn, None, None, None)
    assert torch.allclose(ops.mx4_moe_ffn(x, res, ids, wts, wgu, wd), want, atol=1e-3, rtol=1e-4)
    assert torch.allclose(ops.mx4_moe_layer(x, router, None, k, 4, 2, 2.5, True, False, wgu, wd, n_shared=shared, residual=res), want, atol=1e-3, rtol=1e-4)


def test_choices_outside_the_experts_and_twice_the_same():
    wgu, wd, _ = experts(4, 64, 32)
    x, one = tensor(2, 64, 30), torch.ones(2, 1)
    y = [ops.mx4_moe_ffn(x, None, torch.full((2, 1), e, dtype=torch.int32), one, wgu, wd) for e in range(4)]
    ids = torch.tensor([[1, 1, -1, 9], [3, 4, 0, 0]], dtype=torch.int32)
    out = ops.mx4_moe_ffn(x, None, ids, torch.tensor([[0.5, 0.25, 3.0, 3.0], [1.0, 3.0, 0.5, -0.5]]), wgu, wd)
    assert torch.allclose(out[0], 0.75 * y[1][0], atol=1e-4) and torch.allclose(out[1], y[3][1], atol=1e-4)


def refusals():
    q = ops.mx4_quantize(tensor(16, 64))
    w, pair = ops.mx4_weight(q), ops.mx4_weight(q, q)
    wgu, wd, _ = experts(4, 64, 32)
    x, ids, wts = tensor(2, 64), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, 2)
    router = tensor(4, 64)
    layer = lambda **a: ops.mx4_moe_layer(**{**dict(x=x, w_router=router, bias=None, k=2, n_group=1, topk_group=1, scale=1.0, norm=False, sigmoid=False,  # noqa: E731
                                                    wgu=wgu, wd=wd), **a})
    return {
        "columns that are no blocks": lambda: ops.mx4_quantize(tensor(2, 48)),
        "no columns": lambda: ops.mx4_quantize(tensor(2, 0)),
        "one dimension": lambda: ops.mx4_quantize(tensor(1, 64)[0]),
        "whole numbers": lambda: ops.mx4_quantize(torch.zeros(2, 64, dtype=torch.int32)),
        "64 bits": lambda: ops.mx4_quantize(tensor(2, 64).double()),
        "result type": lambda: ops.mx4_dequantize(q, torch.float64),
        "scales of other blocks": lambda: ops.Mx4Tensor(q.codes, q.scales[:, :1]),
        "codes of another type": lambda: ops.Mx4Tensor(q.codes.int(), q.scales),
        "pair of other sizes": lambda: ops.mx4_weight(q, ops.mx4_quantize(tensor(17, 64))),
        "no rows": lambda: ops.mx4_weight(ops.Mx4Tensor(q.codes[:0], q.scales[:0])),
        "other columns": lambda: ops.mx4_linear(tensor(2, 96), w),
        "fp16 activations": lambda: ops.mx4_linear(x.half(), w),
        "three dimensions": lambda: ops.mx4_linear(x[None], w),
        "a pair as a matrix": lambda: ops.mx4_linear(x, pair),
        "a matrix as a pair": lambda: ops.mx4_gateup(x, w),
        "a tensor as a weight": lambda: ops.mx4_linear(x, q),
        "activation": lambda: ops.mx4_gateup(x, pair, "relu"),
        "residual": lambda: ops.mx4_linear(x, w, residual=tensor(2, 17)),
        "result in fp16": lambda: ops.mx4_linear(x, w, out_dtype=torch.float16),
        "operands of other columns": lambda: ops.mx4_matmul(q, ops.mx4_quantize(tensor(2, 96))),
        "a batch of operands": lambda: ops.mx4_matmul(q, ops.mx4_quantize(tensor(4, 64).view(2, 2, 64))),
        "one matrix as experts": lambda: ops.mx4_moe_ffn(x, None, ids, wts, pair, wd),
        "down of other sizes": lambda: ops.mx4_moe_ffn(x, None, ids, wts, wgu, experts(4, 64, 64)[1]),
        "64-bit ids": lambda: ops.mx4_moe_ffn(x, None, ids.long(), wts, wgu, wd),
        "weights of other tokens": lambda: ops.mx4_moe_ffn(x, None, ids, wts[:1], wgu, wd),
        "residual of another type": lambda: ops.mx4_moe_ffn(x, tensor(2, 64).bfloat16(), ids, wts, wgu, wd),
        "experts without a router row": lambda: layer(n_shared=1),
        "more choices than experts": lambda: layer(k=5),
        "uneven groups": lambda: layer(n_group=3),
        "more choices than the kept groups have": lambda: layer(n_group=4, topk_group=1),
        "bias": lambda: layer(bias=torch.zeros(3)),
    }


@pytest.mark.parametrize("what", sorted(refusals()))
def test_refused(what):
    with pytest.raises(ValueError):
        refusals()[what]()
