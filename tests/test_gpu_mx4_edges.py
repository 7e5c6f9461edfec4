"""4-bit operators where their inputs end: choices without an expert, rows of one token, memory that nobody wrote, scales far apart, strides and
addresses of views.  Limits as in the tests of the single operators."""
import pytest
import torch

from jittorinfer_b200 import ops
from jittorinfer_b200.ops import mx4
from test_gpu_mx4 import DEV, experts, gen, moe_want, randn, within

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
