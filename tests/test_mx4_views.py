"""What the expert layers over 4-bit weights hand to their launches when tensors are views, and what the launches refuse: addresses only, nothing is computed."""
import contextlib
import ctypes as C
import types

import pytest
import torch

from jittorinfer_b200 import build
from jittorinfer_b200.ops import mx4, native, native_mx4

E, D, F, K = 8, 64, 32, 2
ALIGN = -2                     # JIB_E_ALIGN


@pytest.fixture
def calls(monkeypatch):
    """(name, arguments) of the launches; the library is not called."""
    seen = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.append((name, a)) or int(name in ("jib_mx4_moe_sizes", "jib_mx4_gemm_scratch"))

    def launched(rc, what):
        pass
    monkeypatch.setattr(native, "load", lambda: Lib())
    monkeypatch.setattr(native, "_ck", launched)
    monkeypatch.setattr(native, "_stream", lambda: 0)
    monkeypatch.setattr(native, "workspace", lambda dev: types.SimpleNamespace(status=torch.zeros(4, dtype=torch.int32)))
    monkeypatch.setattr(native_mx4, "_on", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(native_mx4, "_few_sizes", {})
    monkeypatch.setattr(native_mx4, "_scratch_bytes", {})
    return seen


def packed(n, k, gated):
    w = mx4.Mx4Weight(n, k, E, gated)
    w.codes = w.scales = w.factors = w.exps = torch.zeros(64, dtype=torch.uint8)
    return w


def view(rows, cols, dtype, offset):
    """Contiguous rows that begin `offset` elements behind an aligned address."""
    return torch.zeros(rows * cols + 8, dtype=dtype)[offset:offset + rows * cols].view(rows, cols)


def layer(T, router, residual=None):
    return native_mx4.moe_layer(torch.zeros(T, D, dtype=torch.bfloat16), router, None, K, 1, 1, 1.0, False, False, packed(F, D, True), packed(D, F, False), 0, False,
                                residual, "silu")


@pytest.mark.parametrize("T,launch,at", [(3, "jib_mx4_moe_prepare", 2), (20, "jib_moe_gate", 1)])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_a_router_at_an_odd_address_is_copied(calls, T, launch, at, offset):
    router = view(E, D, torch.float32, offset)
    layer(T, router)
    given = next(a[at] for name, a in calls if name == launch)
    assert given % 16 == 0 and (given == router.data_ptr()) == (offset == 0)


@pytest.fixture(scope="module")
def lib():
    return C.CDLL(build.build_kernels())


P = C.c_void_p
ALL = 1 << 20                  # an aligned address that is not read


@pytest.mark.parametrize("odd", [0, 1])
def test_a_router_at_an_odd_address_is_refused(lib, odd):
    a = [P(ALL), P(ALL)]
    a[odd] = P(ALL + 4)
    x, w = a
    f, z = C.c_float(1.0), C.c_longlong(D)
    assert lib.jib_mx4_moe_prepare(x, z, w, P(ALL), P(ALL), P(ALL), 4, 3, D, E, None) == ALIGN
    for T in (3, 20):
        assert lib.jib_moe_gate(x, w, None, None, P(ALL), P(ALL), P(ALL), T, D, E, K, 1, 1, f, 0, 0, 0, 0, 0, None) == ALIGN
        assert lib.jib_moe_gate_sort(x, w, None, None, P(ALL), P(ALL), P(ALL), T, D, E, K, 1, 1, f, 0, 0, 0, 0, 0, 0, E, P(ALL), P(ALL), P(ALL), P(ALL), None) == ALIGN
    assert lib.jib_moe_route_fused(x, w, None, P(ALL), P(ALL), P(ALL), P(ALL), P(ALL), P(ALL), P(ALL), 3, D, E, K, 1, 1, f, 0, 0, 0, 0, 0, E, None, f, None, None) == ALIGN


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_a_residual_at_an_odd_address_is_copied_for_the_weighted_sum(calls, offset):
    residual = view(20, D, torch.bfloat16, offset)
    layer(20, torch.zeros(E, D), residual)
    given = next(a[4] for name, a in calls if name == "jib_moe_combine")
    assert given % 16 == 0 and (given == residual.data_ptr()) == (offset == 0)


@pytest.mark.parametrize("odd", range(4))
def test_rows_at_an_odd_address_are_refused_by_the_weighted_sum(lib, odd):
    y, shared, residual, out = (P(ALL + 2 * (i == odd)) for i in range(4))
    assert lib.jib_moe_combine(y, P(ALL), P(ALL), shared, residual, out, 20, K, D, 20 * K, None) == ALIGN
    assert lib.jib_moe_combine_norm(y, P(ALL), P(ALL), shared, residual, P(ALL), out, P(ALL), 20, K, D, C.c_float(1e-6), None) == ALIGN


# ---- sizes of buffers -------------------------------------------------------------------------------------------------------------
def test_sizes_are_asked_for_on_each_device(calls):
    """Tiles, splits and partial sums go by a device's SMs."""
    w, down = packed(F, D, True), packed(D, F, False)
    for dev in ("cpu", "meta"):
        for _ in range(2):
            native_mx4._scratch(20, w, True, torch.device(dev))
            native_mx4._few(torch.zeros(3, D, dtype=torch.bfloat16, device=dev), w, down, K)
    assert [name for name, _ in calls] == ["jib_mx4_gemm_scratch", "jib_mx4_moe_sizes"] * 2


def test_a_buffer_that_is_too_small_is_refused(lib):
    SCRATCH = -6               # JIB_E_SCRATCH
    need = lib.jib_mx4_gemm_scratch
    need.restype, need.argtypes = C.c_longlong, [C.c_longlong] + [C.c_int] * 4
    d = native.Mx4Desc()
    d.x, d.w, d.w_scales, d.out, d.status, d.ldx, d.ldo, d.T, d.N, d.K, d.batch, d.max_rows = ALL, ALL, ALL, ALL, ALL, 2048, 512, 40, 512, 2048, 1, 40
    n = need(40, 512, 2048, 0, 0)
    assert n > 2 * 40 * 2048 + 4 * 40 * 512             # planes of x and, K being split, sums
    assert lib.jib_mx4_gemm(C.byref(d), None, P(ALL), C.c_longlong(n - 1), None, C.c_longlong(0), 0, None) == SCRATCH
    m, sizes = native.Mx4MoeDesc(), (C.c_longlong * 4)()
    assert lib.jib_mx4_moe_sizes(3, D, F, E, K, sizes) == 1
    for name, kind in m._fields_:
        if kind is C.c_void_p:
            setattr(m, name, ALL)
    m.T, m.d, m.F, m.E, m.k, m.n_group, m.topk_group, m.scale, m.part_floats = 3, D, F, E, K, 1, 1, 1.0, sizes[2] - 1
    assert lib.jib_mx4_moe(C.byref(m), None) == SCRATCH
