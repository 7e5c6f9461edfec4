"""ctypes front-end of the kernels over microscaled 4-bit tensors (see ``ops.mx4`` for the operators and their checks)."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional

import torch

from . import native as nat
from .mx4 import COLS, MX4_MAX_CHOICES as MAX_CHOICES, MX4_MAX_EXPERTS as MAX_EXPERTS, MX4_MAX_GROUPS as MAX_GROUPS, Mx4Tensor, Mx4Weight, scale_rows

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
# Tokens of a layer in two launches, us, as tiles in brackets: 8 of width 2048, 64 + 2 experts of 1408 67.6 (69.3), one 33.8 (38.5); of 5120, 160 + 2 of 1536
# 154.6 (159.3) and 53.4 (71.1); of 1024, 16 + 2 of 512 28.9 (30.9) and 25.6 (26.2); of 2048, 128 of 768 59.8 (66.3) and 34.6 (36.1).  9, with a second tile of 8
# rows here: 98 (73).
FEW_TOKENS = 8
PAD = 32                                     # rows of an expert are padded to in grouped products (csrc/kernels/mx4_gemm.cu)
_NO_SWITCH = contextlib.nullcontext()
_current = nat._device or torch.cuda.current_device


def _on(t: torch.Tensor):
    """The tensor's device as the current one: launches go to the current device's stream."""
    return _NO_SWITCH if t.get_device() == _current() else torch.cuda.device(t.device)


def quantize(x: torch.Tensor) -> Mx4Tensor:
    *lead, cols = x.shape
    x2 = x if len(lead) == 1 else x.reshape(-1, cols)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    codes = torch.empty(*lead, cols // 2, dtype=torch.uint8, device=x.device)
    scales = scale_rows(lead, cols // 32, x.device)
    with _on(x):
        nat._ck(nat.load().jib_mx4_quantize(x2.data_ptr(), TYPES[x.dtype], x2.stride(0), codes.data_ptr(), scales.data_ptr(), scales.stride(-2), x2.shape[0], cols,
                                            nat._stream()), "mx4_quantize")
    return Mx4Tensor._of(codes, scales)


def dequantize(q: Mx4Tensor, dtype: torch.dtype) -> torch.Tensor:
    out = torch.empty(q.shape, dtype=dtype, device=q.codes.device)
    cols = out.shape[-1]
    with _on(out):
        nat._ck(nat.load().jib_mx4_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), q.scales.stride(-2), out.data_ptr(), TYPES[dtype], out.numel() // cols, cols,
                                              nat._stream()), "mx4_dequantize")
    return out


def pack(w: Mx4Weight, q: Mx4Tensor, up: Optional[Mx4Tensor]) -> None:
    E, R, members = w.matrices, w.rows, (q,) if up is None else (q, up)
    w.codes = torch.empty(E, w.chunks, R, COLS // 2, dtype=torch.uint8, device=q.device)
    w.scales = torch.empty(E, w.chunks, R, COLS // 32, dtype=torch.uint8, device=q.device)
    lost = None
    if w.batch:                    # only layers of experts have a form for a few tokens
        w.factors = torch.empty_like(w.scales)
        w.exps = torch.empty(E, R, dtype=torch.int32, device=q.device)
        lost = torch.zeros(1, dtype=torch.int32, device=q.device)
    with _on(q.codes):
        for m, t in enumerate(members):
            nat._ck(nat.load().jib_mx4_pack(t.codes.data_ptr(), t.scales.data_ptr(), t.scales.stride(-2), w.codes.data_ptr(), w.scales.data_ptr(),
                                            nat._p(w.factors), nat._p(w.exps), nat._p(lost), E, w.n, w.k, len(members), m, nat._stream()), "mx4_pack")
        # (read once, when weights are laid out; a graph that does so cannot say yet)
        w.far = lost is not None and (torch.cuda.is_current_stream_capturing() or bool(lost.item()))


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Rows that the kernels can read: contiguous, 16-byte steps."""
    ok = x.stride(1) == 1 and x.stride(0) >= x.shape[1] and (x.stride(0) * x.element_size()) % 16 == 0 and x.data_ptr() % 16 == 0
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _vectors(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _desc(w: Mx4Weight, out: torch.Tensor, residual: Optional[torch.Tensor], act: Optional[str]) -> "nat.Mx4Desc":
    d = nat.Mx4Desc()
    d.w, d.w_scales = w.codes.data_ptr(), w.scales.data_ptr()
    d.out, d.ldo, d.out_f32 = out.data_ptr(), out.stride(0), int(out.dtype == torch.float32)
    if residual is not None:
        d.residual, d.ldr, d.res_f32 = residual.data_ptr(), residual.stride(0), int(residual.dtype == torch.float32)
    d.T, d.N, d.K, d.batch, d.max_rows = out.shape[0], w.n, w.k, 1, out.shape[0]
    d.gated, d.act = int(w.gated), nat.ACTS[act or "silu"]
    d.status = nat.workspace(out.device).status.data_ptr()
    return d


_scratch_bytes: dict = {}        # (rows, n, k, gated, grouped, device): tiles and splits go by a device's SMs


def _scratch(rows: int, w: Mx4Weight, grouped: bool, device) -> torch.Tensor:
    key = (rows, w.n, w.k, int(w.gated), int(grouped), device)
    n = _scratch_bytes.get(key)
    if n is None:
        if len(_scratch_bytes) > 4096:
            _scratch_bytes.clear()
        n = _scratch_bytes[key] = nat.load().jib_mx4_gemm_scratch(*key[:5])
    return torch.empty(n, dtype=torch.uint8, device=device)


def product(x: torch.Tensor, w: Mx4Weight, residual: Optional[torch.Tensor], dtype: torch.dtype, act: Optional[str]) -> torch.Tensor:
    x = _rows(x)
    out = torch.empty(x.shape[0], w.n, dtype=dtype, device=x.device)
    if residual is not None and residual.stride(1) != 1:
        residual = residual.contiguous()
    if x.shape[0]:
        with _on(x):
            d = _desc(w, out, residual, act)
            if x.dtype == torch.bfloat16:
                scratch = _scratch(x.shape[0], w, False, x.device)
                d.x, d.ldx = x.data_ptr(), x.stride(0)
                nat._ck(nat.load().jib_mx4_gemm(C.byref(d), None, scratch.data_ptr(), scratch.numel(), None, 0, 0, nat._stream()), "mx4_gemm")
            else:
                d.x, d.ldx = x.data_ptr(), x.stride(0)
                nat._ck(nat.load().jib_mx4_product_simt(C.byref(d), nat._stream()), "mx4_product_simt")
    return out


def _grouped_simt(x: torch.Tensor, w: Mx4Weight, seg: torch.Tensor, src: Optional[torch.Tensor], rows: int, act: Optional[str]) -> torch.Tensor:
    """fp32 rows sorted by expert: expert e's are seg[e] .. seg[e + 1] - 1; row r is computed from x[src[r]] (without ``src`` x[r])."""
    out = torch.empty(rows, w.n, dtype=x.dtype, device=x.device)
    d = _desc(w, out, None, act)
    d.x, d.ldx, d.seg, d.src, d.batch, d.max_rows = x.data_ptr(), x.stride(0), seg.data_ptr(), nat._p(src), w.batch, rows
    nat._ck(nat.load().jib_mx4_product_simt(C.byref(d), nat._stream()), "mx4_grouped_simt")
    return out


def _grouped(x: torch.Tensor, wgu: Mx4Weight, wd: Mx4Weight, pad, src: int, pairs: int, act: str) -> torch.Tensor:
    """The experts' results, bf16 rows in the padded order ``pad`` = (first, count, capacity); row r is computed from x[src[r]].  Hidden units go from product to
    product as planes where the first can write them.

    Results are rounded to bf16 as those of the layer over bf16 weights are: 515 tokens of width 2048 write and read 19 MB of them, twice that in fp32.  With
    the hidden units' rounding the layer is 0.0020 from the definition in 64 bits there (rms, relative); 0.0017 is the rounding of its own result."""
    first, count, cap = pad
    L, stream = nat.load(), nat._stream()
    scratch, then = _scratch(cap, wgu, True, x.device), _scratch(cap, wd, True, x.device)
    joined = L.jib_mx4_gemm_joins(wgu.n, 1)
    h = torch.empty(0 if joined else cap, wgu.n, dtype=torch.bfloat16, device=x.device)
    y = torch.empty(cap, wd.n, dtype=torch.bfloat16, device=x.device)
    d = _desc(wgu, h, None, act)
    d.T, d.x, d.ldx, d.seg, d.src, d.batch, d.max_rows = cap, x.data_ptr(), x.stride(0), first, src, wgu.batch, pairs
    nat._ck(L.jib_mx4_gemm(C.byref(d), count, scratch.data_ptr(), scratch.numel(), then.data_ptr() if joined else None, then.numel(), 0, stream), "mx4_grouped")
    d = _desc(wd, y, None, None)
    d.x, d.ldx, d.seg, d.batch, d.max_rows = h.data_ptr(), wgu.n, first, wd.batch, pairs
    nat._ck(L.jib_mx4_gemm(C.byref(d), count, then.data_ptr(), then.numel(), None, 0, joined, stream), "mx4_grouped")
    return y


def matmul(a: Mx4Tensor, b: Mx4Tensor, dtype: torch.dtype) -> torch.Tensor:
    T, K = a.shape
    N = b.shape[0]
    out = torch.empty(T, N, dtype=dtype, device=a.device)
    if T and N:
        with _on(out):
            nat._ck(nat.load().jib_mx4_matmul(a.codes.data_ptr(), a.scales.data_ptr(), a.scales.stride(0), b.codes.data_ptr(), b.scales.data_ptr(),
                                              b.scales.stride(0), out.data_ptr(), N, int(dtype == torch.float32), T, N, K,
                                              nat.workspace(out.device).status.data_ptr(), nat._stream()), "mx4_matmul")
    return out


_few_sizes: dict = {}        # (tokens, width, hidden, experts, choices, device) -> bytes of xf and h, floats of part, ints of sync, or None


def _few(x: torch.Tensor, wgu: Mx4Weight, wd: Mx4Weight, k: int):
    """The buffers' sizes where a layer of few tokens runs as two launches."""
    if x.dtype != torch.bfloat16 or x.shape[0] > FEW_TOKENS or wgu.far or wd.far:
        return None
    key = (x.shape[0], wgu.k, wgu.n, wgu.batch, k, x.device)
    if key not in _few_sizes:
        s = (C.c_longlong * 4)()
        _few_sizes[key] = tuple(s) if nat.load().jib_mx4_moe_sizes(*key[:5], s) else None
    return _few_sizes[key]


def _few_layer(x, residual, wgu: Mx4Weight, wd: Mx4Weight, sizes, act: str, m, w_router: Optional[torch.Tensor]) -> torch.Tensor:
    """Both launches; ``m`` holds what says which experts."""
    T, d = x.shape
    xf, h, part, sync = sizes
    out = torch.empty(T, d, dtype=x.dtype, device=x.device)
    E = w_router.shape[0] if w_router is not None else 0
    scratch = torch.empty(xf + h + 4 * (part + sync + T * E), dtype=torch.uint8, device=x.device)
    m.out, m.xf = out.data_ptr(), scratch.data_ptr()
    m.h, m.part, m.sync, m.part_floats = m.xf + xf, m.xf + xf + h, m.xf + xf + h + 4 * part, part
    if E:
        m.logits = m.sync + 4 * sync
    if residual is not None:
        m.residual, m.ldr = residual.data_ptr(), residual.stride(0)
    m.gu, m.gu_factors, m.gu_exp = wgu.codes.data_ptr(), wgu.factors.data_ptr(), wgu.exps.data_ptr()
    m.down, m.down_factors, m.down_exp = wd.codes.data_ptr(), wd.factors.data_ptr(), wd.exps.data_ptr()
    m.status = nat.workspace(x.device).status.data_ptr()
    m.T, m.d, m.F, m.E, m.act = T, d, wgu.n, wgu.batch, nat.ACTS[act]
    L, stream = nat.load(), nat._stream()
    nat._ck(L.jib_mx4_moe_prepare(x.data_ptr(), x.stride(0), nat._p(w_router), m.logits, m.xf, m.sync, sync, T, d, E, stream), "mx4_moe_prepare")
    nat._ck(L.jib_mx4_moe(C.byref(m), stream), "mx4_moe")
    return out


def moe_ffn(x, residual, ids, wts, wgu, wd, act, n_shared=0):
    x = _rows(x)
    T, k = ids.shape
    if T == 0:
        return torch.empty_like(x)
    if residual is not None and residual.stride(1) != 1:
        residual = residual.contiguous()
    if T * k > 1 << 28:
        raise ValueError(f"mx4_moe_ffn: {T} tokens of {k} choices in one call")
    if wgu.batch > MAX_EXPERTS:
        raise ValueError(f"mx4_moe_ffn: {wgu.batch} experts, at most {MAX_EXPERTS}")
    if k == 0:
        return torch.zeros_like(x) if residual is None else residual.clone(memory_format=torch.contiguous_format)
    with _on(x):
        sizes = _few(x, wgu, wd, k)
        if sizes is not None:
            m = nat.Mx4MoeDesc()
            m.ids, m.wts, m.k = ids.data_ptr(), wts.data_ptr(), k
            return _few_layer(x, residual, wgu, wd, sizes, act, m, None)
        E, n = wgu.batch, T * k
        if x.dtype == torch.bfloat16:
            cap = (n + min(E, n) * (PAD - 1) + PAD - 1) // PAD * PAD
            table = torch.empty(2 * E + 1 + cap + n, dtype=torch.int32, device=x.device)       # first, count, token of each row, row of each pair
            first = table.data_ptr()
            count, row_src, pair_row = first + 4 * (E + 1), first + 4 * (2 * E + 1), first + 4 * (2 * E + 1 + cap)
            nat._ck(nat.load().jib_mx4_sort(ids.data_ptr(), n, k, E, first, count, row_src, pair_row, nat._stream()), "mx4_sort")
            routed = T * (k - n_shared) * E // (E - n_shared)       # the rows were there no shared experts: what the tiles are chosen for
            y = _grouped(x, wgu, wd, (first, count, cap), row_src, routed, act)
            return nat.moe_combine(y, table[2 * E + 1 + cap:].view(T, k), wts, None, None if residual is None else _vectors(residual))
        seg, src, dest = nat.moe_permute(ids, 0, E)
        h = _grouped_simt(x, wgu, seg, src, n, act)
        y = _grouped_simt(h, wd, seg, None, n, None)
        # a choice without an expert has no row: what stands in its place, and its weight, may be no number
        out = torch.where((dest >= 0)[..., None], y[dest.clamp(min=0).long()] * wts[..., None], 0.0).sum(1)
        return out if residual is None else out + residual


def moe_layer(x, w_router, bias, k, n_group, topk_group, scale, norm, sigmoid, wgu, wd, n_shared, group_top2, residual, act):
    x = _rows(x)
    T, d = x.shape
    if T == 0:
        return torch.empty_like(x)
    if k + n_shared > MAX_CHOICES or wgu.batch > MAX_EXPERTS or n_group > MAX_GROUPS:
        raise ValueError(f"mx4_moe_layer: {k} + {n_shared} of {wgu.batch} experts in {n_group} groups; at most {MAX_CHOICES} of {MAX_EXPERTS} in {MAX_GROUPS}")
    with _on(x):
        w_router = _vectors(w_router)
        if x.stride(0) != d:           # (a single row counts as contiguous whatever its stride)
            x = x.clone(memory_format=torch.contiguous_format) if T > 1 else x.as_strided((1, d), (d, 1))
        sizes = _few(x, wgu, wd, k + n_shared)
        if sizes is not None:
            if residual is not None and residual.stride(1) != 1:
                residual = residual.contiguous()
            m = nat.Mx4MoeDesc()
            m.bias, m.k, m.n_group, m.topk_group, m.scale = nat._p(bias), k, n_group, topk_group, scale
            m.norm, m.sigmoid, m.n_shared, m.group_top2 = int(norm), int(sigmoid), n_shared, int(group_top2)
            return _few_layer(x, residual, wgu, wd, sizes, act, m, w_router)
        ids, wts = nat.moe_gate(x, w_router, bias, k, n_group, topk_group, scale, norm, sigmoid, n_shared, group_top2)
    return moe_ffn(x, residual, ids, wts, wgu, wd, act, n_shared)
