"""Microscaled 4-bit floating point: tensors, weights laid out for the products, and the operators over them.

A value is an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times the power of two that its block of 32 columns shares (E8M0, a
byte less 127; 255 makes the block NaN).  Activations are bf16 (or fp32) in ``mx4_linear``, ``mx4_gateup`` and the MoE layers;
``mx4_matmul`` multiplies two 4-bit operands.  CUDA tensors go to the kernels in ``csrc/kernels/mx4*.cu``, CPU tensors to plain PyTorch; fp32
activations are multiplied in fp32.

What the kernels do to bf16 activations.  Tiled products take them as two planes of 8 bits: a value is exact down to 2^-11 of the largest magnitude among its
32 columns and within 2^-21 of that below.  Layers of up to 8 tokens take them as fp16 scaled by a power of two: exact down to 2^-29 of a row's
largest magnitude and within 2^-39 of it below; hidden units have 11 bits each, and sixteen neighbours that are all below 2^-24 of a token's largest in an
expert count as 0.  Sums are fp32.
A row with an infinity or NaN gives results that are not finite, and no other row's.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import reference as ref

BLOCK = 32                     # columns that share a scale
COLS = 128                     # columns of a packed chunk (csrc/kernels/mx4.cuh)
ACTS = ("silu", "gelu_tanh")
MX4_MAX_EXPERTS, MX4_MAX_CHOICES, MX4_MAX_GROUPS = 256, 32, 32          # of a layer, of a token: what the gate and the sort take (csrc/kernels/moe.cu)
_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


_kernels = _front = None          # native_mx4 once its library is loaded; the package


def _native(t: torch.Tensor):
    """The kernels' bindings for a tensor that goes to them, else None."""
    global _kernels, _front
    if not t.is_cuda:
        return None
    if _kernels is None:
        from .. import ops
        _front = ops
        if ops.force_torch():
            return None
        ops.nat()
        from . import native_mx4
        _kernels = native_mx4
    return None if _front._FORCE_TORCH else _kernels


def scale_rows(lead, blocks: int, device) -> torch.Tensor:
    """Room for the scales of rows, a view: each row starts at a multiple of 16 bytes."""
    if blocks % 16 == 0:
        return torch.empty(*lead, blocks, dtype=torch.uint8, device=device)
    return torch.empty(*lead, (blocks + 15) // 16 * 16, dtype=torch.uint8, device=device)[..., :blocks]


def _laid_out(s: torch.Tensor) -> bool:
    ld, want = s.stride(-2), s.stride(-2)
    if s.stride(-1) != 1 or ld % 16 or ld < s.shape[-1] or s.data_ptr() % 16:
        return False
    for i in range(s.dim() - 2, -1, -1):
        if s.stride(i) != want:
            return False
        want *= s.shape[i]
    return True


class Mx4Tensor:
    """Rows of 4-bit values: ``codes`` uint8 [..., cols / 2] (the lower half of a byte is the even column), ``scales`` uint8 [..., cols / 32].  They are kept
    as the kernels read them: codes dense and 16-byte aligned, scale rows at multiples of 16 bytes; tensors that are otherwise are copied."""
    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.device != scales.device:
            raise ValueError("codes and scales are uint8 tensors of one device")
        if codes.dim() < 2 or codes.shape[-1] == 0 or codes.shape[-1] % (BLOCK // 2) or \
                tuple(scales.shape) != (*codes.shape[:-1], codes.shape[-1] * 2 // BLOCK):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not blocks of {BLOCK} columns")
        codes = codes.contiguous()
        self.codes = codes if codes.data_ptr() % 16 == 0 else codes.clone()
        if not _laid_out(scales):
            rows = scale_rows(scales.shape[:-1], scales.shape[-1], scales.device)
            rows.copy_(scales)
            scales = rows
        self.scales = scales

    @classmethod
    def _of(cls, codes: torch.Tensor, scales: torch.Tensor) -> "Mx4Tensor":
        """From tensors that are laid out as they have to be."""
        q = cls.__new__(cls)
        q.codes, q.scales = codes, scales
        return q

    @property
    def shape(self) -> Tuple[int, ...]:
        return (*self.codes.shape[:-1], self.codes.shape[-1] * 2)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


class Mx4Weight:
    """A matrix [n, k], or ``batch`` of them, or as many gated pairs, in the order in which the products read it.  On the GPU ``codes`` and ``scales`` hold
    chunks of 128 columns, rows within them (of a pair 16 of each matrix in turn), ``factors`` and ``exps`` of a batch the scales again as expert layers of a
    few tokens need them; ``far`` says that some of its weights lie too far below their row's largest scale for those, which then do not read it;
    elsewhere ``plain`` holds the tensors."""
    __slots__ = ("n", "k", "batch", "gated", "codes", "scales", "factors", "exps", "far", "plain")

    def __init__(self, n, k, batch, gated):
        self.n, self.k, self.batch, self.gated = n, k, batch, gated
        self.codes = self.scales = self.factors = self.exps = self.plain = None
        self.far = False

    @property
    def device(self) -> torch.device:
        return self.codes.device if self.codes is not None else self.plain[0].device

    @property
    def matrices(self) -> int:
        return self.batch or 1

    @property
    def chunks(self) -> int:
        return (self.k + COLS - 1) // COLS

    @property
    def rows(self) -> int:
        """Rows of a matrix or pair as they are laid out."""
        return (self.n + 15) // 16 * 32 if self.gated else (self.n + 31) // 32 * 32

    def nbytes(self) -> int:
        if self.codes is not None:
            return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.factors, self.exps) if t is not None)
        return sum(p.nbytes() for p in self.plain)

    def values(self, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, ...]:
        """The matrices [(batch,) n, k] (a pair: gate, up) as plain tensors."""
        if self.codes is None:
            return tuple(_dequantize(p, dtype) for p in self.plain)
        return tuple(_unpack(self, m).to(dtype) for m in range(2 if self.gated else 1))


# ---- plain PyTorch ---------------------------------------------------------------------------------------------------------------
def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp64 for integers e."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)


def _quantize(x: torch.Tensor) -> Mx4Tensor:
    b = x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK).double()
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(top)
    top = torch.where(bad, torch.ones_like(top), top)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32)).clamp(-127, 127)
    y = b * _pow2(-e)[..., None]
    a = y.abs()
    a = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) * 2, torch.round(a / 2) * 4)).clamp(max=12)       # twice the value
    code = torch.where(a <= 4, a, torch.where(a == 6, 5.0, torch.where(a == 8, 6.0, 7.0)))
    code = torch.where(bad[..., None], torch.zeros_like(code), code + 8 * torch.signbit(y)).to(torch.uint8).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return Mx4Tensor(code[..., 0] | (code[..., 1] << 4), torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8))


def _dequantize(q: Mx4Tensor, dtype: torch.dtype) -> torch.Tensor:
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), dtype=torch.float64, device=q.device)
    v = torch.stack((table[(q.codes & 15).long()], table[(q.codes >> 4).long()]), -1).reshape(*q.shape[:-1], -1, BLOCK)
    s = torch.where(q.scales == 255, torch.full_like(q.scales, 0, dtype=torch.float64).fill_(float("nan")), _pow2(q.scales.int() - 127))
    return (v * s[..., None]).reshape(q.shape).to(dtype)


def _unpack(w: Mx4Weight, member: int) -> torch.Tensor:
    """fp32 [(batch,) n, k] from the packed bytes (the inverse of the kernel that lays them out)."""
    def rows(x):           # [e, chunks, rows, columns] -> [e, n, chunks, columns]
        x = x.transpose(1, 2)
        if w.gated:
            x = x.reshape(w.matrices, -1, 2, 16, *x.shape[2:])[:, :, member].flatten(1, 2)
        return x[:, :w.n]
    code = rows(w.codes)
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), dtype=torch.float64, device=w.device)
    v = torch.stack((table[(code & 15).long()], table[(code >> 4).long()]), -1).reshape(*code.shape[:3], COLS // BLOCK, BLOCK)

    def scaled(s):
        return (v * s[..., None]).reshape(w.matrices, w.n, -1)[..., :w.k]
    e = rows(w.scales).int()
    nan = torch.full(e.shape, float("nan"), dtype=torch.float64, device=w.device)
    out = scaled(torch.where(e == 255, nan, _pow2(e - 127)))
    if w.factors is not None:
        f, unit = rows(w.factors).int() >> 2, _pow2(rows(w.exps[:, None, :, None]))
        again = scaled(torch.where(f == 31, nan, torch.where(f > 0, _pow2(f - 15), torch.zeros_like(nan))) * unit)
        largest = out.nan_to_num(0.0).abs().amax(-1, keepdim=True)
        lost = (again == 0) & (out.abs() < 2.0 ** -24 * largest)          # scales more than 27 binades below the largest are 0 in the second form
        if not bool(((out == again) | (out.isnan() & again.isnan()) | lost).all()):
            raise RuntimeError("the two forms of a packed weight's scales differ")
    out = out.float()
    return out if w.batch else out[0]


def _act(z: torch.Tensor, act: str) -> torch.Tensor:
    return torch.nn.functional.silu(z) if act == "silu" else torch.nn.functional.gelu(z, approximate="tanh")


# ---- checks ----------------------------------------------------------------------------------------------------------------------
def _check_rows(x: torch.Tensor, k: int, what: str) -> None:
    if x.dim() != 2 or x.shape[1] != k:
        raise ValueError(f"{what}: activations {tuple(x.shape)} for {k} columns")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{what}: activations are bf16 or fp32, not {x.dtype}")


def _check_weight(x: torch.Tensor, w: Mx4Weight, gated: bool, batched: bool, what: str) -> None:
    if not isinstance(w, Mx4Weight) or w.gated != gated or (w.batch is not None) != batched:
        raise ValueError(f"{what}: needs {'a batch of ' if batched else ''}{'gated pairs' if gated else 'matrices'} from mx4_weight")
    if w.device != x.device:
        raise ValueError(f"{what}: weights on {w.device}, activations on {x.device}")


def _check_residual(residual: Optional[torch.Tensor], rows: int, cols: int, x: torch.Tensor, what: str) -> None:
    if residual is not None and (tuple(residual.shape) != (rows, cols) or residual.dtype not in (torch.bfloat16, torch.float32) or residual.device != x.device):
        raise ValueError(f"{what}: residual {tuple(residual.shape)} {residual.dtype} for a result of {(rows, cols)}")


def _check_out(out_dtype: Optional[torch.dtype], x_dtype: torch.dtype, what: str) -> torch.dtype:
    dtype = out_dtype or x_dtype
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{what}: results are bf16 or fp32, not {dtype}")
    return dtype


# ---- operators -------------------------------------------------------------------------------------------------------------------
def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """bf16, fp16 or fp32 [..., cols] to 4 bits, cols a multiple of 32.  A block's scale is 2^(floor(log2 of its largest magnitude) - 2), at least
    2^-127; a value goes to the nearest code, ties to the even one, at most 6.  A block with an infinity or NaN becomes NaN."""
    if x.dtype not in _TYPES:
        raise ValueError(f"mx4_quantize: bf16, fp16 or fp32, not {x.dtype}")
    if x.dim() < 2 or x.shape[-1] == 0 or x.shape[-1] % BLOCK:
        raise ValueError(f"mx4_quantize: rows of whole blocks of {BLOCK}, not {tuple(x.shape)}")
    n = _native(x)
    return n.quantize(x) if n else _quantize(x)


def mx4_dequantize(q: Mx4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values as bf16, fp16 or fp32 (rounded where the type cannot hold them)."""
    if dtype not in _TYPES:
        raise ValueError(f"mx4_dequantize: bf16, fp16 or fp32, not {dtype}")
    n = _native(q.codes)
    return n.dequantize(q, dtype) if n else _dequantize(q, dtype)


def mx4_weight(q: Mx4Tensor, up: Optional[Mx4Tensor] = None) -> Mx4Weight:
    """Lays a matrix [n, k] or a batch of them [e, n, k] out for the products, once; with ``up`` a gated pair (gate, up).  The tensors are not needed
    afterwards (on the CPU they are kept as they are)."""
    if len(q.shape) not in (2, 3) or 0 in q.shape or (up is not None and (up.shape != q.shape or up.device != q.device)):
        raise ValueError(f"mx4_weight: {q.shape}" + (f" and {up.shape}" if up is not None else ""))
    batch = q.shape[0] if len(q.shape) == 3 else None
    w = Mx4Weight(q.shape[-2], q.shape[-1], batch, up is not None)
    n = _native(q.codes)
    if n:
        n.pack(w, q, up)
    else:
        w.plain = (q,) if up is None else (q, up)
    return w


def mx4_linear(x: torch.Tensor, w: Mx4Weight, residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x w^T + residual (bf16 or fp32; one row expanded over the tokens is a bias); ``out_dtype`` bf16 or fp32, default x's."""
    _check_weight(x, w, False, False, "mx4_linear")
    _check_rows(x, w.k, "mx4_linear")
    _check_residual(residual, x.shape[0], w.n, x, "mx4_linear")
    dtype = _check_out(out_dtype, x.dtype, "mx4_linear")
    n = _native(x)
    if n:
        return n.product(x, w, residual, dtype, None)
    y = x.float() @ w.values()[0].T
    return (y if residual is None else y + residual.float()).to(dtype)


def mx4_gateup(x: torch.Tensor, w: Mx4Weight, act: str = "silu", out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x Wg^T) * (x Wu^T); ``act`` "silu" or "gelu_tanh"."""
    _check_weight(x, w, True, False, "mx4_gateup")
    _check_rows(x, w.k, "mx4_gateup")
    if act not in ACTS:
        raise ValueError(f"mx4_gateup: activation {act!r}, not one of {ACTS}")
    dtype = _check_out(out_dtype, x.dtype, "mx4_gateup")
    n = _native(x)
    if n:
        return n.product(x, w, None, dtype, act)
    g, u = w.values()
    return (_act(x.float() @ g.T, act) * (x.float() @ u.T)).to(dtype)


def mx4_matmul(a: Mx4Tensor, b: Mx4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b^T for a [t, k] and b [n, k] in 4 bits; the result [t, n] is bf16 or fp32."""
    if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[1] != b.shape[1] or a.device != b.device:
        raise ValueError(f"mx4_matmul: {a.shape} on {a.device} and {b.shape} on {b.device}")
    dtype = _check_out(out_dtype, torch.bfloat16, "mx4_matmul")
    n = _native(a.codes)
    if n:
        return n.matmul(a, b, dtype)
    return (_dequantize(a, torch.float32) @ _dequantize(b, torch.float32).T).to(dtype)


def _check_moe(x, wgu, wd, residual, act, what):
    _check_weight(x, wgu, True, True, what)
    _check_weight(x, wd, False, True, what)
    _check_rows(x, wgu.k, what)
    if (wd.n, wd.k, wd.batch) != (wgu.k, wgu.n, wgu.batch):
        raise ValueError(f"{what}: {wd.batch} down matrices {(wd.n, wd.k)} for {wgu.batch} pairs {(wgu.n, wgu.k)}")
    if act not in ACTS:
        raise ValueError(f"{what}: activation {act!r}, not one of {ACTS}")
    _check_residual(residual, x.shape[0], x.shape[1], x, what)
    if residual is not None and residual.dtype != x.dtype:
        raise ValueError(f"{what}: residual {residual.dtype} beside activations {x.dtype}")


def _moe_plain(x, residual, ids, wts, wgu, wd, act):
    g, u = wgu.values()
    d, = wd.values()
    out = torch.zeros(x.shape, dtype=torch.float32, device=x.device) if residual is None else residual.float()
    for e in range(wgu.batch):
        share = torch.where(ids == e, wts, torch.zeros_like(wts)).sum(-1)
        rows = torch.nonzero((ids == e).any(-1))[:, 0]
        if rows.numel():
            xr = x[rows].float()
            h = (_act(xr @ g[e].T, act) * (xr @ u[e].T)).to(x.dtype).float()
            out = out.index_add(0, rows, share[rows, None] * (h @ d[e].T))
    return out.to(x.dtype)


def mx4_moe_ffn(x: torch.Tensor, residual: Optional[torch.Tensor], ids: torch.Tensor, wts: torch.Tensor, wgu: Mx4Weight, wd: Mx4Weight,
                act: str = "silu") -> torch.Tensor:
    """residual + sum over the choices of a token of wts * down(act(gate) * up), x's dtype.

    ``ids`` int32, ``wts`` fp32 [tokens, k]; an id outside the experts counts for nothing, its weight neither.  ``residual`` may be None.  Up to 8 bf16 tokens
    run as two launches, unless weights lie more than 27 binades below the largest scale of their row.  More tokens' hidden units and each expert's result
    before the weighted sum are rounded to x's dtype."""
    _check_moe(x, wgu, wd, residual, act, "mx4_moe_ffn")
    if ids.dim() != 2 or ids.shape[0] != x.shape[0] or ids.shape != wts.shape or ids.dtype != torch.int32 or wts.dtype != torch.float32 or \
            ids.device != x.device or wts.device != x.device:
        raise ValueError(f"mx4_moe_ffn: ids {tuple(ids.shape)} {ids.dtype} and weights {tuple(wts.shape)} {wts.dtype} for {x.shape[0]} tokens")
    n = _native(x)
    return n.moe_ffn(x, residual, ids.contiguous(), wts.contiguous(), wgu, wd, act) if n else _moe_plain(x, residual, ids, wts, wgu, wd, act)


def mx4_moe_layer(x: torch.Tensor, w_router: torch.Tensor, bias: Optional[torch.Tensor], k: int, n_group: int, topk_group: int, scale: float, norm: bool,
                  sigmoid: bool, wgu: Mx4Weight, wd: Mx4Weight, n_shared: int = 0, group_top2: bool = False,
                  residual: Optional[torch.Tensor] = None, act: str = "silu") -> torch.Tensor:
    """A whole MoE layer: router, choice of experts, their products, weighted sum and residual.  The gate's arguments are those of ``moe_gate``; the
    last ``n_shared`` experts of the weights take every token with weight 1.  On the GPU at most 32 choices, shared ones among them, of 256 experts in 32
    groups.  Launches and roundings as in ``mx4_moe_ffn``."""
    _check_moe(x, wgu, wd, residual, act, "mx4_moe_layer")
    E = w_router.shape[0] if w_router.dim() == 2 else -1
    if w_router.dim() != 2 or w_router.shape[1] != x.shape[1] or E + n_shared != wgu.batch or n_shared < 0 or w_router.dtype != torch.float32 or \
            w_router.device != x.device:
        raise ValueError(f"mx4_moe_layer: router {tuple(w_router.shape)} {w_router.dtype} and {n_shared} shared experts for {wgu.batch} of width {x.shape[1]}")
    if bias is not None and (tuple(bias.shape) != (E,) or bias.dtype != torch.float32 or bias.device != x.device):
        raise ValueError(f"mx4_moe_layer: bias {tuple(bias.shape)} {bias.dtype} for {E} experts")
    if k < 1 or n_group < 1 or E % n_group or not 1 <= topk_group <= n_group or k > topk_group * (E // n_group):
        raise ValueError(f"mx4_moe_layer: {k} of {E} experts in {topk_group} of {n_group} groups")
    n = _native(x)
    if n:
        return n.moe_layer(x, w_router, bias if bias is None else bias.contiguous(), k, n_group, topk_group, scale, norm, sigmoid, wgu, wd,
                           n_shared, group_top2, residual, act)
    ids, wts = ref.moe_gate(x, w_router, bias, k, n_group, topk_group, scale, norm, sigmoid, n_shared, group_top2)
    return _moe_plain(x, residual, ids, wts, wgu, wd, act)
