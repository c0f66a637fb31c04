"""8-bit products with a float32 scale for each block of 128, with gradients.

Beside the MX tiers (a power-of-two scale for each 32 elements), this is the
form in which 8-bit weights are usually stored and trained: e4m3 payloads,
a scale for each 128 values along a row of the left operand, and for each
128 x 128 tile of the right one.

    top = max(max |x| over the block, 2**-100)
    scale = top / 448;  q = e4m3(x * (448 / top));  x ~ q * scale

in float32, each step rounded to nearest. A block with a NaN or an infinity
stands for NaN. On a GPU the matrix unit adds the products of 8 neighbours
along k with 13 bits behind the largest one's power of two, and these sums in
float32. GPU tensors run the HIP kernels (csrc/fp8.hip,
csrc/grouped_core.h), CPU tensors plain torch.
"""

from __future__ import annotations

import dataclasses
import math
from typing import Optional, Union

import torch

from .backend import require_ext, use_hip
from .grouped import (check_capture, check_offsets, check_out_dtype,
                      needs_grad, product_type, refuse_tangents, rows_product,
                      weights_product)

BLOCK = 128
_MAX = 448.0
_TOP_MIN = 2.0 ** -100
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _ceil128(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


@dataclasses.dataclass
class Fp8Blocks:
    """A matrix, or a stack of them, in e4m3 with block scales.

    data: float8_e4m3fn [..., rows, cols], contiguous.
    scale: float32, contiguous, column blocks first: [..., ceil(cols / 128),
    rows] for kind "row", [..., ceil(cols / 128), ceil(rows / 128)] for
    kind "tile"."""
    data: torch.Tensor
    scale: torch.Tensor
    kind: str

    def __post_init__(self):
        if self.kind not in ("row", "tile"):
            raise ValueError(f'kind must be "row" or "tile", got '
                             f'{self.kind!r}')
        d, s = self.data, self.scale
        if d.dtype != torch.float8_e4m3fn or s.dtype != torch.float32:
            raise TypeError(f"data must be float8_e4m3fn and scale float32, "
                            f"got {d.dtype} and {s.dtype}")
        if d.dim() < 2:
            raise ValueError("data must have at least two dimensions")
        r = d.shape[-2] if self.kind == "row" else _ceil128(d.shape[-2])
        want = tuple(d.shape[:-2]) + (_ceil128(d.shape[-1]), r)
        if tuple(s.shape) != want:
            raise ValueError(f"scale must be {want} for data "
                             f"{tuple(d.shape)}, got {tuple(s.shape)}")
        if d.device != s.device:
            raise ValueError("data and scale must be on one device")
        if not (d.is_contiguous() and s.is_contiguous()):
            raise ValueError("data and scale must be contiguous")

    @classmethod
    def _made(cls, data, scale, kind) -> "Fp8Blocks":
        """Blocks that were made here and need no checks."""
        q = object.__new__(cls)
        q.data, q.scale, q.kind = data, scale, kind
        return q

    @property
    def shape(self) -> torch.Size:
        return self.data.shape

    @property
    def device(self) -> torch.device:
        return self.data.device

    def transpose(self) -> "Fp8Blocks":
        """The transposed matrices (kind "tile"): the same values, copied."""
        if self.kind != "tile":
            raise ValueError('only kind "tile" can be transposed')
        d = self.data
        if use_hip(d):
            n, r, c = math.prod(d.shape[:-2]), d.shape[-2], d.shape[-1]
            d = require_ext().fp8_turn(d.view(n, r, c)).view(
                *d.shape[:-2], c, r)
        else:
            d = d.view(torch.uint8).transpose(-1, -2).contiguous().view(
                torch.float8_e4m3fn)
        return Fp8Blocks(d, self.scale.transpose(-1, -2).contiguous(), "tile")

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the blocks stand for."""
        s = self.scale.transpose(-1, -2)
        s = s.repeat_interleave(BLOCK, -1)[..., :self.shape[-1]]
        if self.kind == "tile":
            s = s.repeat_interleave(BLOCK, -2)[..., :self.shape[-2], :]
        return (self.data.float() * s).to(dtype)


def _cpu_quantize(x: torch.Tensor, kind: str) -> Fp8Blocks:
    r, c = x.shape[-2:]
    h = 1 if kind == "row" else BLOCK
    v = torch.nn.functional.pad(x.float(), (0, -c % BLOCK, 0, -r % h))
    v = v.reshape(*x.shape[:-2], v.shape[-2] // h, h, v.shape[-1] // BLOCK,
                  BLOCK)
    top = v.abs().amax((-3, -1), keepdim=True) if v.numel() else \
        v.new_zeros(*v.shape[:-3], 1, v.shape[-2], 1)
    top = torch.maximum(top, torch.full_like(top, _TOP_MIN))
    most = torch.full_like(top, _MAX)  # true divisions on every device
    q = (v * (most / top)).to(torch.float8_e4m3fn)
    q = q.reshape(*q.shape[:-4], q.shape[-4] * h,
                  q.shape[-2] * BLOCK).view(torch.uint8)[..., :r, :c]
    s = (top / most).squeeze(-1).squeeze(-2).transpose(-1, -2)
    return Fp8Blocks(q.contiguous().view(torch.float8_e4m3fn),
                     s.contiguous(), kind)


def _check_values(x: torch.Tensor, name: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got "
                        f"{x.dtype}")
    if x.layout != torch.strided:
        raise TypeError(f"{name} must be dense")


def quantize_fp8(x: torch.Tensor, kind: str = "row") -> Fp8Blocks:
    """x [rows, cols], or a stack [n, rows, cols], in e4m3 with a scale for
    each 128 values along a row (kind "row": left operands) or for each
    128 x 128 tile (kind "tile": right operands). Not differentiable."""
    _check_values(x, "x")
    if kind not in ("row", "tile"):
        raise ValueError(f'kind must be "row" or "tile", got {kind!r}')
    if x.dim() not in (2, 3):
        raise ValueError(f"x must be [rows, cols] or [n, rows, cols], got "
                         f"{tuple(x.shape)}")
    x = x.detach()
    if not use_hip(x):
        return _cpu_quantize(x, kind)
    e = require_ext()
    if kind == "tile":
        q, s, _, _ = e.fp8_quantize_tile(x if x.dim() == 3 else x[None],
                                         False)
        return Fp8Blocks._made(q, s, kind) if x.dim() == 3 else \
            Fp8Blocks._made(q[0], s[0], kind)
    if x.dim() == 2:
        q, s = e.fp8_quantize_row(x)
        return Fp8Blocks._made(q, s, kind)
    n, r, c = x.shape
    q, s = e.fp8_quantize_row(x.reshape(n * r, c))
    s = s.reshape(s.shape[0], n, r).transpose(0, 1).contiguous()
    return Fp8Blocks(q.view(n, r, c), s, kind)


def _product(a, bt: Fp8Blocks, offsets, out_dtype):
    """a @ bt[group]^T; a: blocks, or values to be quantized; bt [groups, n,
    k] or [n, k]."""
    blocks = isinstance(a, Fp8Blocks)
    if not use_hip(bt.data):
        q = a if blocks else _cpu_quantize(a, "row")
        w = bt.dequantize()
        return rows_product(q.dequantize(),
                            (w if w.dim() == 3 else w[None]).transpose(1, 2),
                            offsets, out_dtype)
    return require_ext().grouped_rows_fp8(
        a.data if blocks else a,
        a.scale if blocks else None, bt.data, bt.scale, offsets, out_dtype,
        None, False)


class _CpuFp8Matmul(torch.autograd.Function):
    """Fp8Matmul of csrc/ext_grouped.cpp for CPU tensors."""

    @staticmethod
    def forward(ctx, a, w, frozen, offsets, out_dtype):
        q = _cpu_quantize(w, "tile") if frozen is None else frozen
        ctx.q, ctx.frozen = q, frozen is not None
        ctx.save_for_backward(a, w, offsets)
        return _product(a, q, offsets, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        a, w, offsets = ctx.saved_tensors
        da = dw = None
        if ctx.needs_input_grad[0]:
            da = _product(grad, ctx.q.transpose(), offsets, a.dtype)
        if not ctx.frozen and ctx.needs_input_grad[1]:
            # in the operands' own type: the sum runs over rows, along which
            # neither has its scales
            groups = 1 if w.dim() == 2 else w.shape[0]
            ty = product_type(grad, a.dtype)
            dw = weights_product(grad.to(ty), a.to(ty), offsets, groups,
                                 w.dtype).reshape(w.shape)
        return da, dw, None, None, None


def _differentiable(a, w, frozen, offsets, out_dtype):
    if not use_hip(a):
        return _CpuFp8Matmul.apply(a, w, frozen, offsets, out_dtype)
    q, s = (None, None) if frozen is None else (frozen.data, frozen.scale)
    return require_ext().fp8_matmul(a, w, q, s, offsets, out_dtype)


def fp8_matmul(a: Union[torch.Tensor, Fp8Blocks],
               bt: Union[torch.Tensor, Fp8Blocks],
               offsets: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """a @ bt^T in 8 bits. The sums are float32 ones, but for what a GPU's
    matrix unit cuts off the products of 8 neighbours (above).

    a [rows, k]: a tensor, quantized here by rows, or blocks of kind "row".
    bt [n, k], or [groups, n, k] with offsets (see grouped_matmul): a tensor,
    quantized here by tiles, or blocks of kind "tile" that a program keeps.
    The result has a's type (bfloat16 for blocks) or out_dtype; rows of no
    group are zeros.

    Differentiable in the operands given as tensors: the gradient of a is an
    8-bit product too (the result's gradient quantized by rows, bt by the
    same tiles), that of bt a product in a's type."""
    if isinstance(a, Fp8Blocks):
        if a.kind != "row":
            raise ValueError('blocks of a must be of kind "row"')
    else:
        _check_values(a, "a")
    if isinstance(bt, Fp8Blocks):
        if bt.kind != "tile":
            raise ValueError('blocks of bt must be of kind "tile"')
    else:
        _check_values(bt, "bt")
    if len(a.shape) != 2:
        raise ValueError(f"a must be [rows, k], got {tuple(a.shape)}")
    if len(bt.shape) != (2 if offsets is None else 3):
        raise ValueError(f"bt must be [n, k], or [groups, n, k] with "
                         f"offsets, got {tuple(bt.shape)}")
    if a.shape[-1] != bt.shape[-1]:
        raise ValueError(f"a has {a.shape[-1]} columns, bt {bt.shape[-1]}")
    if a.device != bt.device:
        raise ValueError(f"a is on {a.device}, bt on {bt.device}")
    if offsets is not None:
        check_offsets(offsets, bt.shape[0], a.shape[0], a.device)
    out_dtype = check_out_dtype(
        out_dtype, torch.bfloat16 if isinstance(a, Fp8Blocks) else a.dtype)
    refuse_tangents(a, bt)
    if isinstance(a, Fp8Blocks):
        if isinstance(bt, torch.Tensor):
            if bt.requires_grad and torch.is_grad_enabled():
                raise ValueError("the gradient of bt needs a as a tensor")
            bt = quantize_fp8(bt, "tile")
        return _product(a, bt, offsets, out_dtype)
    if isinstance(bt, torch.Tensor):
        if bt.dtype != a.dtype:
            raise TypeError(f"a is {a.dtype}, bt {bt.dtype}")
        if needs_grad(a, bt):
            check_capture(a, bt)
            return _differentiable(a, bt, None, offsets, out_dtype)
        bt = quantize_fp8(bt, "tile")
    elif needs_grad(a):
        check_capture(a)
        return _differentiable(a, None, bt, offsets, out_dtype)
    return _product(a, bt, offsets, out_dtype)
