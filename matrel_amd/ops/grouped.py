"""Products of ragged row groups, with gradients.

`grouped_matmul` multiplies the rows of each group by the group's own matrix
in ONE launch, where `gemm_bt_batch` (csrc/ext.cpp) takes a list of
tile-aligned block products and launches one kernel for each. Groups are
given as CSR-style offsets that stay on the device: group g is the rows
[offsets[g], offsets[g + 1]). Groups may be empty or hold one row; no size
has to be a multiple of anything.

GPU tensors run the HIP kernels (csrc/grouped_core.h), CPU tensors plain
torch. Sums are float32 and are rounded once to the result's type.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .backend import require_ext, use_hip

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def check_offsets(offsets: torch.Tensor, groups: int, rows: int,
                  device: torch.device) -> None:
    """Offsets: int32/int64 [groups + 1] beside the operands. The values are
    looked at on the CPU only; on a GPU the kernels hold them to [0, rows]."""
    if not isinstance(offsets, torch.Tensor):
        raise TypeError("offsets must be a tensor")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got "
                        f"{offsets.dtype}")
    if offsets.dim() != 1 or offsets.numel() != groups + 1:
        raise ValueError(f"offsets must hold groups + 1 = {groups + 1} "
                         f"values, got shape {tuple(offsets.shape)}")
    if offsets.device != device:
        raise ValueError(f"offsets are on {offsets.device}, the operands "
                         f"on {device}")
    if not offsets.is_cuda:
        v = offsets.tolist()
        if any(x > y for x, y in zip(v, v[1:])) or v[0] < 0 or v[-1] > rows:
            raise ValueError(f"offsets must rise within [0, {rows}]")


def check_out_dtype(out_dtype: Optional[torch.dtype],
                    default: torch.dtype) -> torch.dtype:
    if out_dtype is None:
        return default
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be bfloat16, float16 or float32, "
                        f"got {out_dtype}")
    return out_dtype


def needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def refuse_tangents(*operands) -> None:
    """Forward-mode tangents, which requires_grad does not show: the kernels
    carry none, and a result without one would count as constant."""
    if forward_ad._current_level < 0:
        return
    for t in operands:
        if isinstance(t, torch.Tensor) \
                and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("grouped and 8-bit products have no "
                                      "forward-mode derivative")


def check_capture(*operands) -> None:
    """Autograd runs a node of a backward pass on the stream of its forward
    pass, and a leaf's accumulation on the stream of the graph that met it
    first. A backward pass captured while an operand or a leaf behind it (a
    view's, say) has nodes outside would make the capture wait for that
    stream, which ends the process: it is refused here, before anything is
    recorded."""
    if not operands[0].is_cuda or not require_ext().capturing(operands[0]):
        return
    for t in operands:
        if require_ext().held_by_other_stream(t):
            raise RuntimeError(
                "an autograd graph built outside of this capture still "
                "holds an operand: free it (its loss and outputs) before "
                "capturing, or capture grouped_matmul_grads instead")


def _cpu_rows(a, b, offsets, out_dtype):
    out = a.new_zeros(a.shape[0], b.shape[2], dtype=torch.float32)
    v = [0, a.shape[0]] if offsets is None else offsets.tolist()
    for g, (lo, hi) in enumerate(zip(v, v[1:])):
        out[lo:hi] = a[lo:hi].float() @ b[g].float()
    return out.to(out_dtype)


def _cpu_weights(a, b, offsets, groups, out_dtype):
    out = a.new_zeros(groups, a.shape[1], b.shape[1], dtype=torch.float32)
    v = [0, a.shape[0]] if offsets is None else offsets.tolist()
    for g, (lo, hi) in enumerate(zip(v, v[1:])):
        out[g] = a[lo:hi].float().t() @ b[lo:hi].float()
    return out.to(out_dtype)


def rows_product(a, b, offsets, out_dtype):
    """c[t] = a[t] @ b[group of t]; offsets None: one group of all rows."""
    if not use_hip(a):
        return _cpu_rows(a, b, offsets, out_dtype)
    return require_ext().grouped_rows(a, b, offsets, out_dtype)


def weights_product(a, b, offsets, groups, out_dtype):
    """c[g] = a_g^T @ b_g over the rows of each group."""
    if not use_hip(a):
        return _cpu_weights(a, b, offsets, groups, out_dtype)
    return require_ext().grouped_weights(a, b, offsets, groups, out_dtype)


def _check(a, b, offsets):
    if not (isinstance(a, torch.Tensor) and isinstance(b, torch.Tensor)):
        raise TypeError("a and b must be tensors")
    if a.dim() != 2 or b.dim() != 3:
        raise ValueError(f"a must be [rows, k] and b [groups, k, n], got "
                         f"{tuple(a.shape)} and {tuple(b.shape)}")
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"a has {a.shape[1]} columns, b's matrices "
                         f"{b.shape[1]} rows")
    if a.dtype not in _TYPES or b.dtype != a.dtype:
        raise TypeError(f"a and b must both be bfloat16, float16 or "
                        f"float32, got {a.dtype} and {b.dtype}")
    if a.layout != torch.strided or b.layout != torch.strided:
        raise TypeError("a and b must be dense")
    if a.device != b.device:
        raise ValueError(f"a is on {a.device}, b on {b.device}")
    check_offsets(offsets, b.shape[0], a.shape[0], a.device)


def grouped_matmul_grads(grad: torch.Tensor, a: torch.Tensor,
                         b: torch.Tensor, offsets: torch.Tensor
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(d_a, d_b) of grouped_matmul(a, b, offsets) for the gradient `grad` of
    its result. Builds no autograd graph, so it can be captured at any time."""
    _check(a, b, offsets)
    if tuple(grad.shape) != (a.shape[0], b.shape[2]) \
            or grad.device != a.device:
        raise ValueError(f"grad must be {(a.shape[0], b.shape[2])} on "
                         f"{a.device}, got {tuple(grad.shape)} on "
                         f"{grad.device}")
    if use_hip(a):
        refuse_tangents(grad, a, b)
    with torch.no_grad():
        grad = grad.to(product_type(grad, a.dtype))
        return (_grad_a(grad, b, offsets), _grad_b(grad, a, b, offsets))


def product_type(grad: torch.Tensor, dtype: torch.dtype) -> torch.dtype:
    """The one type of a gradient's product: the operands' dtype, to which a
    wider result's gradient is rounded. It can lie outside of float16's range
    (the products of 1e5 and 1e-4 are not infinite): all is multiplied in
    float32 there."""
    if dtype == torch.float16 and grad.dtype != dtype:
        return torch.float32
    return dtype


def _grad_a(grad, b, offsets):
    return rows_product(grad, b.to(grad.dtype).transpose(1, 2), offsets,
                        b.dtype)


def _grad_b(grad, a, b, offsets):
    a = a.to(grad.dtype)
    # in the memory order of b, so that an optimizer walks both alike
    if b.stride(1) == 1 and b.shape[1] > 1:
        return weights_product(grad, a, offsets, b.shape[0],
                               b.dtype).transpose(1, 2)
    return weights_product(a, grad, offsets, b.shape[0], b.dtype)


class _CpuGroupedMatmul(torch.autograd.Function):
    """GroupedMatmul of csrc/ext_grouped.cpp for CPU tensors."""

    @staticmethod
    def forward(ctx, a, b, offsets, out_dtype):
        ctx.save_for_backward(a, b, offsets)
        return rows_product(a, b, offsets, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        a, b, offsets = ctx.saved_tensors
        grad = grad.to(product_type(grad, a.dtype))
        da = _grad_a(grad, b, offsets) if ctx.needs_input_grad[0] else None
        db = _grad_b(grad, a, b, offsets) if ctx.needs_input_grad[1] else None
        return da, db, None, None


def grouped_matmul(a: torch.Tensor, b: torch.Tensor, offsets: torch.Tensor,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """c[t] = a[t] @ b[g] for the rows t of group g = [offsets[g],
    offsets[g + 1]).

    a [rows, k]; b [groups, k, n], contiguous along k or n (pass stored
    [groups, n, k] weights as w.transpose(1, 2): nothing is copied); offsets
    int32/int64 [groups + 1], rising within [0, rows], on the operands'
    device. bfloat16, float16 or float32 operands of one type; the result
    has that type, or out_dtype. Rows of no group are zeros. Differentiable
    in a and b."""
    _check(a, b, offsets)
    out_dtype = check_out_dtype(out_dtype, a.dtype)
    if use_hip(a):
        refuse_tangents(a, b)
    if not needs_grad(a, b):
        return rows_product(a, b, offsets, out_dtype)
    if not use_hip(a):
        return _CpuGroupedMatmul.apply(a, b, offsets, out_dtype)
    check_capture(a, b)
    return require_ext().grouped_matmul(a, b, offsets, out_dtype)
