"""Row operators in front of the sparse layers: residual + RMS norm, and e4m3 rows.

``rms_norm`` adds the residual, norms the row and writes only the columns the
next layer reads (its alive list), so the layer needs no gather: its output
goes into :func:`~ghostweight_triton_b200.kernels.matmul.packed_linear` as it
is. ``rms_norm_q8`` writes those columns as e4m3 with one scale per row, the
operand of :func:`~ghostweight_triton_b200.kernels.matmul.packed_linear_q8`;
``quantize_rows`` does the same without the norm (hidden activations, and
weights once through ``pack_weight_q8``). They are extensions: the reference
leaves the norm and the residual to torch and gathers the whole normed row
again (ghostweight_triton/kernels/gather.py:139-146).

Like the sparse forwards they have no backward pass: activations that require
gradients are refused, parameters are taken as constants.
"""

from __future__ import annotations

import math

import torch

from ghostweight_triton_b200 import _native
from ghostweight_triton_b200.kernels._args import leading, out_matrix, refuse_grad, refuse_grad_out, rows, written
from ghostweight_triton_b200.kernels.gather import PACK_ALIGN, _round_up

# e4m3 rows keep a stride of a multiple of 128 bytes: one k-block of the
# e4m3 product, so every TMA row starts 128-byte aligned. Padding is zero.
PACK_ALIGN_Q8 = 128


def _alive(alive_indices: torch.Tensor, dev: int) -> torch.Tensor:
    """The list as contiguous int64 on CUDA device `dev`."""
    assert alive_indices.dim() == 1, f"alive_indices must be one list, got shape {tuple(alive_indices.shape)}"
    if alive_indices.dtype is not torch.int64 or not alive_indices.is_cuda or alive_indices.get_device() != dev:
        assert not alive_indices.is_floating_point() and alive_indices.dtype is not torch.bool, \
            f"alive_indices must be integers, got {alive_indices.dtype}"
        alive_indices = alive_indices.to(device=torch.device("cuda", dev), dtype=torch.int64)
    return alive_indices if alive_indices.is_contiguous() else alive_indices.contiguous()


def _norm(x, weight, eps, residual, alive_indices, residual_out, q8):
    # Small calls are bound by this function, not by the kernel (4 us for one
    # row of 4096): attribute reads and integer compares, no tensor operation
    # that the operands do not need.
    assert x.is_cuda and x.dim() >= 1, "rms_norm runs on CUDA (sm_100) only"
    dtype = x.dtype
    if dtype not in _native.DTYPE_CODES:
        _native.dtype_code(dtype)                # raises
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        refuse_grad(x=x, residual=residual)
    dev = x.get_device()
    flat = x.dim() == 2
    shape = x.shape
    cols = shape[-1]
    assert cols > 0, "the norm of a row without columns is undefined"
    assert eps >= 0.0, f"eps must not be negative, got {eps}"
    if flat and x.is_contiguous():
        x_2d, M, ldx = x, shape[0], cols
    else:
        x_2d = rows(x, cols)
        M, ldx = x_2d.shape[0], leading(x_2d)
    if weight is not None:
        assert weight.dim() == 1 and weight.numel() == cols, (
            f"weight must have shape ({cols},), got {tuple(weight.shape)}")
        assert weight.is_cuda and weight.get_device() == dev, "weight must be on x's device"
        if weight.dtype is not dtype:
            weight = weight.detach().to(dtype)
        if not weight.is_contiguous():
            weight = weight.contiguous()
    total = r_2d = None
    ldr = lds = 0
    given = residual_out
    if residual is not None:
        assert (residual.shape == shape and residual.dtype is dtype and residual.is_cuda
                and residual.get_device() == dev), "residual must have x's shape, dtype and device"
        if flat and residual.is_contiguous():
            r_2d, ldr = residual, cols
        else:
            r_2d = rows(residual, cols)
            ldr = leading(r_2d)
        if residual_out is None:
            total = residual_out = x.new_empty(shape)
            lds = cols
        else:
            refuse_grad_out("residual_out", residual_out)
            total = out_matrix("residual_out", residual_out, x, x_2d, r_2d)
            lds = leading(total)
    else:
        assert residual_out is None, "residual_out needs a residual"
    idx, n, ld = None, cols, cols
    if alive_indices is not None:
        idx = _alive(alive_indices, dev)
        n = idx.numel()
        ld = (n + PACK_ALIGN - 1) // PACK_ALIGN * PACK_ALIGN
    scale = None
    if q8:
        ld = (n + PACK_ALIGN_Q8 - 1) // PACK_ALIGN_Q8 * PACK_ALIGN_Q8
        buf = torch.empty((M, ld), dtype=torch.float8_e4m3fn, device=x.device)
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        buf = x.new_empty((M, ld))
    if M:
        _native.rms_norm(x_2d, M, cols, ldx, r_2d, ldr, total, lds, weight, eps, idx, n, buf, ld, scale)
        if given is not None:
            written(given)
    y = buf if ld == n else buf.narrow(1, 0, n)
    if not flat:
        y = y.view(*shape[:-1], n)
        scale = scale.view(shape[:-1]) if q8 else None
    if residual is None:
        return (y, scale) if q8 else (y,)
    return (y, scale, residual_out) if q8 else (y, residual_out)


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    residual: torch.Tensor | None = None,
    alive_indices: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
):
    """Residual addition and root-mean-square norm, over the alive columns only.

    s = x + residual;  y[..., j] = s[..., alive[j]] * rsqrt(mean(s ** 2) + eps) * weight[alive[j]]

    Parameters
    ----------
    x             : [..., K], fp16, bf16 or fp32; rows may be strided.
    weight        : [K] or None (ones); converted to x's dtype.
    eps           : added to the mean square (taken over all K columns, in fp32).
    residual      : optional, x's shape and dtype.
    alive_indices : optional [K_alive], any integer dtype: the columns of the
                    output, in any order. An index outside [0, K) gives a zero
                    column and raises the device error word.
    residual_out  : where s goes (rounded once); x or residual itself updates
                    that tensor in place. A new tensor by default.

    Returns
    -------
    y [..., K_alive] without a residual, else (y, s). With a list, y is a view
    of rows padded to a multiple of 64 elements with zeros, which
    ``packed_linear`` takes without a copy.
    """
    out = _norm(x, weight, eps, residual, alive_indices, residual_out, q8=False)
    return out[0] if residual is None else out


def rms_norm_q8(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    residual: torch.Tensor | None = None,
    alive_indices: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
):
    """:func:`rms_norm` with the output in e4m3 and one scale per row.

    scale = max(max|y| / 448, 2^-126) over the row's outputs, q = y / scale
    rounded to e4m3 from fp32. Returns (q [..., K_alive] float8_e4m3fn, scale
    [...] float32), and s behind them when a residual is given. q is a view of
    rows padded to a multiple of 128 bytes with zeros.
    """
    return _norm(x, weight, eps, residual, alive_indices, residual_out, q8=True)


def quantize_rows(
    x: torch.Tensor,
    alive_indices: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of x [..., K] (its alive columns) in e4m3 with one scale each.

    Returns (q [..., K_alive] float8_e4m3fn, scale [...] float32) with
    q * scale ~ x[..., alive], as :func:`rms_norm_q8` rounds its output.
    Columns outside the list are not looked at.
    """
    assert x.is_cuda and x.dim() >= 1, "quantize_rows runs on CUDA (sm_100) only"
    _native.dtype_code(x.dtype)
    if torch.is_grad_enabled():
        refuse_grad(x=x)
    shape = x.shape
    flat = x.dim() == 2
    cols = shape[-1]
    idx, n = None, cols
    if alive_indices is not None:
        idx = _alive(alive_indices, x.get_device())
        n = idx.numel()
    M = shape[0] if flat else math.prod(shape[:-1])
    ld = _round_up(n, PACK_ALIGN_Q8)
    buf = torch.empty((M, ld), dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    if M:
        if not (flat and x.is_contiguous()):
            x = rows(x, cols) if cols else x.reshape(M, 0)
        _native.quantize_rows(x, idx, n, buf, scale)
    q = buf if ld == n else buf.narrow(1, 0, n)
    if not flat:
        q, scale = q.view(*shape[:-1], n), scale.view(shape[:-1])
    return q, scale


def pack_weight_q8(weight: torch.Tensor, alive_indices: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Pack the alive input columns of a linear weight in e4m3 for ``packed_linear_q8``.

    ``weight`` is [N, K] (nn.Linear orientation, any strides), rounded from its
    own dtype. Returns (W' [N, K_alive] float8_e4m3fn, a view of rows padded to
    a multiple of 128 bytes with zeros, and the scales [N]).
    """
    assert weight.ndim == 2 and weight.is_cuda
    return quantize_rows(weight.detach(), alive_indices)
