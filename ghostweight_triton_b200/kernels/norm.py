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
from ghostweight_triton_b200.kernels._args import out_matrix, refuse_grad, rows
from ghostweight_triton_b200.kernels.gather import PACK_ALIGN, _round_up

# e4m3 rows keep a stride of a multiple of 128 bytes: one k-block of the
# e4m3 product, so every TMA row starts 128-byte aligned. Padding is zero.
PACK_ALIGN_Q8 = 128


def _alive(alive_indices: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor | None:
    if alive_indices is None:
        return None
    assert alive_indices.ndim == 1, f"alive_indices must be one list, got shape {tuple(alive_indices.shape)}"
    if alive_indices.dtype is not torch.int64 or alive_indices.device != x.device:
        assert not alive_indices.is_floating_point() and alive_indices.dtype is not torch.bool, \
            f"alive_indices must be integers, got {alive_indices.dtype}"
        alive_indices = alive_indices.to(device=x.device, dtype=torch.int64)
    return alive_indices.contiguous()


def _norm(x, weight, eps, residual, alive_indices, residual_out, q8):
    assert x.ndim >= 1 and x.is_cuda, "rms_norm runs on CUDA (sm_100) only"
    _native.dtype_code(x.dtype)
    refuse_grad(x=x, residual=residual)
    cols = x.shape[-1]
    assert cols > 0, "the norm of a row without columns is undefined"
    assert eps >= 0.0, f"eps must not be negative, got {eps}"
    lead = x.shape[:-1]
    x_2d = rows(x, cols)
    if weight is not None:
        assert weight.shape == (cols,), f"weight must have shape ({cols},), got {tuple(weight.shape)}"
        assert weight.device == x.device, "weight must be on x's device"
        weight = weight.detach()
        if weight.dtype is not x.dtype:
            weight = weight.to(x.dtype)
        weight = weight.contiguous()
    total = r_2d = None
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype is x.dtype and residual.device == x.device, (
            "residual must have x's shape, dtype and device")
        r_2d = rows(residual, cols)
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        total = out_matrix("residual_out", residual_out, x, x_2d, r_2d)
    else:
        assert residual_out is None, "residual_out needs a residual"
    idx = _alive(alive_indices, x)
    n = cols if idx is None else idx.numel()
    M = x_2d.shape[0]
    if q8:
        buf = torch.empty((M, _round_up(n, PACK_ALIGN_Q8)), dtype=torch.float8_e4m3fn, device=x.device)
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        buf = torch.empty((M, n if idx is None else _round_up(n, PACK_ALIGN)), dtype=x.dtype, device=x.device)
        scale = None
    if M:
        _native.rms_norm(x_2d, r_2d, total, weight, eps, idx, n, buf, scale)
    y = buf if buf.shape[1] == n else buf[:, :n]
    if x.ndim != 2:
        y = y.view(*lead, n)
        scale = scale.view(lead) if q8 else None
    out = (y, scale) if q8 else (y,)
    return out if residual is None else (*out, residual_out)


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
    assert x.ndim >= 1 and x.is_cuda, "quantize_rows runs on CUDA (sm_100) only"
    _native.dtype_code(x.dtype)
    refuse_grad(x=x)
    cols = x.shape[-1]
    lead = x.shape[:-1]
    idx = _alive(alive_indices, x)
    n = cols if idx is None else idx.numel()
    M = math.prod(lead)
    buf = torch.empty((M, _round_up(n, PACK_ALIGN_Q8)), dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    if M:
        _native.quantize_rows(rows(x, cols) if cols else x.reshape(M, 0), idx, n, buf, scale)
    q = buf if buf.shape[1] == n else buf[:, :n]
    if x.ndim != 2:
        q, scale = q.view(*lead, n), scale.view(lead)
    return q, scale


def pack_weight_q8(weight: torch.Tensor, alive_indices: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Pack the alive input columns of a linear weight in e4m3 for ``packed_linear_q8``.

    ``weight`` is [N, K] (nn.Linear orientation, any strides), rounded from its
    own dtype. Returns (W' [N, K_alive] float8_e4m3fn, a view of rows padded to
    a multiple of 128 bytes with zeros, and the scales [N]).
    """
    assert weight.ndim == 2 and weight.is_cuda
    return quantize_rows(weight.detach(), alive_indices)
