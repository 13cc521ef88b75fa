"""Argument checks shared by the operator wrappers (host side, no kernel)."""

from __future__ import annotations

import torch

from ghostweight_triton_b200 import _native


def refuse_grad(**tensors: torch.Tensor | None) -> None:
    """Raise if a tensor would need a gradient that the operator cannot give."""
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} requires a gradient, and this operator has no backward pass: "
                                   "call it under torch.no_grad() or on detached tensors")


def refuse_grad_out(what: str, out: torch.Tensor) -> None:
    """Raise if results written into `out` would be lost to its gradient."""
    if out.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} requires a gradient, and this operator has no backward pass: "
                           "call it under torch.no_grad() or on detached tensors")


# Called for every given tensor that a kernel has written: the autograd engine and the
# caches of packed weights see the write by the tensor's version.
written = torch.autograd.graph.increment_version


class Kept:
    """Tensors that one call makes and later calls use again, on any stream: another stream
    than theirs waits until they are made, and the allocator for that stream's work before it
    hands their memory out again. A capture takes them as they are (it starts when the device
    is idle).
    """

    def __init__(self, tensors):
        self.tensors = list(tensors)
        self.device = self.tensors[0].device
        self.streams = {_native._stream(self.device)}      # that the tensors are ordered on
        self.made = torch.cuda.current_stream(self.device).record_event()

    def on_this_stream(self) -> None:
        raw = _native._stream(self.device)
        if raw not in self.streams and not _native._capturing():
            stream = torch.cuda.current_stream(self.device)
            stream.wait_event(self.made)
            for t in self.tensors:
                t.record_stream(stream)
            self.streams.add(raw)


def rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t as a row-major [rows, cols] matrix (copied only when its strides are not such)."""
    t = t.reshape(-1, cols)
    if (t.stride(1) != 1 and cols > 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def leading(m: torch.Tensor) -> int:
    """Leading dimension of a row-major matrix (torch gives matrices of one row any stride)."""
    return max(m.stride(0), m.shape[1])


def _span(m: torch.Tensor) -> tuple[int, int]:
    return m.data_ptr(), m.data_ptr() + ((m.shape[0] - 1) * m.stride(0) + m.shape[1]) * m.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two row-major matrices share memory. Columns side by side in one buffer do
    not; matrices whose rows interleave at different strides are taken to."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    # At one stride, the rows of a take the bytes [0, wa) of every period and those of b
    # [d, d + wb): apart if that ends behind the first and before the next period's.
    pitches = {t.stride(0) * t.element_size() for t in (a, b) if t.shape[0] > 1}
    if len(pitches) != 1:
        return True
    pitch = pitches.pop()
    d = (b0 - a0) % pitch
    return d < a.shape[1] * a.element_size() or d + b.shape[1] * b.element_size() > pitch


def in_place_or_apart(what: str, out: torch.Tensor, *inputs: torch.Tensor | None) -> None:
    """Assert that the matrix `out` takes the very place of an input matrix or none of its
    memory (each element is read before it is written only if both have the same rows)."""
    for t in inputs:
        if t is None or (t.data_ptr() == out.data_ptr() and t.shape == out.shape
                         and (t.shape[0] <= 1 or t.stride(0) == out.stride(0))):
            continue
        assert not overlap(out, t), f"{what} overlaps an input without being the same rows"


def out_matrix(what: str, out: torch.Tensor, like: torch.Tensor, *inputs: torch.Tensor | None) -> torch.Tensor:
    """`out` as a matrix that results of `like`'s shape and type can be written to: rows that
    do not overlap one another, and in_place_or_apart with the input matrices."""
    assert out.shape == like.shape and out.dtype is like.dtype and out.device == like.device, (
        f"{what} must have shape {tuple(like.shape)}, dtype {like.dtype} and be on {like.device}")
    cols = like.shape[-1]
    m = out.view(-1, cols) if out.is_contiguous() and cols else out
    assert m.ndim == 2 and (m.stride(1) == 1 or cols <= 1) and (m.shape[0] <= 1 or m.stride(0) >= cols), (
        f"{what} must be a row-major matrix (or contiguous)")
    in_place_or_apart(what, m, *inputs)
    return m


def residual_matrix(residual: torch.Tensor, shape: tuple[int, int], like: torch.Tensor) -> torch.Tensor:
    """The residual [M, N] of a product as a row-major matrix."""
    assert residual.dtype is like.dtype and residual.get_device() == like.get_device(), (
        f"residual must be {like.dtype} on {like.device}, got {residual.dtype} on {residual.device}")
    assert residual.shape == shape, f"residual must have shape {tuple(shape)}, got {tuple(residual.shape)}"
    if torch.is_grad_enabled():
        refuse_grad(residual=residual)
    if residual.is_contiguous():
        return residual
    if (residual.stride(1) != 1 and shape[1] > 1) or (shape[0] > 1 and residual.stride(0) < shape[1]):
        residual = residual.contiguous()
    return residual
