"""CPU: the outputs and operands that the products refuse (host checks, no kernel)."""

from __future__ import annotations

import random

import pytest
import torch

from ghostweight_triton_b200.kernels import _args
from ghostweight_triton_b200.kernels.matmul import _apart_from, _operands_ok, _product_out

F16 = torch.float16


@pytest.mark.parametrize("out", [
    torch.empty(2, 16, dtype=torch.uint8),                      # smaller in every way
    torch.empty(3, 48, dtype=F16),                              # a row short
    torch.empty(4, 47, dtype=F16),                              # a column short
    torch.empty(4, 49, dtype=F16),
    torch.empty(4 * 48, dtype=F16),
    torch.empty(4, 48, dtype=torch.bfloat16),
    torch.empty(4, 48, dtype=torch.float32),
    torch.empty(4, 48, dtype=F16, device="meta"),               # another device
    torch.empty(48, 4, dtype=F16).t(),                          # columns of adjacent elements
    torch.empty(1, 48, dtype=F16).expand(4, 48),                # one row four times
    torch.empty(4 * 48, dtype=F16).as_strided((4, 48), (40, 1)),     # rows that overlap
])
@pytest.mark.parametrize("with_residual", [False, True])
def test_outputs_refused(out, with_residual):
    x = torch.empty(4, 32, dtype=F16)
    with pytest.raises(AssertionError):
        _product_out(out, torch.empty(4, 48, dtype=F16) if with_residual else None, 4, 48, x)


def test_outputs_taken():
    x = torch.empty(4, 32, dtype=F16)
    for out in (torch.empty(4, 48, dtype=F16), torch.empty(4, 60, dtype=F16)[:, 5:53], torch.empty(9, 48, dtype=F16)[::2][:4]):
        assert _product_out(out, None, 4, 48, x)[0] is out
        assert _product_out(out, torch.empty(4, 48, dtype=F16), 4, 48, x)[0] is out
    new, _ = _product_out(None, None, 4, 48, x)
    assert new.shape == (4, 48) and new.dtype is F16
    column = torch.empty(4, 3, dtype=F16)[:, 1:2]
    assert _product_out(column, None, 4, 1, x)[0] is column


def test_columns_side_by_side():
    """Output and residual in the halves of one buffer share no element."""
    x = torch.empty(6, 32, dtype=F16)
    buf = torch.empty(6, 100, dtype=F16)
    for out, residual in ((buf[:, 48:96], buf[:, :48]), (buf[:, :48], buf[:, 52:]), (buf[:, 10:58], buf[:, 58:]),
                          (buf[:1, 48:96], buf[:1, :48])):
        n = min(out.shape[1], residual.shape[1])
        out, residual = out[:, :n], residual[:, :n]
        y, r = _product_out(out, residual, len(out), n, x)
        assert y is out and r is residual
    for out, residual in ((buf[:, 47:95], buf[:, :48]), (buf[1:, :48], buf[:5, 2:50]), (buf[:5, 60:], buf[1:, 50:90])):
        with pytest.raises(AssertionError, match="overlaps"):
            _product_out(out, residual, len(out), out.shape[1], x)


def test_overlap_against_the_elements():
    """Random windows of one buffer: never called apart when an element is in both, and
    called overlapping exactly then where their rows have one stride."""
    rng = random.Random(1)
    buf = torch.empty(400, dtype=F16)

    def window():
        rows, ld = rng.randint(1, 5), rng.randint(1, 12)
        return buf.as_strided((rows, rng.randint(1, ld)), (ld, 1), rng.randint(0, 60))

    def elements(m):
        return {m.storage_offset() + r * m.stride(0) + c for r in range(m.shape[0]) for c in range(m.shape[1])}

    one_stride = 0
    for _ in range(20000):
        a, b = window(), window()
        shared = bool(elements(a) & elements(b))
        got = _args.overlap(a, b)
        assert got == _args.overlap(b, a) and (got or not shared)
        if a.shape[0] > 1 and b.shape[0] > 1 and a.stride(0) == b.stride(0):
            one_stride += 1
            assert got == shared
    assert one_stride > 500


def test_operands_leave_the_output():
    """An operand that shares memory with the output is copied at its strides, a weight refused."""
    buf = torch.arange(8 * 40, dtype=F16).view(8, 40)
    w = torch.zeros(16, 24, dtype=F16)
    for x, out in ((buf[:, :24], buf[:, :16]), (buf[:, :24], buf[:, 20:36]), (buf[1:2, :24], buf[:, :16]), (buf[1:2], buf[:, 3:19])):
        copy = _apart_from(out, x, w)
        assert copy.data_ptr() != x.data_ptr() and torch.equal(copy, x) and not _args.overlap(copy, out)
        assert copy.shape == x.shape and copy.stride() == x.stride()
    for x, out in ((buf[:, :24], buf[:, 24:]), (buf[:4, :24], buf[4:, :16]), (buf[:0], buf), (torch.zeros(8, 24), buf)):
        assert _apart_from(out, x, w) is x
    with pytest.raises(AssertionError, match="w_packed"):
        _apart_from(w[:8, :16], buf[:, :24], w)


def weights_and_biases_refused(N, K, dtype):
    """(weight, bias) pairs that a product of K columns and N features must not read."""
    w = torch.zeros(N, K, dtype=dtype)
    b = torch.zeros(N, dtype=dtype)
    return [(w[:, : K - 1], b), (w[:, : K // 2], None), (w.float() if dtype is not torch.float32 else w.half(), b),
            (torch.zeros(K, N, dtype=dtype).t(), b), (w[:1].expand(N, K), b), (w.view(-1).as_strided((N // 2, K), (K // 2, 1)), None),
            (w, b[: N - 1]), (w, torch.zeros(2 * N, dtype=dtype)[::2]), (w, b.double()), (w, b[:1].expand(N))]


def test_operands_that_end_too_early():
    for w, b in weights_and_biases_refused(16, 24, F16):
        with pytest.raises(AssertionError, match="must"):
            _operands_ok(w, 24, b, F16, -1)
    w, b = torch.zeros(16, 24, dtype=F16), torch.zeros(16, dtype=F16)
    assert _operands_ok(w, 24, b, F16, -1) == 24
    assert _operands_ok(w[:, :20], 20, None, F16, -1) == 24           # rows with a gap
    assert _operands_ok(w, 20, b, F16, -1) == 24                     # wider: the first columns
    assert _operands_ok(torch.zeros(1, 24, dtype=F16).t().contiguous().t(), 24, None, F16, -1) == 24
    assert _operands_ok(torch.zeros(16, 64, dtype=F16)[:, :0], 0, b, F16, -1) == 64
    assert _operands_ok(torch.zeros(0, 24, dtype=F16), 24, None, F16, -1) == 24
