"""CPU: the outputs and operands that the products refuse (host checks, no kernel)."""

from __future__ import annotations

import pytest
import torch

from ghostweight_triton_b200.kernels.matmul import _product_out

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
