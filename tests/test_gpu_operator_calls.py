"""GPU: calls of the operators around a layer that their documentation allows and the
operators' own test files do not make, against the formulas in 64 bits (the bounds are
those files')."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from tests.test_gpu_prenorm import block, exact, inputs

pytestmark = pytest.mark.gpu


def check_block(y, m, x, r, eps):
    """The 16-bit block's bound (see test_gpu_prenorm)."""
    s, want, h, N, H, W2 = exact(m, x, r, eps)
    u = torch.finfo(x.dtype).eps / 2
    dh = 1.13 * 1.1 * u * N + u * h.abs() + 1e-5 * N
    bound = dh @ W2.abs().t() + 1.1 * u * H / 16 + 2 * u * want.abs() + u * s.abs() + 1e-6
    err = (y.double() - want).abs()
    assert bool((err <= bound).all()), f"off by {(err / bound).max().item():.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_with_the_norms_default_eps(dtype):
    """Rows of about 1e-3, where eps = 2^-23 (fp32's, in which torch norms 16-bit rows) counts."""
    m = block(128, 256, dtype, 2, eps=None)
    x, r = inputs(9, 128, dtype, 2)
    x, r = (x.float() * 1e-3).to(dtype), (r.float() * 1e-3).to(dtype)
    with torch.no_grad():
        check_block(m(x, residual=r), m, x, r, 2.0 ** -23)
        n = m.norm(x).double()
    d = x.double()
    want = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 2.0 ** -23) * m.norm.weight.double()
    assert bool(((n - want).abs() <= 3 * torch.finfo(dtype).eps / 2 * want.abs() + 1e-6).all())
