"""CPU: what a pre-norm block takes from its modules, without a kernel."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from ghostweight_triton_b200 import GhostLinear
from ghostweight_triton_b200.fuse import GhostPreNormMLP


def block(norm, D=16, F=32, **kw):
    return GhostPreNormMLP(norm, GhostLinear(D, F), GhostLinear(F, D), "gelu", **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_default_eps_is_the_norms(dtype):
    """nn.RMSNorm without eps: rows of values next to sqrt(eps), where eps decides the result.

    The formula in 64 bits with the block's eps against the norm itself: each of its
    (at most three) roundings to dtype is off by half a step of the value."""
    torch.manual_seed(0)
    norm = nn.RMSNorm(16, dtype=dtype)
    x = (1e-3 * torch.randn(8, 16)).to(dtype)
    d = x.double()
    want = d / torch.sqrt((d * d).mean(-1, keepdim=True) + block(norm)._eps())
    err = (norm(x).double() - want).abs()
    assert bool((err <= 3 * torch.finfo(dtype).eps / 2 * want.abs() + 1e-6).all())
    assert block(nn.RMSNorm(16, eps=1e-3))._eps() == 1e-3
