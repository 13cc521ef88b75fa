"""CPU: what a pre-norm block takes from its modules, without a kernel."""

from __future__ import annotations

import copy

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


class OnePlusWeight(nn.Module):
    """x / rms(x) * (1 + weight): the gain is stored as its distance from one."""

    def __init__(self, D, eps=1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.zeros(D))
        self.eps = eps

    def forward(self, x):
        n = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + self.eps)
        return (n * (1.0 + self.weight.float())).type_as(x)


class EpsOutside(nn.Module):
    def __init__(self, D, eps=1e-5):
        super().__init__()
        self.weight, self.eps = nn.Parameter(torch.ones(D)), eps

    def forward(self, x):
        return x / (x.square().mean(-1, keepdim=True).sqrt() + self.eps) * self.weight


class MeanSubtracting(nn.Module):
    def __init__(self, D, eps=1e-6):
        super().__init__()
        self.weight, self.eps = nn.Parameter(torch.ones(D)), eps

    def forward(self, x):
        x = x - x.mean(-1, keepdim=True)
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * self.weight


class InFloat(nn.Module):
    """The usual form: statistics in fp32, the gain in the parameter's type; variance_epsilon."""

    def __init__(self, D, dtype=torch.float32):
        super().__init__()
        self.weight = nn.Parameter(1 + 0.1 * torch.randn(D, dtype=dtype))
        self.variance_epsilon = 1e-5

    def forward(self, x):
        f = x.to(torch.float32)
        f = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + self.variance_epsilon)
        return self.weight * f.to(x.dtype)


@pytest.mark.parametrize("norm", [
    OnePlusWeight(16), EpsOutside(16), MeanSubtracting(16), nn.GroupNorm(1, 16, affine=False), nn.GroupNorm(4, 16, affine=False),
    nn.BatchNorm1d(16, affine=False), nn.BatchNorm1d(16, affine=False).eval(), nn.RMSNorm(8, elementwise_affine=False),
    nn.InstanceNorm1d(16), nn.LayerNorm(16, elementwise_affine=False), nn.Identity()])
def test_norms_refused(norm):
    with pytest.raises(AssertionError, match="norm must"):
        block(norm)


@pytest.mark.parametrize("precision", ["input", "e4m3"])
def test_norms_taken(precision):
    torch.manual_seed(1)
    for norm in (nn.RMSNorm(16), nn.RMSNorm(16, eps=1e-5), nn.RMSNorm(16, eps=0.0), nn.RMSNorm((16,), elementwise_affine=False),
                 nn.RMSNorm(16, dtype=torch.bfloat16), InFloat(16), InFloat(16, torch.float16)):
        with torch.no_grad():
            if getattr(norm, "weight", None) is not None:
                norm.weight.copy_(torch.randn(16))
        keep = {k: v.clone() for k, v in norm.state_dict().items()}
        m = block(norm, precision=precision)
        assert m.norm is norm and all(torch.equal(v, keep[k]) and v.dtype == keep[k].dtype for k, v in norm.state_dict().items())
    meta = block(nn.RMSNorm(16, device="meta"))      # tried when it has values
    assert not meta._norm_known and block(nn.RMSNorm(16))._norm_known


@pytest.mark.parametrize("gain", [0.0, -1.0])
def test_the_gain_does_not_hide_the_form(gain):
    """A norm is told by its form whatever its weight is when the block is built."""
    for norm, ok in ((nn.RMSNorm(16, eps=0.5), True), (OnePlusWeight(16), False), (MeanSubtracting(16), False)):
        nn.init.constant_(norm.weight, gain)
        if ok:
            assert block(norm)._norm_known
        else:
            with pytest.raises(AssertionError, match="norm must"):
                block(norm)


def test_replicas_and_copies_are_known():
    m = block(nn.RMSNorm(16))
    replica = m._replicate_for_data_parallel()       # what nn.DataParallel makes, with norms of its own
    replica._modules["norm"] = nn.RMSNorm(16)
    assert replica._norm_known and copy.deepcopy(m)._norm_known
    m.norm = nn.RMSNorm(16)
    assert not m._norm_known
