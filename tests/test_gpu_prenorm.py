"""GPU: a pre-norm MLP block as one chain of the row operators and products.

    s = x + r;  y = s + proj(act(fc(norm(s))))

The 16-bit chain is checked against the formula in 64 bits. Each of its
intermediate results is rounded to the input's type: the normed row and the
hidden row by half a step (u = finfo.eps / 2) of each value, and y once. A
product carries a relative perturbation d of its operand's values into at most
d sum |a| |w|, the GELU multiplies by at most 1.13; the fp32 sums in between
are off by (K + 16) 2^-23 of the same sums, far below u. So with N = |n| |W1|^T + |b1|
and H = |h| |W2|^T + |b2| (in 64 bits, with the exact n and h):

    dh <= 1.13 (1.1 u N) + u |h| + 1e-5 N;   |y - exact| <= dh |W2|^T + 1.1 u H 2^-4 + 2 u |y|

with 1.1 for the second order and the fp32 sums. s is rounded once more before it
is added (u |s|), which 2 u |y| + u |s| covers.

The e4m3 chain is checked against the same operators called one by one (bit for
bit), which have their own tests, and against the 16-bit chain in norm: each of
its four roundings to e4m3 is off by at most 2^-4 of a value or 2^-10 of the
row's scale, so independent errors leave a relative error of the branch
(without s) below 4 x 2^-4.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn as nn

from ghostweight_triton_b200 import GhostLinear
from ghostweight_triton_b200.fuse import GhostPreNormMLP
from ghostweight_triton_b200.kernels.matmul import packed_linear_q8
from ghostweight_triton_b200.kernels.norm import pack_weight_q8, quantize_rows, rms_norm_q8

pytestmark = pytest.mark.gpu


def block(D, F, dtype, seed, bias=True, activation="gelu_tanh", dropout=None, precision="input", eps=1e-5, dead=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    norm = nn.RMSNorm(D, eps=eps, device="cuda", dtype=dtype)
    fc = GhostLinear(D, F, bias=bias, threshold=0.0, device="cuda", dtype=dtype)
    proj = GhostLinear(F, D, bias=bias, threshold=0.0, device="cuda", dtype=dtype)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * torch.randn(D, generator=g, device="cuda"))
        for m in (fc, proj):
            m.weight.copy_(torch.randn(m.weight.shape, generator=g, device="cuda") / math.sqrt(m.in_features))
            if bias:
                m.bias.copy_(0.1 * torch.randn(m.out_features, generator=g, device="cuda"))
            m.weight[:, torch.randperm(m.in_features, generator=g, device="cuda")[: int(m.in_features * dead)]] = 0
            m.freeze_weight_mask()
    return GhostPreNormMLP(norm, fc, proj, activation, dropout, precision).eval()


def inputs(M, D, dtype, seed, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed + 100)
    x = torch.randn(M, D, generator=g, device="cuda").to(dtype)
    return x, torch.randn(M, D, generator=g, device="cuda").to(dtype) if residual else None


def exact(m, x, r, eps):
    s = x.double() if r is None else x.double() + r.double()
    n = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * m.norm.weight.double()
    W1, W2 = m.fc.weight.double(), m.proj.weight.double()
    b1 = m.fc.bias.double() if m.fc.bias is not None else torch.zeros(W1.shape[0], device="cuda").double()
    b2 = m.proj.bias.double() if m.proj.bias is not None else torch.zeros(W2.shape[0], device="cuda").double()
    v = n @ W1.t() + b1
    if m.activation == "gelu_tanh":
        h = 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    else:
        h = 0.5 * v * (1 + torch.erf(v / math.sqrt(2.0)))
    N = n.abs() @ W1.abs().t() + b1.abs()
    H = h.abs() @ W2.abs().t() + b2.abs()
    return s, s + h @ W2.t() + b2, h, N, H, W2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,D,F", [(1, 256, 512), (3, 100, 300), (17, 768, 1000), (300, 512, 2048), (2100, 1024, 2304)])
def test_block_matches_the_formula(M, D, F, dtype):
    for activation, bias, residual in (("gelu_tanh", True, True), ("gelu", False, False)):
        m = block(D, F, dtype, M + D, bias, activation)
        x, r = inputs(M, D, dtype, M, residual)
        keep = x.clone()
        with torch.no_grad():
            y = m(x, residual=r)
        s, want, h, N, H, W2 = exact(m, x, r, 1e-5)
        u = torch.finfo(dtype).eps / 2
        dh = 1.13 * 1.1 * u * N + u * h.abs() + 1e-5 * N
        bound = dh @ W2.abs().t() + 1.1 * u * H / 16 + 2 * u * want.abs() + u * s.abs() + 1e-6
        err = (y.double() - want).abs()
        assert y.dtype is dtype and bool((err <= bound).all()), f"off by {(err / bound).max().item():.3g} of the bound"
        assert torch.equal(x, keep)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 30, 500, 2100])
def test_e4m3_block_is_its_operators(M, dtype):
    D, F = 512, 1024
    m = block(D, F, dtype, M, precision="e4m3")
    plain = block(D, F, dtype, M)
    x, r = inputs(M, D, dtype, M)
    with torch.no_grad():
        y = m(x, residual=r)
        a1, a2 = m.fc._frozen_indices, m.proj._frozen_indices
        q, sc, s = rms_norm_q8(x, m.norm.weight, 1e-5, residual=r, alive_indices=a1)
        w1, s1 = pack_weight_q8(m.fc.weight[a2], a1)
        pad = -a2.numel() % 64
        h = packed_linear_q8(q, sc, w1, s1, bias=m.fc.bias[a2], activation="gelu_tanh", dtype=dtype)
        h = torch.cat([h, h.new_zeros(M, pad)], 1)
        w2, s2 = pack_weight_q8(m.proj.weight, a2)
        hq, hs = quantize_rows(h)
        want = packed_linear_q8(hq[:, : a2.numel()], hs, w2, s2, bias=m.proj.bias, residual=s)
        assert torch.equal(y, want)
        ref = plain(x, residual=r)
    branch = ref.double() - s.double()
    assert ((y.double() - s.double() - branch).norm() / branch.norm()).item() < 4 / 16


def test_weight_updates_and_dropout():
    m = block(256, 512, torch.bfloat16, 5, precision="e4m3")
    x, r = inputs(20, 256, torch.bfloat16, 5)
    with torch.no_grad():
        first = m(x, residual=r)
        m.proj.weight.mul_(2.0)                      # seen by itself
        second = m(x, residual=r)
        assert not torch.equal(first, second)
        m.proj.weight.data.mul_(0.5)                 # not seen: told
        m.refresh_packed()
        assert torch.equal(m(x, residual=r), first)
        d = block(256, 512, torch.bfloat16, 5, dropout=nn.Dropout(1.0))
        d.train()
        assert torch.equal(d(x, residual=r), (x.float() + r.float()).to(torch.bfloat16))
        lead = m(x.view(2, 10, 256), residual=r.view(2, 10, 256))
        assert lead.shape == (2, 10, 256) and torch.equal(lead.view(20, 256), first)
        assert m(x[:0]).shape == (0, 256)


def test_captured():
    for precision in ("input", "e4m3"):
        m = block(512, 1024, torch.float16, 7, precision=precision)
        x, r = inputs(40, 512, torch.float16, 7)
        with torch.no_grad():
            m(x, residual=r)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = m(x, residual=r)
            x2, r2 = inputs(40, 512, torch.float16, 8)
            x.copy_(x2)
            r.copy_(r2)
            graph.replay()
            assert torch.equal(y, m(x2, residual=r2))


def test_refusals():
    good = block(128, 256, torch.float16, 9)
    x, r = inputs(4, 128, torch.float16, 9)
    with pytest.raises(ValueError):
        GhostPreNormMLP(good.norm, good.fc, good.proj, "gelu", precision="int8")
    for norm in (nn.LayerNorm(128), nn.RMSNorm(64)):
        with pytest.raises(AssertionError):
            GhostPreNormMLP(norm, good.fc, good.proj, "gelu")
    with pytest.raises(AssertionError):
        GhostPreNormMLP(good.norm, good.fc, GhostLinear(256, 64, device="cuda", dtype=torch.float16), "gelu")
    with torch.no_grad():
        with pytest.raises(AssertionError):
            good(x.float())
        with pytest.raises(AssertionError):
            good(x, residual=r[:2])
    with pytest.raises(RuntimeError, match="no backward"):
        good(x.requires_grad_())
    good.fc.unfreeze_mask()
    with torch.no_grad(), pytest.raises(RuntimeError, match="frozen"):
        good(x)


@pytest.mark.parametrize("precision", ["input", "e4m3"])
def test_two_streams_at_once(precision):
    """Blocks of one module running on two streams together give what each gives alone."""
    m = block(512, 1024, torch.bfloat16, 31, precision=precision)
    for M in (1, 40, 700):
        data = [inputs(M, 512, torch.bfloat16, seed) for seed in (1, 2)]
        with torch.no_grad():
            want = [m(x, r) for x, r in data]
            torch.cuda.synchronize()
            streams = [torch.cuda.Stream(), torch.cuda.Stream()]
            got = [[], []]
            for _ in range(20):
                for i, stream in enumerate(streams):
                    with torch.cuda.stream(stream):
                        got[i].append(m(*data[i]))
            torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(y, want[i]) for y in got[i])
