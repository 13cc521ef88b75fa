"""GPU: the residual added in the epilogue of every product, against the formula in 64 bits.

    y = act(x[:, alive] W'^T + b) + r

Tolerance: the fp32 sum of K' products takes at most K' additions (in any
order, each off by at most 2^-23 of the running sum, which is at most the sum
of the products' magnitudes S), the bias, the residual and the activation a
few more, and the result is rounded once to y's type (half a step of it):

    |err| <= finfo.eps / 2 |y| + (K' + 16) 2^-23 (S + |b|) 1.13 + 1e-5 |v| + 2^-22 (|act| + |r|)

1.13 bounds the slope of the GELU, 1e-5 |v| the fast exponential of its tanh
form (v the value before it). The smallest subnormals of the type add half of
themselves.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn as nn

from ghostweight_triton_b200 import GhostLinear, _native
from ghostweight_triton_b200.fuse import GhostMLPChain
from ghostweight_triton_b200.kernels.gather import pack_weight, pack_weight_dev
from ghostweight_triton_b200.kernels.matmul import ghost_linear, ghost_linear_dev, packed_linear

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def half(K, seed, runs=False):
    g = gen(seed)
    if runs:
        keep = torch.randperm(K // 64, generator=g, device="cuda")[: max(1, K // 128)].sort().values
        return (keep[:, None] * 64 + torch.arange(64, device="cuda")).reshape(-1)
    return torch.randperm(K, generator=g, device="cuda")[: (K + 1) // 2].sort().values


def act64(v, activation):
    if activation == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2.0)))
    if activation == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def check(y, a, w, bias, activation, residual):
    """y against act(a w^T + bias) + residual of the given operands, all in 64 bits."""
    a, w = a.double(), w.double()
    b = bias.double() if bias is not None else torch.zeros(w.shape[0], dtype=torch.float64, device=w.device)
    r = residual.double() if residual is not None else torch.zeros((), dtype=torch.float64, device=w.device)
    v = a @ w.t() + b
    s = a.abs() @ w.abs().t() + b.abs()
    z = act64(v, activation)
    want = z + r
    info = torch.finfo(y.dtype)
    bound = (info.eps / 2 * want.abs() + 1.13 * (a.shape[1] + 16) * 2.0 ** -23 * s + 1e-5 * v.abs()
             + 2.0 ** -22 * (z.abs() + r.abs())) * (1 + info.eps) + info.smallest_normal * info.eps / 2
    err = (y.double() - want).abs()
    assert y.shape == want.shape
    assert bool((err <= bound).all()), f"off by {(err / bound).max().item():.3g} of the bound"


# One shape at least for each GEMM kernel (decode with its own gather, decode, cluster
# split-K, single-CTA, CTA pairs with whole and with half tiles, 192-wide pairs, fp32).
SHAPES = [(1, 256, 512), (1, 100, 77), (3, 1000, 600), (16, 640, 768), (17, 129, 1000), (32, 2304, 768),
          (40, 768, 512), (100, 513, 700), (300, 1024, 640), (517, 2050, 320), (1024, 4096, 256),
          (4096, 768, 200), (2300, 3968, 260), (1290, 72, 128)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_ghost_linear(M, N, K, dtype):
    g = gen(M + N + K)
    x, r, b = randn(g, M, K, dtype=dtype), randn(g, M, N, dtype=dtype), randn(g, N, dtype=dtype)
    w = randn(g, N, K, dtype=dtype) / math.sqrt(K)
    idx = half(K, K)
    wp = pack_weight(w, idx)
    for activation, bias in ((None, b), ("gelu_tanh", b), ("gelu", None)):
        y = ghost_linear(x, wp, idx, bias=bias, activation=activation, residual=r)
        check(y, x[:, idx], w[:, idx], bias, activation, r)
    # Without one nothing changes: the same bits as a residual of zeros gives for None.
    plain = ghost_linear(x, wp, idx, bias=b)
    assert torch.equal(plain, ghost_linear(x, wp, idx, bias=b, residual=torch.zeros_like(r)))
    # In place, and with rows that are neither adjacent nor aligned.
    acc = r.clone()
    y = ghost_linear(x, wp, idx, bias=b, out=acc, residual=acc)
    assert y is acc
    check(acc, x[:, idx], w[:, idx], b, None, r)
    big = torch.full((M, N + 3), 5.0, dtype=dtype, device="cuda")
    big[:, 1: N + 1] = r
    y = ghost_linear(x, wp, idx, bias=b, residual=big[:, 1: N + 1])
    check(y, x[:, idx], w[:, idx], b, None, r)
    ghost_linear(x, wp, idx, bias=b, residual=big[:, 1: N + 1], out=big[:, 1: N + 1])
    check(big[:, 1: N + 1], x[:, idx], w[:, idx], b, None, r)
    assert bool((big[:, 0] == 5).all()) and bool((big[:, N + 1:] == 5).all())
    assert _native.device_error() == 0


@pytest.mark.parametrize("strategy", ["fused", "pregather", "overlap", "runs"])
@pytest.mark.parametrize("M,N,K", [(2, 256, 512), (24, 512, 640), (130, 520, 512), (2048, 2304, 512)])
def test_strategies(M, N, K, strategy):
    g = gen(M)
    dt = torch.bfloat16
    x, r, b = randn(g, M, K, dtype=dt), randn(g, M, N, dtype=dt), randn(g, N, dtype=dt)
    w = randn(g, N, K, dtype=dt) / math.sqrt(K)
    idx = half(K, K, runs=strategy == "runs")
    y = ghost_linear(x, pack_weight(w, idx), idx, bias=b, activation="gelu", strategy=strategy, residual=r)
    check(y, x[:, idx], w[:, idx], b, "gelu", r)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(5, 200, 300), (300, 768, 512), (2048, 2304, 300)])
@pytest.mark.parametrize("alive", [0, 1, 150])
def test_count_on_the_device(M, N, K, alive, dtype):
    g = gen(M + alive)
    x, r, b = randn(g, M, K, dtype=dtype), randn(g, M, N, dtype=dtype), randn(g, N, dtype=dtype)
    w = randn(g, N, K, dtype=dtype) / math.sqrt(K)
    buf = torch.zeros(K, dtype=torch.int64, device="cuda")
    idx = torch.randperm(K, generator=g, device="cuda")[:alive].sort().values
    buf[:alive] = idx
    count = torch.tensor([alive], dtype=torch.int32, device="cuda")
    y = ghost_linear_dev(x, pack_weight_dev(w, buf, count), buf, count, bias=b, residual=r)
    check(y, x[:, idx], w[:, idx], b, None, r)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_empty_alive_list(dtype):
    g = gen(1)
    x, r, b = randn(g, 7, 64, dtype=dtype), randn(g, 7, 50, dtype=dtype), randn(g, 50, dtype=dtype)
    idx = torch.empty(0, dtype=torch.int64, device="cuda")
    w = torch.empty(50, 64, dtype=dtype, device="cuda")
    y = ghost_linear(x, pack_weight(w, idx), idx, bias=b, activation="gelu", residual=r)
    check(y, x[:, :0], torch.empty(50, 0, device="cuda", dtype=dtype), b, "gelu", r)
    none = ghost_linear(x[:0], pack_weight(w, idx), idx, residual=r[:0])
    assert none.shape == (0, 50)


@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (16, 768, 768), (200, 1000, 333), (1024, 4096, 512)])
def test_packed_linear(M, N, K):
    g = gen(N)
    for dt in (torch.float16, torch.bfloat16):
        a, r, b = randn(g, M, (K + 7) // 8 * 8, dtype=dt), randn(g, M, N, dtype=dt), randn(g, N, dtype=dt)
        a = a[:, :K]                                 # aligned rows with a gap: taken as they are
        w = randn(g, N, K, dtype=dt) / math.sqrt(K)
        wp = pack_weight(w, torch.arange(K, device="cuda"))
        out = torch.empty(M, N, dtype=dt, device="cuda")
        y = packed_linear(a, wp, bias=b, activation="gelu_tanh", residual=r, out=out)
        assert y is out
        check(y, a, w, b, "gelu_tanh", r)
        if K % 8 == 0:
            assert torch.equal(packed_linear(a.contiguous(), wp, bias=b), packed_linear(a, wp, bias=b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("mode", ["frozen", "frozen-runs", "dynamic", "synchronous", "dense"])
@pytest.mark.parametrize("M", [1, 16, 90, 1100])
def test_ghost_linear_module(M, mode, dtype):
    g = gen(M)
    K, N = 512, 384
    layer = GhostLinear(K, N, threshold=0.0, device="cuda", dtype=dtype, activation="gelu")
    dead = torch.zeros(K, dtype=torch.bool, device="cuda")
    if mode == "frozen-runs":
        dead.view(-1, 64)[::2] = True
    elif mode != "dense":
        dead[torch.randperm(K, generator=g, device="cuda")[: K // 2]] = True
    x = randn(g, M, K, dtype=dtype)
    with torch.no_grad():
        layer.weight.copy_(randn(g, N, K, dtype=dtype) / math.sqrt(K))
        layer.bias.copy_(randn(g, N, dtype=dtype))
        layer.weight[:, dead] = 0
        x[:, dead] = 0
    if mode.startswith("frozen"):
        layer.freeze_weight_mask()
    elif mode == "synchronous":
        layer.sync_free = False
    r = randn(g, M, N, dtype=dtype)
    with torch.no_grad():
        for _ in range(3):                           # the second call of a frozen layer takes its fast path
            y = layer(x, residual=r)
            torch.cuda.synchronize()
            if mode == "dense" and _ > 0:
                # F.linear and F.gelu round before the addition: three roundings instead of one.
                want = torch.nn.functional.gelu(x.double() @ layer.weight.double().t() + layer.bias.double()) + r.double()
                scale = (x.double().abs() @ layer.weight.double().abs().t() + layer.bias.double().abs())
                bound = torch.finfo(dtype).eps * (want.abs() + scale) + (K + 16) * 2.0 ** -22 * scale + 1e-5
                assert bool(((y.double() - want).abs() <= bound).all())
            else:
                check(y, x, layer.weight, layer.bias, "gelu", r)
        plain = layer(x)
        assert plain.shape == (M, N)
        y3 = layer(x.view(1, M, K), residual=r.view(1, M, N))
        assert y3.shape == (1, M, N)
    for bad in (r[:, :-1], r.double(), r.cpu(), r[None]):
        with pytest.raises(AssertionError), torch.no_grad():
            layer(x, residual=bad)
    with pytest.raises(RuntimeError, match="no backward"):
        layer(x, residual=r.clone().requires_grad_())


@pytest.mark.parametrize("dropout", [None, nn.Dropout(0.5)])
def test_mlp_chain(dropout):
    g = gen(3)
    dt = torch.float16
    fc = GhostLinear(256, 512, device="cuda", dtype=dt)
    proj = GhostLinear(512, 256, device="cuda", dtype=dt)
    with torch.no_grad():
        for m in (fc, proj):
            m.weight.copy_(randn(g, *m.weight.shape, dtype=dt) / 16)
            m.bias.copy_(randn(g, m.out_features, dtype=dt))
            m.weight[:, torch.randperm(m.in_features, generator=g, device="cuda")[: m.in_features // 2]] = 0
            m.freeze_weight_mask()
        chain = GhostMLPChain(fc, proj, "gelu_tanh", dropout).eval()
        x, r = randn(g, 2, 30, 256, dtype=dt), randn(g, 2, 30, 256, dtype=dt)
        y = chain(x, residual=r)
        plain = chain(x)
        # One rounding (of the sum) against two (of the product, then of the sum).
        err = (y.double() - (plain.double() + r.double())).abs()
        assert bool((err <= 2.0 ** -11 * (plain.double().abs() + y.double().abs()) + 1e-7).all())
        if dropout is not None:
            chain.train()
            y = chain(x, residual=torch.zeros_like(r))
            assert 0.3 < (y == 0).float().mean().item() < 0.7
        with pytest.raises(AssertionError):
            chain(x, residual=r[:1])


def test_captured():
    g = gen(5)
    dt = torch.bfloat16
    K, N = 512, 768
    w, b = randn(g, N, K, dtype=dt) / 16, randn(g, N, dtype=dt)
    idx = half(K, 1)
    wp = pack_weight(w, idx)
    for M in (1, 8, 64, 2048):
        x, r = randn(g, M, K, dtype=dt), randn(g, M, N, dtype=dt)
        ghost_linear(x, wp, idx, bias=b, residual=r)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ghost_linear(x, wp, idx, bias=b, residual=r)
            z = ghost_linear(x, wp, idx, bias=b, residual=y)      # the previous kernel's output as residual
        for _ in range(2):
            x.copy_(randn(g, M, K, dtype=dt))
            r.copy_(randn(g, M, N, dtype=dt))
            graph.replay()
            check(y, x[:, idx], w[:, idx], b, None, r)
            check(z, x[:, idx], w[:, idx], b, None, y)


def test_residual_from_the_previous_kernel():
    """Back-to-back calls whose residual is the call before's output: the epilogue waits for it."""
    g = gen(6)
    dt = torch.float16
    for M, N, K in ((1, 4096, 1024), (16, 4096, 2048), (256, 1024, 1024), (2048, 4096, 256)):
        x, b = randn(g, M, K, dtype=dt), randn(g, N, dtype=dt)
        w = randn(g, N, K, dtype=dt) / math.sqrt(K)
        idx = half(K, 2)
        wp = pack_weight(w, idx)
        outs = [randn(g, M, N, dtype=dt)]
        for _ in range(6):
            outs.append(ghost_linear(x, wp, idx, bias=b, residual=outs[-1]))
        for before, after in zip(outs, outs[1:]):
            check(after, x[:, idx], w[:, idx], b, None, before)


def test_refusals():
    dt = torch.float16
    x = torch.zeros(8, 64, dtype=dt, device="cuda")
    idx = torch.arange(32, device="cuda")
    wp = pack_weight(torch.zeros(48, 64, dtype=dt, device="cuda"), idx)
    r = torch.zeros(8, 48, dtype=dt, device="cuda")
    for bad in (r[:, :40], r[:4], r.float(), r.cpu(), r[None]):
        with pytest.raises(AssertionError):
            ghost_linear(x, wp, idx, residual=bad)
        with pytest.raises(AssertionError):
            packed_linear(x[:, :32], wp, residual=bad)
    big = torch.zeros(9, 48, dtype=dt, device="cuda")
    with pytest.raises(AssertionError, match="overlaps"):
        ghost_linear(x, wp, idx, residual=big[:8], out=big[1:])
    with pytest.raises(RuntimeError, match="no backward"):
        ghost_linear(x, wp, idx, residual=r.clone().requires_grad_())
    with torch.no_grad():
        ghost_linear(x, wp, idx, residual=r.clone().requires_grad_())
    assert ghost_linear(x, wp, idx, residual=r[:1].expand(8, 48)).shape == (8, 48)


def test_fp32_more_row_tiles_than_a_grid_dimension():
    """65536 tiles of 64 rows and a part of one: past the second grid dimension's limit."""
    M, K = 65536 * 64 + 5, 4
    g = gen(3)
    x, r = randn(g, M, K, dtype=torch.float32), randn(g, M, 1, dtype=torch.float32)
    w = randn(g, 1, K, dtype=torch.float32)
    idx = torch.tensor([0, 2, 3], device="cuda")
    packed = pack_weight(w, idx)
    y = ghost_linear(x, packed, idx, residual=r)
    check(y, x[:, idx], w[:, idx], None, None, r)
