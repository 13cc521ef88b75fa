"""GPU: the e4m3 product with scales, against the formula in 64 bits on the same e4m3 values.

    y = act(sa[m] sw[n] sum_j a[m, j] w[n, j] + b[n]) + r[m, n]

Tolerance: a product of two e4m3 values (4 significant bits each) is exact in
fp32; the sum of K of them takes at most K additions in any order, each off by
at most 2^-23 of the running sum, which is at most the sum S of the products'
magnitudes; the two scalings, the bias, the residual and the activation add a
few more, and the result is rounded once to y's type (half a step of it):

    |err| <= finfo.eps / 2 |y| + (K + 16) 2^-23 (S + |b|) 1.13 + 1e-5 |v| + 2^-22 (|act| + |r|)

with S scaled, 1.13 bounding the slope of the GELU and 1e-5 |v| the fast
exponential of its tanh form (v the value before it).
"""

from __future__ import annotations

import math

import pytest
import torch

from ghostweight_triton_b200 import _native
from ghostweight_triton_b200.kernels.matmul import packed_linear, packed_linear_q8
from ghostweight_triton_b200.kernels.norm import pack_weight_q8, quantize_rows, rms_norm_q8

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def operand(g, rows, cols, garbage=True):
    """Random e4m3 rows 16-byte aligned, with scales; behind the last column stand NaN bytes."""
    ld = (cols + 15) // 16 * 16
    buf = torch.full((rows, ld), 0x7F, dtype=torch.uint8, device="cuda")
    buf[:, :cols] = (60 * randn(g, rows, cols)).clamp(-448, 448).to(E4M3).view(torch.uint8)
    scale = torch.exp(randn(g, rows) * 2) / 60
    return buf.view(E4M3)[:, :cols], scale


def act64(v, activation):
    if activation == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2.0)))
    if activation == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def check(y, a, sa, w, sw, bias=None, activation=None, residual=None):
    a64, w64 = a.to(torch.float32).double(), w.to(torch.float32).double()
    scale = torch.outer(sa.double(), sw.double())
    b = 0.0 if bias is None else bias.double()
    r = torch.zeros((), dtype=torch.float64, device="cuda") if residual is None else residual.double()
    v = (a64 @ w64.t()) * scale + b
    s = (a64.abs() @ w64.abs().t()) * scale + (0.0 if bias is None else bias.double().abs())
    z = act64(v, activation)
    want = z + r
    info = torch.finfo(y.dtype)
    bound = (info.eps / 2 * want.abs() + 1.13 * (a.shape[1] + 16) * 2.0 ** -23 * s + 1e-5 * v.abs()
             + 2.0 ** -22 * (z.abs() + r.abs())) * (1 + info.eps) + info.smallest_normal * info.eps / 2
    err = (y.double() - want).abs()
    assert y.shape == want.shape
    assert bool((err <= bound).all()), f"off by {(err / bound).max().item():.3g} of the bound"


# One shape at least for each kernel: decode, cluster split-K, single CTA, CTA pairs
# (whole and half tiles, 192 wide), and the smallest sizes.
SHAPES = [(1, 1, 1), (1, 256, 512), (1, 100, 77), (3, 1000, 601), (16, 640, 1536), (17, 129, 2000), (32, 2304, 768),
          (40, 768, 1024), (100, 513, 700), (300, 1024, 1280), (517, 2050, 640), (1024, 4096, 256), (4096, 768, 200),
          (2300, 3968, 260), (1290, 72, 128), (130, 40, 33)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K):
    for dtype in (torch.float16, torch.bfloat16):
        g = gen(M + N + K)
        (a, sa), (w, sw) = operand(g, M, K), operand(g, N, K)
        # Outputs of a few units, within fp16's range.
        sa, sw = sa / sa.mean(), sw / sw.mean() / (60 * 60 * math.sqrt(K) * 8)
        b, r = randn(g, N, dtype=dtype), randn(g, M, N, dtype=dtype)
        y = packed_linear_q8(a, sa, w, sw, dtype=dtype)
        check(y, a, sa, w, sw)
        y = packed_linear_q8(a, sa, w, sw, bias=b, activation="gelu_tanh", residual=r)
        assert y.dtype is dtype
        check(y, a, sa, w, sw, b, "gelu_tanh", r)
        acc = r.clone()
        y = packed_linear_q8(a, sa, w, sw, bias=b, activation="gelu", residual=acc, out=acc)
        assert y is acc
        check(acc, a, sa, w, sw, b, "gelu", r)
        big = torch.full((M, N + 3), 5.0, dtype=dtype, device="cuda")
        packed_linear_q8(a, sa, w, sw, bias=b.float(), residual=r, out=big[:, 1: N + 1])
        check(big[:, 1: N + 1], a, sa, w, sw, b, None, r)
        assert bool((big[:, 0] == 5).all()) and bool((big[:, N + 1:] == 5).all())
    assert _native.device_error() == 0


def test_operands_as_the_row_operators_write_them():
    g = gen(2)
    x, W = randn(g, 45, 700, dtype=torch.bfloat16), randn(g, 260, 700, dtype=torch.bfloat16)
    idx = torch.randperm(700, generator=g, device="cuda")[:333].sort().values
    gain = 1 + 0.1 * randn(g, 700, dtype=torch.bfloat16)
    a, sa = rms_norm_q8(x, gain, alive_indices=idx)
    w, sw = pack_weight_q8(W, idx)
    check(packed_linear_q8(a, sa, w, sw), a, sa, w, sw)
    # Against the product of the unrounded operands: each is within 2^-4 of its value (or
    # 2^-10 of its row's scale), so their products are within a little over twice that.
    n = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6) * gain.double()
    n, v = n[:, idx], W.double()[:, idx]
    da = torch.maximum(n.abs() / 16, sa.double()[:, None] / 1024) * 1.0001
    dw = torch.maximum(v.abs() / 16, sw.double()[:, None] / 1024) * 1.0001
    bound = da @ v.abs().t() + n.abs() @ dw.t() + da @ dw.t()
    err = (packed_linear_q8(a, sa, w, sw).double() - n @ v.t()).abs()
    assert bool((err <= bound + 2.0 ** -8 * (n @ v.t()).abs() + 1e-3).all())


def test_rows_that_tma_cannot_load_are_copied():
    g = gen(3)
    base_a = (60 * randn(g, 9, 131)).to(E4M3)
    base_w = (60 * randn(g, 33, 131)).to(E4M3)
    sa, sw = torch.rand(9, device="cuda", generator=g) / 500, torch.rand(33, device="cuda", generator=g) / 500
    for a, w in ((base_a, base_w), (base_a[:, 1:], base_w[:, 1:]),
                 (base_a.t().contiguous().t(), base_w.t().contiguous().t())):
        check(packed_linear_q8(a, sa, w, sw), a, sa, w, sw)
    strided = torch.stack([sa, sa], 1)[:, 0]
    check(packed_linear_q8(base_a, strided, base_w, sw), base_a, sa, base_w, sw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_no_columns_and_no_rows(dtype):
    g = gen(4)
    b, r = randn(g, 50, dtype=dtype), randn(g, 7, 50, dtype=dtype)
    a, w = torch.empty(7, 0, device="cuda").to(E4M3), torch.empty(50, 0, device="cuda").to(E4M3)
    sa, sw = torch.ones(7, device="cuda"), torch.ones(50, device="cuda")
    y = packed_linear_q8(a, sa, w, sw, bias=b, activation="gelu", residual=r)
    check(y, a, sa, w, sw, b, "gelu", r)
    a, w = torch.empty(0, 32, device="cuda").to(E4M3), torch.empty(50, 32, device="cuda").to(E4M3)
    assert packed_linear_q8(a, sa[:0], w, sw, bias=b).shape == (0, 50)


def test_extreme_scales_and_nan():
    """The scales' product may leave fp32's range while the result does not; a NaN row stays one row."""
    g = gen(5)
    for M in (4, 200, 2048):
        (a, _), (w, _) = operand(g, M, 256), operand(g, 2304, 256)
        sa = torch.full((M,), 2.0 ** -120, device="cuda")
        sw = torch.full((2304,), 2.0 ** 105, device="cuda")
        check(packed_linear_q8(a, sa, w, sw), a, sa, w, sw)
        sa[1] = float("nan")
        y = packed_linear_q8(a, sa, w, sw)
        assert y[1].isnan().all() and not y[[0, 2, 3]].isnan().any()
        # A row of zeros as quantize_rows writes it.
        q, s = quantize_rows(torch.zeros(M, 256, device="cuda", dtype=torch.bfloat16))
        assert (packed_linear_q8(q, s, w, sw) == 0).all()


def test_captured_chain():
    """Norm, product, rounding of the hidden rows, product with the residual, in one graph."""
    g = gen(7)
    dt = torch.bfloat16
    K, F = 512, 1024
    idx = torch.randperm(K, generator=g, device="cuda")[: K // 2].sort().values
    w1, s1 = pack_weight_q8(randn(g, F, K, dtype=dt) / 16, idx)
    w2, s2 = pack_weight_q8(randn(g, K, F, dtype=dt) / 16, torch.arange(F, device="cuda"))
    for M in (1, 30, 300, 2048):
        x, r = randn(g, M, K, dtype=dt), randn(g, M, K, dtype=dt)
        for captured in (False, True):
            graph = torch.cuda.CUDAGraph()

            def chain():
                q, s, h = rms_norm_q8(x, None, residual=r, alive_indices=idx)
                f = packed_linear_q8(q, s, w1, s1, activation="gelu_tanh", dtype=dt)
                p, t = quantize_rows(f)
                return q, s, h, f, p, t, packed_linear_q8(p, t, w2, s2, residual=h)

            if captured:
                torch.cuda.synchronize()
                with torch.cuda.graph(graph):
                    out = chain()
                x.copy_(randn(g, M, K, dtype=dt))
                graph.replay()
            else:
                out = chain()
            q, s, h, f, p, t, y = out
            check(f, q, s, w1, s1, None, "gelu_tanh")
            check(y, p, t, w2, s2, None, None, h)
            assert bool(((h.double() - x.double() - r.double()).abs() <= 2.0 ** -8 * (x + r).double().abs() * 1.01).all())


def test_repeated_calls_agree_to_the_bit():
    g = gen(8)
    for M, N, K in ((16, 4096, 2048), (256, 1024, 2048), (2048, 4096, 512)):
        (a, sa), (w, sw) = operand(g, M, K), operand(g, N, K)
        first = packed_linear_q8(a, sa, w, sw)
        for _ in range(3):
            assert torch.equal(first, packed_linear_q8(a, sa, w, sw))


def test_refusals():
    g = gen(9)
    (a, sa), (w, sw) = operand(g, 8, 64), operand(g, 48, 64)
    r = torch.zeros(8, 48, dtype=torch.bfloat16, device="cuda")
    bad_calls = [dict(a=a.float()), dict(a=a[None]), dict(a_scale=sa[:-1]), dict(a_scale=sa.half()), dict(a_scale=sa.cpu()),
                 dict(w_packed=w.view(torch.uint8)), dict(w_packed=w[:, :32]), dict(w_scale=sw[:1]),
                 dict(bias=torch.zeros(47, device="cuda")), dict(bias=torch.zeros(48)), dict(residual=r[:, :47]),
                 dict(residual=r.half(), dtype=torch.bfloat16), dict(out=r.half(), dtype=torch.bfloat16), dict(out=r[:7]),
                 dict(a=a.cpu(), a_scale=sa.cpu())]
    base = dict(a=a, a_scale=sa, w_packed=w, w_scale=sw)
    for bad in bad_calls:
        with pytest.raises(AssertionError):
            packed_linear_q8(**{**base, **bad})
    with pytest.raises(TypeError):
        packed_linear_q8(**base, dtype=torch.float32)
    with pytest.raises(ValueError):
        packed_linear_q8(**base, activation="relu")
    with pytest.raises(RuntimeError, match="no backward"):
        packed_linear_q8(**base, residual=r.clone().requires_grad_())
    lib = _native.load()
    call = lambda **k: lib.gw_packed_gemm_q8(
        k.get("a", a.data_ptr()), sa.data_ptr(), 8, k.get("K", 64), k.get("lda", 64), w.data_ptr(), sw.data_ptr(), 48,
        k.get("ldw", 64), None, 0, None, 0, r.data_ptr(), k.get("dtype", 1), 48, None)
    assert call(dtype=2) == _native.GW_ERR_DTYPE and call(lda=63) == _native.GW_ERR_SHAPE
    assert call(lda=72) == _native.GW_ERR_ALIGN and call(ldw=72) == _native.GW_ERR_ALIGN
    assert call(a=a.data_ptr() + 4) == _native.GW_ERR_ALIGN and call(a=None) == _native.GW_ERR_NULL
    assert call(K=-1) == _native.GW_ERR_SHAPE


@pytest.mark.parametrize("N", [32768, 32771])
def test_outputs_past_32_bits(N):
    """More than 2^31 outputs, and a residual of as many (N odd: rows of 2-byte alignment)."""
    M, K = 65600, 64
    g = gen(N)
    (a, sa), (w, sw) = operand(g, M, K), operand(g, N, K)
    sa, sw = sa / sa.mean(), sw / sw.mean() / (60 * 60 * math.sqrt(K) * 8)
    acc = torch.randn(M, N, generator=g, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([0, 1, 40000, M - 200, M - 2, M - 1], device="cuda")
    r = acc[rows]
    packed_linear_q8(a, sa, w, sw, residual=acc, out=acc)
    check(acc[rows], a[rows], sa[rows], w, sw, None, None, r)
    assert _native.device_error() == 0
