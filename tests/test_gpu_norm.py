"""GPU: residual + RMS norm and e4m3 rows over the alive columns, against their formulas in 64 bits.

    s = x + r;  y[m, j] = s[m, c_j] / sqrt(mean_k s[m, k]^2 + eps) * g[c_j]
    scale[m] = max(max_j |y[m, j]| / 448, 2^-126);  q[m, j] = e4m3(y[m, j] / scale[m])

Tolerances. A rounding to the output type is off by at most half a step:
finfo.eps / 2 of the value, or half the smallest subnormal. In front of it
stand fp32 operations, each off by 2^-24 of its result: the addition of r; the
sum of squares, where one thread adds at most ceil(K / 32) terms and the
threads' sums are joined in at most 10 steps, so that it is off by at most
(K / 32 + 13) 2^-24 and its inverse square root by half of that; the mean, the
eps, rsqrtf (2 steps of 2^-23), and the two products. `slack(K)` is their sum,
rounded up. e4m3 halves a step of 2^-3 (2^-4 of the value), or 2^-10 below
2^-6; its scale is off by the slack alone, and moves q by the slack as well.
"""

from __future__ import annotations

import math

import pytest
import torch

from ghostweight_triton_b200 import _native
from ghostweight_triton_b200.kernels.norm import pack_weight_q8, quantize_rows, rms_norm, rms_norm_q8

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
EPS = 1e-6


def slack(K: int) -> float:
    return ((K / 32 + 13) / 2 + 12) * 2.0 ** -24


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def make(M, K, dtype, seed, residual=True):
    g = gen(seed)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    r = (2 * torch.randn(M, K, generator=g, device="cuda")).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(dtype)
    return x, r, w


def alive(kind, K, seed):
    g = gen(seed + 77)
    if kind == "all":
        return None
    if kind == "half":
        return torch.randperm(K, generator=g, device="cuda")[: (K + 1) // 2].sort().values
    if kind == "one":
        return torch.tensor([K - 1], device="cuda")
    if kind == "empty":
        return torch.empty(0, dtype=torch.int64, device="cuda")
    if kind == "unsorted":
        return torch.randint(0, K, (max(1, K - 1),), generator=g, device="cuda")
    if kind == "longer":                     # repeats: more outputs than columns
        return torch.randint(0, K, (2 * K + 3,), generator=g, device="cuda")
    if kind == "blocks":
        keep = torch.arange(0, max(1, K // 128), 2, device="cuda")
        return (keep[:, None] * 128 + torch.arange(128, device="cuda")).reshape(-1).clamp_max(K - 1)
    raise AssertionError(kind)


def reference(x, r, w, idx, eps=EPS, norm=True):
    s = x.double() if r is None else x.double() + r.double()
    y = s
    if norm:
        y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.double()
    return (y if idx is None else y[..., idx]), s


def close(got, want, dtype, extra):
    """got rounds want once to dtype, with fp32 errors of `extra` relative in front."""
    info = torch.finfo(dtype)
    bound = want.abs() * (info.eps / 2 + extra * (1 + info.eps)) + info.smallest_normal * info.eps / 2
    err = (got.double() - want).abs()
    assert got.dtype is dtype and got.shape == want.shape
    assert bool((err <= bound).all()), f"off by {(err / bound).max().item():.3g} of the bound"


def close_q8(q, scale, want, extra, tiny=0.0):
    """`tiny`: what a product of fp32 subnormals may be off by, absolutely."""
    want_scale = (want.abs().amax(-1) / 448).clamp_min(2.0 ** -126) if want.shape[-1] else \
        torch.full(want.shape[:-1], 2.0 ** -126, dtype=torch.float64, device=want.device)
    assert q.dtype is torch.float8_e4m3fn and scale.dtype is torch.float32
    assert q.shape == want.shape and scale.shape == want.shape[:-1]
    assert bool(((scale.double() - want_scale).abs() <= want_scale * (extra + 2.0 ** -23) + tiny / 448).all())
    s = scale.double().unsqueeze(-1)
    bound = torch.maximum(want.abs() / 16, s / 1024) + want.abs() * 2 * (extra + 2.0 ** -23) + 2 * tiny
    err = (q.float().double() * s - want).abs()
    assert bool((err <= bound).all()), f"off by {(err / bound).max().item():.3g} of the bound"


def padding_is_zero(t, n, align):
    """Behind the n columns of a padded view, up to the next multiple of align, stand zeros."""
    ld = t.stride(0) if t.shape[0] > 1 else -(-n // align) * align
    if t.shape[0] and ld > n:
        raw = t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t
        whole = torch.as_strided(raw, (t.shape[0], ld), (ld, 1))
        assert not bool(whole[:, n:].any())


SHAPES = [(1, 1), (3, 2), (1, 7), (5, 8), (33, 31), (2, 64), (7, 100), (64, 768), (9, 1111), (3, 4096),
          (130, 2048), (2, 8200), (1, 16384), (3, 28672), (2, 50001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", SHAPES)
@pytest.mark.parametrize("kind", ["all", "half", "unsorted"])
def test_rms_norm(M, K, dtype, kind):
    x, r, w = make(M, K, dtype, M * 31 + K)
    idx = alive(kind, K, K)
    y, s = rms_norm(x, w, EPS, residual=r, alive_indices=idx)
    want, total = reference(x, r, w, idx)
    close(y, want, dtype, slack(K))
    close(s, total, dtype, 2.0 ** -24)
    if idx is not None:
        padding_is_zero(y, idx.numel(), 64)
    y1 = rms_norm(x, None, 1e-3, alive_indices=idx)
    close(y1, reference(x, None, None, idx, 1e-3)[0], dtype, slack(K))
    assert _native.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", SHAPES)
@pytest.mark.parametrize("kind", ["all", "half", "unsorted"])
def test_rms_norm_q8(M, K, dtype, kind):
    x, r, w = make(M, K, dtype, M * 37 + K)
    idx = alive(kind, K, K + 1)
    q, scale, s = rms_norm_q8(x, w, EPS, residual=r, alive_indices=idx)
    want, total = reference(x, r, w, idx)
    close_q8(q, scale, want, slack(K))
    close(s, total, dtype, 2.0 ** -24)
    padding_is_zero(q, want.shape[-1], 128)
    q, scale = quantize_rows(x, idx)
    close_q8(q, scale, reference(x, None, None, idx, norm=False)[0], 0.0)
    padding_is_zero(q, want.shape[-1], 128)


@pytest.mark.parametrize("kind", ["one", "empty", "longer", "blocks"])
@pytest.mark.parametrize("M,K", [(1, 5), (17, 200), (4, 4096), (2, 30000)])
def test_lists(M, K, kind):
    x, r, w = make(M, K, torch.bfloat16, 5)
    idx = alive(kind, K, 9)
    want, total = reference(x, r, w, idx)
    y, s = rms_norm(x, w, EPS, residual=r, alive_indices=idx.to(torch.int32))
    close(y, want, torch.bfloat16, slack(K))
    close(s, total, torch.bfloat16, 2.0 ** -24)
    q, scale, s = rms_norm_q8(x, w, EPS, residual=r, alive_indices=idx)
    close_q8(q, scale, want, slack(K))
    close(s, total, torch.bfloat16, 2.0 ** -24)
    q, scale = quantize_rows(x, idx)
    close_q8(q, scale, reference(x, None, None, idx, norm=False)[0], 0.0)
    if kind == "longer":
        padding_is_zero(y, idx.numel(), 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 64), (1000, 256), (4099, 96), (700, 1024), (300, 4096), (160, 13)])
def test_many_rows(M, K, dtype):
    """More rows than CTAs run at once, so that each CTA takes several."""
    x, r, w = make(M, K, dtype, 3)
    idx = alive("half", K, 3)
    y, s = rms_norm(x, w, EPS, residual=r, alive_indices=idx)
    want, total = reference(x, r, w, idx)
    close(y, want, dtype, slack(K))
    close(s, total, dtype, 2.0 ** -24)
    q, scale = quantize_rows(x, idx)
    close_q8(q, scale, reference(x, None, None, idx, norm=False)[0], 0.0)
    x2 = x.repeat(20, 1)
    y2 = rms_norm(x2, w, EPS)
    close(y2, reference(x2, None, w, None)[0], dtype, slack(K))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,off,ld", [(64, 0, 96), (64, 1, 97), (100, 8, 128), (333, 3, 400), (2048, 4, 2056)])
def test_strides(K, off, ld, dtype):
    g = gen(K)
    big = torch.randn(9, ld, generator=g, device="cuda").to(dtype)
    other = torch.randn(9, ld + 5, generator=g, device="cuda").to(dtype)
    x, r = big[:, off: off + K] if off + K <= ld else big[:, :K], other[:, :K]
    w = torch.randn(K + 1, generator=g, device="cuda").to(dtype)[1:]
    idx = alive("half", K, 1)
    for i in (None, idx):
        y, s = rms_norm(x, w, EPS, residual=r, alive_indices=i)
        want, total = reference(x, r, w, i)
        close(y, want, dtype, slack(K))
        close(s, total, dtype, 2.0 ** -24)
        q, scale = quantize_rows(x, i)
        close_q8(q, scale, reference(x, None, None, i, norm=False)[0], 0.0)
    # Columns as rows, and one row for every row: neither is row-major.
    xt = torch.randn(K, 9, generator=g, device="cuda").to(dtype).t()
    close(rms_norm(xt, w, EPS), reference(xt, None, w, None)[0], dtype, slack(K))
    xe = x[:1].expand(9, K)
    close(rms_norm(xe, w, EPS), reference(xe, None, w, None)[0], dtype, slack(K))


def test_leading_dimensions():
    x, r, w = make(24, 96, torch.float16, 1)
    idx = alive("half", 96, 1)
    want, total = reference(x, r, w, idx)
    y, s = rms_norm(x.view(2, 3, 4, 96), w, EPS, residual=r.view(2, 3, 4, 96), alive_indices=idx)
    assert y.shape == (2, 3, 4, 48) and s.shape == (2, 3, 4, 96)
    close(y.reshape(24, 48), want, torch.float16, slack(96))
    close(s.reshape(24, 96), total, torch.float16, 2.0 ** -24)
    q, scale = quantize_rows(x.view(2, 12, 96), idx)
    assert q.shape == (2, 12, 48) and scale.shape == (2, 12)
    y0 = rms_norm(x[0], w, EPS)
    assert y0.shape == (96,)
    q0, s0 = quantize_rows(x[0])
    assert q0.shape == (96,) and s0.shape == ()
    none = rms_norm(x[:0], w, EPS, residual=r[:0], alive_indices=idx)
    assert none[0].shape == (0, 48) and none[1].shape == (0, 96)
    q, scale = quantize_rows(x[:0])
    assert q.shape == (0, 96) and scale.shape == (0,)


@pytest.mark.parametrize("K", [40, 768, 4096, 50001])
@pytest.mark.parametrize("which", ["x", "residual"])
def test_sum_in_place(K, which):
    x, r, w = make(37, K, torch.bfloat16, 2)
    idx = alive("half", K, 2)
    want, total = reference(x, r, w, idx)
    xi, ri = x.clone(), r.clone()
    out = xi if which == "x" else ri
    y, s = rms_norm(xi, w, EPS, residual=ri, alive_indices=idx, residual_out=out)
    assert s is out
    close(y, want, torch.bfloat16, slack(K))
    close(s, total, torch.bfloat16, 2.0 ** -24)
    assert torch.equal(ri if which == "x" else xi, r if which == "x" else x)
    xi, ri = x.clone(), r.clone()
    out = xi if which == "x" else ri
    q, scale, s = rms_norm_q8(xi, w, EPS, residual=ri, residual_out=out)
    close_q8(q, scale, reference(x, r, w, None)[0], slack(K))
    close(s, total, torch.bfloat16, 2.0 ** -24)


def test_rows_behind_the_output_stay():
    """residual_out may be rows of a larger buffer: what lies around them is left as it was."""
    x, r, w = make(6, 100, torch.float16, 8)
    big = torch.full((10, 128), 7.0, dtype=torch.float16, device="cuda")
    out = big[2:8, 10:110]
    _, s = rms_norm(x, w, EPS, residual=r, residual_out=out)
    close(s, x.double() + r.double(), torch.float16, 2.0 ** -24)
    keep = torch.ones_like(big, dtype=torch.bool)
    keep[2:8, 10:110] = False
    assert bool((big[keep] == 7.0).all())


def test_non_finite_and_tiny_rows():
    """One row's NaN or infinity touches no other row; dead columns count in the mean, not in
    the largest value; zeros and subnormals keep their scale."""
    K = 96
    x, _, w = make(8, K, torch.float32, 4, residual=False)
    idx = torch.arange(0, K, 2, device="cuda")
    x[1, 3] = float("nan")          # dead column
    x[2, 4] = float("nan")          # alive
    x[3, 5] = float("inf")          # dead
    x[4, 6] = float("-inf")         # alive
    x[5] = 0.0
    x[6] = 1e-42                    # subnormal in fp32
    y = rms_norm(x, w, EPS, alive_indices=idx)
    want = reference(x, None, w, idx)[0]
    for row in (0, 5, 7):
        close(y[row: row + 1], want[row: row + 1], torch.float32, slack(K))
    assert y[1].isnan().all() and y[2].isnan().all()
    assert (y[3] == 0).all()                                   # finite / sqrt(inf)
    assert y[4, 3].isnan() and (y[4, [0, 1, 2, 4]] == 0).all()
    q, scale = quantize_rows(x, idx)
    plain = x.double()[:, idx]
    for row in (0, 1, 3, 5, 6, 7):                             # dead NaN and infinity are not looked at
        close_q8(q[row: row + 1], scale[row: row + 1], plain[row: row + 1], 0.0)
    back = q.float() * scale[:, None]
    assert back[2].isnan().all() and back[4].isnan().all()
    assert scale[5] == 2.0 ** -126 and (q[5].float() == 0).all()
    qn, sn = rms_norm_q8(x, w, EPS, alive_indices=idx)
    backn = qn.float() * sn[:, None]
    assert backn[1].isnan().all() and backn[2].isnan().all() and backn[4].isnan().all()
    close_q8(qn[[0, 5, 7]], sn[[0, 5, 7]], want[[0, 5, 7]], slack(K))


def test_large_values_saturate_nothing():
    """The largest value of a row is 448 scales, in every type's upper range."""
    for dtype, big in ((torch.float16, 65504.0), (torch.bfloat16, 3.0e38), (torch.float32, 3.3e38)):
        x = torch.full((3, 64), -big, device="cuda").to(dtype)
        x[:, 1] = 1.0
        q, scale = quantize_rows(x)
        assert (q[:, 0].float() == -448).all()
        close_q8(q, scale, x.double(), 0.0)


@pytest.mark.parametrize("K", [96, 2000])
def test_tiny_rows_q8(K):
    """Rows down to the subnormals: the factors between them and e4m3 stay within fp32.

    The product of x with the weight rounds to a multiple of 2^-149 there, so it is off by up
    to 2^-150, which the norm's factor (at most 1 / sqrt(eps)) enlarges."""
    _, _, w = make(1, K, torch.float32, 14, residual=False)
    x = torch.randn(12, K, device="cuda", generator=gen(15))
    x *= torch.logspace(-44, -33, 12, device="cuda")[:, None]
    q, scale = rms_norm_q8(x, w, EPS)
    close_q8(q, scale, reference(x, None, w, None)[0], slack(K) + 2.0 ** -20, 2.0 ** -150 / math.sqrt(EPS))
    q, scale = quantize_rows(x)
    close_q8(q, scale, x.double(), 2.0 ** -20)


def test_bad_indices():
    x, r, w = make(4, 64, torch.bfloat16, 6)
    idx = torch.tensor([0, 64, 5, -1, 1 << 40, 63], device="cuda")
    _native.device_error()
    y, s = rms_norm(x, w, EPS, residual=r, alive_indices=idx)
    assert _native.device_error() == _native.DEVICE_ERR_BAD_INDEX
    want, total = reference(x, r, w, idx.clamp(0, 63))
    want[:, [1, 3, 4]] = 0
    close(y, want, torch.bfloat16, slack(64))
    close(s, total, torch.bfloat16, 2.0 ** -24)
    q, scale = quantize_rows(x, idx)
    assert _native.device_error() == _native.DEVICE_ERR_BAD_INDEX
    plain = x.double()[:, idx.clamp(0, 63)]
    plain[:, [1, 3, 4]] = 0
    close_q8(q, scale, plain, 0.0)


def test_offsets_past_32_bits():
    """Rows that lie more than 2^31 elements apart."""
    K, ld = 200, (1 << 30) + 72
    buf = torch.empty(2 * ld + K, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (3, K), (ld, 1))
    src, r, w = make(3, K, torch.bfloat16, 12)
    x.copy_(src)
    idx = alive("half", K, 12)
    want, total = reference(src, r, w, idx)
    y, s = rms_norm(x, w, EPS, residual=r, alive_indices=idx, residual_out=x)
    close(y, want, torch.bfloat16, slack(K))
    close(x, total, torch.bfloat16, 2.0 ** -24)
    x.copy_(src)
    q, scale = quantize_rows(x)
    close_q8(q, scale, src.double(), 0.0)


def test_pack_weight_q8():
    w = torch.randn(300, 500, device="cuda", generator=gen(1)).half()
    idx = alive("half", 500, 4)
    for weight in (w, w.t().contiguous().t(), torch.nn.Parameter(w)):
        q, scale = pack_weight_q8(weight, idx)
        close_q8(q, scale, w.double()[:, idx], 0.0)
        padding_is_zero(q, idx.numel(), 128)


def test_captured_and_on_another_stream():
    x, r, w = make(65, 640, torch.float16, 21)
    idx = alive("half", 640, 21)
    rms_norm(x, w, EPS, residual=r, alive_indices=idx)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, s = rms_norm(x, w, EPS, residual=r, alive_indices=idx)
    torch.cuda.current_stream().wait_stream(side)
    close(y, reference(x, r, w, idx)[0], torch.float16, slack(640))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y, s = rms_norm(x, w, EPS, residual=r, alive_indices=idx)
        q, scale = quantize_rows(y)
    for seed in (22, 23):
        x2, r2, _ = make(65, 640, torch.float16, seed)
        x.copy_(x2)
        r.copy_(r2)
        graph.replay()
        want, total = reference(x2, r2, w, idx)
        close(y, want, torch.float16, slack(640))
        close(s, total, torch.float16, 2.0 ** -24)
        close_q8(q, scale, y.double(), 0.0)


def test_repeated_calls_agree_to_the_bit():
    x, r, w = make(500, 4096, torch.bfloat16, 30)
    idx = alive("half", 4096, 30)
    first = rms_norm_q8(x, w, EPS, residual=r, alive_indices=idx)
    for _ in range(3):
        again = rms_norm_q8(x, w, EPS, residual=r, alive_indices=idx)
        assert torch.equal(first[0].view(torch.uint8), again[0].view(torch.uint8))
        assert torch.equal(first[1], again[1]) and torch.equal(first[2], again[2])


def test_refusals():
    x, r, w = make(4, 64, torch.float16, 1)
    idx = torch.arange(5, device="cuda")
    for bad in (dict(weight=w[:-1]), dict(weight=w.cpu()), dict(residual=r[:, :-1]), dict(residual=r.float()),
                dict(residual=r[:3]), dict(residual=r.cpu()), dict(alive_indices=idx.float()),
                dict(alive_indices=idx.bool()), dict(alive_indices=idx[:, None]), dict(eps=-1.0),
                dict(residual_out=r), dict(residual=r, residual_out=r.float()),
                dict(residual=r, residual_out=torch.empty(64, 4, dtype=torch.float16, device="cuda").t()),
                dict(residual=r, residual_out=torch.empty(1, 64, dtype=torch.float16, device="cuda").expand(4, 64))):
        with pytest.raises(AssertionError):
            rms_norm(x, **bad)
        with pytest.raises(AssertionError):
            rms_norm_q8(x, **bad)
    big = torch.zeros(8, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(AssertionError, match="overlaps"):
        rms_norm(big[:4], w, residual=r, residual_out=big[1:5])
    with pytest.raises(AssertionError):
        rms_norm(x[:, :0])
    for fn in (rms_norm, rms_norm_q8, quantize_rows):
        with pytest.raises(TypeError):
            fn(torch.zeros(2, 8, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="no backward"):
            fn(x.clone().requires_grad_())
        with torch.no_grad():
            fn(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no backward"):
        rms_norm(x, w, residual=r.clone().requires_grad_())
    y = rms_norm(x, torch.nn.Parameter(w))          # a parameter is a constant here
    assert not y.requires_grad
