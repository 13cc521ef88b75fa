"""GPU: calls of the operators around a layer that their documentation allows and the
operators' own test files do not make, against the formulas in 64 bits (the bounds are
those files')."""

from __future__ import annotations

import copy
import io

import pytest
import torch
import torch.nn as nn

from ghostweight_triton_b200 import GhostLinear, _native
from ghostweight_triton_b200.fuse import GhostMLPChain, GhostPreNormMLP
from ghostweight_triton_b200.kernels.gather import pack_weight
from ghostweight_triton_b200.kernels.matmul import (ghost_linear, ghost_linear_dev, ghost_linear_pipelined,
                                                    ghostweight_matmul, packed_linear, packed_linear_q8)
from ghostweight_triton_b200.kernels.norm import pack_weight_q8, quantize_rows, rms_norm, rms_norm_q8
from tests.test_gpu_prenorm import block, exact, inputs
from tests.test_gpu_residual import check
from tests.test_prenorm_cpu import OnePlusWeight
from tests.test_products_cpu import weights_and_biases_refused

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


def operands(M, N, K, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    idx = torch.arange(K, device="cuda")
    return rnd(M, K), pack_weight(rnd(N, K), idx), idx


def test_outputs_refused():
    """Every product's `out`, with and without a residual, before anything is launched."""
    M, N, K = 8, 48, 64
    x, w, idx = operands(M, N, K)
    count = torch.tensor([K], dtype=torch.int32, device="cuda")
    qa, sa = quantize_rows(x)
    qw, sw = quantize_rows(w)
    res = torch.zeros(M, N, dtype=x.dtype, device="cuda")
    calls = [lambda out, r: ghost_linear(x, w, idx, out=out, residual=r),
             lambda out, r: ghost_linear_dev(x, w, idx, count, out=out, residual=r),
             lambda out, r: packed_linear(x, w, out=out, residual=r),
             lambda out, r: packed_linear_q8(qa, sa, qw, sw, dtype=x.dtype, out=out, residual=r),
             lambda out, r: ghost_linear_pipelined([(x, w, idx, out)])]
    for out in (torch.empty(M - 1, N, dtype=x.dtype, device="cuda"), torch.empty(M, N - 1, dtype=x.dtype, device="cuda"),
                torch.empty(M, N, dtype=torch.uint8, device="cuda"), torch.empty(M, N, dtype=x.dtype),
                torch.empty(N, M, dtype=x.dtype, device="cuda").t()):
        for call in calls:
            for r in (None, res):
                with pytest.raises(AssertionError, match="out must be"):
                    call(out, r)


@pytest.mark.parametrize("M,N,K", [(1, 96, 64), (5, 200, 128), (300, 768, 512), (2100, 1000, 256)])
def test_output_beside_the_residual(M, N, K):
    """Output and residual in two column ranges of one buffer; the row operators likewise."""
    for dtype in (torch.float16, torch.float32):
        x, w, idx = operands(M, N, K, dtype)
        buf = torch.randn(M, 2 * N + 3, device="cuda").to(dtype)
        keep = buf.clone()
        y = ghost_linear(x, w, idx, residual=buf[:, :N], out=buf[:, N + 2: 2 * N + 2])
        assert torch.equal(y, ghost_linear(x, w, idx, residual=keep[:, :N].contiguous()))
        keep[:, N + 2: 2 * N + 2] = y
        assert torch.equal(buf, keep)
        n, s = rms_norm(buf[:, :N], residual=keep[:, :N], residual_out=buf[:, N + 1: 2 * N + 1])
        assert torch.equal(s, keep[:, :N] + keep[:, :N]) and torch.equal(buf[:, :N], keep[:, :N])
        # Rounded once; the fp32 sum of N squares is off by at most N 2^-24 of itself (half of that in
        # its root's inverse), the root and the two products by a few 2^-24.
        want = 2 * keep[:, :N].double()
        want /= torch.sqrt((want * want).mean(1, keepdim=True) + 1e-6)
        assert bool(((n.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + (N / 2 + 16) * 2.0 ** -24)
                     * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M", [1, 7, 130, 700, 3000])
def test_output_in_the_operands_place(M, dtype):
    """x + x W'^T written over x (N = K), and over columns of it, equal the same call with an
    output of its own: no tile of x is read after it was overwritten."""
    K = 768
    x, _, _ = operands(M, K, K, dtype)
    w = (torch.randn(K, K, device="cuda") / 28).to(dtype)
    idx = torch.randperm(K, device="cuda")[: K // 2].sort().values
    wp = pack_weight(w, idx)
    count = torch.tensor([idx.numel()], dtype=torch.int32, device="cuda")
    calls = [lambda x, r, out, s=s: ghost_linear(x, wp, idx, residual=r, out=out, strategy=s)
             for s in (("auto",) if dtype is torch.float32 else ("auto", "fused", "overlap"))]
    calls += [lambda x, r, out: ghost_linear_dev(x, wp, idx, count, residual=r, out=out)]
    if dtype is not torch.float32:
        full = pack_weight(w, torch.arange(K, device="cuda"))
        calls += [lambda x, r, out: packed_linear(x, full, residual=r, out=out),
                  lambda x, r, out: ghost_linear(x, full, torch.arange(K, device="cuda"), residual=r, out=out, strategy="runs")]
    for call in calls:
        want = call(x, x, None)
        for _ in range(5):
            y = x.clone()
            assert call(y, y, y) is y and torch.equal(y, want)
            y = x.clone()
            assert torch.equal(call(y, None, y), call(x, None, None))
    if dtype is not torch.float32:
        half = pack_weight(w[:, : K // 2], torch.arange(K // 2, device="cuda"))[: 3 * K // 4]
        for _ in range(3):
            y = x.clone()                            # both operands strided, the output across them
            got = packed_linear(y[:, : K // 2], half, out=y[:, K // 4:])
            assert torch.equal(got, packed_linear(x[:, : K // 2], half))
            assert torch.equal(y[:, : K // 4], x[:, : K // 4])
    with pytest.raises(AssertionError, match="w_packed"):
        ghost_linear(x[:5], wp, idx, out=wp.as_strided((min(M, 5), K), (wp.stride(0) * 2, 1)))


def at_address(ptr, make):
    """A tensor that make() returns at the given address (the allocator hands freed blocks out again)."""
    others = []
    for _ in range(50):
        t = make()
        if t.data_ptr() == ptr:
            return t
        others.append(t)
    return None


@pytest.mark.parametrize("precision", ["input", "e4m3", "chain"])
@pytest.mark.parametrize("what", ["mask", "weight", "proj mask", "bias"])
def test_replaced_tensors_at_the_old_address(what, precision):
    """A mask, weight or bias that replaces another one at its address and version is seen."""
    D, F = 256, 512
    g = torch.Generator(device="cuda").manual_seed(3)
    m = block(D, F, torch.float16, 3, precision="input" if precision == "chain" else precision)
    if precision == "chain":
        m = GhostMLPChain(m.fc, m.proj, "gelu")
    x, _ = inputs(20, D, torch.float16, 3)
    layer = m.proj if what == "proj mask" else m.fc
    other = {"weight": torch.randn(F, D, generator=g, device="cuda").half() / 16,
             "bias": torch.randn(F, generator=g, device="cuda").half(),
             }.get(what, torch.randperm(layer.in_features, generator=g, device="cuda")[: layer.in_features // 2].sort().values)
    with torch.no_grad():
        if what in ("weight", "bias"):
            setattr(m.fc, what, nn.Parameter(torch.randn_like(other), requires_grad=False))
        else:
            layer._set_frozen(other.flip(0).clone())
        m(x)
        torch.cuda.synchronize()
        old = m.fc.weight if what == "weight" else m.fc.bias if what == "bias" else layer._frozen_indices
        ptr, version = old.data_ptr(), old._version
        del old
        if what in ("weight", "bias"):
            setattr(m.fc, what, None)
            new = at_address(ptr, other.clone)
            setattr(m.fc, what, nn.Parameter(other.clone() if new is None else new, requires_grad=False))
            assert new is None or getattr(m.fc, what)._version == version
        else:
            layer.unfreeze_mask()
            new = at_address(ptr, other.clone)
            layer._set_frozen(other.clone() if new is None else new)
        y = m(x)
        m.refresh_packed()
        assert torch.equal(y, m(x))


@pytest.mark.parametrize("updated", [False, True])
@pytest.mark.parametrize("kind", ["input", "e4m3", "chain", "layer"])
def test_captured_first(kind, updated):
    """A capture that has to pack the weights (the first call, or the first one after an update)
    leaves nothing behind that an eager call before the first replay would take as packed."""
    D, F = 512, 1024
    m = block(D, F, torch.float16, 11, precision="e4m3" if kind == "e4m3" else "input")
    if kind == "chain":
        m = GhostMLPChain(m.fc, m.proj, "gelu")
    elif kind == "layer":
        m = m.fc
    fresh = block(D, F, torch.float16, 11, precision="e4m3" if kind == "e4m3" else "input")
    if kind in ("chain", "layer"):
        fresh = GhostMLPChain(fresh.fc, fresh.proj, "gelu") if kind == "chain" else fresh.fc
    x, _ = inputs(40, D, torch.float16, 11)
    weight = m.weight if kind == "layer" else m.proj.weight
    with torch.no_grad():
        if updated:
            m(x)
            for mod in (weight, fresh.weight if kind == "layer" else fresh.proj.weight):
                mod.mul_(-0.5)
        want = fresh(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        assert torch.equal(m(x), want)               # before any replay
        graph.replay()
        assert torch.equal(y, want) and torch.equal(m(x), want)
        x2, _ = inputs(40, D, torch.float16, 12)
        x.copy_(x2)
        graph.replay()
        assert torch.equal(y, fresh(x2))
        del graph
        assert torch.equal(m(x), fresh(x2))


def chain_or_block(kind, D, F, seed):
    m = block(D, F, torch.float16, seed, precision="e4m3" if kind == "e4m3" else "input")
    return GhostMLPChain(m.fc, m.proj, "gelu") if kind == "chain" else m


@pytest.mark.parametrize("kind", ["input", "e4m3", "chain"])
def test_first_use_on_two_streams(kind):
    """The operands are packed on one stream, behind other work, and used at once on a second one."""
    D, F = 512, 1024
    want = chain_or_block(kind, D, F, 21)
    x, _ = inputs(40, D, torch.float16, 21)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        want = want(x)
        for _ in range(3):
            m = chain_or_block(kind, D, F, 21)
            torch.cuda.synchronize()
            with torch.cuda.stream(a):
                torch.cuda._sleep(100_000_000)       # some 50 ms
                first = m(x)
            with torch.cuda.stream(b):
                second = m(x)
            torch.cuda.synchronize()
            assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.parametrize("kind", ["input", "e4m3", "chain"])
def test_replaced_while_another_stream_uses_them(kind):
    """Operands replaced (and their memory handed out again) on the stream that packed them,
    while a call on another stream still has to read them."""
    D, F = 512, 1024
    m = chain_or_block(kind, D, F, 22)
    x, _ = inputs(40, D, torch.float16, 22)
    b = torch.cuda.Stream()
    with torch.no_grad():
        want = m(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(b):
            torch.cuda._sleep(100_000_000)
            y = m(x)
        m.refresh_packed()
        rubbish = [torch.full((n,), 77, dtype=torch.uint8, device="cuda") for n in range(256 * 512, 2 << 20, 64 << 10)]
        m(x)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and len(rubbish)


@pytest.mark.parametrize("kind", ["input", "e4m3", "chain"])
def test_copies_pack_their_own_operands(kind):
    m = chain_or_block(kind, 256, 512, 23)
    x, _ = inputs(5, 256, torch.float16, 23)
    with torch.no_grad():
        want = m(x)
        twin = copy.deepcopy(m)
        buf = io.BytesIO()
        torch.save(m, buf)
        buf.seek(0)
        loaded = torch.load(buf, weights_only=False)
        m.proj.weight.zero_()
        for other in (twin, loaded):
            assert torch.equal(other(x), want)


@pytest.mark.parametrize("parameters", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 40, 700])
def test_e4m3_weights_are_rounded_once(M, parameters):
    """The block's e4m3 weights are the parameters' own, not those of their copy in the input's type."""
    D, F, dtype = 256, 600, torch.bfloat16
    m = block(D, F, parameters, 25, precision="e4m3")
    x, r = inputs(M, D, dtype, 25)
    a1, a2 = m.fc._frozen_indices, m.proj._frozen_indices
    with torch.no_grad():
        q, sc, s = rms_norm_q8(x, m.norm.weight, 1e-5, residual=r, alive_indices=a1)
        h = packed_linear_q8(q, sc, *pack_weight_q8(m.fc.weight[a2], a1), bias=m.fc.bias[a2], activation="gelu_tanh", dtype=dtype)
        h = torch.cat([h, h.new_zeros(M, -a2.numel() % 64)], 1)      # as the block pads them
        hq, hs = quantize_rows(h)
        want = packed_linear_q8(hq[:, : a2.numel()], hs, *pack_weight_q8(m.proj.weight, a2), bias=m.proj.bias, residual=s)
        assert torch.equal(m(x, residual=r), want)
    # Nothing but e4m3 weights, scales and the bias is kept: a byte a weight, rows padded to 128.
    padded = lambda n, to: (n + to - 1) // to * to
    weights = padded(a2.numel(), 64) * padded(a1.numel(), 128) + D * padded(a2.numel(), 128)
    assert sum(t.untyped_storage().nbytes() for t in m._plan.tensors) <= weights + 4 * (D + F) + 2 * F


@pytest.mark.parametrize("precision", ["input", "e4m3"])
@pytest.mark.parametrize("empty", ["fc", "proj", "both"])
def test_masks_that_leave_nothing(empty, precision):
    """fc without a live column gives act(b1) for every row, proj without one leaves s + b2."""
    D, F, dtype = 128, 256, torch.float16
    m = block(D, F, dtype, 26, precision=precision)
    with torch.no_grad():
        for layer, name in ((m.fc, "fc"), (m.proj, "proj")):
            if empty in (name, "both"):
                layer.weight.zero_()
                layer.freeze_weight_mask()
                assert layer._frozen_indices.numel() == 0
        for M in (1, 50, 400):
            x, r = inputs(M, D, dtype, M)
            y = m(x, residual=r)
            if empty == "fc" and precision == "e4m3":
                s, want, *_ = exact(m, x, r, 1e-5)
                branch = want - s                    # two roundings to e4m3: see test_gpu_prenorm
                assert ((y.double() - want).norm() / branch.norm()).item() < 2 / 16
            else:
                check_block(y, m, x, r, 1e-5)


def test_operands_refused():
    """Weights narrower than the product, of another type or device or in overlapping rows, and
    biases that do not hold N values: refused by every 16-bit product before a launch."""
    M, N, K = 8, 48, 64
    x, w, idx = operands(M, N, K)
    count = torch.tensor([K], dtype=torch.int32, device="cuda")
    out = torch.empty(M, N, dtype=x.dtype, device="cuda")
    calls = [lambda w, b: ghost_linear(x, w, idx, bias=b), lambda w, b: ghost_linear_dev(x, w, idx, count, bias=b),
             lambda w, b: packed_linear(x, w, bias=b), lambda w, b: ghost_linear_pipelined([(x, w, idx, out, b)])]
    for bad, b in weights_and_biases_refused(N, K, x.dtype):
        bad = bad.cuda() if bad.stride(0) >= bad.shape[1] and bad.stride(1) == 1 else torch.zeros_like(w).set_(
            torch.zeros(N * K, dtype=bad.dtype, device="cuda").untyped_storage(), 0, bad.shape, bad.stride())
        b = None if b is None else b.cuda() if b.is_contiguous() else torch.zeros(2 * N, dtype=b.dtype, device="cuda")[::2]
        for i, call in enumerate(calls):
            if bad.shape[0] == N or i < 3:
                with pytest.raises(AssertionError, match="must"):
                    call(bad, b)
    for call in calls:
        for bad, b in ((w.cpu(), None), (w, torch.zeros(N, dtype=x.dtype))):
            with pytest.raises(AssertionError, match="must"):
                call(bad, b)
    with pytest.raises(AssertionError, match="alive_indices"):
        ghost_linear(x, w, idx.cpu())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 3, 17, 300, 2100])
def test_packed_linear_takes_any_rows(M, dtype):
    """Rows that TMA cannot load (odd widths, odd offsets, columns of adjacent elements) are copied."""
    for K in (1, 7, 333, 512):
        g = torch.Generator(device="cuda").manual_seed(M + K)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
        N, big = 300, rnd(M + 2, K + 13)
        w, b, r = rnd(N, K) / max(K, 1) ** 0.5, rnd(N), rnd(M, N)
        wp = pack_weight(w, torch.arange(K, device="cuda"))
        flat = rnd(M * K + 1)
        for a in (rnd(M, K), flat[1:].view(M, K), big[1: M + 1, 3: K + 3], big[:M, 8: K + 8], rnd(K, M).t(),
                  rnd(1, K).expand(M, K), rnd(M, 2 * K)[:, ::2], rnd(2 * M, K)[::2]):
            keep = a.clone()
            check(packed_linear(a, wp, bias=b, activation="gelu", residual=r), a, w, b, "gelu", r)
            assert torch.equal(a, keep)
    # What rms_norm writes without a list: rows of the width itself.
    x, weight = rnd(M, 333), rnd(333)
    w = rnd(64, 333) / 18
    n = rms_norm(x, weight)
    check(packed_linear(n, pack_weight(w, torch.arange(333, device="cuda"))), n, w, None, None, None)


@pytest.mark.parametrize("K", [4096, 4100, 4104])
def test_one_row_of_a_padded_buffer(K):
    """A row that torch calls contiguous at whatever stride, over 64-column runs; the layer likewise."""
    g = torch.Generator(device="cuda").manual_seed(K)
    N, dt = 256, torch.bfloat16
    runs = torch.randperm(64, generator=g, device="cuda")[:32].sort().values
    idx = (runs[:, None] * 64 + torch.arange(64, device="cuda")).reshape(-1)
    w = (torch.randn(N, K, generator=g, device="cuda") / 64).to(dt)
    wp = pack_weight(w, idx)
    layer = GhostLinear(K, N, bias=False, device="cuda", dtype=dt)
    with torch.no_grad():
        layer.weight.copy_(w)
        layer._set_frozen(idx)
    for ld in (K, 4104, 4106, 4160):
        big = torch.randn(2, ld, generator=g, device="cuda").to(dt)
        r = torch.randn(1, N, generator=g, device="cuda").to(dt)
        for x in (big[0:1, :K], big.view(-1)[:K].as_strided((1, K), (1, 1))):
            assert x.is_contiguous()
            check(ghost_linear(x, wp, idx, strategy="runs", residual=r), x[:, idx], w[:, idx], None, None, r)
            with torch.no_grad():
                for _ in range(2):
                    check(layer(x, residual=r), x[:, idx], w[:, idx], None, None, r)


def test_norms_told_by_what_they_compute():
    """A norm that multiplies by 1 + weight is refused; one built on the meta device is tried in the first forward."""
    m = block(128, 256, torch.float16, 30)
    with pytest.raises(AssertionError, match="norm must"):
        GhostPreNormMLP(OnePlusWeight(128).cuda(), m.fc, m.proj, "gelu")
    x, r = inputs(4, 128, torch.float16, 30)
    with torch.no_grad():
        for norm, good in ((nn.RMSNorm(128, eps=1e-5, device="meta"), True), (OnePlusWeight(128).to("meta"), False)):
            late = GhostPreNormMLP(norm, m.fc, m.proj, m.activation)
            late.norm.to_empty(device="cuda")
            late.norm.weight.copy_(m.norm.weight)
            if good:
                assert torch.equal(late(x, residual=r), m(x, residual=r))
            else:
                with pytest.raises(AssertionError, match="norm must"):
                    late(x, residual=r)


def writers(M, N, K, g):
    """name -> call that writes an [M, N] fp16 tensor that it is given."""
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
    x, w, idx = rnd(M, K), rnd(N, K) / 16, torch.arange(K, device="cuda")
    wp = pack_weight(w, idx)
    count = torch.tensor([K], dtype=torch.int32, device="cuda")
    qa, qw, s = quantize_rows(x), quantize_rows(w), rnd(M, N)
    return {"ghost_linear": lambda out: ghost_linear(x, wp, idx, out=out),
            "ghost_linear_dev": lambda out: ghost_linear_dev(x, wp, idx, count, out=out),
            "packed_linear": lambda out: packed_linear(x, wp, residual=s, out=out),
            "packed_linear_q8": lambda out: packed_linear_q8(*qa, *qw, out=out),
            "pipelined": lambda out: ghost_linear_pipelined([(x, wp, idx, out)]),
            "rms_norm": lambda out: rms_norm(s, residual=s, residual_out=out),
            "rms_norm_q8": lambda out: rms_norm_q8(s, residual=s, residual_out=out)}


@pytest.mark.parametrize("name", ["ghost_linear", "ghost_linear_dev", "packed_linear", "packed_linear_q8", "pipelined",
                                  "rms_norm", "rms_norm_q8"])
def test_writes_into_given_tensors_are_seen(name):
    """By the caches of packed weights, by autograd, and under inference mode, where nothing is counted."""
    g = torch.Generator(device="cuda").manual_seed(40)
    M, N, K = 64, 256, 128
    write = writers(M, N, K, g)[name]
    buf = torch.randn(M, N, generator=g, device="cuda").half()
    act = torch.randn(9, M, generator=g, device="cuda").half()
    alive = torch.arange(M, device="cuda")
    with torch.no_grad():
        ghostweight_matmul(act, buf, alive)          # buf as a weight: its packed form is kept
        write(buf)
        assert torch.equal(ghostweight_matmul(act, buf, alive), ghostweight_matmul(act, buf.clone(), alive))
    p = torch.randn(M, N, generator=g, device="cuda").half().requires_grad_()
    z = (buf * p).sum()                              # keeps buf for the gradient of p
    write(buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    leaf = buf.clone().requires_grad_()
    before = leaf.detach().clone()
    with pytest.raises(RuntimeError, match="no backward"):
        write(leaf)
    assert torch.equal(leaf, before)
    with torch.no_grad():
        write(leaf)
    with torch.inference_mode():
        inner = torch.empty(M, N, dtype=torch.float16, device="cuda")
        write(inner)
        assert torch.equal(inner, leaf)


def test_precision_and_type_change_between_calls():
    """A block whose precision or input type changes packs what that form needs."""
    m = block(128, 256, torch.float16, 41)
    forms = [("input", torch.float16), ("e4m3", torch.float16), ("e4m3", torch.bfloat16), ("input", torch.bfloat16)]
    want = {}
    with torch.no_grad():
        for precision, dtype in forms:
            twin = copy.deepcopy(m)
            twin.precision = precision
            want[precision, dtype] = twin(*inputs(9, 128, dtype, 41))
        for precision, dtype in forms + forms[::-1] + forms[::2]:
            m.precision = precision
            assert torch.equal(m(*inputs(9, 128, dtype, 41)), want[precision, dtype])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N", [(1, 1214), (20, 1526), (300, 1001), (1600, 2878), (2056, 1214), (2100, 4093), (4097, 767)])
def test_nothing_is_written_beside_the_output(M, N, dtype):
    """Outputs in aligned rows with a gap behind them: the gap keeps its values, where a row ends
    inside a 16-byte unit too."""
    K = 130
    x, w, idx = operands(M, N, K, dtype)
    res = torch.randn(M, N, device="cuda").to(dtype)
    qa, qw = quantize_rows(x), quantize_rows(w)
    calls = [lambda r, out: ghost_linear(x, w, idx, residual=r, out=out),
             lambda r, out: ghost_linear_dev(x, pack_weight(w, idx).as_strided((N, 192), (192, 1)), idx,
                                             torch.tensor([K], dtype=torch.int32, device="cuda"), residual=r, out=out)]
    if dtype is not torch.float32:
        calls += [lambda r, out, s=s: ghost_linear(x, w, idx, residual=r, out=out, strategy=s) for s in ("fused", "overlap")]
        calls += [lambda r, out: packed_linear(x, w, residual=r, out=out),
                  lambda r, out: packed_linear_q8(*qa, *qw, residual=r, dtype=dtype, out=out)]
    ld = (N + 7) // 8 * 8
    for call in calls:
        for pad in (0, 8) if ld > N else (8,):
            for r in (None, res, "in place"):
                buf = torch.full((M + 1, ld + pad), 5.0, dtype=dtype, device="cuda")
                out = buf[:M, :N]
                if r == "in place":
                    out.copy_(res)
                want = call(res if r == "in place" else r, None)
                call(out if r == "in place" else r, out)
                assert torch.equal(out, want)
                assert bool((buf[:, N:] == 5).all()) and bool((buf[M] == 5).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N", [(1, 300), (20, 1526), (300, 1001), (700, 4096), (1600, 2880), (2056, 1214)])
def test_nothing_behind_the_operands_columns_counts(M, N, dtype):
    """NaN behind the last column of both operands, inside the same 16-byte unit and behind it, and in
    the workspace that the gathered columns of x pass through."""
    for K in (1, 63, 130, 333):
        ld = (K + 7) // 8 * 8 + 8
        a = torch.full((M, ld), float("nan"), dtype=dtype, device="cuda")[:, :K]
        w = torch.full((N, ld), float("nan"), dtype=dtype, device="cuda")[:, :K]
        a.copy_(torch.randn(M, K, device="cuda"))
        w.copy_(torch.randn(N, K, device="cuda") / K ** 0.5)
        check(packed_linear(a, w), a, w, None, None, None)
        idx = torch.arange(K, device="cuda")
        for strategy in ("pregather", "overlap", "fused", "auto"):
            for ws in _native._gemm_ws.values():
                ws[4096:].fill_(0xFF)                # behind the header: NaN in both types
            x = a.contiguous()
            check(ghost_linear(x, w, idx, strategy=strategy), a, w, None, None, None)


def test_a_replaced_norm_is_tried():
    m = block(128, 256, torch.float16, 31)
    keys = set(m.state_dict())
    x, r = inputs(4, 128, torch.float16, 31)
    with torch.no_grad():
        m(x, residual=r)
        norm = m.norm
        m.norm = OnePlusWeight(128).cuda()
        with pytest.raises(AssertionError, match="norm must"):
            m(x, residual=r)
        m.norm = nn.RMSNorm(128, eps=1e-3, device="cuda", dtype=torch.float16)
        check_block(m(x, residual=r), m, x, r, 1e-3)
        m.norm = norm
        for other in (m, copy.deepcopy(m)):
            check_block(other(x, residual=r), m, x, r, 1e-5)
            assert set(other.state_dict()) == keys


@pytest.mark.parametrize("M,N", [(300, 1214), (2056, 1214), (2056, 1216), (2100, 4093)])
def test_peer_copies_end_with_the_row(M, N):
    """The output and its copies in other buffers (here on the same GPU), rows that end inside a
    16-byte unit included: nothing behind them is written in any."""
    K = 130
    x, w, idx = operands(M, N, K)
    ld = (N + 7) // 8 * 8 + 8
    bufs = [torch.full((M, ld), 5.0, dtype=x.dtype, device="cuda") for _ in range(3)]
    want = ghost_linear(x, w, idx)
    _native.gather_gemm_peers(x, w, idx, bufs[0][:, :N], [b.data_ptr() for b in bufs[1:]], strategy="pregather")
    for b in bufs:
        assert torch.equal(b[:, :N], want) and bool((b[:, N:] == 5).all())


@pytest.mark.parametrize("bias_type", [torch.float16, torch.float32])
@pytest.mark.parametrize("M", [2, 40, 600])
def test_layer_used_at_once_on_two_streams(M, bias_type):
    """A frozen layer's packed weight (and its bias in x's type), made on one stream behind other work
    and used at once on a second one; the next calls alternate."""
    K, N, dt = 512, 768, torch.float16
    g = torch.Generator(device="cuda").manual_seed(M)
    x, r = torch.randn(M, K, generator=g, device="cuda").to(dt), torch.randn(M, N, generator=g, device="cuda").to(dt)
    w = torch.randn(N, K, generator=g, device="cuda") / 16
    w[:, torch.randperm(K, generator=g, device="cuda")[: K // 2]] = 0
    b = torch.randn(N, generator=g, device="cuda")

    def layer():
        m = GhostLinear(K, N, threshold=0.0, device="cuda", dtype=bias_type)
        m.weight.copy_(w)
        m.bias.copy_(b)
        m.freeze_weight_mask()
        return m

    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        want = layer()(x, residual=r)
        for _ in range(3):
            m = layer()
            torch.cuda.synchronize()
            got = []
            with torch.cuda.stream(a):
                torch.cuda._sleep(100_000_000)       # some 50 ms
                got.append(m(x, residual=r))
            with torch.cuda.stream(c):
                got.append(m(x, residual=r))
            for s in (a, c, a, c):
                with torch.cuda.stream(s):
                    got.append(m(x, residual=r))
            torch.cuda.synchronize()
            assert all(torch.equal(y, want) for y in got)
        # Copies pack anew, and a captured call uses what is kept.
        twin = copy.deepcopy(m)
        m.weight.zero_()
        assert torch.equal(twin(x, residual=r), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = twin(x, residual=r)
        graph.replay()
        assert torch.equal(y, want)


@pytest.mark.parametrize("M", [2, 40, 600])
def test_cached_weight_used_at_once_on_two_streams(M):
    """ghostweight_matmul's packed weight, made on one stream behind other work and used at once on a second."""
    K, N, dt = 512, 768, torch.float16
    g = torch.Generator(device="cuda").manual_seed(M)
    x, w = torch.randn(M, K, generator=g, device="cuda").to(dt), torch.randn(K, N, generator=g, device="cuda").to(dt)
    idx = torch.arange(0, K, 2, device="cuda")
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        want = ghostweight_matmul(x, w.clone(), idx)
        for _ in range(3):
            fresh = w.clone()
            torch.cuda.synchronize()
            got = []
            with torch.cuda.stream(a):
                torch.cuda._sleep(100_000_000)       # some 50 ms
                got.append(ghostweight_matmul(x, fresh, idx))
            for s in (c, a, c):
                with torch.cuda.stream(s):
                    got.append(ghostweight_matmul(x, fresh, idx))
            torch.cuda.synchronize()
            assert all(torch.equal(y, want) for y in got)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("M", [1, 16])
def test_decode_products_over_cold_weights(M, q8):
    """Up to 16 rows with more k-blocks per CTA than the ring has stages, back to back over weights that
    lie in HBM (their loads land in any order): the same bits in every round, and the formula's values."""
    N, K, dt = 4096, 4096, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(M)
    x, r = torch.randn(M, K, generator=g, device="cuda").to(dt), torch.randn(M, N, generator=g, device="cuda").to(dt)
    ws = [(torch.randn(N, K, generator=g, device="cuda") / 64).to(dt) for _ in range(12)]      # 400 MB
    if q8:
        a, packed = quantize_rows(x), [quantize_rows(w) for w in ws]
        call = lambda i: packed_linear_q8(*a, *packed[i], residual=r)
    else:
        call = lambda i: packed_linear(x, ws[i], residual=r)
    first = [call(i) for i in range(len(ws))]
    rounds = [[call(i) for i in range(len(ws))] for _ in range(20)]
    for i, y in enumerate(first):
        assert all(torch.equal(y, later[i]) for later in rounds)
        if not q8:
            check(y, x, ws[i], None, None, r)
