"""Cases of the pre-norm operators around the column-sparse linear layers.

A pre-norm MLP block of a pruned model is a chain of four operators: the residual addition with the root-mean-square
norm, written out over the next layer's alive columns only (``rms_norm``, ``rms_norm_q8``); the rounding of rows to
e4m3 with one scale each, for the weights once and for the hidden activations every pass (``quantize_rows``); and
the matrix product over the alive columns with the bias, the activation and the residual's addition in its epilogue,
from 16/32-bit operands (``ghost_linear``) and from e4m3 operands with scales (``packed_linear_q8``).

``listed()`` holds the cases, ``draw()`` draws more of the same ranges, ``prepare()`` makes a case's inputs,
``run()`` makes one pass (the plain form in 32 bits, or the package's operators where ``own`` is true), ``exact()``
gives the definition's values in 64 bits and ``work()`` the bytes and operations a pass cannot do without.
"""

import math

import torch

own = False

if torch.cuda.is_available():
    DEVICE = torch.device("cuda")
else:
    DEVICE = torch.device("cpu")

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def _norm(name, M, K, dtype, residual, pattern, dead):
    return {"name": name, "op": "norm", "M": M, "K": K, "dtype": dtype, "residual": residual, "pattern": pattern,
            "dead": dead}


def _q8(name, M, K, dtype, norm, residual, pattern, dead):
    return {"name": name, "op": "q8", "M": M, "K": K, "dtype": dtype, "norm": norm, "residual": residual,
            "pattern": pattern, "dead": dead}


def _linear(name, M, N, K, dtype, bias, activation, residual, pattern, dead):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "bias": bias,
            "activation": activation, "residual": residual, "pattern": pattern, "dead": dead}


def _linear_q8(name, M, N, K, dtype, bias, activation, residual):
    return {"name": name, "op": "linear_q8", "M": M, "N": N, "K": K, "dtype": dtype, "bias": bias,
            "activation": activation, "residual": residual}


def listed():
    return [
        # One token of one sequence: the norm in front of a decoding step's layer, latency alone.
        _norm("norm-token", 1, 4096, "bf16", True, "random", 0.5),
        # A prefill of 8 x 512 tokens at width 4096, half of the next layer's columns dead.
        _norm("norm-prefill", 4096, 4096, "fp16", True, "random", 0.5),
        # An odd width and row count in fp32, full output (the last norm of a model, in front of a dense head).
        _norm("norm-odd-fp32", 1000, 1111, "fp32", False, "none", 0.0),
        # The first norm of the e4m3 chain, for 16 sequences decoding at the width of the small GPT-2.
        _q8("q8-norm-decode", 16, 768, "fp16", True, True, "random", 0.5),
        # The same in a long prefill, with 70% of the columns dead in 128-column blocks.
        _q8("q8-norm-prefill", 8192, 8192, "bf16", True, True, "blocks", 0.7),
        # The hidden activations between the two products of the chain (odd rows, every column kept).
        _q8("q8-rows", 1537, 11008, "bf16", False, False, "none", 0.0),
        # One token through a projection with bias and residual: the weights are read once.
        _linear("linear-token", 1, 4096, 4096, "fp16", True, "none", True, "random", 0.5),
        # The second projection of an MLP over a prefill, with bias and residual.
        _linear("linear-prefill", 4096, 4096, 4096, "bf16", True, "none", True, "random", 0.5),
        # An fp32 attention output projection of the small GPT-2, batch 8 x 128 tokens, with the residual.
        _linear("linear-fp32", 1024, 768, 768, "fp32", True, "gelu", True, "random", 0.5),
        # Sixteen sequences decoding through an e4m3 projection: half the weight bytes.
        _linear_q8("q8-linear-decode", 16, 4096, 2048, "bf16", True, "none", True),
        # A few hundred rows (a small batch, odd sizes), with the GELU of an MLP's first projection.
        _linear_q8("q8-linear-batch", 517, 4104, 2043, "fp16", True, "gelu_tanh", False),
        # The large MLP projection: 8192 rows, 28672 features, 30% of 8192 input columns alive.
        _linear_q8("q8-linear-mlp", 8192, 28672, 2432, "bf16", True, "gelu_tanh", False),
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over the logarithm; a third of them multiples of 64, a third of 8."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    step = rng.choice([1, 8, 64])
    return max(lo, min(hi, int(round(v / step)) * step or step))


def draw(rng):
    op = rng.choice(["norm", "q8", "linear", "linear_q8"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    pattern = rng.choice(["none", "random", "random", "blocks"])
    dead = round(rng.uniform(0.05, 0.95), 3) if pattern != "none" else 0.0
    if op in ("norm", "q8"):
        M, K = _size(rng, 1, 16384), _size(rng, 48, 28672)
        while M * K > 8192 * 8192:
            M = max(1, M // 2)
        if pattern == "blocks":
            K = max(128, K // 128 * 128)
        if op == "norm":
            return _drawn(_norm("", M, K, dtype, rng.random() < 0.7, pattern, dead))
        norm = rng.random() < 0.6
        return _drawn(_q8("", M, K, dtype, norm, norm and rng.random() < 0.7, pattern, dead))
    M, N, K = _size(rng, 1, 8192), _size(rng, 32, 16384), _size(rng, 48, 16384)
    most = 8192 * 28672 * 2432 if op == "linear_q8" else 4096 * 8192 * 4096
    while M * N * K > most:
        M = max(1, M // 2)
    act = rng.choice(["none", "gelu", "gelu_tanh"])
    bias, residual = rng.random() < 0.7, rng.random() < 0.7
    if op == "linear_q8":
        return _drawn(_linear_q8("", M, N, K, rng.choice(["fp16", "bf16"]), bias, act, residual))
    if pattern == "none":
        pattern, dead = "random", 0.5
    if pattern == "blocks":
        K = max(128, K // 128 * 128)
    return _drawn(_linear("", M, N, K, dtype, bias, act, residual, pattern, dead))


def _drawn(case):
    del case["name"]
    return case


def _alive_count(case):
    K, pattern = case["K"], case.get("pattern", "none")
    if pattern == "none":
        return K
    unit = 128 if pattern == "blocks" else 1
    units = K // unit
    return max(1, units - int(round(case["dead"] * units))) * unit


# ------------------------------------------------------------------------------------------------ inputs
def _alive(case, gen):
    """The sorted alive columns: random single columns, or whole 128-column blocks."""
    K, n, pattern = case["K"], _alive_count(case), case.get("pattern", "none")
    if pattern == "none":
        return None
    unit = 128 if pattern == "blocks" else 1
    keep = torch.randperm(K // unit, generator=gen, device=DEVICE)[: n // unit].sort().values
    if unit == 1:
        return keep
    return (keep[:, None] * unit + torch.arange(unit, device=DEVICE)).reshape(-1)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _to_e4m3(v):
    """Rows of v as e4m3 in rows of a multiple of 128 bytes, zero behind the last column, and their scales."""
    rows, cols = v.shape
    scale = (v.abs().amax(dim=1) / E4M3_MAX).clamp_min(SCALE_MIN)
    buf = torch.zeros((rows, (cols + 127) // 128 * 128), dtype=torch.uint8, device=v.device)
    buf[:, :cols] = (v / scale[:, None]).to(E4M3).view(torch.uint8)
    return buf.view(E4M3)[:, :cols], scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    if case["op"] in ("norm", "q8"):
        dt, M, K = DTYPES[case["dtype"]], case["M"], case["K"]
        state["idx"] = _alive(case, gen)
        # Activations of a residual stream: a few channels are many times larger than the others.
        channel = torch.where(torch.rand(K, generator=gen, device=DEVICE) < 0.01, 20.0, 1.0)
        state["x"] = (_randn(gen, M, K) * channel).to(dt)
        state["weight"] = (1.0 + 0.1 * _randn(gen, K)).to(dt)
        state["residual"] = (2.0 * _randn(gen, M, K)).to(dt) if case["residual"] else None
        return state
    dt, M, N, K = DTYPES[case["dtype"]], case["M"], case["N"], case["K"]
    state["bias"] = (0.1 * _randn(gen, N)).to(dt) if case["bias"] else None
    state["residual"] = _randn(gen, M, N).to(dt) if case["residual"] else None
    if case["op"] == "linear":
        state["idx"] = _alive(case, gen)
        state["x"] = _randn(gen, M, K).to(dt)
        n = state["idx"].numel()
        # The packed weight a program keeps: the alive columns in rows of a multiple of 64 elements.
        buf = torch.zeros((N, (n + 63) // 64 * 64), dtype=dt, device=DEVICE)
        buf[:, :n] = _randn(gen, N, n).to(dt) / math.sqrt(n)
        state["w"] = buf[:, :n]
    else:
        state["a"], state["a_scale"] = _to_e4m3(_randn(gen, M, K))
        state["w"], state["w_scale"] = _to_e4m3(_randn(gen, N, K) / math.sqrt(K))
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _activate(v, activation):
    if activation == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if activation == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_rows(s, normed):
    """(y, s): the residual sum and its norm over the alive columns, in 32 bits."""
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h
    if normed:
        y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    return (y if s["idx"] is None else y[:, s["idx"]]), h


def _plain_product(s, a, w):
    y = a @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activate(y, s["case"]["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _plain(s):
    op = s["case"]["op"]
    if op == "norm":
        y, h = _plain_rows(s, True)
        dt = s["x"].dtype
        return (y.to(dt),) if s["residual"] is None else (y.to(dt), h.to(dt))
    if op == "q8":
        y, h = _plain_rows(s, s["case"]["norm"])
        scale = (y.abs().amax(dim=1) / E4M3_MAX).clamp_min(SCALE_MIN)
        q = (y / scale[:, None]).to(E4M3)
        return (q, scale) if s["residual"] is None else (q, scale, h.to(s["x"].dtype))
    if op == "linear":
        return _plain_product(s, s["x"][:, s["idx"]].float(), s["w"].float())
    return _plain_product(s, s["a"].float() * s["a_scale"][:, None], s["w"].float() * s["w_scale"][:, None])


def _kernels(s):
    from ghostweight_triton_b200.kernels.matmul import ghost_linear, packed_linear_q8
    from ghostweight_triton_b200.kernels.norm import quantize_rows, rms_norm, rms_norm_q8

    case = s["case"]
    if case["op"] == "norm":
        out = rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], alive_indices=s["idx"])
        return (out,) if s["residual"] is None else out
    if case["op"] == "q8":
        if case["norm"]:
            return rms_norm_q8(s["x"], s["weight"], EPS, residual=s["residual"], alive_indices=s["idx"])
        return quantize_rows(s["x"], alive_indices=s["idx"])
    activation = None if case["activation"] == "none" else case["activation"]
    if case["op"] == "linear":
        return ghost_linear(s["x"], s["w"], s["idx"], bias=s["bias"], activation=activation,
                            strategy="runs" if case["pattern"] == "blocks" else "auto", residual=s["residual"])
    return packed_linear_q8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], activation=activation,
                            residual=s["residual"], dtype=DTYPES[case["dtype"]])


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ the definition
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] in ("norm", "q8"):
        total = s["x"].to(f64)
        if s["residual"] is not None:
            total += s["residual"].to(f64)
        cols = slice(None) if s["idx"] is None else s["idx"]
        if case["op"] == "norm" or case["norm"]:
            power = torch.linalg.vector_norm(total, dim=1).square() / case["K"]
            out = total[:, cols] / torch.sqrt(power + EPS)[:, None] * s["weight"].to(f64)[cols]
        else:
            out = total[:, cols]
        rest = () if s["residual"] is None else (total,)
        if case["op"] == "norm":
            return (out, *rest)
        step = out.abs().max(dim=1).values / E4M3_MAX
        step = torch.where(step < SCALE_MIN, torch.full_like(step, SCALE_MIN), step)
        return ((out / step[:, None]).to(E4M3).to(f64), step, *rest)
    if case["op"] == "linear":
        v = torch.einsum("mk,nk->mn", s["x"].to(f64).index_select(1, s["idx"]), s["w"].to(f64))
    else:
        v = torch.einsum("mk,nk->mn", s["a"].to(f64), s["w"].to(f64))
        v *= torch.outer(s["a_scale"].to(f64), s["w_scale"].to(f64))
    if s["bias"] is not None:
        v += s["bias"].to(f64)
    if case["activation"] == "gelu":
        v = v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
    elif case["activation"] == "gelu_tanh":
        # 0.5 (1 + tanh(u)) is the logistic function of 2 u.
        v = v * torch.sigmoid(math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3))
    if s["residual"] is not None:
        v += s["residual"].to(f64)
    return v


# ------------------------------------------------------------------------------------------------ the work
def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
    M, K, n = case["M"], case["K"], _alive_count(case)
    listing = 8 * n if case.get("pattern", "none") != "none" else 0
    if case["op"] in ("norm", "q8"):
        normed = case["op"] == "norm" or case["norm"]
        # A plain rounding needs the alive columns only; the norm needs the whole row.
        read = (M * K + K) * size if normed else M * n * size
        stream = 2 * M * K * size if case["residual"] else 0
        write = M * n * size if case["op"] == "norm" else M * n + 4 * M
        return {"bytes": read + stream + write + listing, "flops": M * K * (5 if case["residual"] else 4)}
    N = case["N"]
    extra = (N * size if case["bias"] else 0) + (M * N * size if case["residual"] else 0) + M * N * size
    if case["op"] == "linear":
        return {"bytes": (M + N) * n * size + listing + extra, "flops": 2 * M * N * n}
    return {"bytes": (M + N) * (K + 4) + extra, "flops": 2 * M * N * K}
