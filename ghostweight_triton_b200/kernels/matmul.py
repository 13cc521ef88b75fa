"""Fused gather-GEMM on B200.

``ghostweight_matmul`` mirrors ghostweight_triton/kernels/matmul.py:85-142:
C[M, N] = A[:, alive] @ W[alive, :] with fp32 accumulation, cast to A's dtype;
unsorted or repeated indices are fine and an empty index list gives zeros.
On B200 the weight rows are first packed into the K'-major operand (one
transposing gather) and the product runs on the tcgen05 kernel K3
(csrc/gw_gemm_tc.cu). Two strategies feed its A operand: "pregather" gathers
the alive activation columns into a dense scratch matrix and streams both
operands by TMA (two launches; the default when a workspace is affordable),
"fused" has producer warps gather them straight into shared memory (one
launch, no scratch). fp32 inputs use the exact-fp32 kernel, matching the
reference's TF32-off choice for fp32 (matmul.py:127-130).

``ghost_linear`` is the module-level entry: activations [M, K] times an
already packed weight, with bias and optional GELU fused into the epilogue.
"""

from __future__ import annotations

import torch

from ghostweight_triton_b200 import _native
from ghostweight_triton_b200.kernels._args import Kept, in_place_or_apart, overlap, refuse_grad_out, residual_matrix, written
from ghostweight_triton_b200.kernels.gather import pack_weight


def ghostweight_matmul(
    activations: torch.Tensor,
    weights: torch.Tensor,
    alive_indices: torch.Tensor,
    BLOCK_M: int = 64,
    BLOCK_N: int = 64,
    BLOCK_K: int = 32,
    *,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    strategy: str = "auto",
) -> torch.Tensor:
    """Sparse matmul that skips dead neurons.

    Parameters
    ----------
    activations   : [M, K]
    weights       : [K, N]
    alive_indices : [K_alive], any integer dtype (converted to int64)
    BLOCK_M, BLOCK_N, BLOCK_K : accepted for signature compatibility; ignored.
    bias          : optional [N], added in the fp32 epilogue (extension).
    activation    : None, "gelu" or "gelu_tanh", applied after the bias (extension).
    strategy      : "auto" | "pregather" | "fused" | "overlap" | "runs" (extension, see
                    module docstring; "runs" needs an alive list of 64-column runs).

    Returns
    -------
    torch.Tensor [M, N], dtype of ``activations``, contiguous.
    """
    assert activations.ndim == 2 and weights.ndim == 2
    assert activations.is_cuda and weights.is_cuda
    M, K = activations.shape
    K_w, N = weights.shape
    assert K == K_w, f"K mismatch: A K={K}, W K={K_w}"

    if not activations.is_contiguous():
        activations = activations.contiguous()
    if not weights.is_contiguous():
        weights = weights.contiguous()
    if alive_indices.dtype != torch.int64 or alive_indices.device != activations.device:
        alive_indices = alive_indices.to(device=activations.device, dtype=torch.int64)
    if not alive_indices.is_contiguous():
        alive_indices = alive_indices.contiguous()
    if (bias is None and activation is None and strategy == "auto" and M and N
            and activations.get_device() == torch.cuda.current_device()):
        # The reference call without the extensions: the cached packed weight
        # comes with gw_gather_gemm's fixed arguments prepared.
        w_packed, prep = _packed_cache.get_prepared(weights, alive_indices, activations.dtype)
        C = activations.new_empty((M, N))
        if prep is not None:
            _native.gather_gemm_prepared(prep, activations, C)
        else:
            _gemm(activations, w_packed, alive_indices, C, None, None, "auto")
        return C
    C = torch.empty((M, N), dtype=activations.dtype, device=activations.device)
    if M == 0 or N == 0:
        return C
    w_packed = _packed_cache.get(weights, alive_indices, activations.dtype)
    if bias is not None and (bias.dtype != activations.dtype or not bias.is_contiguous()):
        bias = bias.contiguous().to(dtype=activations.dtype)
    _gemm(activations, w_packed, alive_indices, C, bias, activation, strategy)
    return C


class _PackedCache:
    """Packed weights of recent ghostweight_matmul calls.

    The reference API passes the weight [K, N] and the alive list on every
    call, and a loop over layers passes the same tensors again and again; the
    packing (a transposing gather of W[alive, :]) is then done once. An entry
    is used only for the very same tensor objects (held by weak reference, so
    an entry never outlives its weight) at the same in-place version counts
    (any in-place update of either tensor, or of a view sharing their storage,
    changes them), on the same storage (``w.data = ...`` keeps the object and
    its version) and for the same output dtype. Writes through ``w.data``
    change neither, so they need :func:`clear_packed_cache`. Small LRU: at
    most `max_entries` entries and `max_bytes` of packed data.
    """

    def __init__(self, max_entries: int = 32, max_bytes: int = 2 << 30):
        import collections
        import weakref

        self._weakref = weakref
        self._entries: "collections.OrderedDict" = collections.OrderedDict()
        self.max_entries = max_entries
        self.max_bytes = max_bytes
        self.bytes = 0

    def get(self, weights: torch.Tensor, idx: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        return self.get_prepared(weights, idx, dtype, prepare=False)[0]

    def get_prepared(self, weights: torch.Tensor, idx: torch.Tensor, dtype: torch.dtype,
                     prepare: bool = True) -> tuple:
        """(packed weight, the fixed gw_gather_gemm arguments for it without bias,
        activation or strategy choice, or None when the entry is not kept)."""
        key = (id(weights), id(idx), dtype)
        e = self._entries.get(key)
        if e is not None:
            w_ref, i_ref, w_ver, i_ver, packed, prep, ptrs, kept = e
            if (w_ref() is weights and i_ref() is idx and w_ver == weights._version
                    and i_ver == idx._version and ptrs == (weights.data_ptr(), idx.data_ptr())
                    and not _native._capturing()):
                if _native.current_raw_stream(weights.get_device()) not in kept.streams:
                    kept.on_this_stream()
                self._entries.move_to_end(key)
                if prep is None and prepare:
                    prep = e[5] = _native.prepare_gather_gemm(packed, idx, None, None, "auto", dtype)
                return packed, prep
            self._drop(key)
        packed = pack_weight(weights.t(), idx, dtype=dtype)
        if torch.cuda.is_current_stream_capturing():
            return packed, None     # a graph's private pool: do not keep it
        nbytes = packed.untyped_storage().nbytes()
        if nbytes > self.max_bytes:
            return packed, None
        cb = lambda _ref, key=key: self._drop(key)
        prep = _native.prepare_gather_gemm(packed, idx, None, None, "auto", dtype) if prepare else None
        self._entries[key] = [self._weakref.ref(weights, cb), self._weakref.ref(idx, cb),
                              weights._version, idx._version, packed, prep,
                              (weights.data_ptr(), idx.data_ptr()), Kept([packed])]
        self.bytes += nbytes
        while len(self._entries) > self.max_entries or self.bytes > self.max_bytes:
            self._drop(next(iter(self._entries)))
        if key not in self._entries:
            return packed, None
        return packed, prep

    def _drop(self, key) -> None:
        e = self._entries.pop(key, None)
        if e is not None:
            self.bytes -= e[4].untyped_storage().nbytes()

    def clear(self) -> None:
        self._entries.clear()
        self.bytes = 0


_packed_cache = _PackedCache()


def clear_packed_cache() -> None:
    """Forget every packed weight ghostweight_matmul keeps.

    An entry is rebuilt by itself when the weight or the index list is
    replaced, rebound to other storage (``w.data = ...``) or updated in place
    through autograd-visible operations (optimizer steps, ``copy_`` under
    ``no_grad``), which bump the tensor's version counter. In-place writes
    through ``w.data`` bypass that counter; call this after them.
    """
    _packed_cache.clear()


def _gemm(x, w_packed, idx, y, bias, activation, strategy, residual=None, shapes=None):
    """gw_gather_gemm_residual for a contiguous x; y is row-major. shapes: x's and w_packed's."""
    dtype = x.dtype
    (M, K), (N, wk) = shapes or (x.shape, w_packed.shape)
    ldx = K
    if strategy == "runs":
        ldx = max(x.stride(0), K)  # a contiguous x of one row may have any stride
        if x.data_ptr() % 16 or ldx % 8:
            strategy = "auto"      # direct TMA of x needs 16-byte aligned rows
    ldw, uw = w_packed.stride()
    ldy, uy = y.stride()
    n = idx.numel()
    assert idx.dtype is torch.int64 and idx.is_contiguous() and idx.is_cuda, "alive_indices must be contiguous int64 on x's device"
    # _operands_ok for what is usually given; this function is most of a small call's time.
    if not (w_packed.dtype is dtype and w_packed.is_cuda and wk >= n and uw == 1 and ldw >= wk
            and (bias is None or (bias.dtype is dtype and bias.numel() == N and bias.is_cuda and bias.is_contiguous()))):
        ldw = _operands_ok(w_packed, n, bias, dtype, x.get_device())
    if (uy != 1 and N > 1) or dtype not in _native.DTYPE_CODES:
        _native.dtype_code(dtype)                # raises
        _native._rowmajor(y)
    ws_ptr, ws_bytes = None, 0
    if strategy != "fused" and strategy != "runs" and dtype is not torch.float32:
        nbytes = _native.gather_gemm_workspace_bytes(M, n, dtype)
        if nbytes:
            ws = _native.gemm_workspace(x.device, nbytes)
            ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
    r_ptr, ldr = (None, 0) if residual is None else (residual.data_ptr(), residual.stride()[0])
    st = _native._call((_native._api or _native.api()).gw_gather_gemm_residual,
                       (x.data_ptr(), _native.DTYPE_CODES[dtype], M, K, ldx, w_packed.data_ptr(), N, ldw if ldw > n else n,
                        idx.data_ptr(), n, None if bias is None else bias.data_ptr(), _native.epilogue_code(activation),
                        r_ptr, ldr if ldr > N else N, y.data_ptr(), ldy if ldy > N else N, _native.GEMM_STRATEGIES[strategy],
                        ws_ptr, ws_bytes), x.get_device())
    if st:
        _native._check(st, "gw_gather_gemm")


def _operands_ok(w_packed, n, bias, dtype, dev) -> int:
    """The leading dimension of a packed weight [N, n or more] of this type on CUDA device
    `dev`, in row-major rows of their own; asserts this, and that a bias holds N values."""
    N, cols = w_packed.shape
    ld, unit = w_packed.stride()
    assert (w_packed.dtype is dtype and w_packed.get_device() == dev and cols >= n
            and (unit == 1 or cols <= 1) and (ld >= cols or N <= 1)), (
        f"w_packed must be a row-major {dtype} matrix with {n} columns on the activations' device, got "
        f"{w_packed.dtype} {tuple(w_packed.shape)} with strides {w_packed.stride()} on {w_packed.device}")
    if bias is not None:
        assert bias.dtype is dtype and bias.numel() == N and bias.is_contiguous() and bias.get_device() == dev, (
            f"bias must hold {N} contiguous values of {dtype} on the activations' device, got {bias.dtype} "
            f"{tuple(bias.shape)} on {bias.device}")
    return ld if ld > n else n


def index_runs(alive_indices: torch.Tensor, K: int) -> int:
    """Entries of the alive list that keep it from being 64-column runs (0: strategy
    "runs" applies). One device pass and one host synchronisation."""
    return _native.index_runs(alive_indices, K)


def ghost_linear(
    x: torch.Tensor,
    w_packed: torch.Tensor,
    alive_indices: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    out: torch.Tensor | None = None,
    strategy: str = "auto",
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """y = act(x[:, alive] @ w_packed^T + bias) + residual for x [M, K], w_packed [N, K_alive].

    residual [M, N] (x's dtype, rows may be strided) is added in the epilogue,
    in fp32, before the one rounding; ``out`` may be the residual itself. An
    ``out`` that shares memory with x is allowed: x is copied first, since
    tiles of y are written while others still read x.
    """
    assert x.ndim == 2 and x.is_cuda
    if not x.is_contiguous():
        x = x.contiguous()
    shapes = x.shape, w_packed.shape
    M, N = shapes[0][0], shapes[1][0]
    if out is None:
        y = x.new_empty((M, N))
        if residual is not None:
            residual = residual_matrix(residual, (M, N), x)
    else:
        y, residual = _product_out(out, residual, M, N, x)
        x = _apart_from(y, x, w_packed)
    if M and N:
        _gemm(x, w_packed, alive_indices, y, bias, activation, strategy, residual, shapes)
        if out is not None:
            written(out)
    return y


def _product_out(out, residual, M, N, like):
    """(output [M, N], residual as a row-major matrix or None) of a product of `like`'s type
    and device. A given output has that shape, in row-major rows of their own. The output is
    computed through the residual's rows, so it is these rows or lies apart from them."""
    given = residual
    if residual is not None:
        residual = residual_matrix(residual, (M, N), like)
    if out is None:
        return torch.empty((M, N), dtype=like.dtype, device=like.device), residual
    assert out.shape == (M, N) and out.dtype is like.dtype and out.device == like.device, (
        f"out must be {like.dtype} of shape {(M, N)} on {like.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
    assert (out.stride(1) == 1 or N <= 1) and (out.stride(0) >= N or M <= 1), (
        f"out must be a row-major matrix, got strides {out.stride()}")
    refuse_grad_out("out", out)
    if residual is not None:
        in_place_or_apart("out", out, residual)
        assert residual is given or out is not given, "a residual updated in place must have rows of adjacent elements"
    return out, residual


def _apart_from(out: torch.Tensor, x: torch.Tensor, w_packed: torch.Tensor) -> torch.Tensor:
    """x, or a copy of it (at its strides) if the output takes any of its memory: a product
    reads its operands again for every tile, and writes tiles before it has read them all."""
    assert not overlap(out, w_packed), "out shares memory with w_packed"
    if not overlap(out, x):
        return x
    copy = x.new_empty(x.shape[0] * x.stride(0) if x.shape[0] > 1 else max(x.stride(0), x.shape[1]))
    copy = copy.as_strided(x.shape, x.stride())
    return copy.copy_(x)


def ghost_linear_dev(
    x: torch.Tensor,
    w_packed: torch.Tensor,
    alive_buffer: torch.Tensor,
    alive_count: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    out: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """ghost_linear with K' = alive_count[0] read on the device (no host synchronisation).

    w_packed is the [N, round_up(K, 64)] buffer of :func:`pack_weight_dev` for the
    same alive list; alive_buffer's first K' entries are the alive columns.
    """
    assert x.ndim == 2 and x.is_cuda
    x = x.contiguous()
    M = x.shape[0]
    N = w_packed.shape[0]
    y, residual = _product_out(out, residual, M, N, x)
    if out is not None:
        x = _apart_from(y, x, w_packed)
    _operands_ok(w_packed, alive_buffer.numel(), bias, x.dtype, x.get_device())
    if M and N:
        _native.gather_gemm_dev(x, w_packed, alive_buffer, alive_count, y, bias=bias,
                                activation=activation, residual=residual)
        if out is not None:
            written(out)
    return y


def packed_linear(
    a: torch.Tensor,
    w_packed: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """y = act(a @ w_packed^T + bias) + residual for an already compacted a [M, K_alive].

    Both operands arrive by TMA: a's rows may be strided (as ``rms_norm``
    returns them) if they start at multiples of 16 bytes, else they are copied
    into such rows. residual [M, N] and ``out`` as for :func:`ghost_linear`.
    Columns of w_packed from K_alive on are not looked at.
    """
    assert a.ndim == 2 and a.is_cuda
    M, K = a.shape
    N = w_packed.shape[0]
    lda, unit = a.stride()
    if a.data_ptr() % 16 or (unit != 1 and K > 1) or (M > 1 and (lda % 8 or lda < K)):
        lda = (K + 7) // 8 * 8
        buf = a.new_empty((M, lda))              # columns from K on are not looked at
        buf[:, :K] = a
        a = buf[:, :K]
    elif M <= 1:
        lda = (K + 7) // 8 * 8                   # a row's stride may be anything
    dev = a.get_device()
    ldw = _operands_ok(w_packed, K, bias, a.dtype, dev)
    y, residual = _product_out(out, residual, M, N, a)
    if out is not None:
        a = _apart_from(y, a, w_packed)
    if M and N:
        r_ptr, ldr = _native._residual(residual)
        st = _native._call((_native._api or _native.api()).gw_packed_gemm_residual,
                           (a.data_ptr(), _native.dtype_code(a.dtype), M, K, lda, w_packed.data_ptr(), N, ldw,
                            None if bias is None else bias.data_ptr(), _native.epilogue_code(activation), r_ptr, ldr,
                            y.data_ptr(), max(y.stride(0), N)), dev)
        if st:
            _native._check(st, "gw_packed_gemm")
        if out is not None:
            written(out)
    return y


def _q8_operand(what: str, q: torch.Tensor, scale: torch.Tensor, dev: int) -> tuple:
    """(matrix, rows, columns, leading dimension, scales) of an e4m3 operand, in rows that TMA
    can load (16-byte aligned; copied into such rows if they are not)."""
    assert q.dtype is torch.float8_e4m3fn and q.dim() == 2 and q.is_cuda and q.get_device() == dev, (
        f"{what} must be a float8_e4m3fn matrix on one CUDA device with the others, got {q.dtype} "
        f"{tuple(q.shape)} on {q.device}")
    rows, cols = q.shape
    assert (scale.dtype is torch.float32 and scale.dim() == 1 and scale.numel() == rows and scale.is_cuda
            and scale.get_device() == dev), (
        f"{what}_scale must be float32 of shape ({rows},) on {what}'s device")
    if not scale.is_contiguous():
        scale = scale.contiguous()
    ld, unit = q.stride()
    if (unit != 1 and cols > 1) or q.data_ptr() % 16 or (rows > 1 and (ld % 16 or ld < cols)):
        ld = (cols + 15) // 16 * 16
        buf = torch.zeros((rows, ld), dtype=q.dtype, device=q.device)
        buf[:, :cols] = q
        q = buf
    elif rows <= 1:
        ld = (cols + 15) // 16 * 16
    return q, rows, cols, ld, scale


def packed_linear_q8(
    a: torch.Tensor,
    a_scale: torch.Tensor,
    w_packed: torch.Tensor,
    w_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """y = act(a_scale[:, None] * (a @ w_packed^T) * w_scale + bias) + residual in e4m3.

    a [M, K_alive] with a_scale [M] (``rms_norm_q8``, ``quantize_rows``) and
    w_packed [N, K_alive] with w_scale [N] (``pack_weight_q8``) are
    float8_e4m3fn with float32 scales; the sum is accumulated and scaled in
    fp32. ``dtype`` is y's type, float16 or bfloat16 (by default the residual's
    or the output's, else float16 with a float16 bias, else bfloat16); residual
    [M, N] has it too, bias is converted to it. ``out`` may be the residual itself.
    """
    dev = a.get_device() if a.is_cuda else -1
    a, M, K, lda, a_scale = _q8_operand("a", a, a_scale, dev)
    w_packed, N, K_w, ldw, w_scale = _q8_operand("w_packed", w_packed, w_scale, dev)
    assert K == K_w, f"K mismatch: a has {K} columns, w_packed {K_w}"
    if dtype is None:
        dtype = next((t.dtype for t in (residual, out) if t is not None),
                     bias.dtype if bias is not None and bias.dtype is torch.float16 else torch.bfloat16)
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise TypeError(f"unsupported output dtype {dtype}; expected float16 or bfloat16")
    if bias is not None:
        assert bias.dim() == 1 and bias.numel() == N and bias.is_cuda and bias.get_device() == dev, (
            f"bias must have shape ({N},) on a's device")
        if bias.dtype is not dtype or not bias.is_contiguous():
            bias = bias.detach().to(dtype).contiguous()
    if out is None:
        y, ldy = a.new_empty((M, N), dtype=dtype), N
        if residual is not None:
            residual = residual_matrix(residual, (M, N), y)
    else:
        assert out.dtype is dtype and out.is_cuda and out.get_device() == dev, f"out must be {dtype} on a's device"
        y, residual = _product_out(out, residual, M, N, out)
        a = _apart_from(y, a, w_packed)
        ldy = max(y.stride(0), N)
    if M and N:
        _native.packed_gemm_q8(a, a_scale, M, K, lda, w_packed, w_scale, N, ldw, y, ldy, bias, activation, residual)
        if out is not None:
            written(out)
    return y


class _PipeState:
    """Per-device streams, events and x' buffers of ghost_linear_pipelined."""

    def __init__(self, device: torch.device):
        lo, hi = torch.cuda.Stream.priority_range()      # (least, greatest) priority
        self.gemm = torch.cuda.Stream(device, priority=hi)
        self.gather = torch.cuda.Stream(device, priority=lo)
        self.ready = [torch.cuda.Event(), torch.cuda.Event()]
        self.free = [torch.cuda.Event(), torch.cuda.Event()]
        self.bufs: dict = {}

    def xbuf(self, slot: int, dtype: torch.dtype, M: int, ldp: int, device) -> torch.Tensor:
        key = (slot, dtype)
        b = self.bufs.get(key)
        if b is None or b.numel() < M * ldp:
            if b is not None:
                # The gather and GEMM streams may still use the old buffer:
                # the allocator reuses it only after their queued work.
                b.record_stream(self.gather)
                b.record_stream(self.gemm)
            b = self.bufs[key] = torch.empty(M * ldp, dtype=dtype, device=device)
        return b[: M * ldp].view(M, ldp)


_pipe_states: dict = {}


def ghost_linear_pipelined(calls) -> list:
    """Independent gather-GEMM calls with each gather overlapping the previous GEMM.

    ``calls`` is a sequence of ``(x, w_packed, alive_indices, out[, bias[,
    activation]])``, each meaning ``ghost_linear(x, w_packed, alive_indices,
    bias, activation, out=out)``, and the outputs are returned in order. The
    calls must not depend on one another (one call's output is not a later
    call's input): call i+1's gather of x[:, alive] then runs on a
    low-priority stream while call i's GEMM runs on a high-priority one. The
    GEMM keeps the SMs it needs, and the gather fills the registers and issue
    slots it leaves (the GEMM reads only a few percent of HBM bandwidth). x'
    alternates between two buffers, ordered by events. The caller's current
    stream waits for all of it before this returns, and the whole call can be
    captured in a CUDA graph. Calls with at most 4 rows (the decode kernel
    gathers x' itself, one launch), fp32 operands or index lists that are not
    int64 run as ``ghost_linear`` in order on the GEMM stream.
    """
    cur = torch.cuda.current_stream()
    device = cur.device
    st = _pipe_states.get(device.index)
    if st is None:
        st = _pipe_states[device.index] = _PipeState(device)
    norm = []
    for c in calls:
        x, wp, idx, out = c[0], c[1], c[2], c[3]
        bias = c[4] if len(c) > 4 else None
        act = c[5] if len(c) > 5 else None
        assert x.ndim == 2 and x.is_cuda and out is not None
        _product_out(out, None, x.shape[0], wp.shape[0], x)
        _operands_ok(wp, idx.numel(), bias, x.dtype, x.get_device())
        norm.append((x, wp, idx, out, bias, act))
    st.gemm.wait_stream(cur)
    st.gather.wait_stream(cur)
    # Both slots start free, ordered after the caller's work. Recording them
    # here (not reusing an earlier call's events) also keeps every wait inside
    # a CUDA graph capture that this call may be part of.
    for e in st.free:
        e.record(st.gemm)

    def piped(c):
        x, wp, idx, out, bias, act = c
        return (x.shape[0] > 4 and x.dtype is not torch.float32 and x.is_contiguous()
                and idx.dtype is torch.int64 and idx.numel() > 0)

    def gather(i):
        x, wp, idx, _, _, _ = norm[i]
        b = i % 2
        kp = idx.numel()
        ldp = (kp + 63) // 64 * 64
        xg = st.xbuf(b, x.dtype, x.shape[0], ldp, device)[:, :kp]
        st.gather.wait_event(st.free[b])
        with torch.cuda.stream(st.gather):
            _native.gather_columns(x, idx, xg)
            st.ready[b].record(st.gather)
        return xg

    xgs = {}
    if norm and piped(norm[0]):
        xgs[0] = gather(0)
    for i, c in enumerate(norm):
        if i + 1 < len(norm) and piped(norm[i + 1]):
            xgs[i + 1] = gather(i + 1)
        x, wp, idx, out, bias, act = c
        with torch.cuda.stream(st.gemm):
            if i in xgs:
                b = i % 2
                st.gemm.wait_event(st.ready[b])
                if out.numel():
                    _native.packed_gemm(xgs.pop(i), wp, out, bias=bias, activation=act)
                    written(out)
                st.free[b].record(st.gemm)
            else:
                ghost_linear(x, wp, idx, bias=bias, activation=act, out=out)
    cur.wait_stream(st.gemm)
    cur.wait_stream(st.gather)
    return [c[3] for c in norm]
