"""Fused GhostLinear MLP chains: fc -> GELU -> proj without the dead features.

In a transformer MLP the first projection's output goes through an
elementwise activation into the second projection only (GPT-2's
``GPT2MLP``: c_fc -> gelu_new -> c_proj; DistilBERT's ``FFN``: lin1 -> gelu
-> lin2). When both are GhostLinears with frozen masks, the second layer's dead
input features are outputs of the first layer that nothing reads: their
columns of the second weight are zero. The fused chain therefore

* computes only the second layer's alive features in the first GEMM (the rows
  of the first weight restricted to them, packed over the first layer's own
  alive inputs), with the bias and the GELU in its epilogue, so that its output
  already is the second layer's compacted input x'; and
* feeds that straight into the second GEMM (both operands by TMA, no gather).

``GhostPreNormMLP`` puts the residual stream and the root-mean-square norm in
front of the same chain, so that a whole pre-norm MLP block is three launches
(four in e4m3, where the hidden rows are rounded by one of their own): the
residual's addition, the norm and the first layer's gather are one kernel, and
the second addition is the last GEMM's epilogue. Parameters of another type than
the input's add a cast of the norm's weight and one of proj's bias to each call.

One gather launch and the dead part of the first GEMM disappear; the result
equals the unfused chain's (the skipped terms are products with zero weights),
up to the one rounding of the intermediate that the fused GELU saves. This is
an extension: the reference replaces the two projections independently
(ghostweight_triton/replace.py:35-56) and keeps the full intermediate.
"""

from __future__ import annotations

import copy
import math

import torch
import torch.nn as nn

from ghostweight_triton_b200 import _native
from ghostweight_triton_b200.kernels.gather import pack_weight
from ghostweight_triton_b200.kernels._args import Kept, refuse_grad
from ghostweight_triton_b200.kernels.matmul import ghost_linear, packed_linear, packed_linear_q8
from ghostweight_triton_b200.kernels.norm import pack_weight_q8, quantize_rows, rms_norm, rms_norm_q8
from ghostweight_triton_b200.module import GhostLinear

# Activation modules (by class name) that the GEMM epilogue reproduces.
_ACT_BY_CLASS = {
    "NewGELUActivation": "gelu_tanh",     # transformers' gelu_new: tanh approximation
    "GELUTanh": "gelu_tanh",
    "GELUActivation": "gelu",             # exact erf GELU
}


def _epilogue_of(act: nn.Module) -> str | None:
    if isinstance(act, nn.GELU):
        return "gelu_tanh" if act.approximate == "tanh" else "gelu"
    return _ACT_BY_CLASS.get(type(act).__name__)


def _plan_key(form: tuple, *tensors: torch.Tensor | None) -> tuple:
    """What packed operands are made for and from: the tensors themselves (held, so that none
    of them can be freed and another take its address), their versions and storage."""
    return (form, *((t, t._version, t.data_ptr()) for t in tensors if t is not None))


def _same_key(a: tuple, b: tuple) -> bool:
    return (len(a) == len(b) and a[0] == b[0]
            and all(u[0] is v[0] and u[1:] == v[1:] for u, v in zip(a[1:], b[1:])))


class _Plan(Kept):
    """Packed operands kept between calls, with the tensors they were made from (the key)."""

    def __init__(self, key: tuple, operands: tuple):
        super().__init__(t for o in operands for t in (o if isinstance(o, tuple) else (o,)) if t is not None)
        self.key = key
        self.operands = operands

    def take(self) -> tuple:
        self.on_this_stream()
        return self.operands


class GhostMLPChain(nn.Module):
    """fc -> activation -> proj (-> dropout) with proj's dead inputs never computed.

    ``fc`` and ``proj`` are GhostLinears with frozen masks (``proj.in_features ==
    fc.out_features``); they stay registered as submodules, so parameters and
    state-dict keys are unchanged. The packed operands are built on first use and
    rebuilt when a weight or a mask changes. A captured graph reads the operands of
    the call that it captured: capture again after a change.
    """

    precision = "input"                              # of the operands; GhostPreNormMLP has a choice

    def __init__(self, fc: GhostLinear, proj: GhostLinear, activation: str,
                 dropout: nn.Module | None = None):
        super().__init__()
        assert proj.in_features == fc.out_features
        self.fc = fc
        self.proj = proj
        self.activation = activation
        self.dropout = dropout
        self._plan: _Plan | None = None

    def __getstate__(self):
        return {k: None if isinstance(v, _Plan) else v for k, v in self.__dict__.items()}    # copies pack anew

    def refresh_packed(self) -> None:
        """Rebuild the fused operands at the next forward: needed after in-place
        writes through ``weight.data`` or ``bias.data``, which bypass the
        version counters the plan is keyed on."""
        self._plan = None

    def _operands(self, dtype: torch.dtype) -> tuple:
        """(w_fc, b_fc, w_proj) as the products take them, for activations of `dtype`."""
        fc, proj = self.fc, self.proj
        key = _plan_key((dtype, self.precision), fc.weight, proj.weight, fc._frozen_indices, proj._frozen_indices, fc.bias)
        if self._plan is not None and _same_key(self._plan.key, key):
            return self._plan.take()
        with torch.no_grad():
            operands = self._pack(dtype)
        # Under graph capture the packing is only recorded, into the graph's own memory: not kept.
        if not torch.cuda.is_current_stream_capturing():
            self._plan = _Plan(key, operands)
        return operands

    def _pack(self, dtype: torch.dtype) -> tuple:
        # proj's weight packed over its alive inputs, whole buffer: the fused
        # features padded with zero columns to a multiple of 64 (TMA rows).
        wp = pack_weight(self.proj.weight.detach(), self.proj._frozen_indices, dtype=dtype)
        n_pad = wp.stride(0)
        w_proj = wp.as_strided((wp.shape[0], n_pad), (n_pad, 1))
        rows, b_fc = self._features(n_pad, dtype)
        return pack_weight(rows, self.fc._frozen_indices, dtype=dtype), b_fc, w_proj

    def _features(self, n_pad: int, dtype: torch.dtype) -> tuple:
        """Rows of fc's weight (in its own type) and its bias for the features proj reads, and
        zeros up to n_pad of them: their outputs are act(0) = 0."""
        fc, a_proj = self.fc, self.proj._frozen_indices
        rows = fc.weight.detach().index_select(0, a_proj)
        pad = n_pad - rows.shape[0]
        if pad:
            rows = torch.cat([rows, rows.new_zeros(pad, rows.shape[1])])
        b_fc = None
        if fc.bias is not None:
            b_fc = fc.bias.detach().index_select(0, a_proj).to(dtype)
            if pad:
                b_fc = torch.cat([b_fc, b_fc.new_zeros(pad)])
        return rows, b_fc

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """The chain over x [..., in_features]; residual (the output's shape) is added in
        proj's epilogue (behind the dropout, where a training-mode one is active)."""
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.fc.in_features)
        w_fc, b_fc, w_proj = self._operands(x2.dtype)
        h = ghost_linear(x2, w_fc, self.fc._frozen_indices, bias=b_fc, activation=self.activation)
        bias = self.proj.bias
        if bias is not None and bias.dtype != x2.dtype:
            bias = bias.to(x2.dtype)
        if residual is not None:
            assert residual.shape == (*lead, self.proj.out_features), (
                f"residual must have shape {(*lead, self.proj.out_features)}, got {tuple(residual.shape)}")
        identity = self.dropout is None or (isinstance(self.dropout, nn.Dropout) and not self.dropout.training)
        behind = residual is not None and not identity
        fused = None if residual is None or behind else residual.reshape(-1, self.proj.out_features)
        y = packed_linear(h, w_proj, bias=bias, residual=fused)
        if self.dropout is not None and fused is None:
            y = self.dropout(y)
        if behind:
            y = y + residual.reshape(-1, self.proj.out_features)
        return y.reshape(*lead, self.proj.out_features)


class GhostPreNormMLP(GhostMLPChain):
    """s = x + residual;  y = s + proj(activation(fc(rms_norm(s)))).

    ``norm`` is a root-mean-square norm over fc's input features (torch.nn.RMSNorm,
    or a module with ``weight`` and ``eps`` or ``variance_epsilon`` that computes
    x * rsqrt(mean(x^2) + eps) * weight: two rows are tried when the block is built,
    or in its next forward if the norm is on the meta device then or replaced later),
    ``fc`` and ``proj`` are GhostLinears with frozen masks, joined by the GELU
    ``activation`` ("gelu" or "gelu_tanh"); all stay registered, so parameters and
    state-dict keys are theirs. fp16 and bf16 inputs. ``precision="e4m3"`` runs both
    products on e4m3 operands (weights rounded once with a scale per feature,
    activations with one per token), with fp32 sums and the residual stream in
    the input's type.
    """

    def __init__(self, norm: nn.Module, fc: GhostLinear, proj: GhostLinear, activation: str,
                 dropout: nn.Module | None = None, precision: str = "input"):
        super().__init__(fc, proj, activation, dropout)
        if precision not in ("input", "e4m3"):
            raise ValueError(f"precision must be 'input' or 'e4m3', got {precision!r}")
        assert proj.out_features == fc.in_features, "the block adds its output to its input"
        assert not isinstance(norm, nn.LayerNorm) and getattr(norm, "bias", None) is None, (
            "norm must be a root-mean-square norm (no mean, no bias)")
        weight = getattr(norm, "weight", None)
        assert weight is None or weight.shape == (fc.in_features,), (
            f"norm must be over fc's {fc.in_features} input features")
        self.norm = norm
        self.precision = precision
        if weight is None or not weight.is_meta:
            self._try_norm()

    def _eps(self) -> float:
        eps = getattr(self.norm, "eps", getattr(self.norm, "variance_epsilon", None))
        # None: torch.nn.RMSNorm's default, the epsilon of the type it norms 16-bit rows in.
        return torch.finfo(torch.float32).eps if eps is None else float(eps)

    @property
    def _norm_known(self) -> bool:
        """Whether the present norm has been tried (a DataParallel replica's is its module's)."""
        return self.__dict__.get("_tried") is self.norm or getattr(self, "_is_replica", False)

    def _try_norm(self) -> None:
        """Assert that a copy of the norm in fp32, with a gain of its own, computes what rms_norm does,
        of a row of ordinary values whose mean is not zero and of one so small that eps counts."""
        weight = getattr(self.norm, "weight", None)
        device = torch.device("cpu") if weight is None else weight.device
        eps = self._eps()
        row = 1.0 + torch.sin(torch.arange(self.fc.in_features, device=device, dtype=torch.float32))
        x = torch.stack([row, row * math.sqrt(max(eps, 1e-12))])
        want = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + eps)
        try:
            with torch.no_grad():
                twin = copy.deepcopy(self.norm).float()
                if weight is not None:
                    twin.weight.copy_(row - 0.7)
                    want = want * (row - 0.7).double()
                got = twin(x).double()
            same = got.shape == want.shape and bool(((got - want).norm(dim=1) <= 1e-3 * want.norm(dim=1)).all())
        except Exception as e:
            raise AssertionError("norm must take rows of fc's input features") from e
        assert same, "norm must compute x * rsqrt(mean(x^2) + eps) * weight"
        self.__dict__["_tried"] = self.norm          # not a second submodule

    def _pack(self, dtype: torch.dtype) -> tuple:
        if self.precision != "e4m3":
            return super()._pack(dtype)
        # From the parameters' own type, so that they are rounded once. The fused
        # features are padded to a multiple of 64 as in 16 bits; proj's rows, padded
        # with zeros to one of 128, hold as many columns.
        own = lambda w: w if w.dtype in _native.DTYPE_CODES else w.float()
        q, s_proj = pack_weight_q8(own(self.proj.weight), self.proj._frozen_indices)
        n_pad = (q.shape[1] + 63) // 64 * 64
        rows, b_fc = self._features(n_pad, dtype)
        q_proj = q.as_strided((q.shape[0], n_pad), q.stride())
        return pack_weight_q8(own(rows), self.fc._frozen_indices), b_fc, (q_proj, s_proj)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """x [..., features], and optionally a residual of its shape added in front of the norm."""
        assert x.dtype in (torch.float16, torch.bfloat16), f"GhostPreNormMLP runs fp16 and bf16, got {x.dtype}"
        if not (_frozen(self.fc) and _frozen(self.proj)):
            raise RuntimeError("GhostPreNormMLP needs frozen masks on fc and proj (freeze_mask or freeze_weight_mask)")
        refuse_grad(x=x, residual=residual)
        if not self._norm_known:
            self._try_norm()
        features = self.fc.in_features
        x2 = x.reshape(-1, features)
        r2 = None if residual is None else residual.reshape(-1, features)
        norm = dict(weight=getattr(self.norm, "weight", None), eps=self._eps(), residual=r2,
                    alive_indices=self.fc._frozen_indices)
        bias = self.proj.bias
        if bias is not None and bias.dtype != x.dtype:
            bias = bias.to(x.dtype)
        identity = self.dropout is None or (isinstance(self.dropout, nn.Dropout) and not self.dropout.training)
        if self.precision == "e4m3":
            (w_fc, s_fc), b_fc, (w_proj, s_proj) = self._operands(x.dtype)
            q, scale, *rest = rms_norm_q8(x2, **norm)
            s = rest[0] if rest else x2
            h = packed_linear_q8(q, scale, w_fc, s_fc, bias=b_fc, activation=self.activation, dtype=x.dtype)
            q, scale = quantize_rows(h)
            y = packed_linear_q8(q, scale, w_proj, s_proj, bias=bias, residual=s if identity else None, dtype=x.dtype)
        else:
            w_fc, b_fc, w_proj = self._operands(x.dtype)
            out = rms_norm(x2, **norm)
            n, s = out if r2 is not None else (out, x2)
            h = packed_linear(n, w_fc, bias=b_fc, activation=self.activation)
            y = packed_linear(h, w_proj, bias=bias, residual=s if identity else None)
        if not identity:
            y = s + self.dropout(y)
        return y.reshape(x.shape)


def _frozen(m: nn.Module) -> bool:
    return isinstance(m, GhostLinear) and m.mask_frozen and m._frozen_indices is not None


def fuse_mlp_chains(model: nn.Module) -> list[str]:
    """Replace every MLP block whose two projections are frozen GhostLinears joined by
    a GELU with a :class:`GhostMLPChain`; returns the names of the replaced blocks.

    Recognised blocks: modules with ``c_fc``, ``c_proj`` and ``act`` (transformers'
    GPT2MLP) or ``lin1``, ``lin2`` and ``activation`` (DistilBERT's FFN), each with
    an optional ``dropout``. Run it after ``replace_linears(...,
    freeze_from_weight=True)`` (or after freezing the masks).
    """
    replaced = []
    for name, parent in list(model.named_modules()):
        for child_name, child in list(parent.named_children()):
            fc = proj = act = None
            if hasattr(child, "c_fc") and hasattr(child, "c_proj") and hasattr(child, "act"):
                fc, proj, act = child.c_fc, child.c_proj, child.act
            elif hasattr(child, "lin1") and hasattr(child, "lin2") and hasattr(child, "activation"):
                fc, proj, act = child.lin1, child.lin2, child.activation
                if getattr(child, "chunk_size_feed_forward", 0):
                    continue
            if fc is None or not (_frozen(fc) and _frozen(proj)) or fc.activation is not None:
                continue
            epi = _epilogue_of(act) if isinstance(act, nn.Module) else None
            if epi is None or proj.in_features != fc.out_features or proj._frozen_indices.numel() == 0:
                continue
            dropout = getattr(child, "dropout", None)
            setattr(parent, child_name, GhostMLPChain(fc, proj, epi, dropout))
            replaced.append(f"{name}.{child_name}" if name else child_name)
    return replaced
