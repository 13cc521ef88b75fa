"""CPU: the row operators refuse what they do not take, in Python and at the C ABI.

No kernel is launched here: the C entry points check sizes, types and pointers
before they look for a device.
"""

from __future__ import annotations

import pytest
import torch

from ghostweight_triton_b200 import _native
from ghostweight_triton_b200.kernels._args import out_matrix
from ghostweight_triton_b200.kernels.norm import pack_weight_q8, quantize_rows, rms_norm, rms_norm_q8

SHAPE, DTYPE, NULL = _native.GW_ERR_SHAPE, _native.GW_ERR_DTYPE, _native.GW_ERR_NULL


@pytest.mark.parametrize("fn", [rms_norm, rms_norm_q8, quantize_rows])
def test_cpu_tensors_are_rejected(fn):
    with pytest.raises(AssertionError, match="CUDA"):
        fn(torch.randn(4, 8))


def test_pack_rejects_cpu_and_other_ranks():
    with pytest.raises(AssertionError):
        pack_weight_q8(torch.randn(4, 8), torch.arange(4))


def _rms(lib, rows=4, cols=8, ldx=8, dtype=0, r=None, ldr=0, s=None, lds=0, idx=None, n=8, ldy=8, pad=8, y=64):
    return lib.gw_rms_norm(64, dtype, rows, cols, ldx, r, ldr, s, lds, None, 1e-6, idx, n, y, ldy, pad, None)


def test_abi_refusals():
    lib = _native.load()
    assert _rms(lib, dtype=3) == DTYPE and _rms(lib, dtype=-1) == DTYPE
    for bad in (dict(rows=-1), dict(cols=-1), dict(ldx=7), dict(n=-1), dict(pad=7), dict(ldy=7),
                dict(r=64, ldr=7), dict(s=64, lds=7), dict(cols=0, n=0)):
        assert _rms(lib, **bad) == SHAPE, bad
    assert _rms(lib, n=7) == NULL                   # no list: every column
    q = lambda **k: lib.gw_quantize_rows(64, k.get("dtype", 0), 4, 8, k.get("ldx", 8), None, k.get("n", 8), 64,
                                         k.get("ldq", 128), k.get("pad", 128), 64, None)
    assert q(dtype=7) == DTYPE and q(ldx=3) == SHAPE and q(ldq=127) == SHAPE and q(pad=4) == SHAPE
    assert q(n=3) == NULL


def test_residual_out_checks_need_no_gpu():
    _out_rows = lambda out, like, *ins: out_matrix("residual_out", out, like, *ins)
    x = torch.zeros(4, 6)
    r = torch.zeros(4, 6)
    assert _out_rows(x, x, x, r) is not None and _out_rows(torch.empty(4, 6), x, x, r) is not None
    big = torch.zeros(8, 6)
    assert _out_rows(big[4:], big[:4], big[:4], r) is not None
    for out, ins in ((big[1:5], big[:4]), (big[:4].view(-1)[1:1 + 18].view(3, 6), big[:3])):
        with pytest.raises(AssertionError, match="overlaps"):
            _out_rows(out, ins, ins, None)
    with pytest.raises(AssertionError):
        _out_rows(torch.zeros(6, 4).t(), x, x, r)
    with pytest.raises(AssertionError):
        _out_rows(torch.zeros(1, 6).expand(4, 6), x, x, r)
    with pytest.raises(AssertionError):
        _out_rows(torch.zeros(4, 6, dtype=torch.float16), x, x, r)
