"""The linear-layer operators without a GPU: refusals, the C ABI's validation
(nothing is enqueued by any call here) and the exported symbols."""

from __future__ import annotations

import ctypes
import re
import subprocess

import pytest
import torch
from conftest import REPO

import gpumode_qr_b200 as pkg
from gpumode_qr_b200 import _lib, api, layers
from gpumode_qr_b200.build import LIB_PATH

HEADER = REPO / "include" / "qrb200_linear.h"
P = 0x100000  # never dereferenced: every call below fails or returns early


def test_header_symbols_are_exported_and_bound():
    declared = set(re.findall(r"QRB_API\s+[\w\s\*]+?\b(qrbl_\w+)\s*\(", HEADER.read_text()))
    out = subprocess.run(["nm", "-D", "--defined-only", str(LIB_PATH)], capture_output=True, text=True)
    exported = set(re.findall(r"\b(qrbl_\w+)\b", out.stdout))
    assert declared == exported == set(_lib.LINEAR_SIGNATURES)


def test_entry_points_are_public():
    for name in ("linear", "linear_backward", "pack_activation", "unpack_activation",
                 "PackedActivation"):
        assert name in pkg.__all__ and getattr(pkg, name) is getattr(api, name)


def test_struct_layouts_match_the_header():
    text = HEADER.read_text()
    for struct, cls in (("qrbl_linear_args", layers._LinearArgs),
                        ("qrbl_linear_backward_args", layers._BackwardArgs)):
        body = text[:text.index("} " + struct + ";")].rsplit("typedef struct {", 1)[1]
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = [n.strip(" *") for line in body.split(";") if line.strip()
                 for n in line.strip().split(None, 1 if "const" not in line else 2)[-1].split(",")]
        assert names == [f[0] for f in cls._fields_]


def test_cpu_tensors_and_types_are_refused():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    with pytest.raises(ValueError, match="CUDA"):
        api.linear(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        api.linear_backward(torch.randn(4, 6), x, w)
    with pytest.raises(ValueError, match="CUDA"):
        api.pack_activation(x)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        api.linear(x.double(), w.double())
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        api.pack_activation(x.int())
    with pytest.raises(TypeError, match="PackedActivation"):
        api.unpack_activation((x, x))
    with pytest.raises(TypeError):
        api.linear(x.numpy(), w)
    q = api.PackedActivation(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.int8),
                             torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        api.unpack_activation(q)
    with pytest.raises(TypeError, match="packed.dtype"):
        api.unpack_activation(q._replace(dtype=torch.float64))


def _fwd(**kw):
    a = layers._LinearArgs(2, 0, 4, 16, 32, P, 32, P, 32, None, None, 0, P, 16, None, 0, None, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bwd(**kw):
    a = layers._BackwardArgs(2, 4, 4, 16, 32, P, 16, P, 32, None, None, P, 32, P, 16, None, None,
                             P, 32, P, 32, P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    {"dtype": 3}, {"dtype": -1}, {"activation": 5}, {"activation": -1}, {"m": -1}, {"n": -1},
    {"k": -1}, {"x": None}, {"w": None}, {"y": None}, {"ldx": 31}, {"ldw": 31}, {"ldy": 15},
    {"residual": P, "ldr": 15}, {"z": P, "ldz": 15}, {"z_codes": P}, {"z_exponents": P},
    {"x": P + 1}, {"w": P + 1}, {"y": P + 1}, {"bias": P + 1}, {"dtype": 0, "x": P + 2},
    {"ldx": -1, "m": 1}])
def test_forward_validation(bad):
    a = _fwd(**bad)
    assert _lib.lib().qrbl_linear(ctypes.byref(a), None, 0, None) == 1
    assert _lib.lib().qrbl_linear_workspace_bytes(ctypes.byref(a)) == 0


@pytest.mark.parametrize("bad", [
    {"dtype": 7}, {"activation": 9}, {"m": -1}, {"dy": None}, {"x": None}, {"w": None}, {"z": None},
    {"lddy": 15}, {"ldx": 31}, {"ldw": 31}, {"ldz": 15}, {"lddx": 31}, {"lddw": 31},
    {"x_codes": P}, {"z_codes": P}, {"x_codes": P, "x_exponents": P},
    {"z_codes": P, "z_exponents": P}, {"dbias": P + 1}, {"dx": P + 1}, {"dw": P + 1},
    {"z": None, "z_codes": P, "z_exponents": P, "activation": 1}])
def test_backward_validation(bad):
    a = _bwd(**bad)
    assert _lib.lib().qrbl_linear_backward(ctypes.byref(a), None, 0, None) == 1


def test_sizes_workspaces_and_empty_calls():
    L = _lib.lib()
    assert L.qrbl_linear(None, None, 0, None) == 1
    assert L.qrbl_linear_backward(None, None, 0, None) == 1
    # no rows or no columns: nothing to do, and nothing is touched
    assert L.qrbl_linear(ctypes.byref(_fwd(m=0, x=None, y=None)), None, 0, None) == 0
    assert L.qrbl_linear(ctypes.byref(_fwd(n=0, w=None, y=None)), None, 0, None) == 0
    none = {"dx": None, "dw": None, "dbias": None}
    assert L.qrbl_linear_backward(ctypes.byref(_bwd(dy=None, **none)), None, 0, None) == 0
    assert L.qrbl_pack(2, None, 0, 0, 64, None, None, None) == 0
    assert L.qrbl_unpack(2, None, None, 5, 0, None, 0, None) == 0
    # beyond 32-bit coordinates
    big = (1 << 30) + 1
    assert L.qrbl_linear(ctypes.byref(_fwd(k=big, ldx=big, ldw=big)), None, 0, None) == 2
    assert L.qrbl_linear_backward(ctypes.byref(_bwd(m=big)), None, 0, None) == 2
    # an operand that is not 16-byte aligned, or FP32, is staged: a workspace is required
    for a in (_fwd(x=P + 2), _fwd(ldx=33), _fwd(dtype=0)):
        need = L.qrbl_linear_workspace_bytes(ctypes.byref(a))
        assert need > 0
        assert L.qrbl_linear(ctypes.byref(a), None, need, None) == 3
        assert L.qrbl_linear(ctypes.byref(a), P, need - 1, None) == 3
        assert L.qrbl_linear(ctypes.byref(a), P + 4, need, None) == 1
    b = _bwd()
    need = L.qrbl_linear_backward_workspace_bytes(ctypes.byref(b))
    assert need > 0
    assert L.qrbl_linear_backward(ctypes.byref(b), None, need, None) == 3
    assert L.qrbl_linear_backward(ctypes.byref(b), P, need - 1, None) == 3
    assert L.qrbl_linear_backward(ctypes.byref(b), P + 8, need, None) == 1


@pytest.mark.parametrize("args", [
    (3, P, 64, 2, 64, P, P), (2, None, 64, 2, 64, P, P), (2, P, 63, 2, 64, P, P),
    (2, P, 64, -1, 64, P, P), (2, P, 64, 2, 64, None, P), (2, P, 64, 2, 64, P, None),
    (2, P + 1, 64, 2, 64, P, P)])
def test_pack_validation(args):
    dtype, x, ld, rows, cols, codes, exps = args
    assert _lib.lib().qrbl_pack(dtype, x, ld, rows, cols, codes, exps, None) == 1
    assert _lib.lib().qrbl_unpack(dtype, codes, exps, rows, cols, x, ld, None) == 1


def test_injected_failure_enqueues_nothing():
    _lib.set_config("fail_next", 1)
    assert _lib.lib().qrbl_pack(2, P, 64, 2, 64, P, P, None) == 6
    _lib.set_config("fail_next", 1)
    assert _lib.lib().qrbl_linear(ctypes.byref(_fwd()), None, 0, None) == 6
    _lib.set_config("fail_next", 1)
    assert _lib.lib().qrbl_linear_backward(ctypes.byref(_bwd()), None, 0, None) == 6
    assert _lib.get_config("fail_next") == 0
