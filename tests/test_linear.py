"""The linear-layer operators without a GPU: refusals, the C ABI's validation
(nothing is enqueued by any call here) and the exported symbols."""

from __future__ import annotations

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


def _fields(struct: str) -> list[tuple[str, str]]:
    """(name, kind) of a header struct's fields: "i" int32, "q" int64, "P" pointer."""
    text = HEADER.read_text()
    body = text[:text.index("} " + struct + ";")].rsplit("typedef struct {", 1)[1]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    out = []
    for decl in body.split(";"):
        if decl.strip():
            kind = "P" if "*" in decl else {"int32_t": "i", "int64_t": "q"}[decl.split()[0]]
            names = decl.replace("const", "").split(None, 1)[1]
            out += [(n.strip(" *"), kind) for n in names.split(",")]
    return out


def test_struct_layouts_match_the_header():
    import struct

    for name, fields, pack in (("qrbl_linear_args", layers._LINEAR_FIELDS, layers._linear_args),
                               ("qrbl_linear_backward_args", layers._BACKWARD_FIELDS,
                                layers._backward_args)):
        decl = _fields(name)
        assert tuple(n for n, _ in decl) == fields
        values = list(range(1, len(fields) + 1))
        assert pack(*values) == struct.pack("@" + "".join(k for _, k in decl), *values)


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
    a = dict(zip(layers._LINEAR_FIELDS,
                 (2, 0, 4, 16, 32, P, 32, P, 32, 0, 0, 0, P, 16, 0, 0, 0, 0)))
    return layers._linear_args(*{**a, **kw}.values())


def _bwd(**kw):
    a = dict(zip(layers._BACKWARD_FIELDS,
                 (2, 4, 4, 16, 32, P, 16, P, 32, 0, 0, P, 32, P, 16, 0, 0, P, 32, P, 32, P)))
    return layers._backward_args(*{**a, **kw}.values())


@pytest.mark.parametrize("bad", [
    {"dtype": 3}, {"dtype": -1}, {"activation": 5}, {"activation": -1}, {"m": -1}, {"n": -1},
    {"k": -1}, {"x": 0}, {"w": 0}, {"y": 0}, {"ldx": 31}, {"ldw": 31}, {"ldy": 15},
    {"residual": P, "ldr": 15}, {"z": P, "ldz": 15}, {"z_codes": P}, {"z_exponents": P},
    {"x": P + 1}, {"w": P + 1}, {"y": P + 1}, {"bias": P + 1}, {"dtype": 0, "x": P + 2},
    {"ldx": -1, "m": 1}])
def test_forward_validation(bad):
    a = _fwd(**bad)
    assert _lib.lib().qrbl_linear(a, None, 0, None) == 1
    assert _lib.lib().qrbl_linear_workspace_bytes(a) == 0


@pytest.mark.parametrize("bad", [
    {"dtype": 7}, {"activation": 9}, {"m": -1}, {"dy": 0}, {"x": 0}, {"w": 0}, {"z": 0},
    {"lddy": 15}, {"ldx": 31}, {"ldw": 31}, {"ldz": 15}, {"lddx": 31}, {"lddw": 31},
    {"x_codes": P}, {"z_codes": P}, {"x_codes": P, "x_exponents": P},
    {"z_codes": P, "z_exponents": P}, {"dbias": P + 1}, {"dx": P + 1}, {"dw": P + 1},
    {"z": 0, "z_codes": P, "z_exponents": P, "activation": 1}])
def test_backward_validation(bad):
    a = _bwd(**bad)
    assert _lib.lib().qrbl_linear_backward(a, None, 0, None) == 1


def test_sizes_workspaces_and_empty_calls():
    L = _lib.lib()
    assert L.qrbl_linear(None, None, 0, None) == 1
    assert L.qrbl_linear_backward(None, None, 0, None) == 1
    # no rows or no columns: nothing to do, and nothing is touched
    assert L.qrbl_linear(_fwd(m=0, x=0, y=0), None, 0, None) == 0
    assert L.qrbl_linear(_fwd(n=0, w=0, y=0), None, 0, None) == 0
    none = {"dx": 0, "dw": 0, "dbias": 0}
    assert L.qrbl_linear_backward(_bwd(dy=0, **none), None, 0, None) == 0
    assert L.qrbl_pack(2, None, 0, 0, 64, None, None, None) == 0
    assert L.qrbl_unpack(2, None, None, 5, 0, None, 0, None) == 0
    # beyond 32-bit coordinates
    big = (1 << 30) + 1
    assert L.qrbl_linear(_fwd(k=big, ldx=big, ldw=big), None, 0, None) == 2
    assert L.qrbl_linear_backward(_bwd(m=big), None, 0, None) == 2
    # an operand that is not 16-byte aligned, or FP32 of many rows, is staged: a workspace is required
    for a in (_fwd(m=64, x=P + 2), _fwd(m=64, ldx=33), _fwd(m=200, dtype=0)):
        need = L.qrbl_linear_workspace_bytes(a)
        assert need > 0
        assert L.qrbl_linear(a, None, need, None) == 3
        assert L.qrbl_linear(a, P, need - 1, None) == 3
        assert L.qrbl_linear(a, P + 4, need, None) == 1
    b = _bwd()
    need = L.qrbl_linear_backward_workspace_bytes(b)
    assert need > 0
    assert L.qrbl_linear_backward(b, None, need, None) == 3
    assert L.qrbl_linear_backward(b, P, need - 1, None) == 3
    assert L.qrbl_linear_backward(b, P + 8, need, None) == 1


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
    assert _lib.lib().qrbl_linear(_fwd(), None, 0, None) == 6
    _lib.set_config("fail_next", 1)
    assert _lib.lib().qrbl_linear_backward(_bwd(), None, 0, None) == 6
    assert _lib.get_config("fail_next") == 0


@pytest.mark.parametrize("key,good,bad", [("linear_cut", (2256, 2128, 1128, 1064, 0), (1, 1256, -1)),
                                          ("linear_splits", (1, 16, 0), (17, -1)),
                                          ("linear_rows", (0, 32, -1), (33, -2))])
def test_hooks(key, good, bad):
    for v in good:
        _lib.set_config(key, v)
        assert _lib.get_config(key) == v
    for v in bad:
        with pytest.raises(_lib.QRBError):
            _lib.set_config(key, v)
    assert _lib.get_config(key) == good[-1]
