"""Linear layers over libqrb200 (C ABI in ``include/qrb200_linear.h``).

The framework factors statistics ``G G^T`` of weight gradients; these are the
operators around that gradient:

* :func:`linear` — ``z = x W^T + b``, ``y = act(z) + residual`` in one product
  kernel, optionally keeping z for the backward pass;
* :func:`linear_backward` — ``dz = dy act'(z)``, ``dx = dz W``, ``dW = dz^T x``,
  ``db = sum of dz's rows``: dW of an FP32 layer goes straight into
  :func:`.api.gram` or :func:`.api.gram_geqrf`;
* :func:`pack_activation`, :func:`unpack_activation` — a tensor kept in 8 bits
  (plus one exponent for each 32 values of a row) and read back; ``linear``
  writes that form of z from its epilogue, ``linear_backward`` reads it.

All run on the caller's current stream, allocate only their outputs and scratch
(from torch's caching allocator), can be captured into a CUDA graph, and give
the same bits every time (for the same sizes, layouts and arguments). They are
plain functions, like the rest of the library: autograd does not record them,
and arguments that require a gradient are refused while gradients are enabled
(call them under ``torch.no_grad()`` or from an ``autograd.Function``), as are
arguments with a tangent of forward-mode differentiation, which would be lost.
"""

from __future__ import annotations

import struct
from types import SimpleNamespace
from typing import NamedTuple

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_NEED = frozenset(("x", "weight", "bias"))
#: Values of a row that share one exponent in the packed form.
PACK_BLOCK = 32

# The C ABI's argument structs (qrbl_linear_args, qrbl_linear_backward_args) as
# bytes, field by field in the header's order: two int32, then 8 bytes each
# (sizes and strides signed, pointers unsigned, 0 for none).
_LINEAR_FIELDS = ("dtype", "activation", "m", "n", "k", "x", "ldx", "w", "ldw", "bias", "residual",
                  "ldr", "y", "ldy", "z", "ldz", "z_codes", "z_exponents")
_linear_args = struct.Struct("@ii qqq Pq Pq P Pq Pq Pq PP").pack
_BACKWARD_FIELDS = ("dtype", "activation", "m", "n", "k", "dy", "lddy", "x", "ldx", "x_codes",
                    "x_exponents", "w", "ldw", "z", "ldz", "z_codes", "z_exponents", "dx", "lddx",
                    "dw", "lddw", "dbias")
_backward_args = struct.Struct("@ii qqq Pq Pq PP Pq Pq PP Pq Pq P").pack


class PackedActivation(NamedTuple):
    """A tensor in 8 bits: ``codes`` int8 [..., c] and ``exponents`` int8
    [..., ceil(c / 32)]; the values of columns 32 j .. 32 j + 31 are
    ``codes * 2**exponents[..., j]``, exact in ``dtype``, the type packed.
    The code -128 stands for NaN (and for Inf, which comes back as NaN)."""

    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype


_Tensor = torch.Tensor


def _check(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
    """Refuse what the library cannot take. (The entry points look at a plain
    tensor's type, device and requires_grad themselves first: a call's host time
    is most of a small layer's.)"""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (libqrb200 has no CPU path)")
    if like is not None:
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must be {like.dtype} like the others, got {t.dtype}")
        if t.device != like.device:
            raise ValueError(f"{name} must be on {like.device} like the others, got {t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, but autograd does not record this call: "
                           "use torch.no_grad() and linear_backward")


def _refuse_tangents(**tensors) -> None:
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has a tangent, but forward-mode differentiation does not "
                               "pass through this call: give its primal (unpack_dual)")


def _check_packed(name: str, p: PackedActivation, like: torch.Tensor, shape: tuple) -> None:
    codes, exps, dtype = p
    if dtype is not like.dtype:
        raise TypeError(f"{name} was packed from {dtype}, the layer is {like.dtype}")
    dev = like.device
    want = (*shape[:-1], -(-shape[-1] // PACK_BLOCK))
    if (type(codes) is _Tensor and type(exps) is _Tensor and codes.dtype is torch.int8
            and exps.dtype is torch.int8 and codes.device == dev and exps.device == dev
            and codes.shape == shape and exps.shape == want):
        return
    for part, t, s in (("codes", codes, shape), ("exponents", exps, want)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int8:
            raise TypeError(f"{name}.{part} must be an int8 tensor")
        if t.device != dev:
            raise ValueError(f"{name}.{part} must be on {dev}, got {t.device}")
        if t.shape != s:
            raise ValueError(f"{name}.{part} must be {tuple(s)}, got {tuple(t.shape)}")


def _contiguous(p: PackedActivation) -> tuple[torch.Tensor, torch.Tensor]:
    codes, exps, _ = p
    if codes.is_contiguous() and exps.is_contiguous():
        return codes, exps
    return codes.contiguous(), exps.contiguous()


def _rows(t: torch.Tensor, shape: torch.Size, cols: int) -> tuple[torch.Tensor, int, int]:
    """t (of that shape) as [rows, cols] with unit column stride and rows that do
    not overlap (copying only if needed), with its rows and row stride."""
    if len(shape) != 2:
        t = t.reshape(-1, cols) if cols else t.new_empty((shape[:-1].numel(), 0))
        shape = t.shape
    rows = shape[0]
    if t.is_neg():  # a conjugate's .imag is stored negated
        t = t.resolve_neg()
    if t.is_contiguous():
        return t, rows, cols
    row, col = t.stride()
    if (col != 1 and cols > 1) or (row < cols and rows > 1):
        t = t.contiguous()
        row = cols
    return t, rows, row


def _no_activation(name) -> ValueError:
    return ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {name!r}")


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same index and handle without the lazy start (a CUDA tensor is there) and the Stream object
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)
# forward-mode differentiation is on where its level is not negative, read without a call
_level = _forward_ad if hasattr(_forward_ad, "_current_level") else SimpleNamespace(_current_level=0)
_OK, _NEEDS_WORKSPACE = 0, 3  # QRB_OK, QRB_ERR_WORKSPACE


def _run(call, size, args: bytes, like: torch.Tensor, likely: bool = False) -> None:
    """``call`` on the current stream of ``like``'s device, with the workspace
    it asks for (``likely`` some: asked first)."""
    index = like.get_device()
    if index != _current_device():
        with torch.cuda.device(index):
            return _run(call, size, args, like, likely)
    stream = _raw_stream(index)
    need = size(args) if likely else 0
    rc = _NEEDS_WORKSPACE if need else call(args, None, 0, stream)
    if rc == _NEEDS_WORKSPACE:  # nothing was enqueued
        need = need or size(args)
        ws = like.new_empty(need, dtype=torch.uint8)
        rc = call(args, ws.data_ptr(), need, stream)
    if rc != _OK:
        _lib.check(rc)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, activation: str = "none",
           keep: str | None = None):
    """``y = act(x @ weight.T + bias) + residual`` in one product kernel.

    ``x`` is ``[..., k]``, ``weight`` ``[n, k]``, ``bias`` ``[n]``, ``residual``
    ``[..., n]``, all float32, float16 or bfloat16 (one type) on one CUDA device,
    any strides. ``activation`` is ``"none"``, ``"relu"``, ``"gelu"``,
    ``"gelu_tanh"`` or ``"silu"``. Sums are FP32 (FP32 inputs keep their 24
    bits: no TF32; below 2^-110 they lose low ones); y is rounded once. An Inf
    among FP32 inputs may give NaN where the product is Inf: whether it does
    depends on the number of rows.

    ``keep`` also returns the pre-activation ``z = x @ weight.T + bias`` for
    :func:`linear_backward`: ``"plain"`` as a tensor like y, ``"packed"`` as a
    :class:`PackedActivation` (8 bits a value, written from the FP32 sums).
    Returns ``y``, or ``(y, z)`` with ``keep``.
    """
    if type(x) is not _Tensor or x.dtype not in _DTYPES or not x.is_cuda or x.requires_grad:
        _check("x", x)
    dt, dev = x.dtype, x.device
    if (type(weight) is not _Tensor or weight.dtype is not dt or weight.device != dev
            or weight.requires_grad):
        _check("weight", weight, x)
    xs, ws = x.shape, weight.shape
    if len(ws) != 2 or not xs or xs[-1] != ws[1]:
        raise ValueError(f"x must be [..., k] and weight [n, k], got {tuple(xs)} and {tuple(ws)}")
    try:
        act = ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise _no_activation(activation) from None
    if _level._current_level >= 0:
        _refuse_tangents(x=x, weight=weight, bias=bias, residual=residual)
    n, k = ws
    shape = (xs[0], n) if len(xs) == 2 else (*xs[:-1], n)
    x2, m, ldx = _rows(x, xs, k)
    w2, _, ldw = _rows(weight, ws, k)
    bp = rp = ldr = zp = ldz = qp = ep = 0
    if bias is not None:
        if (type(bias) is not _Tensor or bias.dtype is not dt or bias.device != dev
                or bias.requires_grad):
            _check("bias", bias, x)
        if bias.shape != (n,):
            raise ValueError(f"bias must be ({n},), got {tuple(bias.shape)}")
        if bias.stride(0) != 1 or bias.is_neg():
            bias = bias.contiguous().resolve_neg()
        bp = bias.data_ptr()
    if residual is not None:
        if (type(residual) is not _Tensor or residual.dtype is not dt or residual.device != dev
                or residual.requires_grad):
            _check("residual", residual, x)
        rs = residual.shape
        if rs != shape:
            raise ValueError(f"residual must be {shape}, got {tuple(rs)}")
        residual, _, ldr = _rows(residual, rs, n)
        rp = residual.data_ptr()
    z = None
    if keep is not None:
        if keep == "plain":
            z = x.new_empty(*shape)
            zp, ldz = z.data_ptr(), n
        elif keep == "packed":
            z = _empty_packed(shape, x)
            qp, ep = z.codes.data_ptr(), z.exponents.data_ptr()
        else:
            raise ValueError(f"keep must be None, 'plain' or 'packed', got {keep!r}")
    y = x.new_empty(*shape)  # (separate ints: parsed faster than a tuple)
    if m and n:
        L = _lib._lib or _lib.lib()
        _run(L.qrbl_linear, L.qrbl_linear_workspace_bytes,
             _linear_args(_DTYPES[dt], act, m, n, k, x2.data_ptr(), ldx, w2.data_ptr(), ldw,
                          bp, rp, ldr, y.data_ptr(), n, zp, ldz, qp, ep), x)
    return y if keep is None else (y, z)


def linear_backward(dy: torch.Tensor, x: torch.Tensor | PackedActivation | None,
                    weight: torch.Tensor, z: torch.Tensor | PackedActivation | None = None,
                    activation: str = "none", need=("x", "weight", "bias")):
    """Gradients of :func:`linear`: ``(dx, dweight, dbias)``.

    ``dy`` is ``[..., n]``; ``x`` ``[..., k]`` and ``z`` ``[..., n]`` are what the
    forward pass kept, each a tensor or a :class:`PackedActivation`. z is needed
    with an activation, x for dweight. With ``"relu"`` z must not be packed (its
    derivative is z's sign, which values far below their block's largest lose).
    ``need`` names the gradients to compute; the others are None. The residual's
    gradient is ``dy`` itself. ``dz = dy * act'(z)`` is rounded to the layer's
    type before the two products (dbias sums it unrounded); each result is
    rounded once. An Inf among FP32 inputs may give NaN, as in :func:`linear`.
    Packed x is read back into the call's workspace in the layer's type.
    """
    if type(dy) is not _Tensor or dy.dtype not in _DTYPES or not dy.is_cuda or dy.requires_grad:
        _check("dy", dy)
    dt, dev = dy.dtype, dy.device
    if (type(weight) is not _Tensor or weight.dtype is not dt or weight.device != dev
            or weight.requires_grad):
        _check("weight", weight, dy)
    ds, ws = dy.shape, weight.shape
    if len(ws) != 2 or not ds or ds[-1] != ws[0]:
        raise ValueError(f"dy must be [..., n] and weight [n, k], got {tuple(ds)} and {tuple(ws)}")
    try:
        act = ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise _no_activation(activation) from None
    if type(need) is not tuple and not isinstance(need, str):
        need = tuple(need)  # an iterator gives its names once
    if isinstance(need, str) or not _NEED.issuperset(need):
        raise ValueError(f"need must name some of 'x', 'weight' and 'bias', got {need!r}")
    if _level._current_level >= 0:
        _refuse_tangents(dy=dy, weight=weight, x=x if "weight" in need else None,
                         z=z if act else None)
    n, k = ws
    lead = (ds[0],) if len(ds) == 2 else tuple(ds[:-1])
    dy2, m, lddy = _rows(dy, ds, n)
    w2, _, ldw = _rows(weight, ws, k)
    xp = ldx = xq = xe = zp = ldz = zq = ze = dxp = dwp = dbp = 0
    dx = dw = db = None
    if "weight" in need:
        if isinstance(x, PackedActivation):
            _check_packed("x", x, dy, (*lead, k))
            xcodes, xexps = _contiguous(x)
            if k:
                xq, xe = xcodes.data_ptr(), xexps.data_ptr()
        else:
            if x is None:
                raise ValueError("x is needed for the weight's gradient")
            if (type(x) is not _Tensor or x.dtype is not dt or x.device != dev
                    or x.requires_grad):
                _check("x", x, dy)
            xs = x.shape
            if xs != (*lead, k):
                raise ValueError(f"x must be {(*lead, k)}, got {tuple(xs)}")
            x2, _, ldx = _rows(x, xs, k)
            xp = x2.data_ptr()
        dw = dy.new_empty(n, k)
        dwp = dw.data_ptr()
    if act:
        if isinstance(z, PackedActivation):
            if activation == "relu":
                raise ValueError("relu's gradient needs z as a tensor: packed, small values lose "
                                 "their sign")
            _check_packed("z", z, dy, (*lead, n))
            zcodes, zexps = _contiguous(z)
            zq, ze = zcodes.data_ptr(), zexps.data_ptr()
        else:
            if z is None:
                raise ValueError(f"z is needed for the gradient of {activation!r}")
            if (type(z) is not _Tensor or z.dtype is not dt or z.device != dev
                    or z.requires_grad):
                _check("z", z, dy)
            zs = z.shape
            if zs != ds:
                raise ValueError(f"z must be {tuple(ds)}, got {tuple(zs)}")
            z2, _, ldz = _rows(z, zs, n)
            zp = z2.data_ptr()
    if "x" in need:
        dx = dy.new_empty(*lead, k)
        dxp = dx.data_ptr()
    if "bias" in need:
        db = dy.new_empty(n)
        dbp = db.data_ptr()
    L = _lib._lib or _lib.lib()
    _run(L.qrbl_linear_backward, L.qrbl_linear_backward_workspace_bytes,
         _backward_args(_DTYPES[dt], act, m, n, k, dy2.data_ptr(), lddy, xp, ldx, xq, xe,
                        w2.data_ptr(), ldw, zp, ldz, zq, ze, dxp, k, dwp, k, dbp), dy, True)
    return dx, dw, db


def _empty_packed(shape: tuple, like: torch.Tensor) -> PackedActivation:
    blocks = -(-shape[-1] // PACK_BLOCK)
    return PackedActivation(like.new_empty(*shape, dtype=torch.int8),
                            like.new_empty(*shape[:-1], blocks, dtype=torch.int8), like.dtype)


def _on(like: torch.Tensor, call, *args) -> None:
    index = like.get_device()
    if index != _current_device():
        with torch.cuda.device(index):
            return _on(like, call, *args)
    rc = call(*args, _raw_stream(index))
    if rc != _OK:
        _lib.check(rc)


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """``x [..., c]`` (float32, float16 or bfloat16) in 8 bits a value.

    Each 32 values of a row share the step ``2**e``, the smallest with
    ``max |x| <= 127 * 2**e`` (e from -126 to 122, float16 from -24 to 10), and
    are rounded to its nearest multiple (ties to even): the error is at most
    half a step, 1/127 of the block's largest value (one step where e is at its
    upper end, which only the type's largest values reach). Inf and NaN become
    NaN and do not affect the other values.
    """
    if type(x) is not _Tensor or x.dtype not in _DTYPES or not x.is_cuda or x.requires_grad:
        _check("x", x)
    if x.dim() < 1:
        raise ValueError("x must be [..., c], got a scalar")
    if _level._current_level >= 0:
        _refuse_tangents(x=x)
    shape = x.shape
    p = _empty_packed(shape, x)
    if x.numel():
        x2, rows, ld = _rows(x, shape, shape[-1])
        _on(x, _lib.lib().qrbl_pack, _DTYPES[x.dtype], x2.data_ptr(), ld, rows, shape[-1],
            p.codes.data_ptr(), p.exponents.data_ptr())
    return p


def unpack_activation(packed: PackedActivation) -> torch.Tensor:
    """The tensor that ``packed`` stands for, in the type it was packed from."""
    if not isinstance(packed, PackedActivation):
        raise TypeError(f"packed must be a PackedActivation, got {type(packed).__name__}")
    codes, exps, dtype = packed
    if dtype not in _DTYPES:
        raise TypeError(f"packed.dtype must be float32, float16 or bfloat16, got {dtype}")
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda:
        raise ValueError("packed.codes must be a CUDA tensor (libqrb200 has no CPU path)")
    shape = codes.shape
    if not shape:
        raise ValueError("packed.codes must be [..., c], got a scalar")
    x = codes.new_empty(*shape, dtype=dtype)
    _check_packed("packed", packed, x, shape)
    if x.numel():
        codes, exps = _contiguous(packed)
        cols = shape[-1]
        _on(x, _lib.lib().qrbl_unpack, _DTYPES[dtype], codes.data_ptr(), exps.data_ptr(),
            x.numel() // cols, cols, x.data_ptr(), cols)
    return x
