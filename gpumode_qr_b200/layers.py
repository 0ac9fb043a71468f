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
the same bits every time. They are plain functions, like the rest of the
library: autograd does not record them, and arguments that require a gradient
are refused while gradients are enabled (call them under ``torch.no_grad()``
or from an ``autograd.Function``).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
#: Values of a row that share one exponent in the packed form.
PACK_BLOCK = 32

_I64, _P = ctypes.c_int64, ctypes.c_void_p


class _LinearArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("activation", ctypes.c_int32),
                ("m", _I64), ("n", _I64), ("k", _I64),
                ("x", _P), ("ldx", _I64), ("w", _P), ("ldw", _I64), ("bias", _P),
                ("residual", _P), ("ldr", _I64), ("y", _P), ("ldy", _I64), ("z", _P),
                ("ldz", _I64), ("z_codes", _P), ("z_exponents", _P)]


class _BackwardArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("activation", ctypes.c_int32),
                ("m", _I64), ("n", _I64), ("k", _I64),
                ("dy", _P), ("lddy", _I64), ("x", _P), ("ldx", _I64), ("x_codes", _P),
                ("x_exponents", _P), ("w", _P), ("ldw", _I64), ("z", _P), ("ldz", _I64),
                ("z_codes", _P), ("z_exponents", _P), ("dx", _P), ("lddx", _I64), ("dw", _P),
                ("lddw", _I64), ("dbias", _P)]


class PackedActivation(NamedTuple):
    """A tensor in 8 bits: ``codes`` int8 [..., c] and ``exponents`` int8
    [..., ceil(c / 32)]; the values of columns 32 j .. 32 j + 31 are
    ``codes * 2**exponents[..., j]``, exact in ``dtype``, the type packed.
    The code -128 stands for NaN (and for Inf, which comes back as NaN)."""

    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype


def _check(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
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


def _check_packed(name: str, p: PackedActivation, like: torch.Tensor, shape: tuple) -> None:
    if p.dtype != like.dtype:
        raise TypeError(f"{name} was packed from {p.dtype}, the layer is {like.dtype}")
    want = (*shape[:-1], -(-shape[-1] // PACK_BLOCK))
    for part, t, s in (("codes", p.codes, shape), ("exponents", p.exponents, want)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int8:
            raise TypeError(f"{name}.{part} must be an int8 tensor")
        if t.device != like.device:
            raise ValueError(f"{name}.{part} must be on {like.device}, got {t.device}")
        if tuple(t.shape) != tuple(s):
            raise ValueError(f"{name}.{part} must be {tuple(s)}, got {tuple(t.shape)}")


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t as [rows, cols] with unit column stride and rows that do not overlap
    (copying only if needed)."""
    if t.dim() != 2:
        t = t.reshape(-1, cols) if cols else t.new_empty((t.shape[:-1].numel(), 0))
    s = t.stride()
    if (s[1] != 1 and cols > 1) or (s[0] < cols and t.shape[0] > 1):
        t = t.contiguous()
    return t


def _activation(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {name!r}") from None


def _run(size, call, args, dev: torch.device) -> None:
    ref = ctypes.byref(args)
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _run(size, call, args, dev)
    need = size(ref)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.check(call(ref, ws.data_ptr() if need else None, need,
                    torch.cuda.current_stream(dev).cuda_stream))


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, activation: str = "none",
           keep: str | None = None):
    """``y = act(x @ weight.T + bias) + residual`` in one product kernel.

    ``x`` is ``[..., k]``, ``weight`` ``[n, k]``, ``bias`` ``[n]``, ``residual``
    ``[..., n]``, all float32, float16 or bfloat16 (one type) on one CUDA device,
    any strides. ``activation`` is ``"none"``, ``"relu"``, ``"gelu"``,
    ``"gelu_tanh"`` or ``"silu"``. Sums are FP32 (FP32 inputs keep their 24
    bits: no TF32); y is rounded once.

    ``keep`` also returns the pre-activation ``z = x @ weight.T + bias`` for
    :func:`linear_backward`: ``"plain"`` as a tensor like y, ``"packed"`` as a
    :class:`PackedActivation` (8 bits a value, written from the FP32 sums).
    Returns ``y``, or ``(y, z)`` with ``keep``.
    """
    _check("x", x)
    _check("weight", weight, x)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., k] and weight [n, k], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    act = _activation(activation)
    n, k = weight.shape
    shape = (*x.shape[:-1], n)
    x2, w2 = _rows(x, k), _rows(weight, k)
    m = x2.shape[0]
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    a = _LinearArgs(_DTYPES[x.dtype], act, m, n, k, x2.data_ptr(), x2.stride(0), w2.data_ptr(),
                    w2.stride(0), None, None, 0, y.data_ptr(), n)
    if bias is not None:
        _check("bias", bias, x)
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be ({n},), got {tuple(bias.shape)}")
        bias = bias.contiguous()
        a.bias = bias.data_ptr()
    if residual is not None:
        _check("residual", residual, x)
        if tuple(residual.shape) != shape:
            raise ValueError(f"residual must be {shape}, got {tuple(residual.shape)}")
        residual = _rows(residual, n)
        a.residual, a.ldr = residual.data_ptr(), residual.stride(0)
    z = None
    if keep == "plain":
        z = torch.empty(shape, dtype=x.dtype, device=x.device)
        a.z, a.ldz = z.data_ptr(), n
    elif keep == "packed":
        z = _empty_packed(shape, x)
        a.z_codes, a.z_exponents = z.codes.data_ptr(), z.exponents.data_ptr()
    elif keep is not None:
        raise ValueError(f"keep must be None, 'plain' or 'packed', got {keep!r}")
    if m and n:
        L = _lib.lib()
        _run(L.qrbl_linear_workspace_bytes, L.qrbl_linear, a, x.device)
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
    rounded once.
    """
    _check("dy", dy)
    _check("weight", weight, dy)
    if weight.dim() != 2 or dy.dim() < 1 or dy.shape[-1] != weight.shape[0]:
        raise ValueError(f"dy must be [..., n] and weight [n, k], got {tuple(dy.shape)} and "
                         f"{tuple(weight.shape)}")
    act = _activation(activation)
    if isinstance(need, str) or not set(need) <= {"x", "weight", "bias"}:
        raise ValueError(f"need must name some of 'x', 'weight' and 'bias', got {need!r}")
    n, k = weight.shape
    lead = tuple(dy.shape[:-1])
    dy2, w2 = _rows(dy, n), _rows(weight, k)
    m = dy2.shape[0]
    a = _BackwardArgs(_DTYPES[dy.dtype], act, m, n, k, dy2.data_ptr(), dy2.stride(0))
    a.w, a.ldw = w2.data_ptr(), w2.stride(0)
    held = []  # views and copies the call reads
    if "weight" in need:
        if isinstance(x, PackedActivation):
            _check_packed("x", x, dy, (*lead, k))
            codes, exps = x.codes.contiguous(), x.exponents.contiguous()
            held += [codes, exps]
            if k:
                a.x_codes, a.x_exponents = codes.data_ptr(), exps.data_ptr()
        else:
            if x is None:
                raise ValueError("x is needed for the weight's gradient")
            _check("x", x, dy)
            if tuple(x.shape) != (*lead, k):
                raise ValueError(f"x must be {(*lead, k)}, got {tuple(x.shape)}")
            x2 = _rows(x, k)
            held.append(x2)
            a.x, a.ldx = x2.data_ptr(), x2.stride(0)
    if act:
        if isinstance(z, PackedActivation):
            if activation == "relu":
                raise ValueError("relu's gradient needs z as a tensor: packed, small values lose "
                                 "their sign")
            _check_packed("z", z, dy, (*lead, n))
            codes, exps = z.codes.contiguous(), z.exponents.contiguous()
            held += [codes, exps]
            a.z_codes, a.z_exponents = codes.data_ptr(), exps.data_ptr()
        else:
            if z is None:
                raise ValueError(f"z is needed for the gradient of {activation!r}")
            _check("z", z, dy)
            if tuple(z.shape) != (*lead, n):
                raise ValueError(f"z must be {(*lead, n)}, got {tuple(z.shape)}")
            z2 = _rows(z, n)
            held.append(z2)
            a.z, a.ldz = z2.data_ptr(), z2.stride(0)
    dx = dw = db = None
    if "x" in need:
        dx = torch.empty((*lead, k), dtype=dy.dtype, device=dy.device)
        a.dx, a.lddx = dx.data_ptr(), k
    if "weight" in need:
        dw = torch.empty((n, k), dtype=dy.dtype, device=dy.device)
        a.dw, a.lddw = dw.data_ptr(), k
    if "bias" in need:
        db = torch.empty((n,), dtype=dy.dtype, device=dy.device)
        a.dbias = db.data_ptr()
    L = _lib.lib()
    _run(L.qrbl_linear_backward_workspace_bytes, L.qrbl_linear_backward, a, dy.device)
    return dx, dw, db


def _empty_packed(shape: tuple, like: torch.Tensor) -> PackedActivation:
    return PackedActivation(
        torch.empty(shape, dtype=torch.int8, device=like.device),
        torch.empty((*shape[:-1], -(-shape[-1] // PACK_BLOCK)), dtype=torch.int8,
                    device=like.device),
        like.dtype)


def _on(dev: torch.device, call, *args) -> None:
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _on(dev, call, *args)
    _lib.check(call(*args, torch.cuda.current_stream(dev).cuda_stream))


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """``x [..., c]`` (float32, float16 or bfloat16) in 8 bits a value.

    Each 32 values of a row share the step ``2**e``, the smallest with
    ``max |x| <= 127 * 2**e`` (e from -126 to 122, float16 from -24 to 10), and
    are rounded to its nearest multiple (ties to even): the error is at most
    half a step, 1/127 of the block's largest value (one step where e is at its
    upper end, which only the type's largest values reach). Inf and NaN become
    NaN and do not affect the other values.
    """
    _check("x", x)
    if x.dim() < 1:
        raise ValueError("x must be [..., c], got a scalar")
    p = _empty_packed(tuple(x.shape), x)
    if x.numel():
        x2 = _rows(x, x.shape[-1])
        _on(x.device, _lib.lib().qrbl_pack, _DTYPES[x.dtype], x2.data_ptr(), x2.stride(0),
            x2.shape[0], x2.shape[1], p.codes.data_ptr(), p.exponents.data_ptr())
    return p


def unpack_activation(packed: PackedActivation) -> torch.Tensor:
    """The tensor that ``packed`` stands for, in the type it was packed from."""
    if not isinstance(packed, PackedActivation):
        raise TypeError(f"packed must be a PackedActivation, got {type(packed).__name__}")
    if packed.dtype not in _DTYPES:
        raise TypeError(f"packed.dtype must be float32, float16 or bfloat16, got {packed.dtype}")
    codes = packed.codes
    if not isinstance(codes, torch.Tensor) or not codes.is_cuda:
        raise ValueError("packed.codes must be a CUDA tensor (libqrb200 has no CPU path)")
    if codes.dim() < 1:
        raise ValueError("packed.codes must be [..., c], got a scalar")
    x = torch.empty(codes.shape, dtype=packed.dtype, device=codes.device)
    _check_packed("packed", packed, x, tuple(codes.shape))
    if x.numel():
        codes, exps = codes.contiguous(), packed.exponents.contiguous()
        cols = x.shape[-1]
        _on(x.device, _lib.lib().qrbl_unpack, _DTYPES[x.dtype], codes.data_ptr(),
            exps.data_ptr(), x.numel() // cols, cols, x.data_ptr(), cols)
    return x
