"""GPU tests of the linear-layer operators against 64-bit formulas.

Tolerances, elementwise, from arithmetic (u = half a step of the output type):

* a product's FP32 accumulation over k terms, S the sum of |x_i w_i|: the tensor
  core truncates, so every add costs at most one FP32 step 2^-23 of a partial
  sum (at most S). 16-bit layers: k / 16 adds per chain and fewer than 16 within
  an MMA; FP32 layers: chains of 256 values (4 x 4 adds, counted with their
  small products as 24), k / 256 adds of chains, and three dropped products of
  2^-24: ``ACC * S``.
* an activation: slope at most 1.13, its own evaluation below 1e-6 |z| + 1e-7.
* dz is rounded once more to the layer's type (u relative, and for float16 half
  a subnormal step 2^-25): u * (|dz| @ |w|) in dx, likewise in dW; its
  derivative factor is exact to 2e-6 (at most 1.13, so 2e-6 |dy| absolute).
* packing: half a step 2^e (a whole step at the largest exponent).
"""

from __future__ import annotations

import itertools
import math
import threading

import pytest
import torch

from gpumode_qr_b200 import _lib, api, checker, layers

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, HF, FP]
IDS = ["bf16", "fp16", "fp32"]
ACTS = list(layers.ACTIVATIONS)
STEP = 2.0**-23
SUB = {BF: 2.0**-134, HF: 2.0**-25, FP: 2.0**-150}  # half a subnormal step


def u(dt):
    return torch.finfo(dt).eps / 2


def acc(dt, k):
    return STEP * ((24 + k / 256 + 2) if dt == FP else (k / 16 + 18))


def rnd(shape, seed, dt, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dt).to(DEV)


def act64(z, act):
    """(act(z), act'(z)) in the precision of z."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        p = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z**3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def near(got, want, tol, what=""):
    assert got.shape == want.shape
    d = (got.double() - want).abs() - tol
    assert torch.isfinite(got.double()).all(), what
    worst = d.max().item() if d.numel() else -1.0
    assert worst <= 0, f"{what}: over the bound by {worst:.3g} of {tol.flatten()[d.argmax()]:.3g}"


def check_forward(x, w, b, r, act, y, z=None, dt=None):
    dt = dt or x.dtype
    x, w = x.double(), w.double()
    z64 = x @ w.mT
    s = x.abs() @ w.abs().mT
    if b is not None:
        z64, s = z64 + b.double(), s + b.double().abs()
    za = acc(dt, x.shape[-1]) * s
    y64 = act64(z64, act)[0]
    ya = 1.13 * za + (1e-6 * z64.abs() + 1e-7 if act not in ("none", "relu") else 0)
    if r is not None:
        y64 = y64 + r.double()
        ya = ya + 2.0**-23 * (y64.abs() + r.double().abs())
    near(y, y64, u(dt) * y64.abs() * 1.0001 + ya * (1 + u(dt)) + SUB[dt], "y")
    if z is not None:
        near(z, z64, u(dt) * z64.abs() * 1.0001 + za * (1 + u(dt)) + SUB[dt], "z")
    return z64, za


# ---------------------------------------------------------------------------
# forward
# ---------------------------------------------------------------------------
# one row, one column, one value; odd sizes; edges of every tile width; a long
# reduction with few tiles (split); tall and wide
SHAPES = [(1, 1, 1), (1, 4096, 512), (2, 33, 7), (3, 64, 64), (5, 200, 1000), (16, 512, 512),
          (33, 65, 129), (128, 256, 64), (129, 257, 72), (200, 96, 4096), (300, 1000, 40),
          (777, 130, 355), (1024, 513, 136), (8, 8, 8192), (64, 2048, 2048)]


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_sizes(m, n, k, dt):
    x, w = rnd((m, k), 1, dt), rnd((n, k), 2, dt, k**-0.5)
    b, r = rnd((n,), 3, dt), rnd((m, n), 4, dt)
    y = api.linear(x, w, b, r, "silu")
    check_forward(x, w, b, r, "silu", y)
    check_forward(x, w, None, None, "none", api.linear(x, w))


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(3, 96, 64), (150, 264, 96), (20, 64, 4096)])
def test_linear_activations(m, n, k, act, dt):
    x, w, b = rnd((m, k), 5, dt), rnd((n, k), 6, dt, 3 * k**-0.5), rnd((n,), 7, dt)
    y, z = api.linear(x, w, b, None, act, keep="plain")
    check_forward(x, w, b, None, act, y, z)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 32, 16), (3, 40, 64), (130, 264, 96), (257, 77, 64),
                                   (20, 65, 4096), (6, 4096, 1024)])
def test_linear_keeps_z_packed(m, n, k, dt):
    x, w, b, r = rnd((m, k), 8, dt), rnd((n, k), 9, dt, k**-0.5), rnd((n,), 10, dt), rnd((m, n), 11, dt)
    y, p = api.linear(x, w, b, r, "gelu", keep="packed")
    z64, za = check_forward(x, w, b, r, "gelu", y)
    assert p.codes.shape == (m, n) and p.exponents.shape == (m, -(-n // 32)) and p.dtype == dt
    s = torch.ldexp(torch.ones(p.exponents.shape, dtype=torch.float64, device=DEV), p.exponents.int())
    step = s.repeat_interleave(32, dim=1)[:, :n]
    got = api.unpack_activation(p)
    near(got, z64, 0.5 * step + za, "packed z")
    # the step is the smallest that holds the block's largest value
    amax = torch.nn.functional.pad(z64.abs(), (0, -n % 32)).view(m, -1, 32).amax(-1)
    slack = torch.nn.functional.pad(za, (0, -n % 32)).view(m, -1, 32).amax(-1)
    assert (amax - slack <= 127 * s).all() and (amax + slack > 63.5 * s).all()


def test_packed_saturates_beyond_float16():
    # z = 1e5 is finite in FP32 but not in float16: kept as the largest value
    # the packed form has there, not as Inf
    x, w = torch.full((2, 16), 250.0, device=DEV, dtype=HF), torch.full((32, 16), 25.0, device=DEV, dtype=HF)
    y, p = api.linear(x, w, activation="gelu", keep="packed")
    assert torch.isinf(y).all()
    assert (api.unpack_activation(p) == 63 * 1024).all()


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_strides_and_leading_dimensions(dt):
    m, n, k = 37, 48, 80
    big = rnd((m, 3 * k + 5), 12, dt)
    wbig = rnd((n + 3, k + 9), 13, dt, k**-0.5)
    rbig = rnd((m, n + 7), 14, dt)
    bbig = rnd((2 * n,), 15, dt)
    for x, w in ((big[:, 3:3 + k], wbig[1:1 + n, 2:2 + k]),          # rows not 16-byte aligned
                 (big[:, 8:8 + k], wbig[:n, :k]),
                 (big[:, ::3][:, :k], wbig[:n, :k]),                 # column stride 3
                 (big[:, :k].t().contiguous().t(), wbig[:n, :k]),    # column-major
                 (big[:1, :k].expand(m, k), wbig[:n, :k])):          # one row broadcast
        for b, r in ((bbig[1:1 + n], rbig[:, 1:1 + n]), (bbig[::2], rbig[:, :n])):
            y = api.linear(x, w, b, r, "relu")
            check_forward(x, w, b, r, "relu", y)
    x4 = rnd((2, 3, 5, k), 16, dt)
    y4 = api.linear(x4, wbig[:n, :k])
    assert y4.shape == (2, 3, 5, n)
    assert torch.equal(y4.reshape(30, n), api.linear(x4.reshape(30, k), wbig[:n, :k]))
    y1 = api.linear(x4[0, 0, 0], wbig[:n, :k], residual=y4[0, 0, 0])
    assert y1.shape == (n,)
    perm = x4.permute(2, 0, 1, 3)
    assert torch.equal(api.linear(perm, wbig[:n, :k]), y4.permute(2, 0, 1, 3))


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_empty(dt):
    w = rnd((6, 8), 17, dt)
    assert api.linear(torch.empty(0, 8, device=DEV, dtype=dt), w).shape == (0, 6)
    assert api.linear(rnd((3, 8), 1, dt), torch.empty(0, 8, device=DEV, dtype=dt)).shape == (3, 0)
    x0, w0 = torch.empty(3, 0, device=DEV, dtype=dt), torch.empty(70, 0, device=DEV, dtype=dt)
    b, r = rnd((70,), 18, dt), rnd((3, 70), 19, dt)
    y, z = api.linear(x0, w0, b, r, "silu", keep="plain")
    assert torch.equal(z, b.expand(3, 70))
    check_forward(x0, w0, b, r, "silu", y, z)
    y, p = api.linear(x0, w0, b, r, "silu", keep="packed")
    assert torch.equal(api.unpack_activation(p), api.unpack_activation(api.pack_activation(b.expand(3, 70))))


def test_bias_at_any_alignment():
    x, w = rnd((300, 128), 27, BF), rnd((160, 128), 28, BF, 0.1)
    wide = rnd((400,), 29, BF)
    for first in (0, 1, 3, 7):
        b = wide[first:first + 160]
        assert torch.equal(api.linear(x, w, b), api.linear(x, w, b.clone()))
    check_forward(x, w, wide[1:161], None, "none", api.linear(x, w, wide[1:161]))


def test_negated_views():
    """``c.conj().imag`` is a real tensor whose memory holds the values negated."""
    c = torch.complex(rnd((5, 3), 90, FP), rnd((5, 3), 91, FP))
    for cols in (1, 3):
        x, w = c[:, :cols].conj().imag, rnd((4, cols), 92, FP)
        assert x.is_neg()
        check_forward(x, w, None, None, "none", api.linear(x, w))
        p = api.pack_activation(x)
        assert torch.equal(p.codes, api.pack_activation(x.clone()).codes)
    b = c[:1, 0].conj().imag
    w = rnd((1, 3), 93, FP)
    check_forward(c.real, w, b, None, "none", api.linear(c.real, w, b))


@pytest.mark.parametrize("m,n,k", [(60_001, 64, 72), (200_000, 40, 32)])
def test_long_batch_through_a_narrow_layer(m, n, k):
    # one long tile of dW beside hundreds of short ones of dx; thousands of bias sums
    dy, x, w = rnd((m, n), 48, BF), rnd((m, k), 49, BF), rnd((n, k), 50, BF)
    check_backward(dy, x.double(), w, None, "none", *api.linear_backward(dy, x, w))


def test_linear_non_finite_rows_stay_in_their_row():
    for dt in TYPES:
        x, w = rnd((70, 96), 20, dt), rnd((130, 96), 21, dt, 0.1)
        clean, _ = api.linear(x, w, activation="gelu", keep="packed")
        x[3, 5], x[40, 7] = float("nan"), float("inf")
        y, p = api.linear(x, w, activation="gelu", keep="packed")
        rows = torch.ones(70, dtype=torch.bool, device=DEV)
        rows[3] = rows[40] = False
        assert torch.equal(y[rows], clean[rows])
        assert y[3].isnan().all()
        assert not torch.isfinite(y[40][(w[:, 7] > 0)]).any()
        back = api.unpack_activation(p)
        assert back[3].isnan().all() and back[rows].isfinite().all()


def test_linear_in_place_residual():
    x, w = rnd((100, 64), 22, BF), rnd((72, 64), 23, BF, 0.1)
    r = rnd((100, 72), 24, BF)
    want = api.linear(x, w, None, r, "gelu")
    out = r.clone()
    a = layers._linear_args(2, 2, 100, 72, 64, x.data_ptr(), 64, w.data_ptr(), 64, 0,
                            out.data_ptr(), 72, out.data_ptr(), 72, 0, 0, 0, 0)
    assert _lib.lib().qrbl_linear(a, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (130, 100, 72), (16, 48, 4096), (21, 70, 128)])
def test_rows_and_columns_outside_stay_as_they_were(m, n, k, dt):
    # outputs inside larger buffers: only [m, n] is written
    L, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    x, w = rnd((m, k), 25, dt), rnd((n, k), 26, dt, 0.1)
    want = api.linear(x, w)
    for ldy in (n, n + 8, n + 3):
        y = torch.full((m + 200, ldy), 7.0, device=DEV, dtype=dt)
        a = layers._linear_args(layers._DTYPES[dt], 0, m, n, k, x.data_ptr(), k, w.data_ptr(), k,
                                0, 0, 0, y.data_ptr(), ldy, 0, 0, 0, 0)
        need = L.qrbl_linear_workspace_bytes(a)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        assert L.qrbl_linear(a, ws.data_ptr(), need, s) == 0
        assert torch.equal(y[:m, :n], want)
        assert (y[m:] == 7).all() and (y[:, n:] == 7).all()


# ---------------------------------------------------------------------------
# backward
# ---------------------------------------------------------------------------
def check_backward(dy, x64, w, z64, act, dx, dw, db):
    dt, m = dy.dtype, dy.shape[0]
    dy, w = dy.double(), w.double()
    dz = dy * act64(z64, act)[1] if act != "none" else dy
    # dz as the products see it: rounded (or, FP32, split), its factor off by 2e-6
    e = (0 if act == "none" else u(dt) if dt != FP else 0) * dz.abs()
    e = e + (0 if act == "none" else 2e-6 * dy.abs() + SUB[dt])
    if dx is not None:
        s = dz.abs() @ w.abs()
        tol = (e @ w.abs()) + acc(dt, dy.shape[1]) * s
        want = dz @ w
        near(dx, want, u(dt) * want.abs() * 1.0001 + tol * (1 + u(dt)) + SUB[dt], "dx")
    if dw is not None:
        s = dz.abs().mT @ x64.abs()
        tol = (e.mT @ x64.abs()) + acc(dt, m) * s
        want = dz.mT @ x64
        near(dw, want, u(dt) * want.abs() * 1.0001 + tol * (1 + u(dt)) + SUB[dt], "dw")
    if db is not None:  # FP32 sums of 64 rows and of the blocks
        want = dz.sum(0)
        tol = (2e-6 * dy.abs()).sum(0) + 2.0**-24 * (80 + m / 64) * dz.abs().sum(0)
        near(db, want, u(dt) * want.abs() * 1.0001 + tol * (1 + u(dt)) + SUB[dt], "db")


BSHAPES = [(1, 1, 1), (2, 33, 70), (64, 64, 64), (129, 257, 72), (999, 177, 530), (5, 1000, 16),
           (4096, 32, 48), (300, 513, 1024)]


@pytest.mark.parametrize("kept", ["plain", "packed"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", BSHAPES)
def test_backward_sizes(m, n, k, dt, kept):
    dy, x, w, z = (rnd((m, n), 30, dt), rnd((m, k), 31, dt), rnd((n, k), 32, dt, n**-0.5),
                   rnd((m, n), 33, dt, 1.5))
    if kept == "packed":
        x, z = api.pack_activation(x), api.pack_activation(z)
        x64, z64 = api.unpack_activation(x).double(), api.unpack_activation(z).double()
    else:
        x64, z64 = x.double(), z.double()
    for act in ("gelu", "none"):
        dx, dw, db = api.linear_backward(dy, x, w, z if act != "none" else None, act)
        check_backward(dy, x64, w, z64, act, dx, dw, db)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("act,kept", [(a, p) for a in ACTS for p in ("plain", "packed")
                                      if (a, p) not in (("relu", "packed"), ("none", "packed"))])
def test_backward_activations(act, kept, dt):
    m, n, k = 70, 96, 40
    dy, x, w, z = rnd((m, n), 34, dt), rnd((m, k), 35, dt), rnd((n, k), 36, dt), rnd((m, n), 37, dt, 3.0)
    if kept == "packed":
        zp = api.pack_activation(z)
        z64 = api.unpack_activation(zp).double()
    else:
        zp, z64 = z, z.double()
    check_backward(dy, x.double(), w, z64, act, *api.linear_backward(dy, x, w, zp, act))


def test_backward_far_pre_activations():
    # saturated and overflowing z: the derivative is 0 or 1, never NaN
    z = torch.tensor([-3e38, -1e20, -1e4, -200.0, -90.0, -30.0, 0.0, 30.0, 90.0, 1e4, 1e20, 3e38],
                     device=DEV)
    want = (z > 0).float() + 0.5 * (z == 0).float()
    for dt in (FP, BF):
        zz = z.to(dt).reshape(1, -1)
        dy = torch.ones_like(zz)
        eye = torch.eye(12, device=DEV, dtype=dt)
        for act in ("gelu", "gelu_tanh", "silu"):
            dx, _, db = api.linear_backward(dy, None, eye, zz, act, need=("x", "bias"))
            assert (dx.float()[0] - want).abs().max() < 1e-9
            assert (db.float() - want).abs().max() < 1e-9
            y = api.linear(zz, eye, activation=act)
            # z * 1 is a product with zeros beside it: finite z only
            assert (y.float()[0, 3:10] - (z * want)[3:10].to(dt).float()).abs().max() < 1e-9


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp32"])
def test_backward_packed_far_and_non_finite(dt):
    # packed z at the ends of the exponents' range: derivative 0, 1 / 2 or 1; a
    # block with NaN or Inf keeps the others' values; NaN stays in its row of dx
    z = torch.zeros(4, 96, dtype=dt)
    z[0, :32], z[0, 32:64], z[0, 64:] = 3e38, -3e38, 1e-37
    z[1] = torch.linspace(-60, 60, 96).to(dt)
    z[2], z[2, 40], z[2, 41] = 1.0, float("nan"), float("inf")
    zp = api.pack_activation(z.to(DEV))
    back = api.unpack_activation(zp).double()
    assert back[2].isnan().sum() == 2 and (back[2][~back[2].isnan()] == 1).all()
    dy, eye = torch.ones(4, 96, device=DEV, dtype=dt), torch.eye(96, device=DEV, dtype=dt)
    for act in ("gelu", "gelu_tanh", "silu"):
        dx, _, db = api.linear_backward(dy, None, eye, zp, act, need=("x", "bias"))
        want = act64(back, act)[1]
        rows = [0, 1, 3]
        near(dx[rows], want[rows], u(dt) * 1.2 + 2e-6 + 0 * want[rows])
        assert dx[2].isnan().all()
        assert db.isnan().sum() == 2


@pytest.mark.parametrize("need", [c for r in range(4) for c in itertools.combinations(
    ("x", "weight", "bias"), r)])
def test_backward_computes_what_is_needed(need):
    m, n, k = 130, 72, 100
    dy, x, w, z = rnd((m, n), 38, BF), rnd((m, k), 39, BF), rnd((n, k), 40, BF), rnd((m, n), 41, BF)
    full = dict(zip(("x", "weight", "bias"), api.linear_backward(dy, x, w, z, "silu")))
    got = dict(zip(("x", "weight", "bias"),
                   api.linear_backward(dy, x if "weight" in need else None, w, z, "silu", need=need)))
    for name in full:
        assert torch.equal(got[name], full[name]) if name in need else got[name] is None


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_backward_strides(dt):
    m, n, k = 65, 40, 56
    big = rnd((m, 400), 42, dt)
    wbig = rnd((n, k + 5), 43, dt)
    for dy, x, z, w in ((big[:, 1:1 + n], big[:, 100:100 + k], big[:, 203:203 + n], wbig[:, 3:3 + k]),
                        (big[:, :2 * n:2], big[:, 96:96 + k], big[:, 200:200 + n], wbig[:, :k]),
                        (big[:1, :n].expand(m, n), big[:, 96:96 + k], big[:, 200:200 + n], wbig[:, :k])):
        check_backward(dy, x.double(), w, z.double(), "gelu_tanh",
                       *api.linear_backward(dy, x, w, z, "gelu_tanh"))
        check_backward(dy, x.double(), w, z.double(), "none", *api.linear_backward(dy, x, w))
    dy3, x3 = rnd((3, 4, n), 44, dt), rnd((3, 4, k), 45, dt)
    dx, dw, db = api.linear_backward(dy3, x3, wbig[:, :k])
    assert dx.shape == (3, 4, k) and dw.shape == (n, k) and db.shape == (n,)
    check_backward(dy3.reshape(12, n), x3.reshape(12, k).double(), wbig[:, :k], None, "none",
                   dx.reshape(12, k), dw, db)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_backward_empty(dt):
    w = rnd((6, 8), 46, dt)
    e = lambda *s: torch.empty(*s, device=DEV, dtype=dt)  # noqa: E731
    dx, dw, db = api.linear_backward(e(0, 6), e(0, 8), w, e(0, 6), "gelu")
    assert dx.shape == (0, 8) and (dw == 0).all() and (db == 0).all()
    dx, dw, db = api.linear_backward(e(3, 0), e(3, 8), e(0, 8), e(3, 0), "gelu")
    assert (dx == 0).all() and dx.shape == (3, 8) and dw.shape == (0, 8) and db.shape == (0,)
    dy = rnd((3, 6), 47, dt)
    dx, dw, db = api.linear_backward(dy, e(3, 0), e(6, 0))
    assert dx.shape == (3, 0) and dw.shape == (6, 0)
    near(db, dy.double().sum(0), 2e-6 * dy.double().abs().sum(0) + u(dt) * dy.double().sum(0).abs())
    xp, zp = api.pack_activation(e(0, 8)), api.pack_activation(e(0, 6))
    dx, dw, db = api.linear_backward(e(0, 6), xp, w, zp, "silu")
    assert (dw == 0).all() and (db == 0).all()


def test_backward_of_nothing_through_a_wide_layer():
    k = 2**29 + 24  # one row of dW is more than 2^31 bytes
    w = torch.empty(1, k, device=DEV)
    dw = api.linear_backward(w.new_empty(0, 1), w.new_empty(0, k), w, need=("weight",))[1]
    assert dw.shape == (1, k) and not dw.any()


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    # central differences of the FP64 formula's loss sum(y * c) around the FP32 inputs
    m, n, k = 4, 5, 6
    x, w, b, c = rnd((m, k), 50, FP), rnd((n, k), 51, FP), rnd((n,), 52, FP), rnd((m, n), 53, FP)
    _, z = api.linear(x, w, b, None, act, keep="plain")
    dx, dw, db = api.linear_backward(c, x, w, z, act)

    def loss(x, w, b):
        return (act64(x @ w.mT + b, act)[0] * c.double()).sum()

    args = [t.double() for t in (x, w, b)]
    for i, g in enumerate((dx, dw, db)):
        for j in range(g.numel()):
            h = 1e-5
            vals = []
            for sgn in (1, -1):
                moved = [t.clone() for t in args]
                moved[i].view(-1)[j] += sgn * h
                vals.append(loss(*moved).item())
            # h^2 / 6 * |third derivative| and cancellation are below 1e-8; FP32 results 1e-5
            assert abs((vals[0] - vals[1]) / (2 * h) - g.view(-1)[j].item()) < 3e-5


# ---------------------------------------------------------------------------
# packed form
# ---------------------------------------------------------------------------
def pack64(x):
    """Codes and exponents from the definition, in 64 bits on the CPU."""
    lo, hi = (-24, 10) if x.dtype == HF else (-126, 122)
    v = x.detach().cpu().double().reshape(-1, x.shape[-1])
    rows, c = v.shape
    v = torch.nn.functional.pad(v, (0, -c % 32)).view(rows, -1, 32)
    fin = torch.isfinite(v)
    amax = torch.where(fin, v, 0.0).abs().amax(-1)
    e = torch.full(amax.shape, lo)
    for p in range(lo, hi):  # the smallest step that holds amax
        e = torch.where(amax > 127 * 2.0**p, p + 1, e)
    e = e.clamp(lo, hi)
    most = torch.where(e == hi, 63.0, 127.0)[..., None]
    q = torch.where(fin, v, 0.0) / torch.ldexp(torch.ones(e.shape, dtype=torch.float64), e)[..., None]
    q = torch.minimum(torch.maximum(q.round(), -most), most)
    q = torch.where(fin, q, -128.0)
    return (q.view(rows, -1)[:, :c].to(torch.int8).reshape(x.shape),
            e.to(torch.int8).reshape(*x.shape[:-1], -1))


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 64), (4, 200), (1, 5000),
                                   (1000, 40), (130, 257), (2, 3, 48), (17,)])
def test_pack_is_the_definition(shape, dt):
    x = rnd(shape, 60, dt) * torch.exp(2 * rnd((*shape[:-1], 1), 61, FP)).to(dt)
    p = api.pack_activation(x)
    q, e = pack64(x)
    assert torch.equal(p.codes.cpu(), q) and torch.equal(p.exponents.cpu(), e)
    back = api.unpack_activation(p)
    want = torch.ldexp(q.double(), e.int().repeat_interleave(32, dim=-1)[..., :shape[-1]])
    assert back.dtype == dt and torch.equal(back.double().cpu(), want)
    assert torch.equal(api.unpack_activation(api.pack_activation(back)), back)  # nothing lost twice


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_pack_special_values(dt):
    big, tiny = torch.finfo(dt).max, torch.finfo(dt).smallest_normal
    rows = torch.zeros(12, 64, dtype=dt)
    rows[1] = big
    rows[2, ::2] = -big
    rows[3] = tiny
    rows[4, 3], rows[4, 4], rows[4, 5], rows[4, 6] = float("nan"), float("inf"), -float("inf"), 1.0
    rows[5] = float("inf")
    rows[6] = 127.0
    rows[7, :32] = torch.arange(32) * 0.5 + 0.25
    rows[7, 32] = 127 * 2.0**-7
    rows[8] = tiny / 4
    rows[9, 0], rows[9, 1:32] = 1.0, 2.0**-8  # half a step: to even, zero
    rows[10, 0], rows[10, 1:32] = 1.0, 3 * 2.0**-8
    rows[11] = -0.0
    p = api.pack_activation(rows.to(DEV))
    q, e = pack64(rows)
    assert torch.equal(p.codes.cpu(), q) and torch.equal(p.exponents.cpu(), e)
    back = api.unpack_activation(p).cpu()
    assert torch.equal(back.isnan(), ~rows.isfinite())
    assert not back.isinf().any()


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_pack_strides(dt):
    big = rnd((40, 300), 62, dt)
    for x in (big[:, 1:100], big[:, ::3], big.t(), big[:1].expand(40, 300), big[:, 8:136]):
        p = api.pack_activation(x)
        q, e = pack64(x)
        assert torch.equal(p.codes.cpu(), q) and torch.equal(p.exponents.cpu(), e)
    p = api.pack_activation(big)
    # codes and exponents that are views
    wide = api.PackedActivation(p.codes.repeat(1, 2)[:, :300], p.exponents.repeat(1, 2)[:, :10], dt)
    assert torch.equal(api.unpack_activation(wide), api.unpack_activation(p))
    assert api.pack_activation(torch.empty(0, 5, device=DEV, dtype=dt)).codes.shape == (0, 5)
    assert api.unpack_activation(api.pack_activation(torch.empty(3, 0, device=DEV, dtype=dt))).shape == (3, 0)


def test_offsets_beyond_32_bits():
    rows, cols = 70_001, 32_768  # 2.29e9 values
    x = torch.empty(rows, cols, device=DEV, dtype=BF)
    x.copy_(rnd((1, cols), 63, BF).expand(rows, cols))
    x[-1] = rnd((cols,), 64, BF)
    p = api.pack_activation(x)
    del x
    back = api.unpack_activation(p)
    for r in (0, 65_536, rows - 2, rows - 1):
        want = rnd((1, cols), 64 if r == rows - 1 else 63, BF)
        assert torch.equal(back[r:r + 1], api.unpack_activation(api.pack_activation(want)))
    del p, back
    m, n, k = 600_011, 4096, 64  # y and dy: 2.46e9 values
    xs, w = rnd((m, k), 65, BF), rnd((n, k), 66, BF, 0.125)
    y = api.linear(xs, w)
    for r in (slice(0, 200), slice(m - 200, m)):
        check_forward(xs[r], w, None, None, "none", y[r].contiguous())
    dx, _, _ = api.linear_backward(y, None, w, need=("x",))
    for r in (slice(0, 100), slice(m - 100, m)):
        check_backward(y[r].contiguous(), None, w, None, "none", dx[r].contiguous(), None, None)


# ---------------------------------------------------------------------------
# every way a product is cut
# ---------------------------------------------------------------------------
@pytest.fixture
def hooks():
    names = ("linear_cut", "linear_splits", "linear_rows")
    old = {k: _lib.get_config(k) for k in names}
    yield _lib.set_config
    for k, v in old.items():
        _lib.set_config(k, v)


CUTS = [2256, 2128, 1128, 1064]


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("splits", [0, 3])
@pytest.mark.parametrize("cut", CUTS)
def test_forward_cuts(cut, splits, dt, hooks):
    hooks("linear_cut", cut)
    hooks("linear_splits", splits)
    hooks("linear_rows", 0)
    # edges of the tiles, more tiles than SMs, aligned and unaligned rows
    for m, n, k in ((1, 40, 200), (257, 520, 200), (130, 264, 72), (131, 77, 45), (40, 24, 1000),
                    (3000, 1064, 96), (600, 333, 520)):
        x, w = rnd((m, k), 170, dt), rnd((n, k), 171, dt, k**-0.5)
        b, r = rnd((n,), 172, dt), rnd((m, n), 173, dt)
        y, z = api.linear(x, w, b, r, "silu", keep="plain")
        check_forward(x, w, b, r, "silu", y, z)
        check_forward(x, w, None, r, "none", api.linear(x, w, None, r))
        y, p = api.linear(x, w, b, r, "gelu_tanh", keep="packed")
        z64, za = check_forward(x, w, b, r, "gelu_tanh", y)
        s = torch.ldexp(torch.ones(p.exponents.shape, dtype=torch.float64, device=DEV), p.exponents.int())
        near(api.unpack_activation(p), z64, 0.5 * s.repeat_interleave(32, dim=1)[:, :n] + za, "packed z")


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("splits", [0, 3])
@pytest.mark.parametrize("cut", CUTS)
def test_backward_cuts(cut, splits, dt, hooks):
    hooks("linear_cut", cut)
    hooks("linear_splits", splits)
    # either product the longer one; more tiles than SMs in one or both
    for m, n, k in ((257, 136, 520), (1, 40, 24), (1000, 64, 1032), (64, 1000, 1032), (131, 77, 45),
                    (2500, 1100, 1300)):
        dy, x, w, z = (rnd((m, n), 174, dt), rnd((m, k), 175, dt), rnd((n, k), 176, dt, n**-0.5),
                       rnd((m, n), 177, dt))
        check_backward(dy, x.double(), w, z.double(), "silu", *api.linear_backward(dy, x, w, z, "silu"))
        check_backward(dy, x.double(), w, None, "none", *api.linear_backward(dy, x, w))


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_few_rows_and_tiles_agree(dt, hooks):
    m = 8 if dt == FP else 32
    for n, k in ((100, 72), (4096, 512), (33, 1000)):
        x, w = rnd((m, k), 178, dt), rnd((n, k), 179, dt, k**-0.5)
        b, r = rnd((n,), 180, dt), rnd((m, n), 181, dt)
        for rows in (m, 0):
            hooks("linear_rows", rows)
            check_forward(x, w, b, r, "gelu", api.linear(x, w, b, r, "gelu"))


@pytest.mark.parametrize("m,n,k", [(9, 512, 256), (13, 2048, 1024), (32, 70, 999), (33, 1000, 257),
                                   (64, 128, 128), (127, 33, 40), (128, 40, 8)])
def test_fp32_tokens_in_groups(m, n, k):
    """More than eight rows in FP32: groups of four or eight over the grid, the last one cut."""
    x, w = rnd((m, k), 182, FP), rnd((n, k), 183, FP, k**-0.5)
    b, r = rnd((n,), 184, FP), rnd((m, n), 185, FP)
    y, z = api.linear(x, w, b, r, "gelu", keep="plain")
    check_forward(x, w, b, r, "gelu", y, z)
    y, p = api.linear(x, w, b, r, "gelu", keep="packed")
    z64, z_err = check_forward(x, w, b, r, "gelu", y)
    half = torch.ldexp(torch.full(p.exponents.shape, 0.5, dtype=torch.float64, device=DEV),
                       p.exponents.int()).repeat_interleave(32, dim=1)[:, :n]
    near(api.unpack_activation(p), z64, half + z_err, "packed z")
    one = torch.cat([api.linear(x[i:i + 1], w, b, r[i:i + 1], "gelu") for i in (0, m // 2, m - 1)])
    check_forward(x[[0, m // 2, m - 1]], w, b, r[[0, m // 2, m - 1]], "gelu", one)


def test_z_kept_both_ways():
    # the C entry point may ask for z plain and packed at once
    for m, n, k in ((200, 160, 96), (4, 64, 64)):
        x, w = rnd((m, k), 182, BF), rnd((n, k), 183, BF, 0.1)
        y0, z0 = api.linear(x, w, None, None, "silu", keep="plain")
        y, z = torch.empty_like(y0), torch.empty_like(z0)
        p = layers._empty_packed((m, n), x)
        a = layers._linear_args(2, 4, m, n, k, x.data_ptr(), k, w.data_ptr(), k, 0, 0, 0,
                                y.data_ptr(), n, z.data_ptr(), n, p.codes.data_ptr(),
                                p.exponents.data_ptr())
        assert _lib.lib().qrbl_linear(a, None, 0, torch.cuda.current_stream().cuda_stream) == 0
        z64, za = check_forward(x, w, None, None, "silu", y, z)
        s = torch.ldexp(torch.ones(p.exponents.shape, dtype=torch.float64, device=DEV), p.exponents.int())
        near(api.unpack_activation(p), z64, 0.5 * s.repeat_interleave(32, dim=1) + za, "packed z")


# ---------------------------------------------------------------------------
# together, streams, graphs, refusals
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kept", ["plain", "packed"])
def test_two_layers_and_the_statistics_of_their_gradient(kept):
    # x -> gelu(x W1^T + b1) -> (. W2^T + b2) + x, backward, S = dW1 dW1^T, its QR
    m, d, h = 256, 96, 192
    x, w1, b1 = rnd((m, d), 70, FP), rnd((h, d), 71, FP, d**-0.5), rnd((h,), 72, FP, 0.1)
    w2, b2, dy = rnd((d, h), 73, FP, h**-0.5), rnd((d,), 74, FP, 0.1), rnd((m, d), 75, FP)
    a, z = api.linear(x, w1, b1, None, "gelu", keep=kept)
    y = api.linear(a, w2, b2, x)
    ka, kx = (api.pack_activation(a), api.pack_activation(x)) if kept == "packed" else (a, x)
    da, dw2, db2 = api.linear_backward(dy, ka, w2)
    dx, dw1, db1 = api.linear_backward(da, kx, w1, z, "gelu")
    dx = dx + dy

    t = [v.double().requires_grad_() for v in (x, w1, b1, w2, b2)]
    a64 = torch.nn.functional.gelu(t[0] @ t[1].mT + t[2])
    y64 = a64 @ t[3].mT + t[4] + t[0]
    grads = torch.autograd.grad((y64 * dy.double()).sum(), t)
    assert (y - y64).abs().max() < 2e-5 * y64.abs().max()
    # packed: a kept value is off by half a step at most, and a step is at most 1/63.5 of the
    # block's largest, so the root mean square error is below amax / (127 sqrt(3)) = amax / 220.
    # The largest of 32 normal values is 2.5 at most in the root mean square over blocks: 0.0114,
    # 1.2 % of x (rms 1) and 1.8 % of gelu(z) (rms 0.65). gelu' changes by at most 0.8 of z's
    # error, 0.0091, of its rms 0.67: 1.4 % of dz. dw1 has x's and dz's: 2.6 % in sum.
    tol = 2e-5 if kept == "plain" else 0.026
    for got, want in zip((dx, dw1, db1, dw2, db2), grads):
        assert (got - want).norm() <= tol * want.norm()
    H, tau = api.gram_geqrf(dw1)
    assert checker.check(api.gram(dw1), H, tau).passed


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_same_bits_every_time(dt):
    x, w, b = rnd((200, 1000), 80, dt), rnd((130, 1000), 81, dt, 0.03), rnd((130,), 82, dt)
    dy = rnd((200, 130), 83, dt)
    runs = []
    for _ in range(3):
        y, z = api.linear(x, w, b, None, "silu", keep="plain")
        runs.append((y, z, *api.linear_backward(dy, x, w, z, "silu")))
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], r))


def _step(x, w, b, dy):
    y, z = api.linear(x, w, b, x[:, :w.shape[0]], "gelu", keep="packed")
    return (y, *api.linear_backward(dy, api.pack_activation(x), w, z, "gelu"))


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_captured_and_replayed(dt):
    m, n, k = 70, 48, 520
    new = [(rnd((m, k), 90 + i, dt), rnd((n, k), 95 + i, dt, 0.05), rnd((n,), 100 + i, dt),
            rnd((m, n), 105 + i, dt)) for i in range(3)]
    want = [_step(*a) for a in new]
    held = [t.clone() for t in new[0]]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs over the same inputs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*held)
        graphs.append((g, out))
    for i in (1, 2, 0):
        for t, s in zip(held, new[i]):
            t.copy_(s)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want[i]))


def test_other_streams_and_threads():
    dt = BF
    data = [(rnd((300, 256), 110 + i, dt), rnd((192, 256), 120 + i, dt, 0.05), rnd((192,), 130 + i, dt),
             rnd((300, 192), 140 + i, dt)) for i in range(4)]
    want = [_step(*a) for a in data]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got[i] = _step(*data[i])
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for p, q in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_refusals():
    x, w = rnd((4, 8), 150, BF), rnd((6, 8), 151, BF)
    dy, z = rnd((4, 6), 152, BF), rnd((4, 6), 153, BF)
    pk = api.pack_activation
    cases = [
        (TypeError, lambda: api.linear(x, w.half())),
        (TypeError, lambda: api.linear(x, w, rnd((6,), 1, FP))),
        (ValueError, lambda: api.linear(x, w[:, :7])),
        (ValueError, lambda: api.linear(x, w[0])),
        (ValueError, lambda: api.linear(x, w, rnd((5,), 1, BF))),
        (ValueError, lambda: api.linear(x, w, None, rnd((4, 5), 1, BF))),
        (ValueError, lambda: api.linear(x, w, activation="tanh")),
        (ValueError, lambda: api.linear(x, w, activation=None)),
        (ValueError, lambda: api.linear(x, w, keep="fp8")),
        (ValueError, lambda: api.linear(x, w.cpu())),
        (ValueError, lambda: api.linear_backward(dy, x, w, None, "silu")),
        (ValueError, lambda: api.linear_backward(dy, None, w)),
        (ValueError, lambda: api.linear_backward(dy, x[:3], w)),
        (ValueError, lambda: api.linear_backward(dy[:, :5], x, w)),
        (ValueError, lambda: api.linear_backward(dy, x, w, z[:, :5], "silu")),
        (ValueError, lambda: api.linear_backward(dy, x, w, pk(z), "relu")),
        (ValueError, lambda: api.linear_backward(dy, pk(x[:, :7]), w)),
        (TypeError, lambda: api.linear_backward(dy, pk(x.half()), w)),
        (ValueError, lambda: api.linear_backward(dy, x, w, need=("y",))),
        (ValueError, lambda: api.linear_backward(dy, x, w, need="x")),
        (ValueError, lambda: api.unpack_activation(pk(x)._replace(exponents=pk(x).exponents[:3]))),
        (TypeError, lambda: api.unpack_activation(pk(x)._replace(codes=x))),
    ]
    for exc, call in cases:
        with pytest.raises(exc):
            call()
    wg = w.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        api.linear(x, wg)
    with torch.no_grad():
        assert torch.equal(api.linear(x, wg), api.linear(x, w))


def test_withheld_products_time_out_and_the_next_call_works():
    x, w = rnd((300, 512), 160, BF), rnd((300, 512), 161, BF)
    want = api.linear(x, w)
    torch.cuda.synchronize()
    hooks = {"wait_limit": 2_000_000, "test_skip_mma": 1, "sync_check": 1}
    old = {k: _lib.get_config(k) for k in hooks}
    try:
        for k, v in hooks.items():
            _lib.set_config(k, v)
        with pytest.raises(_lib.QRBError) as ei:
            api.linear(x, w)
        assert ei.value.status == 7
    finally:
        for k, v in old.items():
            _lib.set_config(k, v)
        _lib.set_config("device_error", 0)
    assert torch.equal(api.linear(x, w), want)


@pytest.mark.parametrize("cut", CUTS)
def test_products_leave_nothing_in_flight(cut, hooks):
    """Products of fewer, as many and more stages than the ring holds, each followed at
    once by kernels that use the same SMs' shared memory: the same bits every time."""
    hooks("linear_cut", cut)
    hooks("linear_rows", 0)
    G = rnd((4, 128, 128), 190, FP)
    s0 = api.gram(G)
    for k in (64, 192, 256, 512, 1000):
        x, w, dy = rnd((520, k), 191, BF), rnd((264, k), 192, BF, k**-0.5), rnd((520, 264), 193, BF)
        y0, g0 = api.linear(x, w), api.linear_backward(dy, x, w)
        check_forward(x, w, None, None, "none", y0)
        check_backward(dy, x.double(), w, None, "none", *g0)
        runs = []
        for _ in range(40):
            runs += [(api.linear(x, w), api.gram(G), api.linear_backward(dy, x, w), api.gram(G))]
        for y, s, g, t in runs:
            assert torch.equal(y, y0) and torch.equal(s, s0) and torch.equal(t, s0)
            assert all(torch.equal(p, q) for p, q in zip(g, g0))


def long_acc(k):
    """A 16-bit product's sum at any length: chains of at most 8192 values (16 to an MMA,
    fewer than 16 adds within the last), added in FP32, each add half a step."""
    return STEP * (8192 / 16 + 18) + STEP / 2 * (k / 8192 + 1)


@pytest.mark.parametrize("dt", [BF, HF], ids=IDS[:2])
@pytest.mark.parametrize("cut,splits", [(0, 0), (2256, 1), (2128, 1), (1128, 1), (1064, 1), (2256, 3)])
def test_long_reductions_do_not_drift(cut, splits, dt, hooks):
    """Terms of one sign, so that every truncated add would pull the same way."""
    hooks("linear_cut", cut)
    hooks("linear_splits", splits)
    hooks("linear_rows", 0)
    m, n, k = 600_011, 136, 264
    g = torch.Generator(device=DEV).manual_seed(194)
    one = lambda *s: ((torch.rand(*s, device=DEV, generator=g) + 0.5) * m**-0.5).to(dt)  # noqa: E731
    dy, x, w = one(m, n), one(m, k), rnd((n, k), 195, dt)
    dx, dw, _ = api.linear_backward(dy, x, w, need=("x", "weight"))
    want = dy.double().mT @ x.double()
    near(dw, want, (u(dt) * 1.0001 + long_acc(m) * (1 + u(dt))) * want, "dw")
    check_backward(dy[:1000], None, w, None, "none", dx[:1000], None, None)
    # forward, the long axis as k, rows of z beside it (no activation)
    a, b = dy.t().contiguous(), x.t().contiguous()
    y = api.linear(a, b)
    near(y, want, (u(dt) * 1.0001 + long_acc(m) * (1 + u(dt))) * want, "y")


@pytest.mark.parametrize("k", [8191, 8192, 8193, 16_384, 16_385, 24_640])
def test_reductions_about_a_chain_are_exact(k, hooks):
    """Small whole numbers: every partial sum is exact in FP32, so no value may be lost or
    counted twice where one chain ends and the next begins."""
    hooks("linear_splits", 1)
    hooks("linear_rows", 0)
    g = torch.Generator(device=DEV).manual_seed(k)
    whole = lambda *s: torch.randint(-2, 3, s, device=DEV, generator=g).to(BF)  # noqa: E731
    ld = (k + 7) // 8 * 8
    for m, n in ((40, 72), (300, 520), (4000, 1100)):  # more tiles than SMs in the last
        x, w = whole(m, ld)[:, :k], whole(n, ld)[:, :k]
        want = (x.float() @ w.float().mT).to(BF)
        for cut in (0, *CUTS):
            hooks("linear_cut", cut)
            assert torch.equal(api.linear(x, w), want)
            assert torch.equal(api.linear_backward(x.t(), w.t(), w.new_zeros(m, n), need=("weight",))[1],
                               want)


@pytest.mark.parametrize("n", [32, 200])
def test_bias_sums_of_a_long_batch_hold_nothing_up(n, hooks):
    """The sums are added beside the products' tiles: with the waits bounded by 300,000
    clocks (150 us) none runs out over 15,626 blocks' sums of each column."""
    m, k = 2_000_003, 64
    g = torch.Generator(device=DEV).manual_seed(196)
    dy = torch.randint(-2, 3, (m, n), device=DEV, generator=g).to(BF)
    x, w = rnd((m, k), 197, BF), rnd((n, k), 198, BF)
    want = dy.double().sum(0).to(BF)
    limits = {"wait_limit": 300_000, "sync_check": 1}
    old = {key: _lib.get_config(key) for key in limits}
    try:
        for key, v in limits.items():
            _lib.set_config(key, v)
        got = [api.linear_backward(dy, x, w)[2], api.linear_backward(dy, x, w, need=("bias",))[2]]
    finally:
        for key, v in old.items():
            _lib.set_config(key, v)
        _lib.set_config("device_error", 0)
    assert all(torch.equal(db, want) for db in got)


@pytest.mark.parametrize("need", [("x", "bias"), ("weight",), ()])
def test_need_may_be_any_iterable(need):
    dy, x, w = rnd((20, 24), 199, BF), rnd((20, 16), 200, BF), rnd((24, 16), 201, BF)
    want = api.linear_backward(dy, x, w, need=need)
    assert [g is not None for g in want] == [name in need for name in ("x", "weight", "bias")]
    for given in (list(need), set(need), iter(need), (name for name in need), dict.fromkeys(need)):
        for g, h in zip(api.linear_backward(dy, x, w, need=given), want):
            assert h is None if g is None else torch.equal(g, h)
    with pytest.raises(ValueError, match="need"):
        api.linear_backward(dy, x, w, need=iter(("x", "y")))


@pytest.mark.parametrize("act", [["gelu"], {"gelu": 1}, {"gelu"}, 2, b"gelu"])
def test_activations_that_are_no_names_are_refused(act):
    x, w = rnd((4, 8), 202, BF), rnd((6, 8), 203, BF)
    with pytest.raises(ValueError, match="activation must be one of"):
        api.linear(x, w, activation=act)
    with pytest.raises(ValueError, match="activation must be one of"):
        api.linear_backward(rnd((4, 6), 204, BF), x, w, x, act)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as forward_ad

    x, w, b, r = rnd((4, 8), 205, FP), rnd((6, 8), 206, FP), rnd((6,), 207, FP), rnd((4, 6), 208, FP)
    want = api.linear(x, w, b, r)
    with forward_ad.dual_level(), torch.no_grad():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: api.linear(dual(x), w), lambda: api.linear(x, dual(w)),
                     lambda: api.linear(x, w, dual(b)), lambda: api.linear(x, w, b, dual(r)),
                     lambda: api.linear_backward(dual(r), x, w),
                     lambda: api.linear_backward(r, dual(x), w),
                     lambda: api.linear_backward(r, x, dual(w)),
                     lambda: api.linear_backward(r, x, w, dual(r), "gelu"),
                     lambda: api.pack_activation(dual(x))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        # tensors without one, packed ones among them, are taken
        assert torch.equal(api.linear(x, w, b, r), want)
        assert torch.equal(api.linear(forward_ad.unpack_dual(dual(x)).primal, w, b, r), want)
        api.linear_backward(r, api.pack_activation(x), w)
        api.linear_backward(r, dual(x), w, dual(r), need=("x",))  # neither is read
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jvp(lambda t: api.linear(t, w), (x,), (x,))


def test_negated_views_with_unit_stride():
    c = torch.complex(rnd((6, 8), 209, FP), rnd((6, 8), 210, FP)).conj().imag
    x, w = c.as_strided((5, 4), (8, 1)), rnd((6, 4), 211, FP)  # elements of both parts, all negated
    one = c[0, 0].reshape(1)
    assert x.is_neg() and x.stride(1) == 1 and one.is_neg() and one.stride() == (1,)
    check_forward(x, w, None, None, "none", api.linear(x, w))
    check_forward(w, x, None, w[:, :1].expand(6, 5), "none", api.linear(w, x, None, w[:, :1].expand(6, 5)))
    check_forward(x, w[:1], one, x[:, :1], "none", api.linear(x, w[:1], one, x[:, :1]))
    check_backward(x, rnd((5, 3), 212, FP).double(), rnd((4, 3), 213, FP), x.double(), "silu",
                   *api.linear_backward(x, rnd((5, 3), 212, FP), rnd((4, 3), 213, FP), x, "silu"))
    assert torch.equal(api.pack_activation(x).codes, api.pack_activation(x.clone()).codes)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(60_001, 64, 72), (200_000, 40, 32), (100_003, 256, 264)])
def test_long_batch_is_exact_in_whole_numbers(m, n, k, dt):
    """Products and sums of whole numbers up to 2 are exact below 2^24, in every type's
    operands, so dW, db and dx are the exact sums rounded once: no row of the batch may
    be lost, counted twice or added to another."""
    g = torch.Generator(device=DEV).manual_seed(m)
    whole = lambda *s: torch.randint(-2, 3, s, device=DEV, generator=g).to(dt)  # noqa: E731
    dy, x, w = whole(m, n), whole(m, k), whole(n, k)
    dx, dw, db = api.linear_backward(dy, x, w)
    assert torch.equal(dw, (dy.double().mT @ x.double()).to(dt))
    assert torch.equal(db, dy.double().sum(0).to(dt))
    assert torch.equal(dx, (dy.double() @ w.double()).to(dt))


@pytest.mark.parametrize("products", [True, False])
def test_block_sums_of_the_bias_are_joined_in_64_bits(products):
    """Rows of c = (1 + 2^-17) 2^j / 128: a block of 8, 32 or 128 of them has an exact FP32
    sum ((2^17 + 1) i with i <= 128 takes 24 bits), and thousands of blocks an exact FP64
    sum; joined in FP32, each add beyond 128 blocks would lose 2^-17."""
    m, n, k = 1_000_003, 48, 16
    c = (1 + 2.0**-17) / 128 * 2.0 ** (torch.arange(n, dtype=torch.float64, device=DEV) % 5)
    c = c * (1 - 2 * (torch.arange(n, device=DEV) % 2))
    dy = c.float().expand(m, n).contiguous()
    assert torch.equal(dy[0].double(), c)
    x, w = rnd((m, k), 214, FP), rnd((n, k), 215, FP)
    db = api.linear_backward(dy, x, w, need=("x", "weight", "bias") if products else ("bias",))[2]
    assert torch.equal(db, (m * c).float())
