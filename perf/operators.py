"""The linear-layer operators of a training or serving step, measured.

The framework factors the statistics ``G G^T`` of weight gradients. These are
the operators on either side of that gradient: the layer's product with its
epilogue, its backward pass (which makes ``G``), and the layer's activations
kept in 8 bits between the two.

* ``linear``    ``z = x W^T + b``, ``y = act(z) + r``; optionally z is kept for
  the backward pass, in the layer's type or packed to 8 bits.
* ``backward``  from dy and the kept x and z: ``dz = dy act'(z)``,
  ``dx = dz W``, ``dW = dz^T x``, ``db = sum of dz's rows``. The kept tensors
  are plain or packed.
* ``pack``      a tensor packed to 8 bits and read back.

The packed form: per row, blocks of 32 values share a power of two 2^e, the
smallest with ``max |x| <= 127 * 2^e`` (e at least -126, -24 for float16; at
most 122, 10 for float16), and each value is ``round(x / 2^e)`` in 8 bits
(ties to even; at most 63 where e is at its upper end, so that no value read
back overflows its type).
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    def linear(name, m, n, k, dtype, act, bias=True, residual=True, keep="none"):
        return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "act": act,
                "bias": bias, "residual": residual, "keep": keep}

    def backward(name, m, n, k, dtype, act, kept, bias=True):
        return {"name": name, "op": "backward", "m": m, "n": n, "k": k, "dtype": dtype, "act": act,
                "kept": kept, "bias": bias}

    def pack(name, m, k, dtype):
        return {"name": name, "op": "pack", "m": m, "k": k, "dtype": dtype}

    return [
        # serving, one token through a square layer: the weights are read once
        linear("token_4096", 1, 4096, 4096, "bf16", "silu"),
        # the smallest serving call: a few tokens through a narrow layer, latency alone
        linear("tokens_small", 4, 512, 512, "fp16", "gelu"),
        # serving, a batch of sequences at one token each
        linear("tokens_batch", 48, 4096, 1024, "bf16", "none"),
        # a long prompt, or the forward pass of a training step without recomputation
        linear("prompt_4096", 8192, 4096, 4096, "bf16", "gelu_tanh"),
        # training forward: an up-projection that keeps its pre-activation in 8 bits
        linear("train_keep8", 4096, 4096, 1024, "bf16", "gelu", residual=False, keep="packed"),
        # ragged: no size is a multiple of a tile and rows are not 16-byte aligned
        linear("ragged_fp16", 777, 1001, 355, "fp16", "silu", keep="plain"),
        # FP32 layer (the type of the factorization itself)
        linear("fp32_1024", 2048, 1024, 1024, "fp32", "silu"),
        # training backward, kept tensors in the layer's type
        backward("bwd_1024", 4096, 1024, 4096, "bf16", "silu", "plain"),
        # training backward from 8-bit kept tensors: the largest case
        backward("bwd8_4096", 8192, 4096, 4096, "bf16", "gelu", "packed"),
        # a short ragged batch, backward from 8-bit kept tensors
        backward("bwd8_ragged", 999, 177, 530, "fp16", "gelu_tanh", "packed"),
        # FP32 backward: the gradient that goes into the FP32 statistics
        backward("bwd_fp32", 2048, 1024, 512, "fp32", "gelu", "plain"),
        # keeping a layer's input in 8 bits, and reading it back
        pack("pack_8192", 8192, 4096, "bf16"),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; half of them a multiple of 8 (what models use), half as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 16:
        v = v // 8 * 8
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "backward", "backward", "pack"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    wide = 1024 if dtype == "fp32" else 4096
    m, n, k = _size(rng, 1, 8192), _size(rng, 32, wide), _size(rng, 32, wide)
    if op == "pack":
        return {"op": op, "m": m, "k": k, "dtype": dtype}
    if op == "linear":
        keep = rng.choice(["none", "none", "plain", "packed"])
        # packed z: not in FP32, whose last bits decide which side of a code's border z falls;
        # not for relu, whose derivative is z's sign, which small values lose
        if keep == "packed" and (act == "relu" or dtype == "fp32"):
            keep = "plain"
        return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "act": act,
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "keep": keep}
    kept = "plain" if act == "relu" else rng.choice(["plain", "packed"])
    return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "kept": kept,
            "bias": rng.random() < 0.5}


def _blocks(k):
    return -(-k // BLOCK)


def work(case):
    """Bytes: each input read once, each output written once. Flops: the products."""
    m, k, e = case["m"], case["k"], 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "pack":  # x in, codes and exponents out; both in, x out
        return {"bytes": 2 * m * (k * e + k + _blocks(k)), "flops": 0}
    n = case["n"]
    if case["op"] == "linear":
        b = (m * k + n * k + m * n) * e + (n * e if case["bias"] else 0)
        b += m * n * e if case["residual"] else 0
        b += {"none": 0, "plain": m * n * e, "packed": m * (n + _blocks(n))}[case["keep"]]
        return {"bytes": b, "flops": 2 * m * n * k}
    x = m * k * e if case["kept"] == "plain" else m * (k + _blocks(k))
    z = m * n * e if case["kept"] == "plain" else m * (n + _blocks(n))
    z = 0 if case["act"] == "none" else z
    b = m * n * e + x + z + n * k * e + m * k * e + n * k * e + (n * e if case["bias"] else 0)
    return {"bytes": b, "flops": 4 * m * n * k}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, m, k = TYPES[case["dtype"]], case["m"], case["k"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    # activations: columns of different scale, as a layer's channels have
    x = (randn(m, k) * torch.exp(0.5 * randn(k))).to(dt)
    s = {"case": case, "x": x}
    if case["op"] == "pack":
        return s
    n = case["n"]
    s["w"] = (randn(n, k) / math.sqrt(k)).to(dt)
    if case["op"] == "linear":
        s["b"] = (0.1 * randn(n)).to(dt) if case["bias"] else None
        s["r"] = randn(m, n).to(dt) if case["residual"] else None
        return s
    s["dy"] = randn(m, n).to(dt)
    s["z"] = (1.5 * randn(m, n)).to(dt) if case["act"] != "none" else None
    if case["kept"] == "packed":
        s["x"] = _pack(x)
        s["z"] = _pack(s["z"]) if s["z"] is not None else None
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

_RANGE = {torch.bfloat16: (-126, 122), torch.float32: (-126, 122), torch.float16: (-24, 10)}


def _pack(x, dt=None):
    """(codes int8 [m, k], exponents int8 [m, ceil(k / 32)]) of x, to be read back as dt."""
    lo, hi = _RANGE[dt or x.dtype]
    m, k = x.shape
    v = torch.zeros(m, _blocks(k) * BLOCK, device=x.device)
    v[:, :k] = x
    v = v.view(m, -1, BLOCK)
    f, p = torch.frexp(v.abs().amax(dim=-1))  # max |x| = f * 2^p, 0.5 <= f < 1
    e = p - 7 + (f > 127.0 / 128.0).to(p.dtype)
    e = torch.where(f == 0, torch.full_like(e, lo), e.clamp(lo, hi))
    most = torch.where(e == hi, 63.0, 127.0).unsqueeze(-1)
    q = torch.round(torch.ldexp(v, -e.unsqueeze(-1)))
    q = torch.minimum(torch.maximum(q, -most), most)
    return q.view(m, -1)[:, :k].to(torch.int8).contiguous(), e.to(torch.int8)


def _unpack(packed):
    """The FP32 values that codes and exponents stand for."""
    q, e = packed
    e = e.to(torch.int32).repeat_interleave(BLOCK, dim=1)[:, : q.shape[1]]
    return torch.ldexp(q.float(), e)


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain(s):
    c = s["case"]
    dt = TYPES[c["dtype"]]
    if c["op"] == "pack":
        return {"x": _unpack(_pack(s["x"])).to(dt)}
    if c["op"] == "linear":
        z = s["x"].float() @ s["w"].float().t()
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _act(z, c["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        out = {"y": y.to(dt)}
        if c["keep"] == "plain":
            out["z"] = z.to(dt)
        elif c["keep"] == "packed":
            out["z"] = _unpack(_pack(z, dt)).to(dt)
        return out
    x = _unpack(s["x"]) if c["kept"] == "packed" else s["x"].float()
    dz = s["dy"].float()
    if c["act"] != "none":
        z = _unpack(s["z"]) if c["kept"] == "packed" else s["z"].float()
        dz = dz * _act_grad(z, c["act"])
    out = {"dx": (dz @ s["w"].float()).to(dt), "dw": (dz.t() @ x).to(dt)}
    if c["bias"]:
        out["db"] = dz.sum(dim=0, dtype=torch.float64).to(dt)
    return out


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    if not own:
        return _plain(s)
    from gpumode_qr_b200 import api

    c = s["case"]
    if c["op"] == "pack":
        return {"x": api.unpack_activation(api.pack_activation(s["x"]))}
    if c["op"] == "linear":
        keep = c["keep"]
        if keep == "none":
            return {"y": api.linear(s["x"], s["w"], s["b"], s["r"], c["act"])}
        y, z = api.linear(s["x"], s["w"], s["b"], s["r"], c["act"], keep=keep)
        return {"y": y, "z": api.unpack_activation(z) if keep == "packed" else z}
    x, z = s["x"], s["z"]
    if c["kept"] == "packed":
        dt = TYPES[c["dtype"]]
        x = api.PackedActivation(*x, dt)
        z = api.PackedActivation(*z, dt) if z is not None else None
    need = ("x", "weight", "bias") if c["bias"] else ("x", "weight")
    dx, dw, db = api.linear_backward(s["dy"], x, s["w"], z, c["act"], need=need)
    out = {"dx": dx, "dw": dw}
    if c["bias"]:
        out["db"] = db
    return out


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------

def _exact_scale(amax, dtype):
    """log2 of each block's step, from the definition: the smallest e with amax <= 127 * 2^e.
    (The 1e-9 takes log2's own rounding of a power of two back; neighbours are 8e-8 away.)"""
    lo, hi = (-24, 10) if dtype == "fp16" else (-126, 122)
    return torch.ceil(torch.log2((amax / 127).clamp_min(2.0**-300)) - 1e-9).clamp(lo, hi), hi


def _exact_packed(v, dtype):
    m, k = v.shape
    v = torch.nn.functional.pad(v, (0, _blocks(k) * BLOCK - k)).view(m, -1, BLOCK)
    e, hi = _exact_scale(v.abs().amax(dim=2, keepdim=True), dtype)
    step = torch.ldexp(torch.ones_like(e), e.int())
    most = torch.where(e == hi, 63.0, 127.0)
    q = (v / step).round()
    return (torch.maximum(torch.minimum(q, most), -most) * step).view(m, -1)[:, :k]


def _exact_act(z, act):
    phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    # gelu_tanh: z * sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3)
    c = math.sqrt(8 / math.pi)
    s = torch.sigmoid(c * (z + 0.044715 * z**3))
    return z * s, s + z * s * (1 - s) * c * (1 + 0.134145 * z * z)


def exact(case, seed):
    s, dtype = prepare(case, seed), case["dtype"]
    if case["op"] == "pack":
        return {"x": _exact_packed(s["x"].double(), dtype)}
    if case["op"] == "linear":
        z = torch.matmul(s["x"].double(), s["w"].double().mT)
        z = z + (s["b"].double() if s["b"] is not None else 0.0)
        y = _exact_act(z, case["act"])[0] + (s["r"].double() if s["r"] is not None else 0.0)
        out = {"y": y}
        if case["keep"] != "none":
            out["z"] = _exact_packed(z, dtype) if case["keep"] == "packed" else z
        return out

    def read(t):
        if not isinstance(t, tuple):
            return t.double()
        q, e = t
        return torch.ldexp(q.double(), e.int().repeat_interleave(BLOCK, dim=1)[:, : q.shape[1]])

    dz = s["dy"].double()
    if s["z"] is not None:
        dz = dz * _exact_act(read(s["z"]), case["act"])[1]
    out = {"dx": torch.matmul(dz, s["w"].double()), "dw": torch.matmul(dz.mT, read(s["x"]))}
    if case["bias"]:
        out["db"] = dz.sum(dim=0)
    return out
