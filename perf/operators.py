"""The measured cases of the 4-bit and of the dense gated FFN operators, with their plain forms.

Four operators around one FFN's life -- trained dense, pruned to Block-ELL, quantised, served:

  quantize  ``mx_quantize`` and ``mx_dequantize``: rows of activations to microscaled 4-bit floating
            point (groups of 32 features share a power of two) and back
  product   ``mx_matmul``: quantised activations times a Block-ELL weight held in 4 bits
  ffn       ``mx_swiglu``: the SwiGLU FFN on such weights, its hidden state requantised to 4 bits
  gated     ``gated_ffn``: the dense gated FFN in bf16 or fp16, inference or a training step

Sizes come from the repository's benchmark, tests and layer cases.  ``listed()`` holds the fixed
cases, ``draw(rng)`` gives more of the same ranges:

  d_model   512 .. 4096, d_ff 2 .. 4 times that; tiles of 32 or 64, 0.1 .. 1.0 of the column blocks
  tokens    1 .. 16384, odd counts included; padded (all-zero) rows, dead slots, biases
"""

from __future__ import annotations

import os
import sys

import numpy as np
import torch

own = False

_DEV = "cuda"
_GROUP = 32
# most work of a drawn case (the largest listed one takes 1.24e12)
_MAX_DRAW_FLOPS = 6e11


def _kernels():
    pkg = os.path.join(os.getcwd(), "looped-blockell-tpu_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from looped_blockell import kernels

    return kernels


# ------------------------------------------------------------------ cases
def _quantize(name, tokens, d_model, dtype="bfloat16"):
    return dict(name=name, kind="quantize", tokens=tokens, d_model=d_model, dtype=dtype)


def _sparse(name, kind, tokens, d_model, d_ff, tile, density, *, bias=False, residual=False, dead=0.0, pad=0.0):
    """dead: share of pruned slots.  pad: share of all-zero rows (padding tokens) at the end."""
    return dict(name=name, kind=kind, tokens=tokens, d_model=d_model, d_ff=d_ff, tile=tile, density=density, bias=bias,
                residual=residual, dead=dead, pad=pad)


def _gated(name, tokens, d_model, d_ff, *, dtype="bfloat16", act="silu", train=False, residual=False):
    return dict(name=name, kind="gated", tokens=tokens, d_model=d_model, d_ff=d_ff, dtype=dtype, act=act, train=train,
                residual=residual)


def listed():
    return [
        # the activations of 16 sequences generating with the wide model: launches and host work
        _quantize("quantize_16", 16, 4096),
        # the activations of a large batch (the benchmark's headline layer)
        _quantize("quantize_16k", 16384, 1024),
        # one token through the wide model's up projection
        _sparse("product_1_b64", "product", 1, 4096, 14336, 64, 0.10),
        # the headline layer's up projection, with its bias, on a large batch
        _sparse("product_16k_b32", "product", 16384, 1024, 4096, 32, 0.25, bias=True),
        # 16 sequences generating with the wide model, weights streamed from memory
        _sparse("ffn_16_b64", "ffn", 16, 4096, 14336, 64, 0.10),
        # the headline layer on a large batch
        _sparse("ffn_16k_b32", "ffn", 16384, 1024, 4096, 32, 0.25),
        # prompts of odd length through a pruned layer with biases and residual, padded at the end
        _sparse("ffn_4099_b64", "ffn", 4099, 2048, 8192, 64, 0.125, bias=True, residual=True, dead=0.1, pad=0.05),
        # one token through a dense layer
        _gated("gated_1", 1, 2048, 8192),
        # scoring with the dense teacher of the headline layer
        _gated("gated_8k", 8192, 1024, 4096, residual=True),
        # training a small dense model in fp16 on a micro-batch of ragged length
        _gated("gated_train_1999_fp16", 1999, 512, 1792, dtype="float16", act="gelu", train=True, residual=True),
        # one training step of the dense start of the headline layer, 32 sequences of 512
        _gated("gated_train_16k", 16384, 1024, 4096, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    while True:
        kind = rng.choice(["quantize", "product", "ffn", "ffn", "gated", "gated"])
        tokens = _log_int(rng, 1, 16384)
        if rng.random() < 0.5:
            tokens |= 1
        d_model = rng.choice([512, 640, 1024, 1280, 2048, 4096])
        d_ff = int(d_model * rng.choice([2, 3.5, 4]))
        if kind == "quantize":
            c = _quantize(None, tokens, d_model, rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
        elif kind == "gated":
            train = rng.random() < 0.5
            c = _gated(None, max(tokens, 16) if train else tokens, d_model, d_ff, dtype=rng.choice(["bfloat16", "float16"]),
                       act=rng.choice(["silu", "gelu"]), train=train, residual=rng.random() < 0.5)
        else:
            c = _sparse(None, kind, tokens, d_model, d_ff, rng.choice([32, 64]), rng.choice([0.1, 0.125, 0.25, 0.5, 1.0]),
                        bias=rng.random() < 0.5, residual=kind == "ffn" and rng.random() < 0.5,
                        dead=rng.choice([0.0, 0.0, 0.1]), pad=rng.choice([0.0, 0.1]))
        del c["name"]
        if work(c)["flops"] <= _MAX_DRAW_FLOPS:
            return c


def _geometry(c):
    """(name, block rows, column blocks, slots per row) of a sparse case's weights."""
    B, d, ff = c["tile"], c["d_model"], c["d_ff"]
    rf, rm = ff // B, d // B
    up = (rf, rm, max(1, int(rm * c["density"])))
    if c["kind"] == "product":
        return [("w", *up)]
    return [("gate", *up), ("up", *up), ("down", rm, rf, max(1, int(rf * c["density"])))]


def work(c):
    N, d = c["tokens"], c["d_model"]
    if c["kind"] == "quantize":
        # x in; the values that codes and scales stand for out; the 4.25 bits between them once each way
        size = 4 if c["dtype"] == "float32" else 2
        return {"bytes": N * d * (size + 2 + 2 * 17 / 32), "flops": 4.0 * N * d}
    ff = c["d_ff"]
    if c["kind"] == "gated":
        if not c["train"]:
            return {"bytes": 4.0 * N * d + 6.0 * d * ff, "flops": 6.0 * N * d * ff}
        # x and the result's gradient in, result and the input's gradient out; weights in, gradients out
        return {"bytes": 8.0 * N * d + 12.0 * d * ff, "flops": 18.0 * N * d * ff}
    B = c["tile"]
    tiles = sum(R * K for _, R, _, K in _geometry(c))
    out = ff if c["kind"] == "product" else d
    return {"bytes": 2.0 * N * (d + out) + tiles * (B * B * 17 / 32 + 4), "flops": 2.0 * N * tiles * B * B}


# ------------------------------------------------------------------ inputs
def _activations(N, d, g, pad=0.0):
    """Normal values under a log-normal gain per feature: a few channels are much larger than most."""
    x = torch.randn(N, d, device=_DEV, generator=g) * torch.exp(0.7 * torch.randn(d, device=_DEV, generator=g))
    if pad:
        x[N - int(N * pad):] = 0.0
    return x


def _topology(R, C, K, gc):
    """K distinct columns of C per row, unsorted (in order where the row is full)."""
    if K == C:
        return torch.arange(C).repeat(R, 1).to(torch.int32)
    return torch.rand(R, C, generator=gc).argsort(1)[:, :K].to(torch.int32)


def prepare(c, seed):
    g = torch.Generator(device=_DEV).manual_seed(int(seed) & 0x7FFFFFFF)
    gc = torch.Generator().manual_seed((int(seed) + 1) & 0x7FFFFFFF)
    N, d = c["tokens"], c["d_model"]
    if c["kind"] == "quantize":
        return {"kind": "quantize", "x": _activations(N, d, g).to(getattr(torch, c["dtype"]))}
    if c["kind"] == "gated":
        dt, ff = getattr(torch, c["dtype"]), c["d_ff"]
        st = {"kind": "gated", "act": c["act"], "train": c["train"], "residual": c["residual"]}
        st["x"] = torch.randn(N, d, device=_DEV, generator=g).to(dt)
        for n, shape in (("w_gate", (ff, d)), ("w_up", (ff, d)), ("w_down", (d, ff))):
            st[n] = torch.randn(shape, device=_DEV, generator=g).mul_(shape[1] ** -0.5).to(dt)
        if c["train"]:
            st["dy"] = torch.randn(N, d, device=_DEV, generator=g).to(dt)
            for n in ("x", "w_gate", "w_up", "w_down"):
                st[n].requires_grad_(True)
        return st
    B = c["tile"]
    st = {"kind": c["kind"], "residual": c["residual"], "x": _activations(N, d, g, c["pad"]).to(torch.bfloat16)}
    for n, R, C, K in _geometry(c):
        # a weight quantised beforehand: [R, K, B_out, B_in] in groups of 32 input features, their
        # largest magnitudes spread over a few powers of two as those of normal weights are
        codes = torch.randint(0, 256, (R, K, B, B // 2), device=_DEV, dtype=torch.uint8, generator=g)
        scales = torch.randint(118, 121, (R, K, B, B // _GROUP), device=_DEV, dtype=torch.uint8, generator=g)
        cols = _topology(R, C, K, gc)
        if c["dead"]:
            cols[torch.rand(R, K, generator=gc) < c["dead"]] = -1
        st[n] = (codes, scales, cols.to(_DEV))
        st["b_" + n] = torch.randn(R * B, device=_DEV, generator=g) * 0.1 if c["bias"] else None
    return st


# ------------------------------------------------------------------ plain forms
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantized(x):
    """The values that x [N, F] stands for in 4 bits, in 32 bits.  The scaling by powers of two is
    exact, and so are the comparisons with the midpoints."""
    v = x.float().reshape(x.shape[0], -1, _GROUP)
    _, e = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = (e - 3).clamp(-127, 127)
    s = torch.ldexp(torch.ones_like(v[..., :1]), -e)
    a = (v * s).abs()
    # to the nearest of 0, .5, 1, 1.5 | 2, 3 | 4, 6, ties to the even code, beyond 6 to 6
    q = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6)
    return (torch.copysign(q, v) / s).reshape(x.shape[0], -1)


def _dense(codes, scales, cols, C):
    """The dense [R * B, C * B] weight, in 32 bits, that codes and scales in their slots stand for."""
    R, K, B, _ = codes.shape
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    v = table[torch.stack([codes & 15, codes >> 4], -1).long()].reshape(R, K, B, -1, _GROUP)
    v = (v * torch.exp2(scales.float() - 127)[..., None]).reshape(R, K, B, B)
    w = torch.zeros(R, C + 1, B, B, device=codes.device)
    at = torch.where(cols < 0, C, cols).long()
    w.scatter_add_(1, at[:, :, None, None].expand_as(v), v)
    return w[:, :C].transpose(1, 2).reshape(R * B, C * B)


def _mx_product(x, weight, bias):
    xq = _quantized(x)
    y = xq @ _dense(*weight, xq.shape[1] // weight[0].shape[2]).T
    return y if bias is None else y + bias


def _silu(z):
    return z / (1 + torch.exp(-z))


def _act(z, act):
    """The activation and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    k = 0.7978845608028654
    t = torch.tanh(k * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


def _plain_gated(st):
    dt = st["x"].dtype
    x, wg, wu, wd = (st[n].detach().float() for n in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, st["act"])
    h = a * u
    out = h @ wd.T
    if st["residual"]:
        out = out + x
    res = {"out": out.to(dt)}
    if st["train"]:
        dy = st["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * da, dh * a
        dx = dg @ wg + du @ wu
        if st["residual"]:
            dx = dx + dy
        res.update(dx=dx.to(dt), dw_gate=(dg.T @ x).to(dt), dw_up=(du.T @ x).to(dt), dw_down=(dy.T @ h).to(dt))
    return res


def _plain(st):
    if st["kind"] == "gated":
        return _plain_gated(st)
    x = st["x"]
    if st["kind"] == "quantize":
        return {"values": _quantized(x).to(torch.bfloat16)}
    if st["kind"] == "product":
        return {"y": _mx_product(x, st["w"], st["b_w"]).to(torch.bfloat16)}
    h = _silu(_mx_product(x, st["gate"], st["b_gate"])) * _mx_product(x, st["up"], st["b_up"])
    out = _mx_product(h, st["down"], st["b_down"])
    return {"out": (out + x.float() if st["residual"] else out).to(torch.bfloat16)}


def _own(st):
    K = _kernels()
    x = st["x"]
    if st["kind"] == "quantize":
        codes, scales = K.mx_quantize(x)
        return {"values": K.mx_dequantize(codes, scales, torch.bfloat16)}
    if st["kind"] == "product":
        return {"y": K.mx_matmul(x, *st["w"], bias=st["b_w"])}
    if st["kind"] == "ffn":
        return {"out": K.mx_swiglu(x, st["gate"], st["up"], st["down"], add_residual=st["residual"], b_gate=st["b_gate"],
                                   b_up=st["b_up"], b_down=st["b_down"])}
    w = [st[n] for n in ("w_gate", "w_up", "w_down")]
    out = K.gated_ffn(x, *w, activation=st["act"], add_residual=st["residual"])
    if not st["train"]:
        return {"out": out}
    dx, dg, du, dd = torch.autograd.grad(out, [x, *w], st["dy"])
    return {"out": out.detach(), "dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}


def run(st):
    if own:
        return _own(st)
    with torch.no_grad():
        return _plain(st)


# ------------------------------------------------------------------ in 64 bits
def _nearest_e2m1(v):
    """float64 [..., 32] groups -> the nearest 4-bit values times their group's power of two."""
    top = v.abs().amax(-1, keepdim=True)
    p = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    p = p + (top >= 2.0 ** (p + 1)).double() - (top < 2.0 ** p).double()      # log2 is off by a rounding at most
    scale = 2.0 ** torch.where(top > 0, p - 2, torch.full_like(p, -127.0)).clamp(-127, 127)
    a = v.abs() / scale
    lower = torch.zeros_like(a)
    for k in range(1, 8):
        mid = (_E2M1[k - 1] + _E2M1[k]) / 2
        # a tie goes to the even code: up from an odd k - 1, down from an even one
        lower = torch.where((a > mid) | ((a == mid) & (k % 2 == 0)), torch.full_like(a, _E2M1[k]), lower)
    return torch.sign(v) * lower * scale


def _exact_product(x, weight, bias, C):
    codes, scales, cols = weight
    R, K, B, _ = codes.shape
    xq = _nearest_e2m1(x.reshape(x.shape[0], -1, _GROUP)).reshape(x.shape)
    nib = torch.empty(R, K, B, B, dtype=torch.uint8, device=codes.device)
    nib[..., 0::2], nib[..., 1::2] = codes % 16, codes // 16
    mag = torch.tensor(np.array(_E2M1), device=codes.device)[(nib % 8).long()]
    w = torch.where(nib >= 8, -mag, mag) * (2.0 ** (scales.double() - 127)).repeat_interleave(_GROUP, -1)
    live = (cols >= 0).double()
    full = torch.zeros(R, B, C, B, dtype=torch.float64, device=codes.device)
    rows = torch.arange(R, device=codes.device)
    for k in range(K):
        at = cols[:, k].clamp(min=0).long()
        full[rows, :, at] += w[:, k] * live[:, k, None, None]
    y = xq @ full.reshape(R * B, C * B).T
    return y if bias is None else y + bias.double()


def _exact_gated(st):
    x, wg, wu, wd = (st[n].detach().double().requires_grad_(st["train"]) for n in ("x", "w_gate", "w_up", "w_down"))
    act = (lambda z: z * torch.sigmoid(z)) if st["act"] == "silu" else (
        lambda z: z * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    with torch.set_grad_enabled(st["train"]):
        out = (act(x @ wg.T) * (x @ wu.T)) @ wd.T
        if st["residual"]:
            out = out + x
    res = {"out": out.detach()}
    if st["train"]:
        grads = torch.autograd.grad(out, [x, wg, wu, wd], st["dy"].double())
        res.update(zip(("dx", "dw_gate", "dw_up", "dw_down"), grads))
    return res


def exact(c, seed):
    st = prepare(c, seed)
    if c["kind"] == "gated":
        return _exact_gated(st)
    x = st["x"].double()
    with torch.no_grad():
        if c["kind"] == "quantize":
            return {"values": _nearest_e2m1(x.reshape(x.shape[0], -1, _GROUP)).reshape(x.shape)}
        C = {n: C for n, _, C, _ in _geometry(c)}
        if c["kind"] == "product":
            return {"y": _exact_product(x, st["w"], st["b_w"], C["w"])}
        g = _exact_product(x, st["gate"], st["b_gate"], C["gate"])
        u = _exact_product(x, st["up"], st["b_up"], C["up"])
        out = _exact_product(g * torch.sigmoid(g) * u, st["down"], st["b_down"], C["down"])
        return {"out": out + x if c["residual"] else out}
