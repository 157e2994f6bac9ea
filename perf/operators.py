"""Measured cases of the 8-bit linear path: row quantiser, norms with 8-bit output, 8-bit linear layer.

``own = False`` runs each operator in its plain form (elementary torch operations in 32 bits);
``own = True`` makes the calls a user makes of ``streaming_sparse_b200.ops``. Sizes are those of the
streaming DiT's layers: width 1536, feed-forward 8960, 1560 tokens a frame, 4680 a chunk, 32760 a window.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
TINY = 1e-30          # the smallest scale: a row of zeros keeps a finite one
EPS = 1e-6
WIDEST = 8960
MOST_ROWS = 32760


def listed():
    return [
        # one token through the feed-forward's first product: latency, the weights read once
        dict(name="linear-1tok-ffn1", op="linear", rows=1, out=8960, width=1536, dtype="bf16", bias=True, gelu=True),
        # a short prompt, nothing a multiple of a tile, 32-bit output
        dict(name="linear-77tok-odd", op="linear", rows=77, out=1531, width=1549, dtype="fp32", bias=True, gelu=False),
        # a chunk's fused q/k/v product
        dict(name="linear-chunk-qkv", op="linear", rows=4680, out=4608, width=1536, dtype="bf16", bias=True,
             gelu=False),
        # a chunk's second feed-forward product: the long reduction
        dict(name="linear-chunk-ffn2", op="linear", rows=4680, out=1536, width=8960, dtype="fp16", bias=True,
             gelu=False),
        # a whole window through the first feed-forward product: the largest call
        dict(name="linear-window-ffn1", op="linear", rows=32760, out=8960, width=1536, dtype="bf16", bias=True,
             gelu=True),
        # one token between two layers
        dict(name="rms-1tok", op="rms", rows=1, width=1536, dtype="bf16", residual=True, pad=0),
        # odd width, 32-bit stream, rows inside a wider buffer, no residual
        dict(name="rms-odd-fp32", op="rms", rows=1003, width=1537, dtype="fp32", residual=False, pad=5),
        # a whole window's residual add and norm
        dict(name="rms-window", op="rms", rows=32760, width=1536, dtype="bf16", residual=True, pad=0),
        # a frame's affine norm (the cross-attention's input)
        dict(name="adaln-frame-affine", op="adaln", rows=1560, width=1536, dtype="fp16", frame=1560, residual=False,
             affine=True),
        # a chunk's gated residual add, norm and modulation, one set of vectors a frame
        dict(name="adaln-chunk-gate", op="adaln", rows=4680, width=1536, dtype="bf16", frame=1560, residual=True,
             affine=False),
        # a few tokens' activations, rows inside a wider buffer
        dict(name="quant-7tok", op="quant", rows=7, width=8960, dtype="fp16", pad=1536),
        # a chunk's feed-forward activations
        dict(name="quant-chunk-ffn", op="quant", rows=4680, width=8960, dtype="bf16", pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "rms", "rms", "adaln", "quant"])
    rows, width = _log(rng, 1, MOST_ROWS), _log(rng, 64, WIDEST)
    if rng.random() < 0.5:
        width = max(16, width // 16 * 16)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "linear":
        out = _log(rng, 64, WIDEST)
        rows = min(rows, max(1, MOST_ROWS * 8960 * 1536 // (out * width)))
        return dict(op=op, rows=rows, out=out, width=width, dtype=dtype, bias=rng.random() < 0.7,
                    gelu=rng.random() < 0.4)
    rows = min(rows, max(1, MOST_ROWS * 4 * 1536 // width))
    if op == "rms":
        return dict(op=op, rows=rows, width=width, dtype=dtype, residual=rng.random() < 0.6,
                    pad=rng.choice([0, 0, 8, 3]))
    if op == "adaln":
        return dict(op=op, rows=rows, width=width, dtype=rng.choice(["bf16", "fp16"]),
                    frame=max(1, rows // rng.choice([1, 2, 3])), residual=rng.random() < 0.6,
                    affine=rng.random() < 0.4)
    return dict(op=op, rows=rows, width=width, dtype=dtype, pad=rng.choice([0, 0, 16, 7]))


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(g, rows, width, spread=1.0):
    """Rows of different loudness with a few loud channels, as a deep layer's stream has."""
    x = torch.randn(rows, width, device=DEV, generator=g) * spread
    x *= 0.25 + 2 * torch.rand(rows, 1, device=DEV, generator=g)
    loud = torch.randint(0, width, (max(1, width // 256),), device=DEV, generator=g)
    x[:, loud] *= 6
    return x


def _padded(x, dtype, pad):
    """x as rows inside a buffer that is ``pad`` elements wider."""
    buf = torch.zeros(x.shape[0], x.shape[1] + pad, device=DEV, dtype=dtype)
    buf[:, :x.shape[1]] = x
    return buf[:, :x.shape[1]]


def _codes(x):
    """8-bit codes (rows at multiples of 16 bytes) and scales of rows of x."""
    rows, width = x.shape
    s = (x.abs().amax(1) / 127).clamp_min(TINY)
    buf = torch.zeros(rows, -(-width // 16) * 16, device=DEV, dtype=torch.int8)
    buf[:, :width] = torch.round(x / s[:, None]).to(torch.int8)
    return buf[:, :width], s


def prepare(case, seed):
    g = _gen(seed)
    rows, width, dtype = case["rows"], case["width"], TYPES[case["dtype"]]
    st = dict(case)
    if case["op"] == "linear":
        st["x"], st["xs"] = _codes(_activations(g, rows, width))
        st["w"], st["ws"] = _codes(torch.randn(case["out"], width, device=DEV, generator=g) / math.sqrt(width))
        st["b"] = (0.2 * torch.randn(case["out"], device=DEV, generator=g)).to(dtype) if case["bias"] else None
        return st
    st["x"] = _padded(_activations(g, rows, width), dtype, case.get("pad", 0))
    if case["op"] == "quant":
        return st
    st["r"] = None
    if case["residual"]:
        st["r"] = _padded(_activations(g, rows, width, 0.5), dtype, case.get("pad", 0))
    st["w"] = (1 + 0.1 * torch.randn(width, device=DEV, generator=g)).to(dtype)
    if case["op"] == "adaln":
        frames = -(-rows // case["frame"])
        st["b"] = (0.1 * torch.randn(width, device=DEV, generator=g)).to(dtype)
        vectors = 0.3 * torch.randn(frames, 3, width, device=DEV, generator=g)
        st["shift"], st["scale"], st["gate"] = vectors[:, 0], vectors[:, 1], vectors[:, 2]
    return st


def run(state):
    return _own(state) if own else _plain(state)


# -- the framework's operators ------------------------------------------------------------------
def _values(codes, scales, dtype):
    """What the codes stand for."""
    return torch.mul(codes, scales[:, None], out=torch.empty(codes.shape, device=codes.device, dtype=dtype))


def _own(st):
    from streaming_sparse_b200 import ops

    dtype = TYPES[st["dtype"]]
    if st["op"] == "linear":
        return ops.linear_i8(st["x"], st["xs"], st["w"], st["ws"], bias=st["b"], gelu=st["gelu"], out_dtype=dtype)
    if st["op"] == "quant":
        codes, scales = ops.quant_rows(st["x"])
        return {"values": _values(codes, scales, dtype), "scales": scales}
    if st["op"] == "rms":
        got = ops.rms_norm_i8(st["x"], st["w"], EPS, residual=st["r"])
    elif st["affine"]:
        got = ops.adaln_i8(st["x"], eps=EPS, weight=st["w"], bias=st["b"], y=st["r"])
    else:
        got = ops.adaln_i8(st["x"], eps=EPS, shift=st["shift"], scale=st["scale"], frame_tokens=st["frame"],
                           y=st["r"], gate=st["gate"] if st["r"] is not None else None)
    res = {"values": _values(got[0], got[1], dtype), "scales": got[1]}
    if st["r"] is not None:
        res["sum"] = got[2]
    return res


# -- their plain forms ----------------------------------------------------------------------------
def _quantised(t):
    """Codes of the rows of t as floats and their scales; a row that is not finite: zeros and NaN."""
    u = (t.abs().amax(1, keepdim=True) / 127).clamp_min(TINY)
    fine = torch.isfinite(u)
    return torch.where(fine, torch.round(t * (1 / u)), 0.0), torch.where(fine, u, math.nan)


def _by_row(v, st):
    """Row r's vector of the per-frame vectors v."""
    return v[torch.arange(st["rows"], device=DEV) // st["frame"]]


def _plain(st):
    dtype = TYPES[st["dtype"]]
    if st["op"] == "linear":
        v = (st["x"].float() @ st["w"].float().t()) * (st["xs"][:, None] * st["ws"][None, :])
        if st["b"] is not None:
            v = v + st["b"].float()
        if st["gelu"]:
            v = 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
        return v.to(dtype)
    x = st["x"].float()
    if st["op"] == "quant":
        q, u = _quantised(x)
        return {"values": (q * u).to(dtype), "scales": u[:, 0]}
    if st["r"] is not None:
        r = st["r"].float()
        if st["op"] == "adaln" and not st["affine"]:
            r = r * _by_row(st["gate"], st)
        x = x + r
    if st["op"] == "rms":
        q, u = _quantised(x * st["w"].float())
        u = u * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    else:
        z = x - x.mean(1, keepdim=True)
        z = z * torch.rsqrt((z * z).mean(1, keepdim=True) + EPS)
        if st["affine"]:
            z = z * st["w"].float() + st["b"].float()
        else:
            z = z * (1 + _by_row(st["scale"], st)) + _by_row(st["shift"], st)
        q, u = _quantised(z)
    res = {"values": (q * u).to(dtype), "scales": u[:, 0]}
    if st["r"] is not None:
        res["sum"] = x.to(dtype)
    return res


# -- the definition in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    D = torch.float64
    if case["op"] == "linear":
        out = torch.empty(case["rows"], case["out"], device=DEV, dtype=D)
        w = (st["w"].to(D) * st["ws"].to(D).view(-1, 1)).t()
        for i in range(0, case["rows"], 4096):
            y = (st["x"][i:i + 4096].to(D) * st["xs"][i:i + 4096].to(D).view(-1, 1)) @ w
            if st["b"] is not None:
                y += st["b"].to(D)
            if case["gelu"]:
                y = y / (1 + torch.exp(-math.sqrt(8 / math.pi) * (y + 0.044715 * y.pow(3))))
            out[i:i + 4096] = y
        return out
    y = st["x"].to(D)
    frame = torch.arange(case["rows"], device=DEV).div(case.get("frame", 1), rounding_mode="floor")
    total = None
    if st.get("r") is not None:
        add = st["r"].to(D)
        if case["op"] == "adaln" and not case["affine"]:
            add = add * st["gate"].to(D).index_select(0, frame)
        y = total = y + add
    if case["op"] == "rms":
        y = st["w"].to(D) * y / (y.square().mean(1, keepdim=True) + EPS).sqrt()
    elif case["op"] == "adaln":
        var, mean = torch.var_mean(y, 1, correction=0, keepdim=True)
        y = (y - mean) / (var + EPS).sqrt()
        if case["affine"]:
            y = st["b"].to(D) + st["w"].to(D) * y
        else:
            y = st["shift"].to(D).index_select(0, frame) + y * (1 + st["scale"].to(D).index_select(0, frame))
    step = y.abs().max(1, keepdim=True).values / 127
    res = {"values": torch.round(y / step) * step, "scales": step[:, 0]}
    if total is not None:
        res["sum"] = total
    return res


def work(case):
    rows, width, b = case["rows"], case["width"], SIZE[case["dtype"]]
    if case["op"] == "linear":
        n = case["out"]
        return {"bytes": rows * width + n * width + 4 * (rows + n) + (b * n if case["bias"] else 0) + b * rows * n,
                "flops": 2 * rows * n * width}
    nbytes = rows * width * (b + 1) + 4 * rows
    flops = 4 * rows * width
    if case["op"] != "quant":
        flops += 4 * rows * width
        if case["residual"]:
            nbytes += 2 * rows * width * b
            flops += rows * width
        if case["op"] == "rms" or case["affine"]:
            nbytes += width * b * (1 if case["op"] == "rms" else 2)
        else:
            nbytes += 4 * width * -(-rows // case["frame"]) * (3 if case["residual"] else 2)
    return {"bytes": nbytes, "flops": flops}
