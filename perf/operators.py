"""Performance cases of the 8-bit serving path of an encoder block: the norm that hands its rows on in 8 bits, the
quantiser for everything else, and the matrix product that reads both.

  norm      root-mean-square norm of rows, optionally with the residual's addition in front (the sum comes back too),
            its result in the input's type or in 8 bits (e4m3) with one scale per row and 128 channels;
  quantize  a tensor into 8 bits with one scale per row and 128 channels (activations) or per 128 x 128 block (weights);
  linear    a @ w.T of two such tensors, with bias, GELU and residual in the same pass; the result in bfloat16, float32
            or again in 8 bits with scales.

Formulas (all in 32 bits or more, rounded once where they are stored):
  s = x + residual (stored in x's type);  y = s * (mean(s^2) + eps)^-1/2 * weight
  scale = max(amax|block| / 448, 2^-126);  q = e4m3(v / scale);  the value that is meant is q * scale
  out = [gelu](sum_k (qa * scale_a) (qw * scale_w) + bias) + residual

``listed()`` are fixed cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` makes what a program holds
before the call, ``run`` is one pass: through elementary torch operations, or with ``own`` through the package.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128          # channels that share a scale; rows too in a weight
TOP = 448.0          # the largest e4m3 value
LEAST = 2.0 ** -126  # the least scale
EPS = 1e-6
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(name, rows, d, dtype="bf16", residual=True, quantize=True, wider=0):
    c = dict(kind="norm", rows=rows, d=d, dtype=dtype, residual=residual, quantize=quantize, wider=wider)
    return dict(c, name=name) if name else c


def _quantize(name, rows, d, dtype="bf16", weight=False):
    c = dict(kind="quantize", rows=rows, d=d, dtype=dtype, weight=weight)
    return dict(c, name=name) if name else c


def _linear(name, m, n, k, out="bf16", bias=False, gelu=False, residual=False):
    c = dict(kind="linear", m=m, n=n, k=k, out=out, bias=bias, gelu=gelu, residual=residual)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of a generating model: latency alone
        _norm("norm_1x768", 1, 768),
        # 256 images of 197 tokens in front of the MLP of ViT-Tiny
        _norm("norm_50432x192", 256 * 197, 192),
        # eight sequences of 16384 tokens, 768 channels: the longest of the layer benchmark
        _norm("norm_131072x768", 8 * 16384, 768),
        # float32, odd width, nothing fused: a final norm
        _norm("norm_fp32_4099x1001", 4099, 1001, dtype="fp32", residual=False, quantize=False),
        # the weights of a wide layer, once per set of weights or update
        _quantize("quantize_weight_4096x4096", 4096, 4096, weight=True),
        # activations that no norm produced: attention output of the images above in front of the output projection
        _quantize("quantize_rows_50432x768", 256 * 197, 768),
        # one token against a wide layer: reads the weights, computes next to nothing
        _linear("linear_1x4096x4096", 1, 4096, 4096),
        # a few dozen sequences in decoding
        _linear("linear_48x8192x2048", 48, 8192, 2048, bias=True),
        # one image through the packed q, k, v projection of 768 channels
        _linear("linear_197x2304x768", 197, 2304, 768),
        # the MLP of ViT-Tiny on 256 images, first half: narrow, GELU, 8 bits out for the second
        _linear("linear_gelu_fp8_50432x768x192", 256 * 197, 768, 192, out="fp8", bias=True, gelu=True),
        # ragged in every direction, float32 logits
        _linear("linear_fp32_1027x1003x1333", 1027, 1003, 1333, out="fp32", bias=True),
        # a long prompt through a wide layer
        _linear("linear_16384x4096x4096", 16384, 4096, 4096, residual=True),
    ]


MOST_VALUES = 8 * 16384 * 768            # of a norm or a quantiser
MOST_MACS = 16384 * 4096 * 4096


def _between(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind != "linear":
        d = _between(rng, 64, 16384)
        if rng.random() < 0.6:
            d = -(-d // 64) * 64
        most = MOST_VALUES if dtype == "bf16" else MOST_VALUES // 2
        rows = _between(rng, 1, min(131072, most // d))
        if kind == "norm":
            return _norm(None, rows, d, dtype, rng.random() < 0.7, rng.random() < 0.6, rng.choice([0, 0, 64]))
        return _quantize(None, rows, d, dtype, rng.random() < 0.3)
    n, k = _between(rng, 64, 8192), _between(rng, 64, 8192)
    if rng.random() < 0.6:
        n, k = -(-n // 64) * 64, -(-k // 64) * 64
    m = _between(rng, 1, min(65536, MOST_MACS // (n * k)))
    out = rng.choice(["bf16", "bf16", "fp32", "fp8"])
    return _linear(None, m, n, k, out, rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.4)


# ---- the plain form -------------------------------------------------------------------------------------------------

def _by_block(t, rows, cols):
    """(R, C) with zeros around it -> (R / rows, rows, C / cols, cols)."""
    r, c = t.shape
    t = torch.nn.functional.pad(t, (0, -c % cols, 0, -r % rows))
    return t.view(t.shape[0] // rows, rows, t.shape[1] // cols, cols)


def _to_blocks(v, rows):
    """Values in 32 or 64 bits -> (e4m3 values, scales)."""
    b = _by_block(v, rows, BLOCK)
    scale = torch.clamp(b.abs().amax(dim=(1, 3)) * (1.0 / TOP), min=LEAST)
    q = (b * (1.0 / scale)[:, None, :, None]).reshape(b.shape[0] * rows, -1)[:v.shape[0], :v.shape[1]]
    return q.to(E4M3).contiguous(), scale


def _from_blocks(q, scale, rows, dtype):
    s = scale.to(dtype).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    return q.to(dtype) * (s if rows == 1 else s.repeat_interleave(rows, 0)[:q.shape[0]])


def _gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _plain_norm(s, cast, dtype):
    """cast: the type that is computed in."""
    x = s["x"].to(cast)
    total = None
    if s["residual"] is not None:
        total = (x + s["residual"].to(cast)).to(dtype)
        x = total.to(cast)
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s["weight"].to(cast)
    if s["quantize"]:
        y = _to_blocks(y, 1)
    elif cast == torch.float32:
        y = y.to(dtype)
    return y if total is None else (y, total)


def _plain_linear(s, cast):
    out = _from_blocks(*s["a"], 1, cast) @ _from_blocks(*s["w"], BLOCK, cast).t()
    if s["bias"] is not None:
        out += s["bias"].to(cast)
    if s["gelu"]:
        out = _gelu(out)
    if s["residual"] is not None:
        out += s["residual"].to(cast)
    if s["out"] == "fp8":
        return _to_blocks(out, 1)
    return out.to(TYPES[s["out"]]) if cast == torch.float32 else out


# ---- the cases ------------------------------------------------------------------------------------------------------

def _store8(q, scale):
    """As the quantisers hand them on: rows from 16-byte boundaries, the scales of one block of channels side by side."""
    room = torch.zeros(q.shape[0], -(-q.shape[1] // 16) * 16, dtype=torch.uint8, device=q.device)
    room[:, :q.shape[1]] = q.view(torch.uint8)
    return room.view(E4M3)[:, :q.shape[1]], scale.t().contiguous().t()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        dtype = TYPES.get(case["out"], torch.bfloat16)
        a = randn(m, k)
        a *= torch.exp(0.5 * randn(k))                 # some channels are louder than others
        a = _store8(*_to_blocks(a, 1))
        w = _store8(*_to_blocks(randn(n, k) / math.sqrt(k), BLOCK))
        return dict(kind="linear", a=a, w=w, out=case["out"], dtype=dtype, gelu=case["gelu"],
                    bias=(0.5 * randn(n)).to(dtype) if case["bias"] else None,
                    residual=randn(m, n).to(dtype) if case["residual"] else None)
    dtype, rows, d = TYPES[case["dtype"]], case["rows"], case["d"]
    if case["kind"] == "quantize":
        return dict(kind="quantize", x=(randn(rows, d) * torch.exp(0.5 * randn(d))).to(dtype), weight=case["weight"])
    # (`wider`: the rows are a channel slice of a wider tensor)
    x = randn(rows, d + case["wider"]).to(dtype)[:, :d]
    return dict(kind="norm", x=x, weight=(1.0 + 0.2 * randn(d)).to(dtype), quantize=case["quantize"],
                residual=(2.0 * randn(rows, d)).to(dtype) if case["residual"] else None)


def run(state):
    s = state
    if own:
        from convnn_b200 import ops
        if s["kind"] == "norm":
            return ops.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], quantize=s["quantize"])
        if s["kind"] == "quantize":
            return ops.quantize_fp8(s["x"], block_rows=BLOCK if s["weight"] else 1)
        return ops.linear_fp8(s["a"], s["w"], bias=s["bias"], gelu=s["gelu"], residual=s["residual"], dtype=s["dtype"],
                              quantize=s["out"] == "fp8")
    if s["kind"] == "norm":
        return _plain_norm(s, torch.float32, s["x"].dtype)
    if s["kind"] == "quantize":
        return _to_blocks(s["x"].float(), BLOCK if s["weight"] else 1)
    return _plain_linear(s, torch.float32)


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        elt = {"bf16": 2, "fp32": 4, "fp8": 1}[case["out"]]
        side = 4 if case["out"] == "fp32" else 2
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        moved = m * k + n * k + 4 * (m * kb + nb * kb) + elt * m * n
        moved += side * (n * case["bias"] + m * n * case["residual"]) + (4 * m * nb if case["out"] == "fp8" else 0)
        return {"bytes": moved, "flops": 2 * m * n * k}
    rows, d = case["rows"], case["d"]
    elt = 4 if case["dtype"] == "fp32" else 2
    blocks = -(-d // BLOCK)
    if case["kind"] == "quantize":
        scales = (-(-rows // BLOCK) if case["weight"] else rows) * blocks
        return {"bytes": (elt + 1) * rows * d + 4 * scales, "flops": 2 * rows * d}
    moved = elt * rows * d * (3 if case["residual"] else 1) + elt * d
    moved += rows * (d + 4 * blocks) if case["quantize"] else elt * rows * d
    return {"bytes": moved, "flops": (4 + 2 * case["quantize"] + case["residual"]) * rows * d}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _exact_blocks(v, rows):
    """Block by block of channels."""
    q, scales = torch.empty_like(v), []
    of_row = torch.arange(v.shape[0], device=v.device) // rows
    for c in range(0, v.shape[1], BLOCK):
        part = v[:, c:c + BLOCK]
        most = part.abs().max(dim=1).values
        top = torch.zeros(int(of_row[-1]) + 1, dtype=v.dtype, device=v.device)
        top.scatter_reduce_(0, of_row, most, "amax")
        scale = torch.maximum(top / TOP, torch.tensor(LEAST, dtype=v.dtype, device=v.device))
        q[:, c:c + BLOCK] = part / scale[of_row, None]
        scales.append(scale)
    # the nearest of the e4m3 values: steps of 2^-3 relative to the power of two below, of 2^-9 under 2^-6
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return [torch.round(q / step) * step, torch.stack(scales, 1)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return _exact_blocks(s["x"].double(), BLOCK if s["weight"] else 1)
    if case["kind"] == "norm":
        x, total = s["x"].double(), None
        if s["residual"] is not None:
            total = x + s["residual"].double()
            x = total.to(s["x"].dtype).double()        # the stored sum is what is normalised
        mean = torch.einsum("rd,rd->r", x, x) / x.shape[1]
        y = torch.einsum("rd,d,r->rd", x, s["weight"].double(), 1.0 / torch.sqrt(mean + EPS))
        if s["quantize"]:
            y = _exact_blocks(y, 1)
        return y if total is None else [y, total]
    (qa, sa), (qw, sw) = s["a"], s["w"]
    out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    by_n = torch.arange(case["n"], device="cuda") // BLOCK
    for j in range(sa.shape[1]):                       # one block of the sum at a time
        at = slice(BLOCK * j, min(BLOCK * (j + 1), case["k"]))
        part = qa[:, at].double() @ qw[:, at].double().t()
        out.addcmul_(part * sa[:, j, None].double(), sw[by_n, j].double()[None])
    if s["bias"] is not None:
        out += s["bias"].double()
    if s["gelu"]:
        out = out * torch.special.ndtr(out)
    if s["residual"] is not None:
        out += s["residual"].double()
    return _exact_blocks(out, 1) if s["out"] == "fp8" else out
