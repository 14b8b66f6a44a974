"""Microscaled (MX) layers of a decoder: 4-bit weights, 8-bit activations, as timed cases.

A weight row is cut into blocks of 32 values along the inner dimension.  A block holds one power of two
and 32 codes of 4 bits (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).  The rows that a weight is
multiplied with are cut the same way, with codes of 8 bits (E4M3).  ``kind`` says what a case calls:

* ``quantize_weight``  a weight to 4-bit blocks, and the values that they stand for;
* ``quantize_rows``    activations to 8-bit blocks, and the values that they stand for;
* ``linear``           y = x . w^T for fp16 rows x: the rows to 8-bit blocks, then the product;
* ``gated``            y = up * silu(gate), up and gate the halves of such a product.

The scale of a weight block is 2^(floor(log2 m) - 2), m the block's largest magnitude, and values past 6
become 6; the scale of a block of activations is the smallest power of two that leaves m no more than 448.
Values round to the nearest code, ties to the even one.  A block of zeros has the scale 2^-127.
"""

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
MOST_FLOPS = 2 * 8192 * 24576 * 4096  # the largest listed case


def listed():
    return [
        # A weight as it is loaded: an output projection in fp16.
        dict(name="weight_4096x4096", kind="quantize_weight", n_out=4096, n_in=4096, dtype="float16"),
        # The stacked up and gate projections of a checkpoint in bf16.
        dict(name="weight_24576x4096", kind="quantize_weight", n_out=24576, n_in=4096, dtype="bfloat16"),
        # The hidden states of a verify batch, 16 requests of 5 rows.
        dict(name="rows_80x4096", kind="quantize_rows", rows=80, n_in=4096),
        # The FFN's inner activations of a chunk of prompts.
        dict(name="rows_8192x12288", kind="quantize_rows", rows=8192, n_in=12288),
        # One token through a small model's projection: latency alone.
        dict(name="linear_1_1024x1024", kind="linear", rows=1, n_out=1024, n_in=1024),
        # A verify batch through the stacked q, k and v projections.
        dict(name="linear_80_6144x4096", kind="linear", rows=80, n_out=6144, n_in=4096),
        # A full decode batch through the down projection.
        dict(name="linear_128_4096x12288", kind="linear", rows=128, n_out=4096, n_in=12288),
        # The logits of a few rows: the largest weight that a model has.
        dict(name="linear_16_151936x4096", kind="linear", rows=16, n_out=151936, n_in=4096),
        # One ragged prompt, and a vocabulary shard of odd width.
        dict(name="linear_1237_18993x2080", kind="linear", rows=1237, n_out=18993, n_in=2080),
        # A verify batch through the up and gate projections.
        dict(name="gated_80_12288x4096", kind="gated", rows=80, inter=12288, n_in=4096),
        # A small model's decode batch through the same.
        dict(name="gated_33_2816x1024", kind="gated", rows=33, inter=2816, n_in=1024),
        # A chunk of prompts through them: the largest product of a layer.
        dict(name="gated_8192_12288x4096", kind="gated", rows=8192, inter=12288, n_in=4096),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    kind = rng.choice(["quantize_weight", "quantize_rows", "linear", "linear", "gated", "gated"])
    n_in = _spread(rng, 256, 12288, BLOCK)
    if kind == "quantize_weight":
        return dict(kind=kind, n_out=_spread(rng, 16, 24576 * 4096 // n_in), n_in=n_in,
                    dtype=rng.choice(["float16", "bfloat16", "float32"]))
    if kind == "quantize_rows":
        return dict(kind=kind, rows=_spread(rng, 1, 8192), n_in=n_in)
    # decode and verify batches as often as prompts
    rows = _spread(rng, 1, 128) if rng.random() < 0.5 else _spread(rng, 129, 8192)
    if kind == "gated":
        inter = _spread(rng, 256, 16384, 16)
        inter = max(256, min(inter, MOST_FLOPS // (4 * rows * n_in) // 16 * 16))
        return dict(kind=kind, rows=rows, inter=inter, n_in=n_in)
    n_out = _spread(rng, 17, 151936 if rows <= 32 and n_in <= 4096 else 32768)
    return dict(kind=kind, rows=rows, n_out=max(17, min(n_out, MOST_FLOPS // (2 * rows * n_in))), n_in=n_in)


# ---------------------------------------------------------------- the plain form


def _e2m1(v):
    """fp32 [n, k] -> 4-bit codes and scale bytes of its blocks."""
    v = v.view(v.shape[0], -1, BLOCK)
    most = v.abs().amax(-1, keepdim=True)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -127).clamp(min=-127)
    a = v.abs() * torch.exp2(-e.float())
    # the codes' spacing: 0.5 below 2, 1 below 4, 2 from there on
    code = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, 2 + torch.round(a), 4 + torch.round(a / 2)))
    code = code.clamp(max=7).to(torch.uint8) | ((v < 0).to(torch.uint8) << 3)
    return code.view(v.shape[0], -1), (e.squeeze(-1) + 127).to(torch.uint8)


def _e2m1_values(codes, scales):
    """Codes packed by two (the even one in the low half) and scale bytes -> fp32 [n, k]."""
    n = codes.shape[0]
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1)
    return (v.view(n, -1, BLOCK) * torch.exp2(scales.float() - 127)[..., None]).view(n, -1)


def _e4m3_values(x):
    """fp16 [n, k] -> the fp32 values that its 8-bit blocks stand for."""
    v = x.float().view(x.shape[0], -1, BLOCK)
    most = v.abs().amax(-1, keepdim=True)
    m, p = torch.frexp(most)
    e = torch.where(most > 0, p - 9 + (m > 0.875).to(p.dtype), -127).clamp(min=-127).float()
    a = v * torch.exp2(-e)
    step = torch.exp2(torch.frexp(a).exponent.clamp(min=-5).float() - 4)  # 3 bits after the leading one, 2^-9 at least
    return (torch.round(a / step) * step * torch.exp2(e)).view(x.shape)


def _product(x, codes, scales):
    return _e4m3_values(x) @ _e2m1_values(codes, scales).t().contiguous()


# ---------------------------------------------------------------- inputs


def _activations(g, rows, n_in):
    """Hidden states: unit variance, a few channels far larger, and a row of padding at the end of a batch."""
    x = torch.randn(rows, n_in, device=DEV, generator=g)
    x *= torch.where(torch.rand(n_in, device=DEV, generator=g) < 1 / 256, 24.0, 1.0)
    if rows > 8:
        x[-1] = 0
    return x.half()


def _weight(g, n_out, n_in):
    """A trained weight's values, its rows of different norms."""
    w = torch.randn(n_out, n_in, device=DEV, generator=g)
    return w.mul_((0.5 + torch.rand(n_out, 1, device=DEV, generator=g)) * n_in ** -0.5)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, n_in = case["kind"], case["n_in"]
    s = {"case": case}
    if kind == "quantize_weight":
        s["w"] = _weight(g, case["n_out"], n_in).to(getattr(torch, case["dtype"]))
        return s
    s["x"] = _activations(g, case["rows"], n_in)
    if kind == "quantize_rows":
        return s
    n_out = case["n_out"] if kind == "linear" else 2 * case["inter"]
    codes, scales = [], []
    for at in range(0, n_out, 16384):
        c, e = _e2m1(_weight(g, min(16384, n_out - at), n_in))
        codes.append(c[:, 0::2] | (c[:, 1::2] << 4))
        scales.append(e)
    s["codes"], s["scales"] = torch.cat(codes), torch.cat(scales)
    if own:
        from nebulasd_amd.kernels import mxfp4_pack
        s["weight"] = mxfp4_pack(s["codes"], s["scales"])
    return s


# ---------------------------------------------------------------- one pass


def run(s):
    kind = s["case"]["kind"]
    if own:
        from nebulasd_amd import kernels
        if kind == "quantize_weight":
            return kernels.mxfp4_dequantize(kernels.mxfp4_quantize(s["w"]))
        if kind == "quantize_rows":
            return kernels.mxfp8_dequantize(kernels.mxfp8_quantize(s["x"]))
        if kind == "linear":
            return kernels.mxfp4_linear(s["x"], s["weight"])
        return kernels.mxfp4_up_gate_silu_and_mul(s["x"], s["weight"])
    if kind == "quantize_weight":
        c, e = _e2m1(s["w"].float())
        return _e2m1_values(c[:, 0::2] | (c[:, 1::2] << 4), e).bfloat16()
    if kind == "quantize_rows":
        return _e4m3_values(s["x"]).bfloat16()
    y = _product(s["x"], s["codes"], s["scales"])
    if kind == "gated":
        up, gate = y.chunk(2, 1)
        y = up * (gate / (1 + torch.exp(-gate)))
    return y.half()


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    kind, k = case["kind"], case["n_in"]
    if kind == "quantize_weight":
        n = case["n_out"] * k
        size = 4 if case["dtype"] == "float32" else 2
        # the weight in, codes and scales out, and the values that they stand for
        return {"bytes": n * size + n // 2 + n // BLOCK + 2 * n, "flops": 2 * n}
    r = case["rows"]
    if kind == "quantize_rows":
        return {"bytes": 2 * r * k + r * k + r * k // BLOCK + 2 * r * k, "flops": 2 * r * k}
    n = case["n_out"] if kind == "linear" else 2 * case["inter"]
    out = n if kind == "linear" else case["inter"]
    return {"bytes": n * k // 2 + n * k // BLOCK + 2 * r * k + 2 * r * out, "flops": 2 * r * n * k}


# ---------------------------------------------------------------- the same in 64 bits


def _nearest(v, codes, top, largest_at_most):
    """Each block of 32 of v over its scale, to the nearest of the ascending `codes`, ties to the even place."""
    b = v.double().view(v.shape[0], -1, BLOCK)
    most = b.abs().amax(-1, keepdim=True)
    powers = torch.exp2(torch.arange(-127, 128, device=v.device, dtype=torch.float64))
    if largest_at_most:  # the first power of two with most <= top * power
        at = torch.searchsorted(powers * top, most.contiguous())
    else:                # the last one with most >= top * power (top: the largest code's own power of two)
        at = (torch.searchsorted(powers * top, most.contiguous(), right=True) - 1).clamp(min=0)
    scale = powers[at]
    codes = torch.tensor(codes, device=v.device, dtype=torch.float64)
    middle = (codes[1:] + codes[:-1]) / 2
    a = b.abs() / scale
    below, above = torch.searchsorted(middle, a), torch.searchsorted(middle, a, right=True)
    place = torch.where((below != above) & (below % 2 == 1), above, below)  # on a middle: the even one of the two
    return (torch.sign(b) * codes[place] * scale).view(v.shape)


_E2M1 = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
_E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (p - 3) for p in range(-6, 9) for m in range(8)][:-1]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "quantize_weight":
        return torch.cat([_nearest(w, _E2M1, 4.0, False) for w in s["w"].split(4096)])
    x = torch.cat([_nearest(t, _E4M3, 448.0, True) for t in s["x"].split(2048)])
    if case["kind"] == "quantize_rows":
        return x
    out, table = [], torch.tensor(_E2M1 + [-c for c in _E2M1], device=DEV, dtype=torch.float64)
    for codes, scales in zip(s["codes"].split(8192), s["scales"].split(8192)):
        w = table[torch.stack((codes % 16, codes // 16), -1).flatten(1).int()]
        w *= torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)
        out.append(x @ w.t().contiguous())
    y = torch.cat(out, 1)
    if case["kind"] == "gated":
        half = case["inter"]
        y = y[:, :half] * y[:, half:] * torch.sigmoid(y[:, half:])
    return y
