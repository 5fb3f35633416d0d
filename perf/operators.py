"""The measured work of the operators that use MXFP4 weights after a decode: the norm before a product, the product
itself and the gated activation between two products, through the entry points of ``ptwm_amd.api``.

Formats are the OCP microscaling ones: 32 values share a scale byte b that stands for 2^(b - 127) (255: NaN). Weights
are e2m1 codes, two a byte with the first value in the low bits, as a container's nibble chain restores them;
activations in 8 bits are e4m3 codes. A block of activations takes the smallest scale whose largest code, 448, reaches
its largest magnitude.

A case is one call (a pass) of a decoder layer's feed-forward or projection, for one token (a step of generation),
a few (a batch of them) or many (a prompt).
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
EPS = 1e-5
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# Passes over the weights that an exact product takes with operands of 8 significant bits, by the activations' type.
PASSES = {"bf16": 1, "e4m3": 1, "f16": 2, "f32": 3}

OTHER = 3072  # a size that none of this repository's models has: not drawn


def linear(tokens, rows, cols, x, out="bf16", bias=False, name=None):
    c = {"op": "linear", "tokens": tokens, "rows": rows, "cols": cols, "x": x, "out": out, "bias": bias}
    return c if name is None else dict(c, name=name)


def norm(tokens, cols, x, residual, name=None):
    c = {"op": "norm", "tokens": tokens, "cols": cols, "x": x, "residual": residual}
    return c if name is None else dict(c, name=name)


def swiglu(tokens, cols, x, name=None):
    c = {"op": "swiglu", "tokens": tokens, "cols": cols, "x": x}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # A key projection (a quarter of the hidden size) of one token: the smallest product, latency counts.
        linear(1, 1024, 4096, "bf16", name="linear 1024x4096, 1"),
        # The feed-forward's first product for one token, from activations as the model keeps them.
        linear(1, 14336, 4096, "bf16", name="linear 14336x4096, 1"),
        # Its last product for one token, from 8-bit activations: the long reduction.
        linear(1, 4096, 14336, "e4m3", name="linear 4096x14336, 1 e4m3"),
        # A step of generation for a batch of sixteen.
        linear(16, 14336, 4096, "e4m3", name="linear 14336x4096, 16 e4m3"),
        # Odd sizes with a bias: a head of a fine-tuned model over a short ragged batch.
        linear(37, 5001, 3360, "f16", "f16", True, name="linear 5001x3360, 37 f16"),
        # A prompt from activations as the model keeps them.
        linear(512, 14336, 4096, "bf16", name="linear 14336x4096, 512"),
        # A long prompt from 8-bit activations: the largest, bound by the matrix cores.
        linear(2048, 14336, 4096, "e4m3", name="linear 14336x4096, 2048 e4m3"),
        # The norm before a feed-forward for one token: latency.
        norm(1, 4096, "bf16", True, name="norm 1x4096"),
        # For a long prompt.
        norm(2048, 4096, "bf16", True, name="norm 2048x4096"),
        # A model that keeps its residual stream in 32 bits, odd sizes, the first norm (nothing to add yet).
        norm(333, 5024, "f32", False, name="norm 333x5024 f32"),
        # The activation between the products for a small batch of generation.
        swiglu(7, 14336, "f16", name="swiglu 7x14336 f16"),
        # For a long prompt; gate and up are the halves of one product's output.
        swiglu(2048, 14336, "bf16", name="swiglu 2048x14336"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "swiglu"])
    if op == "linear":
        x = rng.choice(["bf16", "bf16", "e4m3", "e4m3", "f16", "f32"])
        out = x if x != "e4m3" and rng.random() < 0.6 else rng.choice(["bf16", "f16", "f32"])
        while True:
            t, n, k = _log_int(rng, 1, 2048), _log_int(rng, 64, 28672), 32 * _log_int(rng, 2, 448)
            if t * n * k * PASSES[x] <= 2048 * 14336 * 4096 and n * k <= 14336 * 4096 and OTHER not in (t, n, k):
                return linear(t, n, k, x, out, rng.random() < 0.4)
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        t, k = _log_int(rng, 1, 4096), 32 * _log_int(rng, 2, 448)
        if t * k * (2 if op == "swiglu" else 1) <= 2048 * 8192 and OTHER not in (t, k):
            return norm(t, k, x, rng.random() < 0.7) if op == "norm" else swiglu(t, k, x)


def _blocks(v):
    """(codes, scales) of float32 rows in blocks of 32."""
    b = v.reshape(v.shape[0], -1, 32)
    bits = b.abs().amax(-1).view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp(0, 254)
    inverse = ((254 - byte) << 23).view(torch.float32)
    broken = bits >= 0x7F800000
    scaled = torch.where(broken.unsqueeze(-1), math.nan, b * inverse.unsqueeze(-1))
    byte = torch.where(broken, 255, byte).to(torch.uint8)
    return scaled.to(torch.float8_e4m3fn).reshape(v.shape), byte.view(torch.float8_e8m0fnu)


def _weights(rows, cols, g):
    """N(0, 0.02) weights as a checkpoint keeps them: the scale leaves the block's largest magnitude in [4, 8), of
    which more than 6 is cut to 6."""
    w = torch.randn((rows, cols // 32, 32), generator=g, device=DEVICE) * 0.02
    e = torch.frexp(w.abs().amax(-1))[1] - 3
    mag = torch.ldexp(w.abs(), -e.unsqueeze(-1))
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEVICE)
    code = (torch.bucketize(mag, bounds, out_int32=True) + 8 * (w < 0)).to(torch.uint8).reshape(rows, cols)
    return code[:, 0::2] | code[:, 1::2] << 4, (e + 127).to(torch.uint8)


def _activations(tokens, cols, g, scale=1.0):
    """Normal values, one channel in 64 ten times as large, as residual streams have them."""
    loud = torch.where(torch.rand(cols, generator=g, device=DEVICE) < 1 / 64, 10.0, 1.0)
    return torch.randn((tokens, cols), generator=g, device=DEVICE) * loud * scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    t, k, kind = case["tokens"], case["cols"], case["x"]
    s = {"case": case}
    if case["op"] == "linear":
        n = case["rows"]
        s["weight"], s["scales"] = _weights(n, k, g)
        x = _activations(t, k, g)
        if kind == "e4m3":
            s["x"], s["x_scales"] = _blocks(x)
        else:
            s["x"], s["x_scales"] = x.to(TYPES[kind]), None
        s["bias"] = torch.randn(n, generator=g, device=DEVICE).to(TYPES[case["out"]]) if case["bias"] else None
        s["out"] = torch.empty((t, n), dtype=TYPES[case["out"]], device=DEVICE)
        return s
    if case["op"] == "norm":
        s["x"] = _activations(t, k, g).to(TYPES[kind])
        s["weight"] = (1 + 0.1 * torch.randn(k, generator=g, device=DEVICE)).to(TYPES[kind])
        s["residual"] = _activations(t, k, g, 4.0).to(TYPES[kind]) if case["residual"] else None
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
    else:
        both = (_activations(t, 2 * k, g) * 2).to(TYPES[kind])  # the halves of one product's output
        s["gate"], s["up"] = both[:, :k], both[:, k:]
    s["codes"] = torch.empty((t, k), dtype=torch.float8_e4m3fn, device=DEVICE)
    s["code_scales"] = torch.empty((t, k // 32), dtype=torch.float8_e8m0fnu, device=DEVICE)
    return s


def _plain_linear(s):
    w, x = s["weight"], s["x"].float()
    value = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEVICE)
    codes = torch.stack((value[(w & 15).int()], value[(w >> 4).int()]), -1)
    scale = s["scales"].view(torch.float8_e8m0fnu).float()
    w = (codes.reshape(w.shape[0], -1, 32) * scale.unsqueeze(-1)).reshape(w.shape[0], -1)
    if s["x_scales"] is not None:
        x = (x.reshape(x.shape[0], -1, 32) * s["x_scales"].float().unsqueeze(-1)).reshape(x.shape)
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["out"].dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from ptwm_amd import api

        if op == "linear":
            api.mxfp4_linear_cuda(s["x"], s["weight"], s["scales"], s["out"], 0, x_scales=s["x_scales"],
                                  bias=s["bias"])
            return s["out"]
        if op == "norm":
            api.rms_norm_mx_cuda(s["x"], s["weight"], s["codes"], s["code_scales"], 0, residual=s["residual"],
                                 sum_out=s["sum"], eps=EPS)
            return {"codes": s["codes"], "scales": s["code_scales"], "sum": s["sum"]}
        api.swiglu_mx_cuda(s["gate"], s["up"], s["codes"], s["code_scales"], 0)
        return {"codes": s["codes"], "scales": s["code_scales"]}
    if op == "linear":
        return _plain_linear(s)
    if op == "norm":
        x, total = s["x"].float(), None
        if s["residual"] is not None:
            x = x + s["residual"].float()
            total = x.to(s["x"].dtype)
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        codes, scales = _blocks(y)
        return {"codes": codes, "scales": scales, "sum": total}
    gate, up = s["gate"].float(), s["up"].float()
    codes, scales = _blocks(gate / (1 + torch.exp(-gate)) * up)
    return {"codes": codes, "scales": scales}


def exact(case, seed):
    """In 64 bits and before the last rounding: the numbers that codes and outputs are rounded from. The scales are
    powers of two, decided by comparison, and have no such number."""
    s = prepare(case, seed)

    def codes_of(y):
        b = y.reshape(y.shape[0], -1, 32)
        m, e = torch.frexp(b.abs().amax(-1) / 448)
        e = torch.where(m > 0.5, e, e - 1).clamp(-127, 127)
        return {"codes": torch.ldexp(b, -e.unsqueeze(-1)).reshape(y.shape), "scales": None}

    if case["op"] == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x += s["residual"].double()
        root = (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / case["cols"] + EPS).sqrt()
        return {**codes_of(x / root * s["weight"].double()), "sum": x if s["residual"] is not None else None}
    if case["op"] == "swiglu":
        return codes_of(s["gate"].double() * torch.sigmoid(s["gate"].double()) * s["up"].double())
    rows = []
    for w, e in zip(s["weight"].split(2048), s["scales"].split(2048)):
        c = torch.stack((w & 15, w >> 4), -1).reshape(w.shape[0], -1, 32).int()
        m, x = (c & 1).double(), (c >> 1) & 3  # e2m1: (1 + m/2) 2^(x - 1), or m/2 where x is 0
        v = torch.where(x > 0, torch.ldexp(1 + m / 2, x - 1), m / 2) * (1 - 2 * (c >> 3))
        rows.append(torch.ldexp(v, e.int().unsqueeze(-1) - 127).reshape(w.shape[0], -1))
    x = s["x"].double()
    if s["x_scales"] is not None:
        e = s["x_scales"].view(torch.uint8).int() - 127
        x = torch.ldexp(x.reshape(x.shape[0], -1, 32), e.unsqueeze(-1)).reshape(x.shape)
    y = torch.cat([x @ w.t() for w in rows], 1)
    return y if s["bias"] is None else y + s["bias"].double()


def work(case):
    t, k, size = case["tokens"], case["cols"], SIZE[case["x"]]
    if case["op"] == "linear":
        n = case["rows"]
        x = t * k * size + (t * k // 32 if case["x"] == "e4m3" else 0)
        out = (t * n + (n if case["bias"] else 0)) * SIZE[case["out"]]
        return {"bytes": n * k // 2 + n * k // 32 + x + out, "flops": 2 * t * n * k}
    codes = t * k + t * k // 32
    if case["op"] == "norm":
        return {"bytes": t * k * size * (3 if case["residual"] else 1) + k * size + codes, "flops": 5 * t * k}
    return {"bytes": 2 * t * k * size + codes, "flops": 6 * t * k}
