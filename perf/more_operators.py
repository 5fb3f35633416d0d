"""The measured work of the operators around MXFP4 tensors that came later than the product with such weights: the
quantisation to MXFP4, the product of two MXFP4 matrices, and a mixture-of-experts layer on MXFP4 experts for a few
tokens, through the entry points of ``ptwm_amd.api``.

Formats are the OCP microscaling ones: 32 values of a row share a scale byte b that stands for 2^(b - 127) (255: NaN);
values are e2m1 codes, two a byte with the first in the low bits.

A case is one call (a pass): a tensor quantised before it is coded, a projection whose activations are held in 4 bits
too, a decoder layer's experts for a step of generation.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E8M0 = torch.float8_e8m0fnu


def quantise(rows, cols, x, saturate=True, name=None):
    c = {"op": "quantise", "rows": rows, "cols": cols, "x": x, "saturate": saturate}
    return c if name is None else dict(c, name=name)


def matmul(tokens, rows, cols, out="bf16", bias=False, name=None):
    c = {"op": "matmul", "tokens": tokens, "rows": rows, "cols": cols, "out": out, "bias": bias}
    return c if name is None else dict(c, name=name)


def moe(tokens, experts, top_k, cols, inner, x="bf16", bias=False, name=None):
    c = {"op": "moe", "tokens": tokens, "experts": experts, "top_k": top_k, "cols": cols, "inner": inner, "x": x,
         "bias": bias}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # One token's activations before a product in 4 bits: the smallest call, latency counts.
        quantise(1, 4096, "bf16", name="quantise 1x4096"),
        # Activations of a short ragged batch that are kept in 32 bits, at odd sizes, with nothing cut off.
        quantise(333, 5024, "f32", False, name="quantise 333x5024 f32"),
        # A feed-forward matrix on its way into a compressed file.
        quantise(14336, 4096, "bf16", name="quantise 14336x4096"),
        # The feed-forward's first product for one token: the weights' way from memory.
        matmul(1, 14336, 4096, name="matmul 14336x4096, 1"),
        # Odd sizes with a bias: a head of a fine-tuned model over a short ragged batch.
        matmul(37, 5001, 3360, "f16", True, name="matmul 5001x3360, 37 f16"),
        # A prompt.
        matmul(512, 14336, 4096, name="matmul 14336x4096, 512"),
        # A long prompt: bound by the matrix cores.
        matmul(2048, 14336, 4096, name="matmul 14336x4096, 2048"),
        # Many small experts, one token: a step of generation that latency bounds.
        moe(1, 128, 8, 2048, 768, name="moe 128x2048x768, 1"),
        # A few large experts, one token: the chosen experts' way from memory.
        moe(1, 8, 2, 4096, 14336, name="moe 8x4096x14336, 1"),
        # Odd sizes, biases, a type with a narrow range: a short ragged batch.
        moe(7, 11, 3, 1120, 1504, "f16", True, name="moe 11x1120x1504, 7 f16"),
        # A batch of sixteen over experts of a middling size: most of them have a token or two.
        moe(16, 32, 4, 4096, 2048, name="moe 32x4096x2048, 16"),
        # The largest batch: every expert is read, with sixteen tokens on average.
        moe(64, 8, 2, 4096, 14336, name="moe 8x4096x14336, 64"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantise", "matmul", "moe", "moe"])
    if op == "quantise":
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        while True:
            t, k = _log_int(rng, 1, 16384), 32 * _log_int(rng, 2, 448)
            if t * k * SIZE[x] <= 14336 * 4096 * 2:
                return quantise(t, k, x, rng.random() < 0.6)
    if op == "matmul":
        while True:
            t, n, k = _log_int(rng, 1, 2048), _log_int(rng, 64, 28672), 32 * _log_int(rng, 2, 448)
            if t * n * k <= 2048 * 14336 * 4096 and n * k <= 14336 * 4096:
                return matmul(t, n, k, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.4)
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        t, e, k = _log_int(rng, 1, 64), _log_int(rng, 2, 128), rng.randint(1, 8)
        h, i = 32 * _log_int(rng, 4, 160), 32 * _log_int(rng, 2, 448)
        if k <= e and e * h * i <= 8 * 4096 * 14336 and t * k * h * i <= 128 * 4096 * 14336:
            return moe(t, e, k, h, i, x, rng.random() < 0.4)


def _codes_of(x, saturate):
    """(codes, scales) of float32 rows. With `saturate` a block's scale leaves its largest magnitude in [4, 8) and what
    is over 6 becomes 6; without it the scale is the smallest with which nothing is over 6."""
    b = x.reshape(x.shape[0], -1, 32)
    bits = b.abs().amax(-1).view(torch.int32)
    e = (bits >> 23) - 2
    if not saturate:
        e = e + ((bits & 0x7FFFFF) > 0x400000).to(torch.int32)
    e = e.clamp(0, 254)
    # by a power of two in two halves: the whole one may be below the normal numbers
    down = (127 - e).unsqueeze(-1)
    half = down >> 1
    power = lambda p: ((p + 127) << 23).view(torch.float32)  # noqa: E731
    v = b.abs() * power(half) * power(down - half)
    # to nearest, a tie to the even code: halves up to 2, wholes up to 4, twos above
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = (torch.round(v / step) * step).clamp(max=6.0)
    table = torch.tensor([0, 1, 2, 3, 4, 4, 5, 5, 6, 6, 6, 6, 7], dtype=torch.uint8, device=x.device)  # by twice the value
    code = table[(v * 2).int()] | (torch.signbit(b).to(torch.uint8) << 3)
    code = code.reshape(x.shape)
    return code[:, 0::2] | code[:, 1::2] << 4, e.to(torch.uint8)


def _activations(tokens, cols, g, scale=1.0):
    """Normal values, one channel in 64 ten times as large, as residual streams have them."""
    loud = torch.where(torch.rand(cols, generator=g, device=DEVICE) < 1 / 64, 10.0, 1.0)
    return torch.randn((tokens, cols), generator=g, device=DEVICE) * loud * scale


def _weights(rows, cols, g):
    return _codes_of(torch.randn((rows, cols), generator=g, device=DEVICE) * 0.02, True)


def _stack(experts, rows, cols, g):
    codes = torch.empty((experts, rows, cols // 2), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((experts, rows, cols // 32), dtype=torch.uint8, device=DEVICE)
    for c, s in zip(codes, scales):
        c[:], s[:] = _weights(rows, cols, g)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "quantise":
        t, k = case["rows"], case["cols"]
        s["x"] = (_activations(t, k, g) * 0.1).to(TYPES[case["x"]])
        s["codes"] = torch.empty((t, k // 2), dtype=torch.uint8, device=DEVICE)
        s["scales"] = torch.empty((t, k // 32), dtype=E8M0, device=DEVICE)
        return s
    if case["op"] == "matmul":
        t, n, k, out = case["tokens"], case["rows"], case["cols"], TYPES[case["out"]]
        s["weight"], s["scales"] = _weights(n, k, g)
        s["x"], s["x_scales"] = _codes_of(_activations(t, k, g), True)
        s["bias"] = torch.randn(n, generator=g, device=DEVICE).to(out) if case["bias"] else None
        s["out"] = torch.empty((t, n), dtype=out, device=DEVICE)
        return s
    t, e, k, h, i, kind = (case[n] for n in ("tokens", "experts", "top_k", "cols", "inner", "x"))
    kind = TYPES[kind]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    s["x"] = _activations(t, h, g).to(kind)
    s["router"] = (normal(e, h) * (1.25 / math.sqrt(h))).to(kind)
    s["gate"], s["gate_scales"] = _stack(e, i, h, g)
    s["up"], s["up_scales"] = _stack(e, i, h, g)
    s["down"], s["down_scales"] = _stack(e, h, i, g)
    for name, shape in (("router_bias", (e,)), ("gate_bias", (e, i)), ("up_bias", (e, i)), ("down_bias", (e, h))):
        s[name] = (0.5 * normal(*shape)).to(kind) if case["bias"] else None
    s["out"] = torch.empty((t, h), dtype=kind, device=DEVICE)
    s["experts"] = torch.empty((t, k), dtype=torch.int32, device=DEVICE)
    s["weights"] = torch.empty((t, k), dtype=torch.float32, device=DEVICE)
    return s


def _values(codes, scales):
    """Float32 values of a matrix in MXFP4."""
    value = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEVICE)
    v = torch.stack((value[(codes & 15).int()], value[(codes >> 4).int()]), -1).reshape(codes.shape[0], -1, 32)
    return (v * scales.view(E8M0).float().unsqueeze(-1)).reshape(codes.shape[0], -1)


def _plain_moe(s):
    case = s["case"]
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    x = s["x"].float()
    # in 64 bits: which of two near experts is chosen is decided by the order of their logits
    logits = s["x"].double() @ s["router"].double().t()
    if s["router_bias"] is not None:
        logits = logits + s["router_bias"].double()
    logits, experts = torch.sort(logits, dim=-1, descending=True, stable=True)  # ties to the lowest index
    logits, experts = logits[:, :k], experts[:, :k]
    p = torch.exp(logits - logits[:, :1])
    weights = (p / p.sum(-1, keepdim=True)).float()

    def expert(rows, at):
        """The outputs of rows of x by expert `at` (a tensor of one index)."""
        pick = lambda name: s[name].index_select(0, at)[0]  # noqa: E731
        part = lambda name, v: v @ _values(pick(name), pick(name + "_scales")).t()  # noqa: E731
        gate, up = part("gate", rows), part("up", rows)
        if s["gate_bias"] is not None:
            gate, up = gate + pick("gate_bias").float(), up + pick("up_bias").float()
        y = part("down", gate / (1 + torch.exp(-gate)) * up)
        return y + pick("down_bias").float() if s["down_bias"] is not None else y

    y = torch.zeros_like(x)
    if t * k <= e:  # each token by its own experts
        for n in range(t):
            for j in range(k):
                y[n] += weights[n, j] * expert(x[n:n + 1], experts[n, j:j + 1])[0]
    else:  # all tokens by every expert, which counts where it is chosen
        for n in range(e):
            share = (weights * (experts == n)).sum(-1, keepdim=True)
            y += share * expert(x, torch.full((1,), n, device=DEVICE))
    return {"out": y.to(s["out"].dtype), "experts": experts.int(), "weights": weights}


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from ptwm_amd import api

        if op == "quantise":
            api.mxfp4_quantise_cuda(s["x"], s["codes"], s["scales"], 0, saturate=s["case"]["saturate"])
            return {"codes": s["codes"], "scales": s["scales"]}
        if op == "matmul":
            api.mxfp4_matmul_cuda(s["x"], s["x_scales"], s["weight"], s["scales"], s["out"], 0, bias=s["bias"])
            return s["out"]
        api.mxfp4_moe_cuda(s["x"], s["router"], s["gate"], s["gate_scales"], s["up"], s["up_scales"], s["down"],
                           s["down_scales"], s["out"], s["case"]["top_k"], 0, router_bias=s["router_bias"],
                           gate_bias=s["gate_bias"], up_bias=s["up_bias"], down_bias=s["down_bias"],
                           experts=s["experts"], weights=s["weights"])
        return {"out": s["out"], "experts": s["experts"], "weights": s["weights"]}
    if op == "quantise":
        # Every step is exact, so the packed bytes themselves have to be the same.
        codes, scales = _codes_of(s["x"].float(), s["case"]["saturate"])
        return {"codes": codes, "scales": scales.view(E8M0)}
    if op == "matmul":
        y = _values(s["x"], s["x_scales"]) @ _values(s["weight"], s["scales"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(s["out"].dtype)
    return _plain_moe(s)


def _exact_values(codes, scales):
    """Float64 values from the codes' bits: (1 + m/2) 2^(x - 1), or m/2 where x is 0."""
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1, 32).int()
    m, x = (c & 1).double(), (c >> 1) & 3
    v = torch.where(x > 0, torch.ldexp(1 + m / 2, x - 1), m / 2) * (1 - 2 * (c >> 3))
    return torch.ldexp(v, scales.int().unsqueeze(-1) - 127).reshape(codes.shape[0], -1)


def exact(case, seed):
    """In 64 bits and before the last rounding. Codes are decided by comparisons with exact numbers, and experts by the
    order of their logits: they have no such value."""
    s = prepare(case, seed)
    if case["op"] == "quantise":
        m, e = torch.frexp(s["x"].double().reshape(case["rows"], -1, 32).abs().amax(-1))  # m in [0.5, 1)
        e = e - 3 if case["saturate"] else torch.where(m > 0.75, e - 2, e - 3)
        return {"codes": None, "scales": torch.ldexp(torch.ones_like(m), e.clamp(-127, 127))}
    if case["op"] == "matmul":
        x = _exact_values(s["x"], s["x_scales"])
        y = torch.cat([x @ _exact_values(w, e).t() for w, e in zip(s["weight"].split(2048), s["scales"].split(2048))], 1)
        return y if s["bias"] is None else y + s["bias"].double()
    x, k = s["x"].double(), case["top_k"]
    logits = torch.nn.functional.linear(x, s["router"].double(),
                                        None if s["router_bias"] is None else s["router_bias"].double())
    best, chosen = logits.topk(k, -1)
    weights = torch.softmax(best, -1)

    def product(rows, name, n):
        y = torch.cat([rows @ _exact_values(c, e).t()
                       for c, e in zip(s[name][n].split(2048), s[name + "_scales"][n].split(2048))], 1)
        return y if s[name + "_bias"] is None else y + s[name + "_bias"][n].double()

    y = torch.zeros_like(x)
    for n in range(case["experts"]):
        rows, slot = torch.nonzero(chosen == n, as_tuple=True)
        if rows.numel():
            gate = product(x[rows], "gate", n)
            h = gate * torch.sigmoid(gate) * product(x[rows], "up", n)
            y[rows] += weights[rows, slot].unsqueeze(-1) * product(h, "down", n)
    return {"out": y, "experts": None, "weights": weights}


def work(case):
    if case["op"] == "quantise":
        t, k = case["rows"], case["cols"]
        return {"bytes": t * k * SIZE[case["x"]] + t * k // 2 + t * k // 32, "flops": 2 * t * k}
    if case["op"] == "matmul":
        t, n, k = case["tokens"], case["rows"], case["cols"]
        out = (t * n + (n if case["bias"] else 0)) * SIZE[case["out"]]
        return {"bytes": (n + t) * (k // 2 + k // 32) + out, "flops": 2 * t * n * k}
    t, e, k, h, i, size = *(case[n] for n in ("tokens", "experts", "top_k", "cols", "inner")), SIZE[case["x"]]
    used = e * (1 - (1 - k / e) ** t)  # experts that have a token, on average
    each = 3 * h * i * 17 // 32 + ((2 * i + h) * size if case["bias"] else 0)
    return {"bytes": int(used * each) + e * h * size + 2 * t * h * size + 8 * t * k,
            "flops": 2 * t * k * 3 * h * i + 2 * t * e * h}
