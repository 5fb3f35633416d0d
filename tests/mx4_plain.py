"""The formulas, in 64 bits, of the quantisation to MXFP4, the product of two MXFP4 matrices and the mixture-of-experts
layer on MXFP4 experts, and the tolerances that follow from how the operators are specified. Used by the tests; runs
wherever its tensors are."""
import torch

import mx_plain as P

MIDDLES = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]  # between neighbouring e2m1 values; the tie goes to the even code


def power(e):
    """2^e in 64 bits, exactly (a device's own power function is not)."""
    return (e.long() + 1023 << 52).view(torch.float64)


def quantise(x, saturate):
    """(codes, scales) as bytes. Every step is exact in 64 bits."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    broken = ~torch.isfinite(b).all(-1)
    m, e = torch.frexp(torch.where(broken, 0.0, top))  # top = m 2^e, m in [0.5, 1)
    e = e - 3 if saturate else torch.where(m > 0.75, e - 2, e - 3)
    e = torch.where(top == 0, -127, e).clamp(min=-127)
    v = b.abs() * power(-e.unsqueeze(-1))
    code = torch.zeros(v.shape, dtype=torch.uint8, device=x.device)
    for i, middle in enumerate(MIDDLES):
        code += ((v > middle) | ((v == middle) & (i % 2 == 1))).to(torch.uint8)
    code |= torch.signbit(b).to(torch.uint8) << 3
    code = torch.where(broken.unsqueeze(-1), 0, code).reshape(x.shape[0], -1)
    return code[:, 0::2] | code[:, 1::2] << 4, torch.where(broken, 255, e + 127).to(torch.uint8)


def check_matmul(out, x, x_scales, codes, scales, bias=None):
    """The sum of a block's products is exact. Each block, each of up to 16 partial sums and the bias enters by one
    addition that loses a unit in the last place (2^-23) of the sum of magnitudes at most, or of the subnormal numbers
    (2^-149) where the sum is among them; one rounding to out's type."""
    x, w = P.weights(x, x_scales), P.weights(codes, scales)
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    u, tiny = P.ROUND[out.dtype]
    summed = (x.shape[1] / 32 + 17) * (2.0**-23 * mag + 2.0**-149)
    off = (out.double() - y).abs() - (u * (y.abs() + summed) + summed + tiny)
    assert not torch.isnan(out).any(), "NaN in the output"
    assert (off <= 0).all(), f"off by {off.max().item()} more than allowed at {off.argmax().item()}"


def route(x, router, bias, top_k):
    """(logits of all experts, the chosen ones' indices, their weights); an expert at minus infinity has the weight 0."""
    logits = x.double() @ router.double().t()
    if bias is not None:
        logits = logits + bias.double()
    logits = logits + 0.0
    best, chosen = torch.sort(logits, dim=-1, descending=True, stable=True)
    best, chosen = best[:, :top_k], chosen[:, :top_k]
    p = torch.where(best == -torch.inf, 0.0, torch.exp(best - best[:, :1]))
    return logits, chosen, torch.where(best == -torch.inf, 0.0, p / p.sum(-1, keepdim=True))


def moe(x, router, gate, gate_scales, up, up_scales, down, down_scales, top_k, router_bias=None, gate_bias=None,
        up_bias=None, down_bias=None, out_type=torch.float32):
    """(out, experts, weights, how far out may be off before its last rounding).

    A sum of n products in 32 bits is off by (n/32 + 128) units of 2^-23 of the sum of magnitudes, as in the product with
    MXFP4 weights. silu is 1.1-Lipschitz; its own steps, the product with u and the weight add (2|g| + 32) 2^-24, the
    weight's softmax (|l - max| + top_k + 16) 2^-24. h goes into the last product with 16 significant bits at least, 24
    where out is float32; the sums of the chosen experts and their biases enter by top_k more additions each."""
    logits, chosen, weights = route(x, router, router_bias, top_k)
    x = x.double()
    y, slack = torch.zeros_like(x), torch.zeros_like(x)
    unit = 2.0**-23
    for e in range(router.shape[0]):
        rows, slot = torch.nonzero((chosen == e) & (logits.gather(1, chosen) != -torch.inf), as_tuple=True)
        if rows.numel() == 0:
            continue
        xs = x[rows]
        steps = xs.shape[1] / 32 + 129

        def inner(w, s, b):
            w = P.weights(w[e], s[e])
            v, mag = xs @ w.t(), xs.abs() @ w.abs().t()
            if b is not None:
                v, mag = v + b[e].double(), mag + b[e].double().abs()
            return v, steps * unit * mag

        g, dg = inner(gate, gate_scales, gate_bias)
        u, du = inner(up, up_scales, up_bias)
        silu = g / (1 + torch.exp(-g))
        p = weights[rows, slot].unsqueeze(-1)
        h = silu * u * p
        far = (logits[rows].amax(-1) - logits[rows, e]).unsqueeze(-1)
        dh = (1.1 * dg * u.abs() + silu.abs() * du + 1.1 * dg * du) * p
        dh += h.abs() * ((2 * g.abs() + 32) + (far + top_k + 16)) * 2.0**-24
        dh += h.abs() * (2.0**-24 if out_type == torch.float32 else 2.0**-16) + 2.0**-133
        w = P.weights(down[e], down_scales[e])
        v, mag = h @ w.t(), (h.abs() + dh) @ w.abs().t()
        if down_bias is not None:
            v, mag = v + p * down_bias[e].double(), mag + p * down_bias[e].double().abs()
        y[rows] += v
        slack[rows] += dh @ w.abs().t() + (top_k * (h.shape[1] / 32 + 2) + 129) * unit * mag
        if down_bias is not None:
            slack[rows] += p * down_bias[e].double().abs() * (far + top_k + 32) * 2.0**-24
    return y, chosen.int(), weights, slack


def check_moe(out, experts, weights, want):
    y, chosen, p, slack = want
    if experts is not None:
        assert torch.equal(experts, chosen), "other experts"
    if weights is not None:
        off = ((weights.double() - p).abs() / p.clamp(min=2.0**-126)).max().item() if p.numel() else 0.0
        assert off <= (p.shape[1] + 64) * 2.0**-23, f"weights off by {off}"
    u, tiny = P.ROUND[out.dtype]
    off = (out.double() - y).abs() - (u * (y.abs() + slack) + slack + tiny)
    assert not torch.isnan(out).any(), "NaN in the output"
    assert (off <= 0).all(), f"off by {off.max().item()} more than allowed at {off.argmax().item()}"


def random_experts(experts, rows, cols, g, device, low=112, high=120):
    """Uniform codes; scales that leave products around one."""
    codes = torch.randint(0, 256, (experts, rows, cols // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(low, high, (experts, rows, cols // 32), generator=g, dtype=torch.uint8)
    return codes.to(device), scales.to(device)
