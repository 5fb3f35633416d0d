"""The MX operators' formulas in 64 bits, and the tolerances that follow from
how the operators are specified: sums in 32 bits, one rounding at the end.
Used by the tests; runs wherever its tensors are."""
import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# half a unit in the last place of 1, and the smallest half step, by type
ROUND = {torch.float32: (2.0**-24, 2.0**-150), torch.float16: (2.0**-11, 2.0**-25),
         torch.bfloat16: (2.0**-8, 2.0**-134)}


def scale_values(b):
    """2^(b-127) of scale bytes, NaN for 255."""
    v = torch.exp2(b.view(torch.uint8).double() - 127)
    return torch.where(b.view(torch.uint8) == 255, torch.full_like(v, float("nan")), v)


def weights(codes, scales):
    w = codes.view(torch.uint8)
    lut = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=w.device)
    v = torch.stack((lut[(w & 15).long()], lut[(w >> 4).long()]), -1).reshape(w.shape[0], -1, 32)
    return (v * scale_values(scales).unsqueeze(-1)).reshape(w.shape[0], -1)


def blocks(codes, scales):
    """The values that e4m3 codes and their scales stand for."""
    v = codes.view(torch.float8_e4m3fn).double().reshape(codes.shape[0], -1, 32)
    return (v * scale_values(scales).unsqueeze(-1)).reshape(codes.shape)


def check_linear(out, x, x_scales, codes, scales, bias=None):
    """out against the product in 64 bits.  Every product is exact in 32 bits;
    an accumulation loses at most one unit in the last place (2^-23) of the
    sum of magnitudes, at least 32 products enter with each, and within an
    instruction at most 128 are added one after the other."""
    x = blocks(x, x_scales) if x_scales is not None else x.double()
    w = weights(codes, scales)
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    steps = x.shape[1] / 32 + 128
    if bias is not None:
        y, mag, steps = y + bias.double(), mag + bias.double().abs(), steps + 1
    u, tiny = ROUND[out.dtype]
    summed = steps * 2.0**-23 * mag
    off = (out.double() - y).abs() - (u * (y.abs() + summed) + summed + tiny)
    assert not torch.isnan(out).any(), "NaN in the output"
    assert (off <= 0).all(), f"off by {off.max().item()} more than allowed at {off.argmax().item()}"


def check_codes(codes, scales, y, delta):
    """codes and scales against y in 64 bits, which the operator knows to a
    relative error delta (a tensor or a number): the scale is the smallest
    that reaches the block's largest magnitude, and a code is off by half a
    step of e4m3 (a relative 2^-4, or 2^-10 of the scale below its normal
    values)."""
    b = scales.view(torch.uint8)
    assert (b < 255).all(), "a NaN scale for finite values"
    s = scale_values(scales).repeat_interleave(32, 1)
    err = delta * y.abs()
    amax = y.abs().reshape(y.shape[0], -1, 32).amax(-1)
    slack = (err + torch.zeros_like(y)).reshape(y.shape[0], -1, 32).amax(-1)
    unit = scale_values(scales)
    assert (amax - slack <= 448 * unit).all(), "a scale that does not reach the largest magnitude"
    assert ((b == 0) | (amax + slack > 224 * unit)).all(), "a scale that is larger than needed"
    off = (blocks(codes, scales) - y).abs() - (2.0**-4 * (y.abs() + err) + err + s * 2.0**-10)
    assert (off <= 0).all(), f"off by {off.max().item()} more than allowed at {off.argmax().item()}"


def norm(x, residual, weight, eps):
    s = x.double() if residual is None else x.double() + residual.double()
    return s, s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps) * weight.double()


def norm_delta(cols):
    """The sum of squares adds cols non-negative terms (relative error cols
    half units at most, halved by the root); the root, its reciprocal, the
    residual's addition and two products add a few units."""
    return (cols / 2 + 16) * 2.0**-24


def swiglu(gate, up):
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def swiglu_delta(gate):
    """exp(-g) is off by its argument's rounding, |g| units; the other steps
    by a unit or two each."""
    return (2 * gate.double().abs() + 16) * 2.0**-24


def random_weights(rows, cols, g, device, low=110, high=126):
    """Uniform codes and scales (any byte is a weight)."""
    codes = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(low, high, (rows, cols // 32), generator=g, dtype=torch.uint8)
    return codes.to(device), scales.to(device)


def random_blocks(tokens, cols, g, device):
    """Finite e4m3 codes and scales around one."""
    codes = torch.randint(0, 127, (tokens, cols), generator=g, dtype=torch.uint8)
    codes |= torch.randint(0, 2, (tokens, cols), generator=g, dtype=torch.uint8) << 7
    scales = torch.randint(115, 124, (tokens, cols // 32), generator=g, dtype=torch.uint8)
    return codes.view(torch.float8_e4m3fn).to(device), scales.view(torch.float8_e8m0fnu).to(device)
