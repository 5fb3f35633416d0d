"""The MX operators on the GPU against their formulas in 64 bits: types, odd
sizes, strides, alignments, infinities and NaN, empty calls, streams, graphs,
offsets past 32 bits."""
import pytest

import mx_plain as P
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def activations(rows, cols, dtype, g, scale=1.0):
    loud = torch.where(torch.rand(cols, generator=g) < 0.05, 20.0, 1.0)
    return (torch.randn(rows, cols, generator=g) * loud * scale).to(dtype).to(D)


def strided(t, pad, shift):
    """The same matrix with `pad` elements between rows, `shift` elements in."""
    rows, cols = t.shape
    if t.element_size() == 1:
        big = torch.full((rows * (cols + pad) + shift + 1,), 0x55, dtype=torch.uint8, device=t.device).view(t.dtype)
    else:
        big = torch.full((rows * (cols + pad) + shift + 1,), 7.0, dtype=t.dtype, device=t.device)
    v = big[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    v.copy_(t) if t.element_size() > 1 else v.view(torch.uint8).copy_(t.view(torch.uint8))
    return v


def code_buffers(rows, cols):
    return (torch.zeros(rows, cols, dtype=torch.uint8, device=D).view(F8),
            torch.zeros(rows, cols // 32, dtype=torch.uint8, device=D).view(E8))


def linear_case(tokens, rows, cols, kind, out, bias, g):
    codes, scales = P.random_weights(rows, cols, g, D)
    x, xs = P.random_blocks(tokens, cols, g, D) if kind == F8 else (activations(tokens, cols, kind, g), None)
    b = torch.randn(rows, generator=g).to(out).to(D) if bias else None
    o = torch.full((tokens, rows), float("nan"), dtype=out, device=D)
    return x, xs, codes, scales, b, o


LINEAR = [  # tokens, rows, cols
    (1, 1, 32), (1, 16, 64), (1, 1024, 4096), (1, 97, 3360), (2, 33, 96), (3, 130, 416), (7, 515, 1024),
    (15, 64, 2080), (16, 256, 512), (17, 1000, 736), (31, 48, 4096), (33, 257, 160), (40, 5001, 288), (63, 96, 992),
    (64, 512, 1024), (65, 640, 1056), (100, 129, 2048), (128, 256, 256), (129, 300, 544), (200, 1111, 224),
    (257, 513, 1120), (300, 2049, 320), (512, 768, 512), (1, 20000, 128), (16, 64, 14336), (256, 64, 8192),
    (1025, 257, 128),
]


@pytest.mark.parametrize("kind", TYPES + [F8], ids=str)
@pytest.mark.parametrize("tokens,rows,cols", LINEAR)
def test_linear_sizes(tokens, rows, cols, kind):
    g = gen(tokens, rows, cols, 1)
    # every output type with every input type over the sizes
    out = TYPES[(tokens + rows + cols // 32 + (TYPES + [F8]).index(kind)) % 3]
    x, xs, codes, scales, b, o = linear_case(tokens, rows, cols, kind, out, rows % 2 == 1, g)
    if out == torch.float16:  # into the type's range
        scales -= 12
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs, bias=b)
    P.check_linear(o, x, xs, codes, scales, b)


# Where the sizes choose another kernel: rows about the limit for one token, LDS about its limit for one, two and four
# tokens, and enough tiles for the large and the middle ones, with row ends inside a step.
@pytest.mark.parametrize("kind", TYPES + [F8], ids=str)
@pytest.mark.parametrize("tokens,rows,cols", [(1, 6144, 160), (1, 6145, 160), (1, 17, 15360), (1, 17, 15392),
                                              (2, 33, 7680), (2, 33, 7712), (4, 100, 3840), (3, 100, 3872),
                                              (5, 40, 2016), (1300, 4100, 192), (1100, 5001, 96), (700, 4500, 160),
                                              (1290, 4110, 416), (640, 4099, 352), (90, 8200, 1184)])
def test_linear_choices(tokens, rows, cols, kind):
    x, xs, codes, scales, b, o = linear_case(tokens, rows, cols, kind, torch.float32, True, gen(tokens, rows, cols, 3))
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs, bias=b)
    P.check_linear(o, x, xs, codes, scales, b)


# Rows of one to three blocks, less than the kernels' step, in every kernel.
@pytest.mark.parametrize("kind", TYPES + [F8], ids=str)
@pytest.mark.parametrize("tokens,rows", [(1, 77), (4, 7000), (19, 515), (70, 6000), (260, 5001), (1500, 3500)])
@pytest.mark.parametrize("cols", [32, 64, 96])
def test_linear_short_rows(tokens, rows, cols, kind):
    x, xs, codes, scales, b, o = linear_case(tokens, rows, cols, kind, torch.float32, True, gen(tokens, rows, cols, 5))
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs, bias=b)
    P.check_linear(o, x, xs, codes, scales, b)
    r = torch.full_like(o, float("nan"))  # the same from places that no load can take whole
    api.mxfp4_linear_cuda(strided(x, 3, 1), strided(codes, 5, 3), strided(scales, 1, 1), r, 0,
                          x_scales=None if xs is None else strided(xs, 1, 1), bias=b)
    assert torch.equal(o, r)


# Rows so far apart that offsets pass 32 bits: the weights', or the activations' and the outputs'.
@pytest.mark.parametrize("kind", TYPES + [F8], ids=str)
@pytest.mark.parametrize("tokens,rows,far", [(3, 530, "weights"), (530, 40, "tokens")])
def test_linear_far_rows(tokens, rows, far, kind):
    def apart(t, stride):
        big = torch.empty((t.shape[0] - 1) * stride + t.shape[1], dtype=t.dtype, device=D)
        v = big.as_strided(t.shape, (stride, 1))
        v.copy_(t)
        return v

    x, xs, codes, scales, b, o = linear_case(tokens, rows, 352, kind, torch.float32, True, gen(tokens, rows, 6))
    far_o = o
    if far == "weights":
        codes = apart(codes, (1 << 23) + 16)
    else:
        x, far_o = apart(x, (1 << 23) + 8), apart(o, (1 << 22) + 4)
    api.mxfp4_linear_cuda(x, codes, scales, far_o, 0, x_scales=xs, bias=b)
    o.copy_(far_o)
    x, codes = x.contiguous(), codes.contiguous()
    P.check_linear(o, x, xs, codes, scales, b)
    del far_o
    torch.cuda.empty_cache()


@pytest.mark.parametrize("out", TYPES, ids=str)
@pytest.mark.parametrize("kind", TYPES + [F8], ids=str)
@pytest.mark.parametrize("tokens", [1, 5, 48, 160])
def test_linear_types(kind, out, tokens):
    x, xs, codes, scales, b, o = linear_case(tokens, 200, 608, kind, out, True, gen(tokens, 2))
    if out == torch.float16:
        scales -= 12
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs, bias=b)
    P.check_linear(o, x, xs, codes, scales, b)


@pytest.mark.parametrize("kind", TYPES + [F8], ids=str)
@pytest.mark.parametrize("tokens,pad,shift", [(1, 32, 1), (3, 5, 3), (20, 1, 7), (70, 33, 1), (150, 9, 5)])
def test_linear_strides_and_alignment(kind, tokens, pad, shift):
    """Rows apart, addresses at the element's alignment only; what lies between the rows stays as it is."""
    rows, cols = 131, 352
    x, xs, codes, scales, b, o = linear_case(tokens, rows, cols, kind, torch.bfloat16, True, gen(tokens, pad))
    want = o.clone()
    api.mxfp4_linear_cuda(x, codes, scales, want, 0, x_scales=xs, bias=b)
    P.check_linear(want, x, xs, codes, scales, b)
    x, codes, scales, o = strided(x, pad, shift), strided(codes, pad, shift), strided(scales, pad, shift), strided(o, pad, shift)
    xs = strided(xs, pad, shift) if xs is not None else None
    b = strided(b[None], 0, shift)[0]
    around = o._base.clone()
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs, bias=b)
    assert torch.equal(o, want)
    now = o._base.clone()
    mask = torch.ones_like(now, dtype=torch.bool)
    mask[shift:shift + tokens * (rows + pad)].view(tokens, rows + pad)[:, :rows] = False
    assert torch.equal(now[mask], around[mask])


def test_linear_accepts_the_byte_types():
    x, xs, codes, scales, _, o = linear_case(4, 64, 128, F8, torch.float32, False, gen(9))
    p = torch.empty_like(o)
    api.mxfp4_linear_cuda(x, codes.view(torch.float4_e2m1fn_x2), scales.view(E8), p, 0, x_scales=xs.view(torch.uint8))
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    assert torch.equal(o, p)


@pytest.mark.parametrize("kind", TYPES + [F8], ids=str)
@pytest.mark.parametrize("tokens", [1, 24, 140])
def test_linear_extreme_scales(kind, tokens):
    """Scales 0 (2^-127) to the largest whose weights are finite, and NaN (255) in one row's block."""
    rows, cols = 96, 256
    g = gen(tokens, 5)
    codes, _ = P.random_weights(rows, cols, g, D)
    scales = torch.randint(0, 20, (rows, cols // 32), generator=g, dtype=torch.uint8).to(D)
    x = (torch.randn(tokens, cols, generator=g) * 1e4).clamp(-6e4, 6e4)
    if kind == F8:
        x, xs = P.random_blocks(tokens, cols, g, D)
        xs.view(torch.uint8).add_(60)
    else:
        x, xs = x.to(kind).to(D), None
    o = torch.empty(tokens, rows, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    # sums of numbers below 2^-126 may lose what lies under the smallest normal number
    y = (P.blocks(x, xs) if xs is not None else x.double()) @ P.weights(codes, scales).t()
    mag = (P.blocks(x, xs) if xs is not None else x.double()).abs() @ P.weights(codes, scales).abs().t()
    assert ((o.double() - y).abs() <= (cols / 32 + 128) * 2.0**-23 * mag + cols * 2.0**-126).all()
    scales = torch.full((rows, cols // 32), 120, dtype=torch.uint8, device=D)
    scales[7, 3] = 255
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    assert torch.isnan(o[:, 7]).all() and not torch.isnan(o[:, :7]).any() and not torch.isnan(o[:, 8:]).any()


@pytest.mark.parametrize("kind", TYPES, ids=str)
@pytest.mark.parametrize("tokens", [2, 40, 130])
def test_linear_infinities_and_nan(kind, tokens):
    """An infinite activation gives an infinity where its weight is not zero, a NaN gives NaN; other tokens are untouched."""
    rows, cols = 64, 128
    g = gen(tokens, 6)
    codes, scales = P.random_weights(rows, cols, g, D)
    codes[:, 20] = 0x20 | torch.where(torch.arange(rows, device=D) % 2 == 0, 1, 9).to(torch.uint8)  # value 40: +-0.5
    x = activations(tokens, cols, kind, g)
    clean = x.clone()
    x[0, 40], x[tokens - 1, 3] = float("inf"), float("nan")
    o, c = torch.empty(tokens, rows, device=D), torch.empty(tokens, rows, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, o)
    api.mxfp4_linear_cuda(clean, codes, scales, c)
    want = torch.where(torch.arange(rows, device=D) % 2 == 0, 1.0, -1.0) * float("inf")
    assert torch.equal(o[0], want) and torch.isnan(o[tokens - 1]).all()
    assert torch.equal(o[1:tokens - 1], c[1:tokens - 1])
    low = torch.full((1, 1), 0x7F800001, dtype=torch.int32, device=D).view(torch.float32)  # NaN in its lowest bits only
    if kind == torch.float32:
        x = clean.clone()
        x[0, 40] = low[0, 0]
        api.mxfp4_linear_cuda(x, codes, scales, o)
        assert torch.isnan(o[0]).all() and torch.equal(o[1:], c[1:])


@pytest.mark.parametrize("low,high", [(100, 108), (104, 136), (103, 104), (130, 137), (0, 255)])
@pytest.mark.parametrize("tokens,rows", [(3, 100), (40, 200), (700, 4500)])
def test_linear_f16_scales_in_and_out_of_the_types_range(tokens, rows, low, high):
    """Weights that f16 holds, below its normal numbers too, and weights that it does not; activations among its smallest."""
    g = gen(tokens, low)
    codes, scales = P.random_weights(rows, 352, g, D, low, high)
    x = torch.randn(tokens, 352, generator=g)
    x[:, ::3] *= 2.0**-20  # below f16's normal numbers
    x = x.to(torch.float16).to(D)
    o = torch.empty(tokens, rows, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, o)
    w = P.weights(codes, scales)
    if high < 255:
        P.check_linear(o, x, None, codes, scales)
    else:  # sums may pass float32's largest number: those that do not are right
        y, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
        small = (mag < 2.0**127) & (w.abs().amax(1) < 2.0**127)
        assert ((o.double() - y).abs() <= (352 / 32 + 129) * 2.0**-23 * mag + 352 * 2.0**-126)[small].all()


def test_linear_e4m3_nan_and_scale_nan():
    x, xs, codes, scales, _, o = linear_case(5, 40, 128, F8, torch.float32, False, gen(11))
    c = torch.empty_like(o)
    api.mxfp4_linear_cuda(x, codes, scales, c, 0, x_scales=xs)
    x.view(torch.uint8)[1, 70] = 0x7F
    xs.view(torch.uint8)[3, 2] = 255
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    for t in range(5):
        assert torch.isnan(o[t]).all() if t in (1, 3) else torch.equal(o[t], c[t])


def test_linear_largest_activations_stay_finite():
    """Activations near the type's largest value, which a rounding of their parts must not lift to infinity."""
    g = gen(12)
    codes, scales = P.random_weights(32, 64, g, D, 60, 62)
    x = torch.full((3, 64), torch.finfo(torch.float32).max, device=D)
    o = torch.empty(3, 32, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, o)
    P.check_linear(o, x, None, codes, scales)


def test_linear_is_the_same_every_time_and_for_every_batch():
    """No order of additions depends on timing; within a batch size a token's result does not depend on the others."""
    x, xs, codes, scales, b, o = linear_case(80, 700, 1280, torch.bfloat16, torch.bfloat16, True, gen(13))
    p = torch.empty_like(o)
    for _ in range(5):
        api.mxfp4_linear_cuda(x, codes, scales, o, 0, bias=b)
        api.mxfp4_linear_cuda(x.flip(0).contiguous(), codes, scales, p, 0, bias=b)
        assert torch.equal(o, p.flip(0))


def test_empty_calls():
    c, s = torch.zeros(8, 32, dtype=torch.uint8, device=D), torch.zeros(8, 2, dtype=torch.uint8, device=D)
    x = torch.zeros(0, 64, device=D)
    api.mxfp4_linear_cuda(x, c, s, torch.zeros(0, 8, device=D))
    api.mxfp4_linear_cuda(torch.zeros(3, 64, device=D), c[:0], s[:0], torch.zeros(3, 0, device=D))
    oc, os_ = code_buffers(0, 64)
    api.rms_norm_mx_cuda(x, torch.ones(64, device=D), oc, os_)
    api.swiglu_mx_cuda(x, x, oc, os_)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (3, 64), (2, 96), (5, 1056), (70, 2048), (9, 2080),
                                       (17, 5024), (4, 8224), (3, 14336), (2, 16416), (300, 512), (1, 70016)])
def test_norm(rows, cols, residual, dtype):
    g = gen(rows, cols)
    x, r = activations(rows, cols, dtype, g), activations(rows, cols, dtype, g, 3.0) if residual else None
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(TYPES[cols // 32 % 3]).to(D)
    codes, scales = code_buffers(rows, cols)
    total = torch.empty_like(x) if rows != 3 else None
    api.rms_norm_mx_cuda(x, w, codes, scales, 0, residual=r, sum_out=total, eps=1e-5)
    s, y = P.norm(x, r, w, 1e-5)
    P.check_codes(codes, scales, y, P.norm_delta(cols))
    if total is not None:
        u, tiny = P.ROUND[dtype]
        assert ((total.double() - s).abs() <= u * s.abs() * (1 + 2.0**-12) + tiny).all()


@pytest.mark.parametrize("cols", [64, 4096, 20000])
@pytest.mark.parametrize("target", ["x", "residual"])
def test_norm_in_place(target, cols):
    """The sum may be written over x or the residual."""
    g = gen(cols, 3)
    x, r = activations(6, cols, torch.bfloat16, g), activations(6, cols, torch.bfloat16, g)
    w = torch.ones(cols, device=D)
    want_c, want_s = code_buffers(6, cols)
    want = torch.empty_like(x)
    api.rms_norm_mx_cuda(x, w, want_c, want_s, 0, residual=r, sum_out=want)
    codes, scales = code_buffers(6, cols)
    out = {"x": x, "residual": r}[target]
    api.rms_norm_mx_cuda(x, w, codes, scales, 0, residual=r, sum_out=out)
    assert torch.equal(out, want)
    assert torch.equal(codes.view(torch.uint8), want_c.view(torch.uint8))
    assert torch.equal(scales.view(torch.uint8), want_s.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pad,shift", [(1, 1), (32, 3), (7, 0)])
def test_norm_and_swiglu_strides(dtype, pad, shift):
    g = gen(pad, shift)
    rows, cols = 11, 736
    x, r = activations(rows, cols, dtype, g), activations(rows, cols, dtype, g)
    w = torch.randn(cols, generator=g).to(dtype).to(D)
    sx, sr, total = strided(x, pad, shift), strided(r, pad + 1, shift), strided(torch.zeros_like(x), pad, shift)
    codes, scales = (strided(t, pad, shift) for t in code_buffers(rows, cols))
    around = codes._base.view(torch.uint8).clone(), scales._base.view(torch.uint8).clone(), total._base.clone()
    api.rms_norm_mx_cuda(sx, w, codes, scales, 0, residual=sr, sum_out=total)
    s, y = P.norm(x, r, w, 1e-6)
    P.check_codes(codes.contiguous(), scales.contiguous(), y, P.norm_delta(cols))
    for t, was in zip((codes, scales, total), around):
        now = t._base.view(torch.uint8) if t.element_size() == 1 else t._base
        mask = torch.ones(now.shape, dtype=torch.bool, device=D)
        n = t.shape[1]
        mask[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n] = False
        assert torch.equal(now[mask], was[mask])
    api.swiglu_mx_cuda(sx, sr, codes, scales)
    P.check_codes(codes.contiguous(), scales.contiguous(), P.swiglu(x, r), P.swiglu_delta(x))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 14336), (7, 96), (33, 1056), (130, 2080), (3, 40000), (600, 64)])
def test_swiglu(rows, cols, dtype):
    g = gen(rows, cols, 7)
    both = activations(rows, 2 * cols, dtype, g, 3.0)
    codes, scales = code_buffers(rows, cols)
    api.swiglu_mx_cuda(both[:, :cols], both[:, cols:], codes, scales)
    P.check_codes(codes, scales, P.swiglu(both[:, :cols], both[:, cols:]), P.swiglu_delta(both[:, :cols]))


def test_activations_zero_infinite_and_nan_blocks():
    """A zero block: scale 0, codes 0.  A block with an infinity or NaN: NaN scale and codes, others as they are."""
    g = gen(21)
    gate, up = activations(4, 256, torch.float32, g), activations(4, 256, torch.float32, g)
    up[0, 32:64] = 0
    gate[1, 70] = float("inf")
    up[2, 100] = float("nan")
    gate[3, 5] = float("-inf")  # -inf * 0
    gate[3, 200] = -200.0       # exp(200) is infinite, the product is zero
    codes, scales = code_buffers(4, 256)
    api.swiglu_mx_cuda(gate, up, codes, scales)
    b, c = scales.view(torch.uint8).cpu(), codes.view(torch.uint8).cpu()
    assert b[0, 1] == 0 and (c[0, 32:64] & 0x7F == 0).all()
    broken = {(1, 2), (2, 3), (3, 0)}
    y = P.swiglu(gate, up)
    for t in range(4):
        for k in range(8):
            if (t, k) in broken:
                assert b[t, k] == 255 and (c[t, 32 * k:32 * k + 32] == 0x7F).all()
            else:
                part = slice(32 * k, 32 * k + 32)
                P.check_codes(codes[t:t + 1, part].contiguous(), scales[t:t + 1, k:k + 1].contiguous(),
                              y[t:t + 1, part], P.swiglu_delta(gate[t:t + 1, part]))
    x = torch.ones(3, 64, device=D)
    x[1, 40] = float("nan")
    x[2, 3] = float("inf")
    oc, os_ = code_buffers(3, 64)
    api.rms_norm_mx_cuda(x, torch.ones(64, device=D), oc, os_)
    b, c = os_.view(torch.uint8).cpu(), oc.view(torch.uint8).cpu()
    assert (b[0] < 255).all() and (b[1] == 255).all() and b[2, 0] == 255
    assert b[2, 1] == 0 and (c[2, 32:] == 0).all()  # 1 / inf
    api.rms_norm_mx_cuda(torch.zeros(3, 64, device=D), torch.ones(64, device=D), oc, os_)
    assert (os_.view(torch.uint8) == 0).all() and (oc.view(torch.uint8) == 0).all()


def test_scale_at_its_boundaries():
    """Largest magnitudes of 448 * 2^k and the next number above, the smallest scale, signs and ties."""
    up = torch.zeros(6, 32, device=D)
    g = torch.full((6, 32), 64.0, device=D)  # exp(-64) vanishes beside 1: the product is 64 * up exactly
    up[0, 0] = 448 / 64
    up[1, 0] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9)) / 64
    up[2, 0] = -448 * 2.0**60
    up[3, 0] = 2.0**-140
    up[4, 0], up[4, 1], up[4, 2] = 448 / 64, 17 / 64, 19 / 64  # 17 and 19 lie between codes 16, 18 and 20: to even
    up[5, 0] = 2.0**-120 / 64
    codes, scales = code_buffers(6, 32)
    api.swiglu_mx_cuda(g, up, codes, scales)
    b, v = scales.view(torch.uint8).cpu().flatten().tolist(), P.blocks(codes, scales).cpu()
    assert b[0] == 127 and v[0, 0] == 448
    assert b[1] == 128 and v[1, 0] == 448
    assert b[2] == 127 + 66 and v[2, 0] == -448 * 2.0**66
    assert b[3] == 0 and v[3, 0] == 2.0**-134 and b[5] == 0 and v[5, 0] == 2.0**-120
    assert v[4, :3].tolist() == [448, 16, 20]


def test_other_streams_and_graph_replays():
    g = gen(31)
    x, xs, codes, scales, b, o = linear_case(6, 384, 512, torch.bfloat16, torch.bfloat16, True, g)
    w = torch.ones(512, device=D, dtype=torch.bfloat16)
    c, s = code_buffers(6, 512)
    total, p = torch.empty_like(x), torch.empty_like(o)
    c2, s2 = code_buffers(6, 192)

    def step():
        api.rms_norm_mx_cuda(x, w, c, s, 0, residual=x, sum_out=total)
        api.mxfp4_linear_cuda(c, codes, scales, o, 0, x_scales=s, bias=b)
        api.swiglu_mx_cuda(o[:, :192], o[:, 192:], c2, s2)
        api.mxfp4_linear_cuda(total, codes, scales, p, 0)

    results = lambda: [t.view(torch.uint8).clone() for t in (c, s, total, o, c2, s2, p)]  # noqa: E731
    step()
    want = results()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for t in (o, p, total):
            t.zero_()
        torch.cuda._sleep(20_000_000)  # what comes next must wait for this
        x.add_(1)
        step()
        moved = results()
    side.synchronize()
    step()
    assert all(torch.equal(a, m) for a, m in zip(results(), moved))
    x.sub_(1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    step()
    want = results()
    for k in range(4):
        x.mul_(-1)
        graph.replay()
        got = results()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, m) for a, m in zip(got, results())), k
    assert all(torch.equal(a, m) for a, m in zip(got, want))


def test_offsets_past_32_bits():
    """Rows 2^31 bytes apart in every operand."""
    far = 1 << 31
    g = gen(41)
    rows, cols = 3, 64
    codes, scales = P.random_weights(rows, cols, g, D)
    big = torch.empty(rows * far, dtype=torch.uint8, device=D)

    def apart(t, at):
        n = t.element_size()
        v = big.view(t.dtype).as_strided(t.shape, (far // n, 1), at // n)
        v.copy_(t) if n > 1 else v.view(torch.uint8).copy_(t.view(torch.uint8))
        return v

    x = activations(rows, cols, torch.bfloat16, g)
    want, o = torch.empty(rows, rows, device=D), torch.zeros(rows, rows, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, want)
    fx, fc, fs, fo = apart(x, 0), apart(codes, 1024), apart(scales, 2048), apart(o, 4096)
    api.mxfp4_linear_cuda(fx, fc, fs, fo)
    assert torch.equal(fo, want)
    q, qs = code_buffers(rows, cols)
    w = torch.ones(cols, device=D)
    fq, fqs = apart(q, 8192), apart(qs, 9216)
    ft = apart(torch.zeros_like(x), 12288)
    api.rms_norm_mx_cuda(x, w, q, qs, 0, residual=x)
    api.rms_norm_mx_cuda(fx, w, fq, fqs, 0, residual=fx, sum_out=ft)
    assert torch.equal(fq.view(torch.uint8), q.view(torch.uint8))
    assert torch.equal(fqs.view(torch.uint8), qs.view(torch.uint8)) and torch.equal(ft, x + x)
    api.swiglu_mx_cuda(x, x, q, qs)
    api.swiglu_mx_cuda(fx, ft, fq, fqs)
    api.swiglu_mx_cuda(x, x + x, q, qs)
    assert torch.equal(fq.view(torch.uint8), q.view(torch.uint8))


def test_refusals():
    x = torch.zeros(4, 64, device=D, dtype=torch.bfloat16)
    c, s = code_buffers(4, 64)
    w = torch.ones(64, device=D)
    wc, ws = torch.zeros(8, 32, dtype=torch.uint8, device=D), torch.zeros(8, 2, dtype=torch.uint8, device=D)
    o = torch.zeros(4, 8, device=D)
    bad = [
        lambda: api.rms_norm_mx_cuda(x, w[:32], c, s),
        lambda: api.rms_norm_mx_cuda(x, w, c[:, :32], s),
        lambda: api.rms_norm_mx_cuda(x, w, c, s[:3]),
        lambda: api.rms_norm_mx_cuda(x, w, c, s, 0, residual=x[:3]),
        lambda: api.rms_norm_mx_cuda(x, w, c, s, 0, sum_out=x.t()),
        lambda: api.rms_norm_mx_cuda(x, w.cpu(), c, s),
        lambda: api.rms_norm_mx_cuda(x[0], w, c, s),
        lambda: api.swiglu_mx_cuda(x, x[:, :32], c, s),
        lambda: api.swiglu_mx_cuda(x, x.expand(4, 64)[:1].expand(4, 64), c, s),
        lambda: api.mxfp4_linear_cuda(x, wc, ws, o[:, :7]),
        lambda: api.mxfp4_linear_cuda(x, wc[:, :16], ws, o),
        lambda: api.mxfp4_linear_cuda(x, wc, ws[:7], o),
        lambda: api.mxfp4_linear_cuda(x, wc, ws, o, 0, bias=torch.zeros(7, device=D)),
        lambda: api.mxfp4_linear_cuda(x, wc, ws, o, 0, x_scales=s),
        lambda: api.mxfp4_linear_cuda(c, wc, ws, o),
        lambda: api.mxfp4_linear_cuda(x, wc, ws, o.t().contiguous().t()),
        lambda: api.mxfp4_linear_cuda(x, wc.reshape(-1), ws, o),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")
    wrong_type = [
        lambda: api.rms_norm_mx_cuda(c, w, c, s),
        lambda: api.rms_norm_mx_cuda(x, w, x, s),
        lambda: api.rms_norm_mx_cuda(x, c.view(-1)[:64], c, s),
        lambda: api.rms_norm_mx_cuda(x, w, c, s, 0, residual=x.float()),
        lambda: api.swiglu_mx_cuda(x, x.half(), c, s),
        lambda: api.mxfp4_linear_cuda(x.double(), wc, ws, o),
        lambda: api.mxfp4_linear_cuda(x, wc.to(torch.int32), ws, o),
        lambda: api.mxfp4_linear_cuda(x, wc, ws, o.double()),
        lambda: api.mxfp4_linear_cuda(x, wc, ws, torch.zeros(4, 8, device=D).to(F8)),
        lambda: api.mxfp4_linear_cuda(x, wc, ws, o, 0, bias=torch.zeros(8, device=D, dtype=torch.float16)),
    ]
    for k, call in enumerate(wrong_type):
        with pytest.raises(TypeError):
            call()
            pytest.fail(f"call {k} was not refused")
