"""The product of two MXFP4 matrices on the GPU against the formula in 64 bits."""
import pytest

import mx4_plain as Q
import mx_plain as P
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
E8 = torch.float8_e8m0fnu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def case(tokens, rows, cols, out, bias, g, low=112, high=128):
    x, xs = P.random_weights(tokens, cols, g, D, low, high)
    w, s = P.random_weights(rows, cols, g, D, low, high)
    b = torch.randn(rows, generator=g).to(out).to(D) if bias else None
    return x, xs, w, s, torch.full((tokens, rows), float("nan"), dtype=out, device=D), b


SIZES = [(1, 1, 32), (1, 16, 64), (1, 1024, 4096), (1, 97, 3360), (2, 33, 96), (3, 130, 416), (7, 515, 1024),
         (15, 64, 2080), (16, 256, 512), (17, 1000, 736), (31, 48, 4096), (33, 257, 160), (40, 5001, 288), (63, 96, 992),
         (64, 512, 1024), (65, 640, 1056), (100, 129, 2048), (128, 256, 256), (129, 300, 544), (200, 1111, 224),
         (257, 513, 1120), (300, 2049, 320), (512, 768, 512), (1, 20000, 128), (16, 64, 14336), (256, 64, 8192),
         (1025, 257, 128), (1290, 4110, 416), (640, 4099, 672), (2048, 2304, 1056), (1100, 5001, 96), (700, 3000, 2048),
         (5, 9001, 1184), (130, 8200, 1184)]


@pytest.mark.parametrize("tokens,rows,cols", SIZES)
def test_sizes(tokens, rows, cols):
    out = TYPES[(tokens + rows + cols // 32) % 3]
    x, xs, w, s, o, b = case(tokens, rows, cols, out, rows % 2 == 1, gen(tokens, rows, cols),
                             *((112, 122) if out == torch.float16 else (112, 128)))
    api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
    Q.check_matmul(o, x, xs, w, s, b)


@pytest.mark.parametrize("out", TYPES, ids=str)
@pytest.mark.parametrize("tokens,rows", [(1, 77), (4, 7000), (19, 515), (70, 6000), (260, 5001), (1500, 3500)])
@pytest.mark.parametrize("cols", [32, 64, 96, 128, 160, 256])
def test_short_rows(tokens, rows, cols, out):
    x, xs, w, s, o, b = case(tokens, rows, cols, out, True, gen(tokens, rows, cols), 112, 122)
    api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
    Q.check_matmul(o, x, xs, w, s, b)


def strided(t, pad, shift):
    rows, cols = t.shape
    big = torch.full((rows * (cols + pad) + shift,), 0x5A, dtype=torch.uint8, device=D)
    v = big[shift:].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v


@pytest.mark.parametrize("tokens,rows,cols", [(1, 131, 352), (3, 1030, 160), (20, 300, 1184), (70, 131, 2208),
                                              (150, 131, 352), (700, 3001, 256), (1290, 4110, 416), (640, 4099, 672)])
@pytest.mark.parametrize("pad,shift", [(1, 1), (5, 3), (16, 16), (33, 8)])
def test_strides_and_alignment(tokens, rows, cols, pad, shift):
    """The same result from any place, and nothing written between the outputs' rows."""
    x, xs, w, s, o, b = case(tokens, rows, cols, torch.bfloat16, True, gen(tokens, pad))
    api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
    Q.check_matmul(o, x, xs, w, s, b)
    room = torch.full((tokens * (rows + pad) + shift,), 7.0, dtype=o.dtype, device=D)
    far = room[shift:].view(tokens, rows + pad)[:, :rows]
    api.mxfp4_matmul_cuda(strided(x, pad, shift).view(torch.float4_e2m1fn_x2), strided(xs, pad, shift).view(E8),
                          strided(w, pad, shift), strided(s, pad, shift), far, 0, bias=b)
    assert torch.equal(o, far)
    far.fill_(7.0)
    assert (room == 7.0).all()


@pytest.mark.parametrize("tokens", [1, 20, 300, 1290])
def test_every_scale(tokens):
    """Scales over their whole range, paired so that products lie around one; outputs in the subnormal numbers and at
    the top of the range."""
    rows, cols = 1300, 512
    g = gen(tokens, 1)
    x, xs, w, s, o, _ = case(tokens, rows, cols, torch.float32, False, g)
    e = torch.randint(4, 250, (cols // 32,), generator=g).to(D)
    xs = (e + torch.randint(-3, 4, xs.shape, generator=g).to(D)).to(torch.uint8)
    s = (254 - e + torch.randint(-1, 2, s.shape, generator=g).to(D)).clamp(0, 254).to(torch.uint8)
    api.mxfp4_matmul_cuda(x, xs, w, s, o)
    Q.check_matmul(o, x, xs, w, s)
    for shift in (-100, 90):
        low = (xs.int() + shift).clamp(0, 254).to(torch.uint8)
        y = P.weights(x, low) @ P.weights(w, s).t()
        if y.abs().max() < 2.0**126:
            api.mxfp4_matmul_cuda(x, low, w, s, o)
            Q.check_matmul(o, x, low, w, s)
    zero = torch.zeros_like(s)  # 2^-127 by 2^-20 and less: below all numbers, or the smallest of them
    api.mxfp4_matmul_cuda(x, torch.full_like(xs, 105), w, zero, o)
    Q.check_matmul(o, x, torch.full_like(xs, 105), w, zero)


@pytest.mark.parametrize("tokens,rows,cols", [(1, 64, 352), (20, 131, 1184), (300, 515, 352), (1290, 4110, 416)])
def test_broken_scales(tokens, rows, cols):
    """A NaN scale makes its row of outputs NaN, or its column, and leaves the others."""
    x, xs, w, s, o, _ = case(tokens, rows, cols, torch.float32, False, gen(rows))
    api.mxfp4_matmul_cuda(x, xs, w, s, o)
    clean = o.clone()
    xs[tokens // 2, cols // 32 - 1], s[rows // 3, 0] = 255, 255
    api.mxfp4_matmul_cuda(x, xs, w, s, o)
    assert torch.isnan(o[tokens // 2]).all() and torch.isnan(o[:, rows // 3]).all()
    o[tokens // 2], o[:, rows // 3] = clean[tokens // 2], clean[:, rows // 3]
    assert torch.equal(o, clean)


@pytest.mark.parametrize("far", ["x", "weight", "scales", "out"])
@pytest.mark.parametrize("tokens,rows", [(9, 40), (40, 9), (300, 1100)])
def test_rows_far_apart(far, tokens, rows):
    cols = 352

    def apart(t):
        stride = (9 << 30) // t.shape[0] // t.element_size() // 4 * 4  # 9 GiB in all
        v = torch.empty((t.shape[0] - 1) * stride + t.shape[1], dtype=t.dtype, device=D).as_strided(t.shape, (stride, 1))
        v.copy_(t)
        return v

    x, xs, w, s, o, b = case(tokens, rows, cols, torch.bfloat16, True, gen(tokens, 7))
    want = (x, xs, w, s, b)
    if far == "x":
        x, xs = apart(x), apart(xs)
    elif far == "weight":
        w = apart(w)
    elif far == "scales":
        s = apart(s)
    else:
        o = apart(o)
    api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
    Q.check_matmul(o.contiguous(), *want)
    del x, xs, w, s, o
    torch.cuda.empty_cache()


def test_streams_and_graphs():
    for tokens in (1, 30, 700):
        x, xs, w, s, o, b = case(tokens, 3000, 1056, torch.bfloat16, True, gen(tokens))
        api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
        want, p = o.clone(), torch.zeros_like(o)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            api.mxfp4_matmul_cuda(x, xs, w, s, p, 0, bias=b)
        stream.synchronize()
        assert torch.equal(p, want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            api.mxfp4_matmul_cuda(x, xs, w, s, p, 0, bias=b)
        for k in range(4):
            x.random_(generator=torch.Generator(device=D).manual_seed(k))
            api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
            p.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(p, o)


def test_refusals():
    x, xs, w, s, o, b = case(4, 8, 64, torch.bfloat16, True, gen(1))
    for bad, kw, error in [((x.float(), xs, w, s, o), {}, TypeError), ((x, xs[:3], w, s, o), {}, ValueError),
                           ((x, xs, w[:, :16], s, o), {}, ValueError), ((x, xs, w, s[:, :1], o), {}, ValueError),
                           ((x, xs, w, s, o[:, :7]), {}, ValueError), ((x, xs, w, s, o.double()), {}, TypeError),
                           ((x, xs, w, s, o), dict(bias=b.float()), TypeError),
                           ((x, xs, w, s, o), dict(bias=b[:7]), ValueError), ((x, None, w, s, o), {}, TypeError)]:
        with pytest.raises(error):
            api.mxfp4_matmul_cuda(*bad, 0, **kw)
    api.mxfp4_matmul_cuda(x[:0], xs[:0], w, s, o[:0])
    api.mxfp4_matmul_cuda(x, xs, w[:0], s[:0], o[:, :0].contiguous())
