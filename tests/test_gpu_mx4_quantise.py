"""Quantisation to MXFP4 on the GPU: byte for byte what the formula in 64 bits gives."""
import pytest

import mx4_plain as Q
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
E8 = torch.float8_e8m0fnu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def buffers(rows, cols):
    return (torch.full((rows, cols // 2), 0xAA, dtype=torch.uint8, device=D),
            torch.full((rows, cols // 32), 0xAA, dtype=torch.uint8, device=D))


def check(x, saturate):
    codes, scales = buffers(*x.shape)
    api.mxfp4_quantise_cuda(x, codes, scales, 0, saturate=saturate)
    want = Q.quantise(x, saturate)
    assert torch.equal(scales, want[1])
    assert torch.equal(codes, want[0])
    return codes, scales


@pytest.mark.parametrize("saturate", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (2, 64), (3, 96), (7, 5024), (64, 32), (33, 2080), (333, 160),
                                       (1000, 1056), (4099, 32), (5, 131072)])
def test_sizes(rows, cols, dtype, saturate):
    g = gen(rows, cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-14, 9, (rows, cols // 32), generator=g)
                                                          ).repeat_interleave(32, 1)
    check(x.to(dtype).to(D), saturate)


@pytest.mark.parametrize("saturate", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_ties_and_neighbours(dtype, saturate):
    """The middles between codes, what lies next to them, and both signs, at scales over the type's whole range."""
    eps = torch.finfo(dtype).eps
    m = torch.tensor([0.0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], dtype=torch.float64)
    rows = []
    low, high = (-24, 12) if dtype == torch.float16 else (-149 if dtype == torch.float32 else -133, 125)
    for e in range(low, high):
        for lift in (0, eps, -eps):
            v = torch.cat((m, -m)) * (1 + lift)
            for top in (4.0, 6.0, 7.5):
                v[15], v[31] = top, -top
                rows.append(torch.ldexp(v, torch.tensor(e)))
    check(torch.stack(rows).to(dtype).to(D), saturate)


@pytest.mark.parametrize("saturate", [True, False])
def test_every_bfloat16(saturate):
    """Every finite bf16 value as a block's largest, with every other one below it somewhere."""
    bits = torch.arange(0, 0x7F80, dtype=torch.int32)
    rows = bits.unsqueeze(1) - torch.arange(32) * torch.tensor([1, 7, 31]).repeat_interleave(11)[:32]
    x = rows.clamp(min=0).to(torch.int16).view(torch.bfloat16)
    x[1::2] = -x[1::2]
    check(x.to(D), saturate)


@pytest.mark.parametrize("saturate", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_infinities_nan_and_zeros(dtype, saturate):
    x = torch.randn(8, 128, generator=gen(3)).to(dtype)
    x[0, 5], x[1, 40], x[2, 127] = torch.inf, -torch.inf, torch.nan
    x[3], x[4] = 0.0, -0.0
    x[5, :32] = torch.finfo(dtype).max
    x[6, 64:96] = 0
    x[6, 70] = torch.finfo(dtype).smallest_normal / 8
    codes, scales = check(x.to(D), saturate)
    assert scales[0, 0] == 255 and not codes[0, :16].any() and scales[0, 1] != 255
    assert not scales[3].any() and not codes[3].any() and (codes[4] == 0x88).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pad,shift", [(1, 1), (5, 3), (32, 8)])
def test_strides_and_alignment(dtype, pad, shift):
    """Rows apart, at the element's alignment only; what lies between them stays as it is."""
    rows, cols = 37, 352
    x = torch.randn(rows, cols, generator=gen(pad)).to(dtype).to(D)
    want = Q.quantise(x, True)
    big = torch.full((rows * (cols + pad) + shift,), 9.0, dtype=dtype, device=D)
    xs = big[shift:].view(rows, cols + pad)[:, :cols]
    xs.copy_(x)
    room = [torch.full((rows * (n + pad) + shift,), 0x5A, dtype=torch.uint8, device=D) for n in (cols // 2, cols // 32)]
    views = [r[shift:].view(rows, n + pad)[:, :n] for r, n in zip(room, (cols // 2, cols // 32))]
    api.mxfp4_quantise_cuda(xs, views[0].view(torch.float4_e2m1fn_x2), views[1].view(E8), 0)
    for v, w, r in zip(views, want, room):
        assert torch.equal(v, w)
        v.fill_(0x5A)
        assert (r == 0x5A).all()


def test_rows_far_apart():
    rows, cols = 5, 64
    x = torch.randn(rows, cols, generator=gen(8)).to(D)
    far = torch.empty((rows - 1 << 30) + cols, device=D).as_strided((rows, cols), (1 << 30, 1))
    far.copy_(x)
    codes, scales = buffers(rows, cols)
    api.mxfp4_quantise_cuda(far, codes, scales)
    want = Q.quantise(x, True)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    del far
    torch.cuda.empty_cache()


def test_more_rows_than_a_launch_has_threads_for():
    rows, cols = (1 << 30) + 40, 32  # four threads a row
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=D).normal_()
    codes, scales = buffers(rows, cols)
    api.mxfp4_quantise_cuda(x, codes, scales)
    for at in (0, (1 << 30) - 300, rows - 600):
        want = Q.quantise(x[at:at + 600], True)
        assert torch.equal(codes[at:at + 600], want[0]) and torch.equal(scales[at:at + 600], want[1])
    del x, codes, scales
    torch.cuda.empty_cache()


def test_streams_and_graphs():
    x = torch.randn(64, 2048, generator=gen(9)).to(torch.bfloat16).to(D)
    codes, scales = buffers(64, 2048)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        api.mxfp4_quantise_cuda(x, codes, scales)
    s.synchronize()
    want = Q.quantise(x, True)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        api.mxfp4_quantise_cuda(x, codes, scales)
    for k in range(4):
        x.copy_(torch.randn(64, 2048, generator=gen(k)).to(torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        want = Q.quantise(x, True)
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


def test_refusals():
    x = torch.zeros(4, 64, device=D)
    codes, scales = buffers(4, 64)
    for bad, error in [((x.double(), codes, scales), TypeError), ((x, codes[:, :16], scales), ValueError),
                       ((x, codes, scales[:3]), ValueError), ((x.t().contiguous().t(), codes, scales), ValueError),
                       ((x, codes.float(), scales), TypeError), ((x[0], codes, scales), ValueError)]:
        with pytest.raises(error):
            api.mxfp4_quantise_cuda(*bad)
    with pytest.raises(ValueError, match="on device 0"):
        api.mxfp4_quantise_cuda(x, codes, scales, 1)
    api.mxfp4_quantise_cuda(x[:0], codes[:0], scales[:0])
