"""Every kernel of the product of two MXFP4 matrices, at sizes that reach it (mx4_sizes.py)."""
import pytest

import mx4_plain as Q
import mx4_sizes as S
import mx_plain as P
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["-".join(map(str, s)) + "-" + k for s, k in S.SIZES.items()]


def make(tokens, rows, cols, out, seed, low=112, high=122):
    g = torch.Generator().manual_seed(seed)
    x, xs = P.random_weights(tokens, cols, g, D, low, high)
    w, s = P.random_weights(rows, cols, g, D, low, high)
    return x, xs, w, s, torch.full((tokens, rows), float("nan"), dtype=out, device=D), torch.randn(rows, generator=g).to(out).to(D)


def strided(t, pad, shift):
    rows, cols = t.shape
    big = torch.full((rows * (cols + pad) + shift,), 0xFF, dtype=torch.uint8, device=D)
    v = big[shift:].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v


@pytest.mark.parametrize("size", S.SIZES, ids=IDS)
def test_types_and_places(size):
    """Each output type, and the same results from operands at any place: codes and scales at multiples of 16 bytes,
    codes alone, neither; what lies between the rows (broken scales) is not taken."""
    for n, out in enumerate(TYPES):
        x, xs, w, s, o, b = make(*size, out, n)
        api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
        Q.check_matmul(o, x, xs, w, s, b)
        p = torch.full_like(o, float("nan"))
        for pad, shift, scale_pad, scale_shift in ((16, 32, 16, 48), (32, 16, 3, 1), (5, 3, 16, 0)):
            fit = -(size[2] // 32) % 16  # scales' rows at multiples of 16 bytes
            p.fill_(float("nan"))
            api.mxfp4_matmul_cuda(strided(x, pad, shift), strided(xs, fit + scale_pad, scale_shift), strided(w, pad, shift),
                                  strided(s, fit + scale_pad, scale_shift), p, 0, bias=b)
            assert torch.equal(o, p)
        api.mxfp4_matmul_cuda(x, xs, w, s, p)
        Q.check_matmul(p, x, xs, w, s)


@pytest.mark.parametrize("size", S.SIZES, ids=IDS)
def test_each_scale_is_its_own_block_s(size):
    """Scales that differ by far from block to block, and equal codes, so that a scale in a wrong place shows."""
    tokens, rows, cols = size
    x, xs, w, s, o, _ = make(*size, torch.float32, 9)
    x.fill_(0x22), w.fill_(0x22)  # ones
    g = torch.Generator().manual_seed(cols)
    xs.copy_(torch.randint(100, 150, xs.shape, generator=g, dtype=torch.uint8))
    s.copy_(torch.randint(100, 150, s.shape, generator=g, dtype=torch.uint8))
    api.mxfp4_matmul_cuda(x, xs, w, s, o)
    Q.check_matmul(o, x, xs, w, s)


@pytest.mark.parametrize("size", S.SIZES, ids=IDS)
def test_again_and_from_a_graph(size):
    """The same bits each time: no request is taken before it has come."""
    x, xs, w, s, o, b = make(*size, torch.bfloat16, 4)
    api.mxfp4_matmul_cuda(x, xs, w, s, o, 0, bias=b)
    p = torch.zeros_like(o)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(3):
            api.mxfp4_matmul_cuda(x, xs, w, s, p, 0, bias=b)
    for _ in range(5):
        p.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, p)
