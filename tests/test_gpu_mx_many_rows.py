"""Calls of so many rows that one launch, which holds fewer than 2^32 threads, does not hold them."""
import pytest

import mx_plain as P
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"


@pytest.fixture(autouse=True)
def free_memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def windows(rows, *at):
    """Slices about the given rows that there are, the first and the last ones."""
    return [slice(max(0, a - 300), min(rows, a + 300)) for a in (0, *at, rows) if a <= rows]


def nan_codes(rows, cols):
    return (torch.full((rows, cols), 0x7F, dtype=torch.uint8, device=D),
            torch.full((rows, cols // 32), 255, dtype=torch.uint8, device=D))


def test_norm():
    rows, cols = (1 << 26) + 5, 32  # four rows to 256 threads
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=D).normal_()
    w = torch.rand(cols, device=D) + 0.5
    codes, scales = nan_codes(rows, cols)
    total = torch.zeros_like(x)
    api.rms_norm_mx_cuda(x, w, codes, scales, 0, residual=x, sum_out=total, eps=1e-5)
    whole = not (scales == 255).any().item() and torch.equal(total, x + x)
    assert whole
    for part in windows(rows, 1 << 26):
        y = P.norm(x[part], x[part], w, 1e-5)[1]
        P.check_codes(codes[part], scales[part], y, P.norm_delta(cols))


def test_swiglu():
    rows, cols = 1 << 20, 32800  # a thread to eight values
    gate = torch.empty(rows, cols, dtype=torch.bfloat16, device=D).normal_()
    codes, scales = nan_codes(rows, cols)
    api.swiglu_mx_cuda(gate, gate, codes, scales)
    whole = not any((s == 255).any().item() for s in scales.split(1 << 17))
    assert whole
    for part in windows(rows, (1 << 32) * 8 // cols):
        P.check_codes(codes[part], scales[part], P.swiglu(gate[part], gate[part]), P.swiglu_delta(gate[part]))


def test_linear_of_one_token():
    rows, cols = (1 << 27) + 40, 32  # 16 rows to 512 threads
    codes = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, device=D)
    scales = torch.randint(110, 126, (rows, cols // 32), dtype=torch.uint8, device=D)
    x = torch.randn(1, cols, device=D)
    bias = torch.randn(rows, device=D)
    o = torch.full((1, rows), float("nan"), device=D)
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, bias=bias)
    whole = not torch.isnan(o).any().item()
    assert whole
    for part in windows(rows, 1 << 27):
        P.check_linear(o[:, part], x, None, codes[part], scales[part], bias[part])


@pytest.mark.parametrize("tokens,rows,far", [((1 << 32) // 80 + 33, 80, "weight"), (34, (1 << 28) + 24, "x")])
def test_linear_of_rows_far_apart(tokens, rows, far):
    """16 tokens and 16 rows to 256 threads, where a tile's offsets do not reach."""
    cols = 32
    codes = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, device=D)
    scales = torch.randint(110, 126, (rows, cols // 32), dtype=torch.uint8, device=D)
    x = torch.empty(tokens, cols, dtype=torch.bfloat16, device=D).normal_()
    bias = torch.randn(rows, device=D).to(torch.bfloat16)

    def apart(t):
        big = torch.empty((t.shape[0] - 1 << 27) + t.shape[1], dtype=t.dtype, device=D)
        v = big.as_strided(t.shape, (1 << 27, 1))
        v.copy_(t)
        return v

    o = torch.full((tokens, rows), float("nan"), dtype=torch.bfloat16, device=D)
    api.mxfp4_linear_cuda(apart(x) if far == "x" else x, apart(codes) if far == "weight" else codes, scales, o, 0,
                          bias=bias)
    whole = not any(torch.isnan(p).any().item() for p in o.split(max(1, tokens // 8)))
    assert whole
    for t in windows(tokens, (1 << 32) // 80):
        for r in windows(rows, 1 << 28):
            P.check_linear(o[t, r], x[t], None, codes[r], scales[r], bias[r])
