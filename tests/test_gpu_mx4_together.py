"""The operators on MXFP4 tensors together: weights quantised on the GPU, coded, restored by one decode call and used
where they were restored, by the products of 4-bit operands and by the experts' layer."""
import importlib.util
import os

import pytest

import mx4_plain as Q
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    path = os.path.join(ROOT, "examples", "mxfp4_feed_forward.py")
    spec = importlib.util.spec_from_file_location("feed_forward", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def quantised(x, saturate=True):
    rows, cols = x.shape
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=D)
    scales = torch.empty(rows, cols // 32, dtype=torch.uint8, device=D)
    api.mxfp4_quantise_cuda(x, codes, scales, 0, saturate)
    return codes, scales


@pytest.mark.parametrize("tokens", [1, 19, 300])
def test_feed_forward_in_four_bits(example, tokens):
    hidden, inner = 736, 1120
    g = torch.Generator().manual_seed(tokens)
    w = [(torch.randn(*s, generator=g) * 0.03).to(D) for s in ((2 * inner, hidden), (hidden, inner))]
    made = [t for m in w for t in quantised(m)]
    for m, codes, scales in zip(w, made[::2], made[1::2]):
        want = Q.quantise(m, True)
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    planes, state = example.compress(made)
    gate_up, gate_up_scales, down, down_scales = example.restore(planes, state, [t.shape for t in made])
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16).to(D)
    codes, scales = quantised(x, False)
    both = torch.empty(tokens, 2 * inner, dtype=torch.bfloat16, device=D)
    api.mxfp4_matmul_cuda(codes, scales, gate_up, gate_up_scales, both)
    Q.check_matmul(both, codes, scales, gate_up, gate_up_scales)
    act = both[:, :inner].float()
    act = (act / (1 + torch.exp(-act)) * both[:, inner:].float()).to(torch.bfloat16)
    codes, scales = quantised(act, False)
    out = torch.empty(tokens, hidden, dtype=torch.bfloat16, device=D)
    api.mxfp4_matmul_cuda(codes, scales, down, down_scales, out)
    Q.check_matmul(out, codes, scales, down, down_scales)


@pytest.mark.parametrize("tokens", [1, 9, 80])
def test_experts(example, tokens):
    """Gate and up as halves of one restored tensor; eager, on another stream and replayed, with a shared expert beside."""
    experts, top_k, hidden, inner = 6, 2, 2304, 1152
    g = torch.Generator().manual_seed(tokens)
    w = [(torch.randn(*s, generator=g) * 0.03).to(D) for s in ((experts * 2 * inner, hidden), (experts * hidden, inner))]
    made = [t for m in w for t in quantised(m)]
    planes, state = example.compress(made)
    gu, gus, down, ds = example.restore(planes, state, [t.shape for t in made])
    assert all(torch.equal(a, b) for a, b in zip(made, (gu, gus, down, ds)))
    gu, gus = gu.view(experts, 2 * inner, -1), gus.view(experts, 2 * inner, -1)
    down, ds = down.view(experts, hidden, -1), ds.view(experts, hidden, -1)
    layer = (gu[:, :inner], gus[:, :inner], gu[:, inner:], gus[:, inner:], down, ds)
    router = (torch.randn(experts, hidden, generator=g) / hidden**0.5).to(torch.bfloat16).to(D)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16).to(D)
    out = torch.empty_like(x)
    codes = torch.empty(tokens, hidden // 2, dtype=torch.uint8, device=D)
    scales = torch.empty(tokens, hidden // 32, dtype=torch.uint8, device=D)
    shared = torch.empty(tokens, inner, dtype=torch.bfloat16, device=D)

    def step():
        api.mxfp4_moe_cuda(x, router, *layer, out, top_k)
        api.mxfp4_quantise_cuda(x, codes, scales, 0, False)
        api.mxfp4_matmul_cuda(codes, scales, gu[0, :inner], gus[0, :inner], shared)

    def check():
        Q.check_moe(out, None, None, Q.moe(x, router, *layer, top_k, out_type=out.dtype))
        Q.check_matmul(shared, codes, scales, gu[0, :inner], gus[0, :inner])

    step()
    check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        x.copy_(torch.randn(tokens, hidden, generator=g).to(torch.bfloat16))
        out.fill_(float("nan")), shared.fill_(float("nan"))
        graph.replay()
        check()
        step()
        check()
