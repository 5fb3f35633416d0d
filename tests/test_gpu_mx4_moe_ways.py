"""The experts' layer on the GPU at sizes that reach each way to make its products, with codes at multiples of 16 bytes
and not, scales at any byte, gate and up apart or in one tensor."""
import pytest

import mx4_moe_sizes as S
import mx4_plain as Q
from test_gpu_mx4_moe import BF, D, FL, HF, NAMES, Layer, activations, gen

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPE = {"bf16": BF, "f16": HF, "f32": FL}


def moved(t, pad, shift):
    """The same stack with `pad` bytes between its rows, `shift` bytes into its memory."""
    e, r, c = t.shape
    v = torch.full((e * r * (c + pad) + shift,), 0x77, dtype=torch.uint8, device=D)
    v = v.as_strided((e, r, c), (r * (c + pad), c + pad, 1), shift)
    v.copy_(t)
    return v


@pytest.mark.parametrize("size", S.SIZES, ids=str)
def test_each_way(size):
    tokens, experts, top_k, cols, inner, kind = size
    g = gen(tokens, experts, cols, inner)
    for out in (TYPE[kind], BF if kind == "f32" else FL):
        layer = Layer(experts, top_k, cols, inner, g, BF, out, True)
        x = activations(tokens, cols, TYPE[kind], g)
        want = layer.want(x)
        w = layer.w
        codes = NAMES[0::2]
        for kw in ({}, {n: moved(w[n], 0, 8) for n in codes}, {n: moved(w[n], 5, 3) for n in codes},
                   {n: moved(w[n], 16, 16) for n in codes}, {n: moved(w[n], 1, 2) for n in NAMES[1::2]},
                   dict(up=moved(w["up"], 32, 0)), dict(down=moved(w["down"], 0, 4))):
            Q.check_moe(*layer(x, **kw), want)


@pytest.mark.parametrize("size", S.SIZES, ids=str)
def test_views_of_one_tensor(size):
    """Gate and up as alternate rows give the same bits as apart: both lie at multiples of 16 bytes."""
    tokens, experts, top_k, cols, inner, kind = size
    g = gen(tokens, experts, cols, 5)
    layer = Layer(experts, top_k, cols, inner, g, FL, TYPE[kind], True)
    x = activations(tokens, cols, TYPE[kind], g)
    w = layer.w
    mixed = [torch.stack((w[a], w[b]), 2).flatten(1, 2) for a, b in (("gate", "up"), ("gate_scales", "up_scales"))]
    one = layer(x, gate=mixed[0][:, 0::2], up=mixed[0][:, 1::2], gate_scales=mixed[1][:, 0::2], up_scales=mixed[1][:, 1::2])
    assert all(torch.equal(a, b) for a, b in zip(one, layer(x)))
