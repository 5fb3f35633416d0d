"""The mixture-of-experts layer on the GPU where several tokens meet rows so long that the columns of a workgroup stay
in registers, and just past where they do."""
import pytest

import mx4_plain as Q
from ptwm_amd import api
from test_gpu_mx4_moe import BF, D, FL, HF, NAMES, Layer, activations, gen

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SIZES = [  # tokens, experts, top_k, cols, inner: steps of 256 values, whole and not, for one to four turns of eight wavefronts
    (2, 2, 1, 2176, 1152), (3, 5, 2, 2304, 1280), (9, 9, 3, 4096, 2176), (33, 4, 2, 3968, 2048), (64, 2, 1, 4224, 4224),
    (64, 1, 1, 2176, 8192), (17, 300, 2, 2560, 1152), (40, 6, 6, 8064, 1408), (65, 3, 2, 8192, 2304), (8, 2, 1, 8320, 1280),
    (5, 3, 2, 64, 32768), (4, 2, 2, 96, 32896), (64, 4, 4, 2304, 1024), (64, 40, 32, 2304, 1152), (63, 1024, 2, 64, 1152),
    (16, 8, 2, 5120, 32), (50, 7, 1, 32, 14336),
    # rows of blocks that are no multiple of four: scales at any byte, one to seven blocks in the last step
    (7, 3, 2, 2080, 1056), (30, 4, 2, 2112, 1184), (64, 5, 2, 2144, 1248), (21, 6, 3, 4128, 1504), (40, 2, 1, 5056, 2400),
    (12, 4, 2, 8160, 4320), (10, 2, 1, 3360, 14304), (64, 33, 4, 2272, 1312),
    # many experts
    (63, 1024, 2, 64, 2176), (20, 600, 4, 2080, 64),
]


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("tokens,experts,top_k,cols,inner", SIZES)
def test_sizes(tokens, experts, top_k, cols, inner, dtype):
    g = gen(tokens, experts, cols, inner)
    layer = Layer(experts, top_k, cols, inner, g, dtype, dtype, tokens % 2 == 1)
    layer.check(activations(tokens, cols, dtype, g))


@pytest.mark.parametrize("out", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
def test_types(dtype, out):
    g = gen(21, 4)
    Layer(5, 2, 2432, 1664, g, BF, out, True).check(activations(21, 2432, dtype, g))


@pytest.mark.parametrize("dtype", [BF, FL], ids=str)
def test_all_tokens_to_few_experts(dtype):
    """Experts without a token, one with all of them, more than a workgroup holds at a time."""
    g = gen(8, 8)
    layer = Layer(12, 2, 2304, 1280, g, dtype, dtype, True)
    x = activations(64, 2304, dtype, g)
    layer.bias["router_bias"][:] = -30000.0
    layer.bias["router_bias"][5] = layer.bias["router_bias"][11] = 0.0
    _, chosen, _ = layer.check(x)
    assert set(chosen.flatten().tolist()) == {5, 11}


def test_masked_experts():
    g = gen(15)
    layer = Layer(6, 3, 2304, 1152, g, bias=True)
    x = activations(20, 2304, FL, g)
    layer.bias["router_bias"][torch.tensor([0, 1, 2, 4], device=D)] = -torch.inf
    _, _, weights = layer.check(x)
    assert not weights[:, 2].any()
    layer.bias["router_bias"][:] = -torch.inf
    out, *_ = layer.check(x)
    assert not out.any()


def test_broken_values_stay_where_they_are():
    g = gen(16)
    layer = Layer(5, 2, 2176, 1152, g, FL, BF)
    x = activations(30, 2176, BF, g)
    clean, chosen, _ = layer(x)
    y = x.clone()
    y[1, 7], y[2, 2175] = torch.nan, torch.inf
    out, c, w = layer(y)
    assert torch.isnan(out[1]).all() and ((c >= 0) & (c < 5)).all()
    keep = torch.ones(30, dtype=torch.bool, device=D)
    keep[1:3] = False
    Q.check_moe(out[keep], c[keep], w[keep], layer.want(x[keep]))
    for name in ("gate_scales", "down_scales"):
        s = layer.w[name].clone()
        s[3, :, -1] = 255
        out, *_ = layer(x, **{name: s})
        hit = (chosen == 3).any(-1)
        assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


def test_layouts():
    """Gate and up as halves or alternate rows of one tensor, experts and rows apart, by 2^26 and 2^27 bytes too, scales
    and codes at odd addresses."""
    g = gen(18)
    layer = Layer(3, 2, 2304, 1280, g, BF, BF, True)
    x = activations(18, 2304, BF, g)
    want = layer.want(x)
    w = layer.w
    halves = torch.cat((w["gate"], w["up"]), 1), torch.cat((w["gate_scales"], w["up_scales"]), 1)
    mixed = [torch.stack((w[a], w[b]), 2).flatten(1, 2) for a, b in (("gate", "up"), ("gate_scales", "up_scales"))]
    both = torch.stack((layer.bias["gate_bias"], layer.bias["up_bias"]), 2).flatten(1, 2)

    def apart(t, row, shift=0):
        e, r, c = t.shape
        big = torch.full((e * (r * (c + row) + row) + shift,), 0x5A, dtype=torch.uint8, device=D)
        v = big.as_strided((e, r, c), (r * (c + row) + row, c + row, 1), shift)
        v.copy_(t)
        return v

    i = 1280
    for kw in (dict(gate=halves[0][:, :i], up=halves[0][:, i:], gate_scales=halves[1][:, :i], up_scales=halves[1][:, i:]),
               dict(gate=mixed[0][:, 0::2], up=mixed[0][:, 1::2], gate_scales=mixed[1][:, 0::2], up_scales=mixed[1][:, 1::2],
                    gate_bias=both[:, 0::2], up_bias=both[:, 1::2]),
               {n: apart(v, 16) for n, v in w.items()}, {n: apart(v, 4, 16) for n, v in w.items()},
               {n: apart(v, 3, 5) for n, v in w.items()}, dict(up=apart(w["up"], 32)),
               dict(up_scales=apart(w["up_scales"], 4)), dict(gate_scales=apart(w["gate_scales"], 0, 1))):
        Q.check_moe(*layer(x, **kw), want)


@pytest.mark.parametrize("step", [1 << 26, 1 << 27])
def test_rows_far_apart(step):
    g = gen(19)
    for cols, inner, names in ((2176, 32, NAMES[:4:2]), (32, 1152, NAMES[4:5])):
        layer = Layer(2, 1, cols, inner, g, BF, BF)
        x = activations(12, cols, BF, g)
        kw = {}
        for n in names:
            t = layer.w[n]
            v = torch.empty(31 * step + 2 * t.shape[2], dtype=torch.uint8, device=D)
            kw[n] = v.as_strided(t.shape, (t.shape[2], step, 1))
            kw[n].copy_(t)
        Q.check_moe(*layer(x, **kw), layer.want(x))
        del kw, v
    torch.cuda.empty_cache()


def test_streams_and_graphs():
    """Two streams at once, two graphs replayed in turn with eager calls between, the same bits each time."""
    g = gen(20)
    layer = Layer(8, 2, 2304, 2176, g, BF, BF, True)
    xs = [activations(40, 2304, BF, g) for _ in range(6)]
    want = [layer(x)[0] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for k in range(24):
        with torch.cuda.stream(streams[k % 2]):
            got.append(layer(xs[k % 6])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[k % 6]) for k, a in enumerate(got))
    graphs = []
    for _ in range(2):
        x, o = xs[0].clone(), torch.zeros_like(xs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            api.mxfp4_moe_cuda(x, layer.router, *(layer.w[n] for n in NAMES), o, 2, **layer.bias)
        graphs.append((graph, x, o))
    for k in range(6):
        graph, x, o = graphs[k % 2]
        x.copy_(xs[k])
        o.zero_()
        graph.replay()
        eager = layer(xs[(k + 1) % 6])[0]
        torch.cuda.synchronize()
        assert torch.equal(o, want[k]) and torch.equal(eager, want[(k + 1) % 6])
