"""The mixture-of-experts layer on MXFP4 experts on the GPU against its formula in 64 bits."""
import pytest

import mx4_plain as Q
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
E8 = torch.float8_e8m0fnu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
NAMES = ("gate", "gate_scales", "up", "up_scales", "down", "down_scales")


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


class Layer:
    def __init__(self, experts, top_k, cols, inner, g, router=FL, out=FL, bias=False):
        self.top_k, self.type = top_k, out
        # code values of 3 at most times 2^-7: products of a row of n around sqrt(n) / 50
        low = 127 - 4 - (cols.bit_length() // 2)
        made = (Q.random_experts(experts, inner, cols, g, D, low, low + 4) +
                Q.random_experts(experts, inner, cols, g, D, low, low + 4) +
                Q.random_experts(experts, cols, inner, g, D, 127 - 5 - inner.bit_length() // 2, 127 - 1 - inner.bit_length() // 2))
        self.w = dict(zip(NAMES, made))
        self.router = (torch.randn(experts, cols, generator=g) * 1.5 / cols**0.5).to(router).to(D)
        self.bias = {}
        if bias:
            r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
            self.bias = dict(router_bias=r(experts).to(router).to(D), gate_bias=r(experts, inner).to(out).to(D),
                             up_bias=r(experts, inner).to(out).to(D), down_bias=r(experts, cols).to(out).to(D))

    def __call__(self, x, out=None, **kw):
        n = x.shape[0]
        out = torch.full((n, x.shape[1]), float("nan"), dtype=self.type, device=D) if out is None else out
        experts = torch.full((n, self.top_k), -7, dtype=torch.int32, device=D)
        weights = torch.full((n, self.top_k), float("nan"), device=D)
        a = {**self.w, **self.bias, **kw}
        api.mxfp4_moe_cuda(x, a.pop("router", self.router), *(a.pop(n) for n in NAMES), out, self.top_k, 0,
                           experts=experts, weights=weights, **a)
        return out, experts, weights

    def want(self, x):
        return Q.moe(x, self.router, *(self.w[n] for n in NAMES), self.top_k, out_type=self.type, **self.bias)

    def check(self, x):
        got = self(x)
        Q.check_moe(*got, self.want(x))
        return got


def activations(tokens, cols, dtype, g):
    loud = torch.where(torch.rand(cols, generator=g) < 0.03, 8.0, 1.0)
    return (torch.randn(tokens, cols, generator=g) * loud).to(dtype).to(D)


SIZES = [  # tokens, experts, top_k, cols, inner
    (1, 1, 1, 32, 32), (1, 2, 1, 64, 96), (1, 8, 2, 4096, 1440), (1, 128, 8, 2048, 768), (2, 5, 3, 96, 160),
    (3, 64, 6, 416, 96), (5, 65, 7, 352, 1056), (7, 11, 3, 1120, 1504), (15, 3, 3, 160, 64), (16, 32, 4, 1024, 512),
    (17, 32, 4, 736, 544), (31, 2, 1, 288, 992), (33, 4, 2, 1184, 608), (40, 128, 8, 512, 256), (63, 16, 5, 224, 4096),
    (64, 8, 2, 2080, 1120), (64, 1, 1, 544, 480), (64, 3, 3, 320, 352), (65, 8, 2, 256, 288), (130, 6, 4, 192, 128),
    (4, 1024, 32, 128, 64), (70, 200, 32, 64, 32), (64, 8, 1, 128, 14336), (9, 4, 2, 8192, 64),
]


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("tokens,experts,top_k,cols,inner", SIZES)
def test_sizes(tokens, experts, top_k, cols, inner, dtype):
    g = gen(tokens, experts, cols, inner)
    layer = Layer(experts, top_k, cols, inner, g, dtype, dtype, tokens % 2 == 1)
    layer.check(activations(tokens, cols, dtype, g))


@pytest.mark.parametrize("tokens", [1, 6, 40])
@pytest.mark.parametrize("out", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("router", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
def test_types(dtype, router, out, tokens):
    g = gen(tokens, 4)
    Layer(9, 4, 416, 352, g, router, out, True).check(activations(tokens, 416, dtype, g))


@pytest.mark.parametrize("experts,top_k", [(7, 3), (64, 8), (130, 5), (1024, 32)])
def test_ties(experts, top_k):
    """Whole-number logits, many of them equal: the lowest indices are chosen."""
    g = gen(experts)
    layer = Layer(experts, top_k, 64, 32, g)
    layer.router = torch.randint(-1, 2, (experts, 64), generator=g).float().to(D)
    x = torch.randint(-1, 2, (50, 64), generator=g).float().to(D)
    x[0] = 0  # all alike, zeros of both signs
    x[1] = -0.0
    _, chosen, weights = layer.check(x)
    assert chosen[:2].tolist() == [list(range(top_k))] * 2
    assert ((weights[:2] - 1 / top_k).abs() < 1e-6).all()


def test_near_logits():
    """Logits that 32 bits do not tell apart."""
    layer = Layer(4, 1, 64, 32, gen(2))
    layer.router = torch.zeros(4, 64, device=D)
    layer.router[:, 0], layer.router[:, 1] = 1.0, torch.tensor([0.0, 2.0**-40, 2.0**-41, 2.0**-42], device=D)
    x = torch.zeros(3, 64, device=D)
    x[:, 0], x[:, 1] = 1.0, torch.tensor([1.0, -1.0, 0.0], device=D)
    assert layer.check(x)[1].flatten().tolist() == [1, 0, 0]


def test_masked_experts():
    """A bias of minus infinity keeps an expert out; where too few are left, the others have the weight 0."""
    g = gen(5)
    layer = Layer(6, 3, 96, 64, g, bias=True)
    x = activations(9, 96, FL, g)
    layer.bias["router_bias"][torch.tensor([0, 4], device=D)] = -torch.inf
    _, chosen, weights = layer.check(x)
    assert not ((chosen == 0) | (chosen == 4)).any()
    layer.bias["router_bias"][torch.tensor([1, 2, 3], device=D)] = -torch.inf
    _, chosen, weights = layer.check(x)
    assert (chosen == torch.tensor([5, 0, 1], device=D)).all()
    assert (weights == torch.tensor([1.0, 0, 0], device=D)).all()
    layer.bias["router_bias"][:] = -torch.inf
    out, chosen, weights = layer.check(x)
    assert not out.any() and not weights.any() and (chosen == torch.tensor([0, 1, 2], device=D)).all()


@pytest.mark.parametrize("tokens", [3, 20, 64])
@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
def test_broken_values_stay_where_they_are(tokens, dtype):
    """A token with NaN or an infinity, and an expert with a NaN scale, leave the other tokens as they are."""
    g = gen(tokens, 6)
    layer = Layer(5, 2, 160, 96, g, FL, dtype)
    x = activations(tokens, 160, dtype, g)
    clean, chosen, _ = layer(x)
    y = x.clone()
    y[1, 7], y[2, 159] = torch.nan, torch.inf
    out, c, w = layer(y)
    assert torch.isnan(out[1]).all() and torch.isnan(w[1]).all()
    assert ((c >= 0) & (c < 5)).all()
    keep = torch.ones(tokens, dtype=torch.bool, device=D)
    keep[1:3] = False
    Q.check_moe(out[keep], c[keep], w[keep], layer.want(x[keep]))
    for name in ("gate_scales", "down_scales"):
        s = layer.w[name].clone()
        s[3, :, -1] = 255
        out, *_ = layer(x, **{name: s})
        hit = (chosen == 3).any(-1)
        assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
def test_large_and_small_values(dtype):
    """Activations and weights at the ends of the types' ranges, outputs that overflow excepted."""
    g = gen(12)
    for low, scale in ((100, 2.0**10), (124, 2.0**-10), (127, 2.0**-20 if dtype == HF else 2.0**-60)):
        layer = Layer(3, 2, 128, 96, g, FL, FL)
        for n in ("gate", "up"):
            layer.w[n + "_scales"] = torch.randint(low - 3, low, (3, 96, 4), generator=g, dtype=torch.uint8).to(D)
        layer.router = torch.randn(3, 128, generator=g).to(D) * 0.01 / scale
        layer.check((torch.randn(11, 128, generator=g) * scale).to(dtype).to(D))


def strided(t, pad, shift):
    """A stack with `pad` bytes between rows and experts, `shift` bytes in."""
    e, r, c = t.shape
    big = torch.full((e * (r * (c + pad) + pad) + shift,), 0x5A, dtype=torch.uint8, device=D)
    v = big[shift:].as_strided((e, r, c), (r * (c + pad) + pad, c + pad, 1))
    v = torch.as_strided(big, (e, r, c), (r * (c + pad) + pad, c + pad, 1), shift)
    v.copy_(t)
    return v


@pytest.mark.parametrize("tokens", [1, 7, 33])
@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
def test_layouts(tokens, dtype):
    """Halves and alternate rows of one tensor, any alignment, rows of x and out apart: the same results."""
    g = gen(tokens, 8)
    layer = Layer(6, 2, 352, 224, g, BF, dtype, True)
    x = activations(tokens, 352, dtype, g)
    out, chosen, weights = layer.check(x)
    w = layer.w
    halves = torch.cat((w["gate"], w["up"]), 1), torch.cat((w["gate_scales"], w["up_scales"]), 1)
    mixed = [torch.stack((w[a], w[b]), 2).flatten(1, 2) for a, b in (("gate", "up"), ("gate_scales", "up_scales"))]
    both = torch.stack((layer.bias["gate_bias"], layer.bias["up_bias"]), 2).flatten(1, 2)
    i = 224
    for kw in (dict(gate=halves[0][:, :i], up=halves[0][:, i:], gate_scales=halves[1][:, :i], up_scales=halves[1][:, i:]),
               dict(gate=mixed[0][:, 0::2], up=mixed[0][:, 1::2], gate_scales=mixed[1][:, 0::2].view(E8),
                    up_scales=mixed[1][:, 1::2], gate_bias=both[:, 0::2], up_bias=both[:, 1::2]),
               {n: strided(v, 16, 32) for n, v in w.items()},
               {n: strided(v, 3, 5) for n, v in w.items()},
               {n: strided(v, 0, 1) if n == "down" else v for n, v in w.items()},
               {n: v.view(torch.float4_e2m1fn_x2) if n in ("gate", "up", "down") else v.view(E8) for n, v in w.items()}):
        got = layer(x, **kw)
        assert torch.equal(got[0], out) and torch.equal(got[1], chosen) and torch.equal(got[2], weights)
    for pad, shift in ((1, 1), (8, 8), (3, 2)):
        room = torch.full((tokens * (352 + pad) + shift,), 3.0, dtype=dtype, device=D)
        o = room[shift:].view(tokens, 352 + pad)[:, :352]
        xs = torch.full((tokens * (352 + pad) + shift,), 3.0, dtype=dtype, device=D)[shift:].view(tokens, 352 + pad)[:, :352]
        xs.copy_(x)
        r = torch.zeros(6, 352 + pad, dtype=BF, device=D)[:, :352]
        r.copy_(layer.router)
        got = layer(xs, o, router=r)
        assert torch.equal(got[0], out) and torch.equal(got[2], weights)
        o.fill_(3.0)
        assert (room == 3.0).all()
    same = x.clone()  # in place
    assert torch.equal(layer(same, same)[0], out)


@pytest.mark.parametrize("far", ["experts", "rows", "x"])
def test_far_apart(far):
    """Offsets past 32 bits between experts, rows and tokens."""
    g = gen(3, 3)
    layer = Layer(3, 2, 96, 64, g, FL, FL)
    x = activations(40, 96, FL, g)
    want = layer.check(x)

    def apart(t, dim):
        stride = list(t.stride())
        step = (6 << 30) // t.shape[dim] // 16 * 16
        stride[dim] = step
        if dim == 1:
            stride[0] = 3200  # experts between the rows
        size = 1 + sum((n - 1) * s for n, s in zip(t.shape, stride))
        v = torch.empty(size, dtype=t.dtype, device=D).as_strided(t.shape, stride)
        v.copy_(t)
        return v

    if far == "x":
        xs = torch.empty(39 * (1 << 26) + 96, device=D).as_strided((40, 96), (1 << 26, 1))
        xs.copy_(x)
        got = layer(xs)
    else:
        dim = 0 if far == "experts" else 1
        got = layer(x, **{n: apart(layer.w[n], dim) for n in NAMES})
    assert torch.equal(got[0], want[0])
    del got
    torch.cuda.empty_cache()


def test_without_what_is_optional():
    g = gen(2, 2)
    layer = Layer(4, 2, 64, 64, g)
    x = activations(5, 64, FL, g)
    o = torch.empty(5, 64, device=D)
    api.mxfp4_moe_cuda(x, layer.router, *(layer.w[n] for n in NAMES), o, 2)
    assert torch.equal(o, layer.check(x)[0])
    api.mxfp4_moe_cuda(x[:0], layer.router, *(layer.w[n] for n in NAMES), o[:0], 2)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 8, 2), (1, 128, 8), (20, 8, 2), (64, 16, 4)])
def test_streams_and_graphs(tokens, experts, top_k):
    """Two streams at once, and two graphs replayed in turn with eager calls between."""
    g = gen(tokens, 9)
    layer = Layer(experts, top_k, 512, 256, g, BF, BF)
    xs = [activations(tokens, 512, BF, g) for _ in range(6)]
    want = [layer(x)[0] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k, x in enumerate(xs):
        with torch.cuda.stream(streams[k % 2]):
            got.append(layer(x)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        x, o = xs[0].clone(), torch.zeros_like(xs[0])
        e, w = torch.zeros(tokens, top_k, dtype=torch.int32, device=D), torch.zeros(tokens, top_k, device=D)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            api.mxfp4_moe_cuda(x, layer.router, *(layer.w[n] for n in NAMES), o, top_k, experts=e, weights=w)
            api.mxfp4_moe_cuda(x, layer.router, *(layer.w[n] for n in NAMES), o, top_k)
        graphs.append((graph, x, o))
    for k in range(6):
        graph, x, o = graphs[k % 2]
        x.copy_(xs[k])
        o.zero_()
        graph.replay()
        eager = layer(xs[(k + 1) % 6])[0]
        torch.cuda.synchronize()
        assert torch.equal(o, want[k]) and torch.equal(eager, want[(k + 1) % 6])


def test_same_results_again():
    g = gen(77)
    layer = Layer(16, 4, 1024, 512, g, BF, BF)
    x = activations(48, 1024, BF, g)
    first = layer(x)[0]
    for _ in range(20):
        assert torch.equal(layer(x)[0], first)


def test_refusals():
    g = gen(1)
    layer = Layer(4, 2, 64, 96, g)
    x = activations(3, 64, FL, g)
    for kw, error in [(dict(gate=layer.w["gate"][:3]), ValueError), (dict(up=layer.w["up"][:, :64]), ValueError),
                      (dict(down=layer.w["gate"]), ValueError), (dict(gate=layer.w["gate"].float()), TypeError),
                      (dict(gate_scales=layer.w["gate_scales"][:, :, :1]), ValueError),
                      (dict(router=layer.router[:, :32]), ValueError), (dict(router=layer.router.double()), TypeError),
                      (dict(gate_bias=torch.zeros(4, 96, dtype=BF, device=D)), TypeError),
                      (dict(down_bias=torch.zeros(4, 96, device=D)), ValueError),
                      (dict(router_bias=torch.zeros(3, device=D)), ValueError),
                      (dict(gate=layer.w["gate"].transpose(1, 2).contiguous().transpose(1, 2)), ValueError)]:
        with pytest.raises(error):
            layer(x, **kw)
    o = torch.zeros(3, 64, device=D)
    for top_k, error in ((0, ValueError), (5, ValueError), (33, ValueError), ("2", TypeError)):
        with pytest.raises(error):
            api.mxfp4_moe_cuda(x, layer.router, *(layer.w[n] for n in NAMES), o, top_k)
    with pytest.raises(ValueError):
        api.mxfp4_moe_cuda(x, layer.router, *(layer.w[n] for n in NAMES), o[:2], 2)
    with pytest.raises(ValueError):
        api.mxfp4_moe_cuda(x, layer.router, *(layer.w[n] for n in NAMES), o, 2,
                           experts=torch.zeros(3, 4, dtype=torch.int32, device=D)[:, ::2])
