"""Masked experts and broken values in each of the experts' layer's ways to choose and to add up: a choice within the
inner products or in a launch of its own, a workgroup a pair or an expert, weighted sums at once or afterwards, in memory
that held NaN before."""
import pytest

import mx4_plain as Q
from test_gpu_mx4_moe import BF, D, FL, HF, Layer, activations, gen

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LAYERS = [  # experts, top_k, cols, inner
    (7, 3, 96, 64), (64, 3, 96, 352), (3, 3, 2080, 96), (5, 3, 2304, 1280), (40, 3, 2304, 96), (6, 3, 512, 2304),
]


def leave_nan_behind():
    """Fills what torch's allocator has free, in blocks of many sizes, so that workspaces begin with NaN."""
    kept = [torch.full((1 << k,), float("nan"), device=D) for k in range(7, 22) for _ in range(3)]
    torch.cuda.synchronize()
    del kept


@pytest.mark.parametrize("dtype", [BF, FL], ids=str)
@pytest.mark.parametrize("left", [(2, 1), (2,), ()], ids=lambda v: f"{len(v)} left")
@pytest.mark.parametrize("tokens", [1, 2, 5, 9])
@pytest.mark.parametrize("experts,top_k,cols,inner", LAYERS)
def test_masked_experts(experts, top_k, cols, inner, tokens, left, dtype):
    """Fewer experts than are chosen, or none: the others are chosen with the weight 0, the lowest first."""
    g = gen(experts, tokens, len(left), cols)
    layer = Layer(experts, top_k, cols, inner, g, dtype, dtype, True)
    keep = torch.zeros(experts, dtype=torch.bool, device=D)
    keep[list(left)] = True
    layer.bias["router_bias"][~keep] = -torch.inf
    x = activations(tokens, cols, dtype, g)
    leave_nan_behind()
    out, chosen, weights = layer.check(x)
    others = [e for e in range(experts) if e not in left][: top_k - len(left)]
    assert chosen[:, len(left):].tolist() == [others] * tokens
    assert not weights[:, len(left):].any()
    if left:
        assert ((weights.sum(-1) - 1).abs() < 1e-6).all()
    else:
        assert not out.any()


@pytest.mark.parametrize("dtype", [BF, FL], ids=str)
@pytest.mark.parametrize("tokens", [1, 2, 5, 9])
@pytest.mark.parametrize("experts,top_k,cols,inner", LAYERS)
def test_some_masked_experts(experts, top_k, cols, inner, tokens, dtype):
    """Enough are left: no masked one is chosen."""
    if experts == top_k:
        pytest.skip("all of its experts are chosen")
    g = gen(experts, tokens, 11)
    layer = Layer(experts, top_k, cols, inner, g, dtype, dtype, True)
    masked = torch.randperm(experts, generator=g)[: experts - top_k - (experts > 5)].to(D)
    layer.bias["router_bias"][masked] = -torch.inf
    leave_nan_behind()
    _, chosen, _ = layer.check(activations(tokens, cols, dtype, g))
    assert not torch.isin(chosen, masked).any()


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("broken", [torch.nan, torch.inf], ids=str)
@pytest.mark.parametrize("tokens", [2, 5, 9])
@pytest.mark.parametrize("experts,top_k,cols,inner", LAYERS)
def test_a_broken_token(experts, top_k, cols, inner, tokens, broken, dtype):
    """A token with NaN or an infinity leaves the others as they are, whether they share its experts or not: bit for bit,
    but for the order in which two tokens' experts are added up, which goes by both tokens' choices."""
    g = gen(experts, tokens, 12)
    layer = Layer(experts, top_k, cols, inner, g, FL, dtype)
    x = activations(tokens, cols, dtype, g)
    leave_nan_behind()
    clean, chosen, weights = layer.check(x)
    want = layer.want(x)
    for t in (0, tokens - 1):
        for k in (0, cols - 1):
            y = x.clone()
            y[t, k] = broken
            out, c, w = layer(y)
            rest = torch.arange(tokens, device=D) != t
            assert not torch.isfinite(out[t]).any() or broken == torch.inf
            assert ((c >= 0) & (c < experts)).all()
            Q.check_moe(out[rest], c[rest], w[rest], tuple(v[rest] for v in want))
            assert torch.equal(c[rest], chosen[rest]) and torch.equal(w[rest], weights[rest])
            assert tokens == 2 or torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("dtype", [BF, FL], ids=str)
@pytest.mark.parametrize("tokens", [2, 5, 9])
@pytest.mark.parametrize("experts,top_k,cols,inner", LAYERS)
def test_a_broken_expert(experts, top_k, cols, inner, tokens, dtype):
    """An expert with a NaN scale or bias breaks the tokens that chose it and no others."""
    g = gen(experts, tokens, 13)
    layer = Layer(experts, top_k, cols, inner, g, FL, dtype, True)
    x = activations(tokens, cols, dtype, g)
    clean, chosen, _ = layer.check(x)
    for e in {int(chosen[0, 0]), int(chosen[-1, -1])}:
        hit = (chosen == e).any(-1)
        for name in ("up_scales", "down_scales"):
            s = layer.w[name].clone()
            s[e, :, 0] = 255
            out, c, _ = layer(x, **{name: s})
            assert torch.equal(c, chosen) and torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])
        for name in ("gate_bias", "down_bias"):
            b = layer.bias[name].clone()
            b[e] = torch.nan
            out, c, _ = layer(x, **{name: b})
            assert torch.equal(c, chosen) and torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("tokens", [65, 130])
def test_several_passes_in_place(tokens):
    """out may be x where the tokens are served in several passes too."""
    g = gen(tokens, 14)
    layer = Layer(6, 2, 96, 64, g, FL, BF)
    x = activations(tokens, 96, BF, g)
    want = layer.check(x)
    got = layer(x, x)
    assert torch.equal(x, want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
