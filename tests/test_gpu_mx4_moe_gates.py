"""The experts' layer's activation where exp(-gate) is past 32 bits: silu(g) is -2e-37 at g = -89 and less below, and a
large u makes a value of it."""
import math

import pytest

from test_gpu_mx4_moe import D, FL, NAMES, Layer

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

CODE_OF_ONE = 2


@pytest.mark.parametrize("tokens,cols,inner", [(1, 96, 64), (2, 2080, 96), (7, 96, 1120), (40, 2304, 2304)])
@pytest.mark.parametrize("gate,power", [(-60.0, 40), (-87.0, 60), (-88.0, 100), (-88.5, 100), (-89.0, 100), (-95.0, 110),
                                        (-104.0, 120), (-120.0, 126), (-150.0, 126), (-160.0, 126), (40.0, 3), (0.5, 0)])
def test_gates(gate, power, tokens, cols, inner):
    """h = silu(g) * x 2^power of one product each. The exponential, four factors of it at most, the quotient and the
    products round ten times in all, the exponential by a unit in the last place and by half of one for each unit of its
    argument that is off by half of one: (2 |g| + 32) units of 2^-24."""
    g = torch.Generator().manual_seed(int(-gate * 2 + 100) * 50 + tokens)
    x = 1 + torch.rand(tokens, cols, generator=g)
    x[:, 0] = gate
    zero = lambda r, c: torch.zeros(2, r, c // 2, dtype=torch.uint8)  # noqa: E731
    w = dict(gate=zero(inner, cols), up=zero(inner, cols), down=zero(cols, inner))
    scale = lambda r, c, p: torch.full((2, r, c // 32), 127 + p, dtype=torch.uint8)  # noqa: E731
    w |= dict(gate_scales=scale(inner, cols, 0), up_scales=scale(inner, cols, power), down_scales=scale(cols, inner, 0))
    at = torch.randint(1, cols, (inner,), generator=g)
    w["gate"][:, :, 0] = CODE_OF_ONE
    w["up"][:, torch.arange(inner), at // 2] = (CODE_OF_ONE << 4 * (at % 2)).to(torch.uint8)
    h = torch.randint(0, inner, (cols,), generator=g)
    w["down"][:, torch.arange(cols), h // 2] = (CODE_OF_ONE << 4 * (h % 2)).to(torch.uint8)
    layer = Layer(2, 1, cols, inner, g, FL, FL)
    layer.w = {n: w[n].to(D) for n in NAMES}
    out, *_ = layer(x.to(D))
    want = gate / (1 + math.exp(-gate)) * x.double()[:, at[h]] * 2.0**power
    assert want.abs().min() > 2.0**-126 and want.abs().max() < 2.0**127
    off = ((out.double().cpu() - want).abs() / want.abs()).max().item()
    assert off <= (2 * abs(gate) + 32) * 2.0**-24, off
