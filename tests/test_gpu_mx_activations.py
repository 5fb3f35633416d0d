"""The gated activation's accuracy in 32 bits, seen through the scale that a block takes: one value a block, a few
units on either side of 448, where the next scale begins."""
import pytest

import mx_plain as P
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
# In units of 2^-24: the hardware's exponential 2 (a unit in its last place), its argument's low part 2, the sum with 1,
# the reciprocal 2, the products with gate and up 2, and one for what these multiply to.
UNITS = 10


def one_value_blocks(gate, up, dtype=torch.float32):
    """(scale bytes, codes) of blocks that hold gate[i], up[i] and zeros."""
    g = torch.zeros(gate.numel(), 32, dtype=dtype)
    u = torch.zeros(gate.numel(), 32, dtype=dtype)
    g[:, 5], u[:, 5] = gate, up
    codes = torch.zeros(g.shape, dtype=torch.uint8, device=D)
    scales = torch.zeros(g.shape[0], 1, dtype=torch.uint8, device=D)
    api.swiglu_mx_cuda(g.to(D), u.to(D), codes, scales)
    return scales.cpu()[:, 0], codes, scales


@pytest.mark.parametrize("low,high", [(-85, -60), (-60, -20), (-20, -5), (-5, 0), (0, 5), (5, 85)])
def test_swiglu_rounds_like_32_bits(low, high):
    gen = torch.Generator().manual_seed(low + 100)
    gate = torch.rand(4096, generator=gen) * (high - low) + low
    gate = gate[gate.abs() > 1e-3]
    s = P.swiglu(gate, torch.ones_like(gate))
    for side, byte in ((-1, 127), (1, 128)):
        # up is rounded by a unit, and stays UNITS away from 448 all the same
        up = (448 * (1 + side * (UNITS + 2) * 2.0**-24) / s).float()
        y = P.swiglu(gate, up).abs()
        far = y < 448 * (1 - UNITS * 2.0**-24) if side < 0 else y > 448 * (1 + UNITS * 2.0**-24)
        assert far.all()
        got = one_value_blocks(gate, up)[0]
        assert (got == byte).all(), f"{(got != byte).sum().item()} of {gate.numel()} values of the other scale"


def test_swiglu_of_gates_below_the_normal_numbers():
    """gate / 2 is a number of the type as far as gate is an even multiple of the smallest one."""
    m = torch.arange(1, 4097, dtype=torch.float64)
    gate = torch.cat([m, -m, m * 4096]) * 2.0**-148
    for up in (2.0**100, -1.5 * 2.0**120, 1.0):
        y = torch.zeros(gate.numel(), 32, dtype=torch.float64)
        y[:, 5] = gate / 2 * up
        assert torch.equal(gate.float().double(), gate)
        _, codes, scales = one_value_blocks(gate.float(), torch.full_like(gate, up).float())
        P.check_codes(codes, scales, y.to(D), UNITS * 2.0**-24)
