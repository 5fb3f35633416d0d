"""The mixture-of-experts layer on the GPU where every sum is exact, so that each bit of the activations and of the hidden
values decides.

Gates are 32, whose activation is 32 in 24 bits. A row of `up` adds up one to three activations at places that do not
overlap: an integer of 24 (22 for float16) bits. A row of `down` takes one hidden value, or a pair whose leading bits
cancel: the difference is a whole number up to 255. The chosen experts' weights are 1 or 1/2. So partial sums in any
order are multiples of a power of two below 2^24 of it, which 32 bits hold, and the outputs have to be equal."""
import pytest

import mx4_plain as Q
from test_gpu_mx4_moe import BF, D, FL, HF, NAMES, Layer

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DIGITS = {FL: (24,), HF: (11, 11), BF: (8, 8, 8)}  # bits of an activation, and how many make an integer
CODE_OF_ONE, MINUS = 2, 8


class Exact:
    """Inputs of such a layer. `outputs` of a type of 16 bits are differences of neighbours, of 32 bits single values."""

    def __init__(self, tokens, experts, top_k, cols, inner, kind, out, seed):
        g = torch.Generator().manual_seed(seed)
        pick = lambda low, high, *shape: torch.randint(low, high, shape, generator=g)  # noqa: E731
        digits = DIGITS[kind]
        n, bits, blocks = len(digits), digits[0], cols // 32
        # digit d lies in the blocks whose number is d modulo n, the most significant one first; the first value is the gate
        places = [torch.tensor([c for c in range(1, cols) if c // 32 % n == d]) for d in range(n)]
        # values 2m and 2m + 1 of the last digit's places are near each other; all have their highest bit set
        x = pick(2 ** (bits - 1), 2**bits, tokens, cols).double()
        last = places[-1][: len(places[-1]) // 2 * 2]
        a = pick(2 ** (bits - 1), 2**bits - (256 if bits > 8 else 0), tokens, len(last) // 2).double()
        b = a + pick(1, 256, *a.shape) if bits > 8 else pick(2 ** (bits - 1), 2**bits, *a.shape).double()
        x[:, last[0::2]], x[:, last[1::2]] = a, b
        x = x * torch.where(pick(0, 2, tokens, 1) == 1, 1.0, -1.0)
        x[:, 0] = 32
        self.x = x.to(kind).to(D)
        assert torch.equal(self.x.double().cpu(), x)

        gate, up, down = (torch.zeros(experts, r, c, dtype=torch.uint8)
                          for r, c in ((inner, cols), (inner, cols), (cols, inner)))
        scales = [pick(100, 140, experts, r, c // 32).to(torch.uint8) for r, c in ((inner, cols), (inner, cols), (cols, inner))]
        gate[:, :, 0] = CODE_OF_ONE
        scales[0][:, :, 0] = 127
        # up: rows 2j and 2j + 1 share all but the last digit; an integer times 2^-24 (h: 2^-19)
        rows = torch.arange(inner)
        for e in range(experts):
            for d in range(n - 1):
                c = places[d][pick(0, len(places[d]), inner // 2)].repeat_interleave(2)
                up[e, rows, c] = CODE_OF_ONE
            m = pick(0, len(last) // 2, inner // 2)
            up[e, rows, torch.stack((last[2 * m], last[2 * m + 1]), 1).flatten()] = CODE_OF_ONE
        block = torch.arange(blocks)
        scales[1][:] = (127 - 24 + (n - 1 - block % n) * bits).to(torch.uint8)
        # down, of every top_k-th expert; the others' is zero
        rows = torch.arange(cols)
        power = pick(-8, 9, experts, cols, 1) if out == FL else torch.full((experts, cols, 1), 19)
        scales[2][:] = (127 + power).to(torch.uint8)
        sign = pick(0, 2, experts, cols).to(torch.uint8) * MINUS
        for e in range(0, experts, top_k):
            j = pick(0, inner // 2, cols)
            down[e, rows, 2 * j] = CODE_OF_ONE | sign[e]
            if out != FL:
                down[e, rows, 2 * j + 1] = CODE_OF_ONE | sign[e] ^ MINUS
        pack = lambda t: (t[..., 0::2] | t[..., 1::2] << 4).to(D)  # noqa: E731
        s = [t.to(D) for t in scales]
        self.layer = Layer(experts, top_k, cols, inner, g, FL, out)
        self.layer.w = dict(zip(NAMES, (pack(gate), s[0], pack(up), s[1], pack(down), s[2])))
        # one expert by the logits, another for each token as the activations' common size has no weight; several: all
        # logits zero, the first ones
        r = self.layer.router
        self.layer.router = torch.zeros_like(r) if top_k > 1 else r - r.mean(-1, keepdim=True)

    def check(self, **kw):
        out, experts, weights = self.layer(self.x, **kw)
        y, chosen, p, _ = self.layer.want(self.x)
        assert torch.equal(experts, chosen) and torch.equal(weights.double(), p)
        want = y.to(out.dtype)
        assert torch.equal(out, want), f"{(out != want).sum().item()} of {out.numel()} differ"
        assert (want != 0).double().mean() > 0.9  # few neighbours are alike


SIZES = [  # tokens, experts, top_k, cols, inner: each of the products' kernels, whole steps of rows and not
    (1, 3, 1, 96, 64), (1, 8, 2, 4096, 1440), (1, 128, 8, 2048, 768), (2, 5, 1, 2080, 96), (2, 9, 2, 96, 352),
    (3, 64, 4, 416, 96), (5, 3, 1, 352, 1056), (7, 11, 2, 1120, 1504), (16, 32, 4, 1024, 512), (40, 8, 1, 512, 2048),
    (17, 4, 1, 2304, 1280), (33, 4, 2, 3968, 2176), (64, 2, 1, 4224, 4224), (30, 3, 1, 2080, 3296), (64, 3, 1, 8160, 1056),
    (70, 2, 2, 288, 8192),
]


@pytest.mark.parametrize("kind", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("tokens,experts,top_k,cols,inner", SIZES)
def test_every_bit_counts_in_32_bits(tokens, experts, top_k, cols, inner, kind):
    Exact(tokens, experts, top_k, cols, inner, kind, FL, tokens * cols + inner).check()


@pytest.mark.parametrize("out", [BF, HF], ids=str)
@pytest.mark.parametrize("kind", [BF, FL], ids=str)
@pytest.mark.parametrize("tokens,experts,top_k,cols,inner", SIZES)
def test_every_bit_counts_in_16_bits(tokens, experts, top_k, cols, inner, kind, out):
    Exact(tokens, experts, top_k, cols, inner, kind, out, tokens * cols + inner + 1).check()
