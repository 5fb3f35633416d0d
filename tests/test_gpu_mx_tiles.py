"""The product with MXFP4 weights in each of its kernels over several steps of a row: output types, with a bias and
without, operands at any place and stride, values at the ends of the types' ranges, infinities and NaN.  Sizes and the
kernels that they reach are in mx_sizes.py, which test_mx_choice_cpu.py holds against the library's rules."""
import pytest

import mx_plain as P
import mx_sizes as S
from ptwm_amd import api

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = "cuda:0"
F8 = torch.float8_e4m3fn
KINDS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": F8}
OUTS = [torch.bfloat16, torch.float16, torch.float32]
CASES = [pytest.param(kind, *size, id=f"{kind}-{'x'.join(map(str, size))}") for kind in KINDS for size in S.SIZES[kind]]


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def inputs(kind, tokens, rows, cols, g):
    codes, scales = P.random_weights(rows, cols, g, D)
    if kind == "e4m3":
        return (*P.random_blocks(tokens, cols, g, D), codes, scales)
    loud = torch.where(torch.rand(cols, generator=g) < 0.05, 20.0, 1.0)
    return (torch.randn(tokens, cols, generator=g) * loud).to(KINDS[kind]).to(D), None, codes, scales


def bytes_of(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def apart(t, pad, shift):
    """The same matrix with `pad` elements between rows, `shift` elements in, and the buffer that it lies in."""
    rows, cols = t.shape
    big = torch.full((rows * (cols + pad) + shift,), 85, dtype=bytes_of(t).dtype, device=D)
    v = big[shift:].view(rows, cols + pad)[:, :cols]
    v.copy_(bytes_of(t))
    return v.view(t.dtype), big


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("out", OUTS, ids=str)
@pytest.mark.parametrize("kind,tokens,rows,cols", CASES)
def test_types_places_and_strides(kind, tokens, rows, cols, out):
    g = gen(tokens, rows, cols)
    x, xs, codes, scales = inputs(kind, tokens, rows, cols, g)
    if out == torch.float16:  # into the type's range
        scales -= 12
    for bias in (None, torch.randn(rows, generator=g).to(out).to(D)):
        o = torch.full((tokens, rows), float("nan"), dtype=out, device=D)
        api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs, bias=bias)
        P.check_linear(o, x, xs, codes, scales, bias)
        # rows and places that loads of 16 bytes fit, and that they do not; what lies between rows of the output stays
        for pads, shifts in (((32, 16), (16, 48)), ((3, 5), (1, 3)), ((9, 16), (5, 1))):
            (px, _), (pw, _), (ps, _) = apart(x, pads[0], shifts[0]), apart(codes, pads[1], shifts[1]), apart(scales, 1, 1)
            pxs = None if xs is None else apart(xs, 3, 1)[0]
            po, buffer = apart(o, pads[0], shifts[1])
            want = buffer.clone()
            po.fill_(float("nan"))
            api.mxfp4_linear_cuda(px, pw, ps, po, 0, x_scales=pxs, bias=bias)
            assert same(buffer, want), (pads, shifts)


def half_weights(codes, value):
    """Makes every row's weight `value` +-0.5 times its scale, rows in turn."""
    code = torch.where(torch.arange(codes.shape[0], device=D) % 2 == 0, 1, 9).to(torch.uint8)
    at = value // 2
    codes[:, at] = (codes[:, at] & 0xF0 | code) if value % 2 == 0 else (codes[:, at] & 0x0F | code << 4)


@pytest.mark.parametrize("kind,tokens,rows,cols", CASES)
def test_infinities_and_nan(kind, tokens, rows, cols):
    """They reach every output of their token and no other one's; a row's NaN scale reaches that row alone."""
    x, xs, codes, scales = inputs(kind, tokens, rows, cols, gen(tokens, rows, cols, 1))
    last = cols - 27
    half_weights(codes, last)
    clean = torch.empty(tokens, rows, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, clean, 0, x_scales=xs)
    P.check_linear(clean, x, xs, codes, scales)
    o = torch.empty_like(clean)
    ends = torch.where(torch.arange(rows, device=D) % 2 == 0, 1.0, -1.0) * float("inf")
    broken = x.clone()
    t = tokens - 1  # the last token; the first one where there are more
    if kind == "e4m3":
        broken.view(torch.uint8)[t, last] = 0x7F
        if t:
            xs.view(torch.uint8)[0, 1] = 255
    else:
        broken[t, last] = float("inf")
        if t:
            broken[0, 37] = float("nan")
    api.mxfp4_linear_cuda(broken, codes, scales, o, 0, x_scales=xs)
    assert torch.isnan(o[t]).all() if kind == "e4m3" else torch.equal(o[t], ends)
    if t:
        assert torch.isnan(o[0]).all() and torch.equal(o[1:t], clean[1:t])
    # a NaN scale in the row's first step and in its last one
    x, xs, codes, scales = inputs(kind, tokens, rows, cols, gen(tokens, rows, cols, 1))
    r = rows - 2
    scales[r, cols // 32 - 1] = 255
    scales[7, 2] = 255
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    assert torch.isnan(o[:, r]).all() and torch.isnan(o[:, 7]).all()
    keep = torch.ones(rows, dtype=torch.bool, device=D)
    keep[[r, 7]] = False
    P.check_linear(o[:, keep], x, xs, codes[keep], scales[keep])


@pytest.mark.parametrize("kind,tokens,rows,cols", CASES)
def test_ends_of_the_ranges(kind, tokens, rows, cols):
    """Weights from 2^-128 on; activations up to the type's largest value."""
    g = gen(tokens, rows, cols, 2)
    x, xs, codes, _ = inputs(kind, tokens, rows, cols, g)
    scales = torch.randint(0, 20, (rows, cols // 32), generator=g, dtype=torch.uint8).to(D)
    if kind == "e4m3":
        xs.view(torch.uint8).add_(60)
    else:
        x = (x.float() * 1e4).clamp(-6e4, 6e4).to(x.dtype)
    o = torch.empty(tokens, rows, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    v = P.blocks(x, xs) if xs is not None else x.double()
    w = P.weights(codes, scales)
    # a sum of numbers below 2^-126 may lose, with each product, what lies under the smallest normal number
    room = (cols / 32 + 128) * 2.0**-23 * (v.abs() @ w.abs().t()) + cols * 2.0**-126
    assert ((o.double() - v @ w.t()).abs() <= room).all()
    if kind != "e4m3":
        x = torch.full_like(x, torch.finfo(x.dtype).max) * torch.where(torch.arange(cols, device=D) % 3 == 0, -1, 1)
        # cols products of 2^128 and a weight stay finite with weights up to 6 * 2^-16
        scales = torch.randint(100, 112, (rows, cols // 32), generator=g, dtype=torch.uint8).to(D)
        api.mxfp4_linear_cuda(x.to(KINDS[kind]), codes, scales, o)
        P.check_linear(o, x.to(KINDS[kind]), None, codes, scales)


@pytest.mark.parametrize("kind", KINDS)
def test_streams_and_graph_replays(kind):
    calls = []
    for tokens, rows, cols in S.SIZES[kind]:
        x, xs, codes, scales = inputs(kind, tokens, rows, cols, gen(tokens, rows, cols, 3))
        calls.append((x, codes, scales, torch.empty(tokens, rows, device=D, dtype=torch.bfloat16), xs))

    def step():
        for x, codes, scales, o, xs in calls:
            api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)

    def turn():  # the weights of the other sign, outputs cleared
        for _, codes, _, o, _ in calls:
            codes ^= 0x88
            o.zero_()

    results = lambda: [c[3].clone() for c in calls]  # noqa: E731
    step()
    first = results()
    turn()
    step()
    second = results()
    turn()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # what comes next must wait for this
        turn()
        step()
        moved = results()
    side.synchronize()
    assert all(map(torch.equal, moved, second)) and not any(map(torch.equal, moved, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        turn()
        graph.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, results(), first if k % 2 == 0 else second)), k


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,rows", [(1, 131), (1, 9001), (3, 131), (20, 131)])
def test_last_tokens_of_sequences(kind, tokens, rows):
    """hidden[:, -1] of [tokens, 2048, 4096], rows 2^23 elements apart: the same kernel and bits as packed rows."""
    x, xs, codes, scales = inputs(kind, tokens, rows, 4096, gen(tokens, rows, 4))
    hidden = torch.zeros(tokens, 2048, 4096, dtype=bytes_of(x).dtype, device=D)
    hidden[:, -1] = bytes_of(x)
    last = hidden.view(x.dtype)[:, -1]
    assert last.stride(0) == 2048 * 4096
    o, p = torch.empty(tokens, rows, device=D), torch.empty(tokens, rows, device=D)
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    P.check_linear(o, x, xs, codes, scales)
    api.mxfp4_linear_cuda(last, codes, scales, p, 0, x_scales=xs)
    assert torch.equal(o, p)


@pytest.mark.parametrize("kind,operand", [(k, o) for k in KINDS for o in S.FAR_COUNTS if o != "x_scales" or k == "e4m3"])
def test_strides_about_the_reach_of_a_tile(kind, operand):
    x, xs, codes, scales = inputs(kind, *S.FAR, gen(5))
    o, p = (torch.empty(S.FAR[:2], device=D) for _ in range(2))
    api.mxfp4_linear_cuda(x, codes, scales, o, 0, x_scales=xs)
    P.check_linear(o, x, xs, codes, scales)
    all_ = {"x": x, "weight": codes, "scales": scales, "x_scales": xs}
    t = all_[operand]
    stride = S.far_stride(operand, t.element_size())
    for beyond in (0, 1):
        big = torch.empty((t.shape[0] - 1) * (stride + beyond) + t.shape[1], dtype=bytes_of(t).dtype, device=D)
        v = big.as_strided(t.shape, (stride + beyond, 1))
        v.copy_(bytes_of(t))
        call = {**all_, operand: v.view(t.dtype)}
        api.mxfp4_linear_cuda(call["x"], call["weight"], call["scales"], p, 0, x_scales=call["x_scales"])
        del big, v, call
        if beyond:
            P.check_linear(p, x, xs, codes, scales)
        else:
            assert torch.equal(o, p)
    torch.cuda.empty_cache()
