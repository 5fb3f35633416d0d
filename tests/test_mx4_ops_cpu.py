"""CPU checks of the later MX operators' boundary (quantisation to MXFP4, product of two MXFP4 matrices,
mixture-of-experts layer): arguments are refused before any device is touched, and the tests' own formulas hold on
values worked by hand."""
import ctypes as C

import pytest

import mx4_plain as Q
import mx_plain as P
from ptwm_amd import _native, api

torch = pytest.importorskip("torch")

A = 1 << 20  # an address that no refused call reads


def quantise_args(**kw):
    a = dict(dtype=6, x=A, x_stride=64, codes=A, codes_stride=32, scales=A, scales_stride=2, rows=4, cols=64,
             saturate=1, stream=0, device=0)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


def matmul_args(**kw):
    a = dict(x=A, x_stride=32, x_scales=A, x_scales_stride=2, weight=A, weight_stride=32, scales=A, scales_stride=2,
             out_dtype=6, bias=0, out=A, out_stride=8, tokens=4, rows=8, cols=64, stream=0, device=0)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


def moe_call(**kw):
    inner, cols = kw.get("inner", 96), kw.get("cols", 64)
    c = _native.Mxfp4Moe(x=A, x_stride=cols, router=A, router_stride=cols, out=A, out_stride=cols, workspace=A,
                         workspace_bytes=1 << 40, tokens=4, experts=8, top_k=2, cols=cols, inner=inner, x_dtype=6,
                         router_dtype=1, out_dtype=4)
    for name, rows, n in (("gate", inner, cols), ("up", inner, cols), ("down", cols, inner)):
        setattr(c, name, _native.Experts(codes=A, codes_stride=n // 2, codes_expert=rows * n // 2, scales=A,
                                         scales_stride=n // 32, scales_expert=rows * n // 32))
    for name, v in kw.items():
        at, field = (getattr(c, name.split("__")[0]), name.split("__")[1]) if "__" in name else (c, name)
        setattr(at, field, v)
    return c


@pytest.mark.parametrize("rc,kw", [
    (-5, dict(dtype=29)), (-5, dict(dtype=0)), (-1, dict(cols=0)), (-1, dict(cols=48)), (-1, dict(x=0)),
    (-1, dict(codes=0)), (-1, dict(scales=0)), (-1, dict(x_stride=63)), (-1, dict(codes_stride=31)),
    (-1, dict(scales_stride=1)), (-1, dict(rows=1 << 31)), (-1, dict(cols=1 << 31)), (0, dict(rows=0)),
])
def test_quantise_refusals(rc, kw):
    assert _native.lib().ptwm_mi355x_mxfp4_quantise_cuda(*quantise_args(**kw)) == rc


@pytest.mark.parametrize("rc,kw", [
    (-5, dict(out_dtype=29)), (-5, dict(out_dtype=31)), (-1, dict(cols=0)), (-1, dict(cols=63)), (-1, dict(x=0)),
    (-1, dict(x_scales=0)), (-1, dict(weight=0)), (-1, dict(scales=0)), (-1, dict(out=0)), (-1, dict(x_stride=31)),
    (-1, dict(x_scales_stride=1)), (-1, dict(weight_stride=31)), (-1, dict(scales_stride=1)), (-1, dict(out_stride=7)),
    (-1, dict(tokens=1 << 31)), (-1, dict(rows=1 << 31)), (0, dict(tokens=0)), (0, dict(rows=0)),
])
def test_matmul_refusals(rc, kw):
    assert _native.lib().ptwm_mi355x_mxfp4_matmul_cuda(*matmul_args(**kw)) == rc


@pytest.mark.parametrize("rc,kw", [
    (-5, dict(x_dtype=29)), (-5, dict(router_dtype=13)), (-5, dict(out_dtype=31)), (-1, dict(reserved=1)),
    (-1, dict(cols=0)), (-1, dict(cols=48)), (-1, dict(inner=0)), (-1, dict(inner=40)), (-1, dict(cols=131104)),
    (-1, dict(inner=131104)), (-1, dict(experts=0)), (-1, dict(experts=1025)), (-1, dict(top_k=0)),
    (-1, dict(top_k=9)), (-1, dict(top_k=33, experts=64)), (-1, dict(tokens=1 << 31)), (-1, dict(x=0)),
    (-1, dict(router=0)), (-1, dict(out=0)), (-1, dict(x_stride=63)), (-1, dict(router_stride=63)),
    (-1, dict(out_stride=63)), (-1, dict(gate__codes=0)), (-1, dict(up__scales=0)), (-1, dict(down__codes=0)),
    (-1, dict(gate__codes_stride=31)), (-1, dict(up__scales_stride=1)), (-1, dict(down__codes_stride=47)),
    (-1, dict(down__scales_stride=2)), (-1, dict(workspace=0)), (-1, dict(workspace=A + 16)),
    (-1, dict(workspace_bytes=100)), (0, dict(tokens=0)),
])
def test_moe_refusals(rc, kw):
    assert _native.lib().ptwm_mi355x_mxfp4_moe_cuda(C.byref(moe_call(**kw)), 0, 0) == rc


def test_moe_workspace():
    L = _native.lib()
    need = lambda **kw: L.ptwm_mi355x_mxfp4_moe_workspace(C.byref(moe_call(**kw)))  # noqa: E731
    assert need() > 0 and need(tokens=1) <= need(tokens=64) == need(tokens=1000)
    assert need(workspace=0, workspace_bytes=0, x=0) == need()  # addresses are not looked at
    assert need(top_k=0) == -1 and need(x_dtype=2) == -5
    assert L.ptwm_mi355x_mxfp4_moe_workspace(None) == -1 and L.ptwm_mi355x_mxfp4_moe_cuda(None, 0, 0) == -1
    assert L.ptwm_mi355x_mxfp4_moe_cuda(C.byref(moe_call(workspace_bytes=need() - 1)), 0, 0) == -1


def test_tensors_of_the_host_are_refused():
    x, c, s = torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="not on a GPU"):
        api.mxfp4_quantise_cuda(x, c, s)
    with pytest.raises(ValueError, match="not on a GPU"):
        api.mxfp4_matmul_cuda(c, s, c, s, torch.zeros(2, 2))
    with pytest.raises(ValueError, match="not on a GPU"):
        api.mxfp4_moe_cuda(x, x, *[c.unsqueeze(0), s.unsqueeze(0)] * 3, x, 1)
    with pytest.raises(TypeError, match="missing argument 'scales'"):
        api.mxfp4_quantise_cuda(x, c)
    with pytest.raises(ValueError, match="blocks of 32"):
        api.mxfp4_quantise_cuda(x[:, :33], c, s)
    with pytest.raises(ValueError, match="blocks of 16"):
        api.mxfp4_matmul_cuda(c[:, :8], s, c[:, :8], s, torch.zeros(2, 2))


def test_plain_formulas_on_values_worked_by_hand():
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :14] = torch.tensor([7.0, 6.0, 5.0, -5.1, 3.5, 2.5, 1.75, 1.25, 0.75, -0.25, 0.26, -0.0, 4.9, 3.4])
    codes, scales = Q.quantise(x, True)
    assert scales.tolist() == [[127]]  # 7 is in [4, 8)
    got = torch.stack((codes & 15, codes >> 4), -1).reshape(-1)[:14].tolist()
    assert got == [7, 7, 6, 8 + 7, 6, 4, 4, 2, 2, 8, 1, 8, 6, 5]
    codes, scales = Q.quantise(x, False)
    assert scales.tolist() == [[128]]  # 7 is above 6
    assert P.weights(codes, scales)[0, :4].tolist() == [8.0, 6.0, 4.0, -6.0]  # 3.5 is nearer to 4 by the tie, 2.5 to 2
    assert Q.quantise(torch.zeros(1, 32), True)[1].item() == 0
    x[0, 20] = torch.nan
    codes, scales = Q.quantise(x, True)
    assert scales.item() == 255 and not codes.any()

    x = torch.tensor([[1.0] + [0.0] * 31])
    router = torch.zeros(3, 32)
    router[:, 0] = torch.tensor([0.0, 2.0, 2.0])
    logits, chosen, weights = Q.route(x, router, None, 2)
    assert chosen.tolist() == [[1, 2]] and weights.tolist() == [[0.5, 0.5]]
    assert Q.route(x, router, torch.tensor([0.0, -torch.inf, -torch.inf]), 2)[2].tolist() == [[1.0, 0.0]]
    one = torch.zeros(3, 32, 16, dtype=torch.uint8)
    one[:, 0, 0] = 2  # the first value of the first row is 1
    y, *_ = Q.moe(x, router, one, torch.full((3, 32, 1), 127, dtype=torch.uint8), one,
                  torch.full((3, 32, 1), 128, dtype=torch.uint8), one, torch.full((3, 32, 1), 127, dtype=torch.uint8), 2)
    assert abs(y[0, 0].item() - 2 / (1 + 2.718281828459045**-1)) < 1e-12 and not y[0, 1:].any()
