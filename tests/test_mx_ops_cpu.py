"""CPU checks of the MX operators' boundary: arguments are refused before any
device is touched, and the tests' own formulas hold on values worked by hand."""
import pytest

import mx_plain as P
from ptwm_amd import _native, api

torch = pytest.importorskip("torch")

A = 1 << 20  # an address that no refused call reads


def norm_args(**kw):
    a = dict(dtype=6, x=A, x_stride=64, residual=0, residual_stride=0, weight_dtype=6, weight=A, eps=1e-6, sum=0,
             sum_stride=0, codes=A, codes_stride=64, scales=A, scales_stride=2, rows=4, cols=64, stream=0, device=0)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


def swiglu_args(**kw):
    a = dict(dtype=6, gate=A, gate_stride=64, up=A, up_stride=64, codes=A, codes_stride=64, scales=A,
             scales_stride=2, rows=4, cols=64, stream=0, device=0)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


def linear_args(**kw):
    a = dict(x_dtype=6, x=A, x_stride=64, x_scales=0, x_scales_stride=0, weight=A, weight_stride=32, scales=A,
             scales_stride=2, out_dtype=6, bias=0, out=A, out_stride=8, tokens=4, rows=8, cols=64, stream=0, device=0)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("rc,kw", [
    (-5, dict(dtype=29)), (-5, dict(dtype=13)), (-5, dict(weight_dtype=22)), (-1, dict(cols=0)), (-1, dict(cols=48)),
    (-1, dict(x=0)), (-1, dict(weight=0)), (-1, dict(codes=0)), (-1, dict(scales=0)), (-1, dict(x_stride=63)),
    (-1, dict(residual=A, residual_stride=32)), (-1, dict(sum=A, sum_stride=32)), (-1, dict(codes_stride=63)),
    (-1, dict(scales_stride=1)), (-1, dict(rows=1 << 31)), (-1, dict(cols=1 << 31)), (0, dict(rows=0)),
])
def test_norm_refusals(rc, kw):
    assert _native.lib().ptwm_mi355x_rms_norm_mx_cuda(*norm_args(**kw)) == rc


@pytest.mark.parametrize("rc,kw", [
    (-5, dict(dtype=29)), (-5, dict(dtype=0)), (-1, dict(cols=0)), (-1, dict(cols=33)), (-1, dict(gate=0)),
    (-1, dict(up=0)), (-1, dict(codes=0)), (-1, dict(scales=0)), (-1, dict(gate_stride=0)), (-1, dict(up_stride=63)),
    (-1, dict(codes_stride=1)), (-1, dict(scales_stride=1)), (-1, dict(rows=1 << 40)), (0, dict(rows=0)),
])
def test_swiglu_refusals(rc, kw):
    assert _native.lib().ptwm_mi355x_swiglu_mx_cuda(*swiglu_args(**kw)) == rc


@pytest.mark.parametrize("rc,kw", [
    (-5, dict(x_dtype=30)), (-5, dict(x_dtype=31)), (-5, dict(out_dtype=29)), (-1, dict(cols=0)), (-1, dict(cols=63)),
    (-1, dict(x=0)), (-1, dict(weight=0)), (-1, dict(scales=0)), (-1, dict(out=0)), (-1, dict(x_stride=63)),
    (-1, dict(weight_stride=31)), (-1, dict(scales_stride=1)), (-1, dict(out_stride=7)),
    (-1, dict(x_dtype=29)),                                     # 8-bit activations without scales
    (-1, dict(x_scales=A, x_scales_stride=2)),                  # scales without 8-bit activations
    (-1, dict(x_dtype=29, x_scales=A, x_scales_stride=1)), (-1, dict(tokens=1 << 31)), (-1, dict(rows=1 << 31)),
    (0, dict(tokens=0)), (0, dict(rows=0)),
])
def test_linear_refusals(rc, kw):
    assert _native.lib().ptwm_mi355x_mxfp4_linear_cuda(*linear_args(**kw)) == rc


def test_tensors_of_the_host_are_refused():
    x, c, s = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="not on a GPU"):
        api.rms_norm_mx_cuda(x, torch.ones(64), c, s)
    with pytest.raises(ValueError, match="not on a GPU"):
        api.swiglu_mx_cuda(x, x, c, s)
    with pytest.raises(ValueError, match="not on a GPU"):
        api.mxfp4_linear_cuda(x, torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8),
                              torch.zeros(2, 8))
    with pytest.raises(TypeError):
        api.swiglu_mx_cuda(c, c, c, s)
    with pytest.raises(ValueError, match="blocks of 32"):
        api.swiglu_mx_cuda(x[:, :33], x[:, :33], c, s)


def test_plain_formulas_on_values_worked_by_hand():
    codes = torch.zeros(1, 16, dtype=torch.uint8)
    codes[0, 0], codes[0, 1] = 0x72, 0xF9          # 1, 6; -0.5, -6
    scales = torch.tensor([[128]], dtype=torch.uint8)
    assert P.weights(codes, scales)[0, :4].tolist() == [2.0, 12.0, -1.0, -12.0]
    y = torch.zeros(1, 32, dtype=torch.float64)
    y[0, 0] = 448.0
    good = torch.zeros(1, 32, dtype=torch.uint8)
    good[0, 0] = 0x7E
    P.check_codes(good, torch.tensor([[127]], dtype=torch.uint8), y, 0.0)
    with pytest.raises(AssertionError, match="larger than needed"):
        P.check_codes(good, torch.tensor([[128]], dtype=torch.uint8), y, 0.0)
    with pytest.raises(AssertionError, match="does not reach"):
        P.check_codes(good, torch.tensor([[126]], dtype=torch.uint8), y, 0.0)
    y[0, 1] = 100.0                                # a code that is missing
    with pytest.raises(AssertionError, match="more than allowed"):
        P.check_codes(good, torch.tensor([[127]], dtype=torch.uint8), y, 0.0)
