"""Views whose sign torch keeps as a flag beside the memory (the imaginary part of a conjugate) are refused: an operator
that reads the memory would take them with the other sign."""
import pytest

from ptwm_amd import api

torch = pytest.importorskip("torch")


def test_lazily_negated_views_are_refused():
    x = torch.ones(2, 64, dtype=torch.complex64).conj().imag.as_strided((2, 64), (128, 1))
    assert x.is_neg()
    plain, c, s = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    w, ws = torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(64, 2, dtype=torch.uint8)
    calls = [
        lambda: api.swiglu_mx_cuda(x, plain, c, s),
        lambda: api.rms_norm_mx_cuda(x, torch.ones(64), c, s),
        lambda: api.mxfp4_linear_cuda(x, w, ws, torch.zeros(2, 64)),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="negated"):
            call()
