"""diffphycon_amd.sequence where a call is allowed but unusual, against the definitions in 64 bits (tests/sequence_oracle.py)."""
import math

import pytest
import torch

import sequence_oracle as O
from test_gpu_sequence import TYPES, _check_attention, _gen, _randn, _within, dev  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("C", [8, 32, 128, 512, 2048, 16384, 32768])
@pytest.mark.parametrize("pad", [0, 1])
def test_layer_norm_gradient_of_a_far_constant_row(C, pad, t, dev):
    """Rows of 2^100: x - mean is 0, while mean / sqrt(eps) is beyond fp32's range; lanes past the row's end must not bring that in.  With xh = 0 the
    gradient is rstd (g - mean(g)), off by a sum of C terms and a few operations."""
    from diffphycon_amd import sequence as S
    g = _gen(C)
    x = torch.full((5, C + pad), 2.0 ** 100, dtype=t, device=dev)[:, :C]
    dy, w = _randn(g, 5, C, dtype=t), _randn(g, C, dtype=t, shift=1.0)
    y, st = S.layer_norm_forward(x, w, eps=1e-20)
    assert not y.any()
    dx, dw, db = S.layer_norm_backward(dy, x, st, w)
    z = dy.double() * w.double()
    rstd, mean, size = 1e-20 ** -0.5, z.mean(1, keepdim=True), z.abs().mean(1, keepdim=True)
    value = rstd * (z - mean)
    _within("dx", dx, value, O.add_rounding(value, rstd * O.E * (6 * z.abs() + (C + 10) * size), t))
    assert not dw.any()
    _within("db", db, dy.double().sum(0), O.add_rounding(dy.double().sum(0), 9 * O.E * dy.double().abs().sum(0), t))
