"""spinn_hip_linear_i8 of few rows into very many columns, as a vocabulary's layer has."""
import pytest
import torch

from tests.decodeops import BF16, F32, NAMES, HALF_STEP, assert_close, gen, randn
from tests.test_gpu_linear_i8 import ints, layer, padded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 16, 17, 64, 65, 128, 129])
@pytest.mark.parametrize("n,k", [(32769, 200), (40000, 64), (100003, 130)])
def test_exact_sums(hip, m, n, k):
    g = gen(m + n)
    x, w = ints(g, m, k), ints(g, n, k)
    one = torch.ones(n, device="cuda")
    y = layer(hip, padded(x), one[:m], w.cuda(), one, F32, k=k)
    assert torch.equal(y, (x.cuda().double() @ w.cuda().double().t().contiguous()).float())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m", [3, 40, 100])
def test_scales_bias_and_residual(hip, dtype, m):
    """The sum's conversion, two scales, bias and residual are five roundings of 2^-24 of the magnitudes' sum; then the result's."""
    n, k = 50001, 96
    g = gen(m)
    x, w = ints(g, m, k), ints(g, n, k)
    sx, sw = torch.rand(m, generator=g) + 0.5, (torch.rand(n, generator=g) + 0.5) / 50000
    bias, res = randn(g, n, dtype=dtype), randn(g, m, n, dtype=dtype)
    y = layer(hip, padded(x), sx.cuda(), w.cuda(), sw.cuda(), dtype, bias=bias.cuda(), res=res.cuda(), k=k)
    v = (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()
    off = 5 * 2.0 ** -24 * (v.abs() + bias.double().abs() + res.double().abs())
    ref = v + bias.double() + res.double()
    assert_close(y, ref, off + HALF_STEP[dtype] * (ref.abs() + off) + 1e-37, f"wide {m}")
