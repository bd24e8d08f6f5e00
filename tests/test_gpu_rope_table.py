"""The frequencies that spinn_hip_rope_table lays out, against 80 decimal digits: angles are exact to 2^-32 of a turn at any position."""
import ctypes as C
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch

from tests.decodeops import F32
from tests.test_gpu_rope import desc, run, table

pytestmark = pytest.mark.gpu

getcontext().prec = 80
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798214808651")


def turns(d):
    """Turns a position of each pair, by the definition, of the descriptor's own numbers."""
    base, factor, low, high = (Decimal(float(v)) for v in (d.base, d.factor, d.low, d.high))
    out = []
    for i in range(d.rot_dim // 2):
        f = (base.ln() * -2 * i / d.rot_dim).exp() / (2 * PI)
        if d.scaling == 1:
            f /= factor
        elif d.scaling == 2:
            t = min(max((d.trained * f - low) / (high - low), Decimal(0)), Decimal(1))
            f = t * f + (1 - t) * f / factor
        out.append(f)
    return out


@pytest.mark.parametrize("scaling", ["plain", "linear", "parts"])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1.0, 0.5, 0.01, 1e-9, 1e30])
@pytest.mark.parametrize("rot", [2, 6, 64, 128, 510, 512])
def test_frequencies(hip, scaling, base, rot):
    """A position of up to 2^31 multiplies an entry's error of 2^-63 to 2^-32."""
    d = desc(hip, F32, 1, rot, rot, False, scaling, base)
    if scaling != "plain":
        d.factor = 3.7
    got = table(hip, d).cpu().numpy().view(np.uint64).tolist()
    for i, (a, f) in enumerate(zip(got, turns(d))):
        far = (Decimal(a) - f % 1 * 2 ** 64) % 2 ** 64
        assert min(far, 2 ** 64 - far) <= 2, (i, float(min(far, 2 ** 64 - far)))


@pytest.mark.parametrize("base", [10000.0, 0.01])
def test_the_farthest_positions(hip, base):
    """(cos, sin) of the angles themselves. 2^-32 of a turn is 2^-29; sines and cosines of a quarter turn in fp32 are off by 2^-21 at most."""
    far = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 12345, 2 ** 27 + 1]
    d = desc(hip, F32, 1, 64, 64, True, base=base, strides=(64, 64, 64, 64))
    x = torch.tensor([1.0, 0.0], device="cuda").repeat(len(far), 32)
    y = torch.zeros_like(x)
    run(hip, d, torch.tensor(far, dtype=torch.int32, device="cuda"), table(hip, d), x, y)
    for t, p in enumerate(far):
        angle = np.array([float(p * f % 1) for f in turns(d)]) * 2 * np.pi
        got = y[t].cpu().double().numpy()
        assert np.abs(got[0::2] - np.cos(angle)).max() <= 2.0 ** -21
        assert np.abs(got[1::2] - np.sin(angle)).max() <= 2.0 ** -21
