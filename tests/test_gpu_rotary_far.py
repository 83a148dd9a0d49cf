"""Rotary positions far out: the sine and cosine against 50 digits, within what cvcuda/Rotary.h says of them."""
import importlib
import math
from decimal import Decimal, getcontext

import pytest
import torch

pytestmark = pytest.mark.gpu
getcontext().prec = 60
TURN = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494")


@pytest.mark.parametrize("base", [10000.0, 500000.0, 2.0, 7.0])
@pytest.mark.parametrize("dims", [64, 128, 256])
def test_angles_of_far_positions(cv, gpu, dims, base):
    api = importlib.import_module("cvcuda_amd.pyapi")
    positions = [0, 1, 12345, 1 << 20, (1 << 24) + 3, 1 << 28, (1 << 31) - 1]
    x = torch.zeros((len(positions), 1, dims), device="cuda")
    x[..., :dims // 2] = 1                                       # (cosine, sine)
    out = torch.empty_like(x)
    api.rotary_into(api.as_tensor(out, "TWE"), api.as_tensor(x, "TWE"), api.as_tensor(torch.tensor(positions, device="cuda")), base=base)
    out = out.double().cpu()
    for i in range(dims // 2):
        f = (Decimal(base).ln() * (Decimal(-2 * i) / Decimal(dims))).exp()
        for n, position in enumerate(positions):
            angle = float((Decimal(position) * f) % TURN)
            # (the sine's and cosine's polynomials and reduction: 8 roundings)
            bound = 8 * 2.0 ** -24 + position * 2.0 ** -52
            assert abs(out[n, 0, i] - math.cos(angle)) <= bound, (position, i)
            assert abs(out[n, 0, dims // 2 + i] - math.sin(angle)) <= bound, (position, i)
