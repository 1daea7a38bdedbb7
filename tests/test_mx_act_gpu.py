"""Activations of the microscaled product where test_mx_gpu does not look: gates whose exponential is near the end of fp32, and
weights that run in several K slices."""

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib
from tensorfold_b200.cuda.kernels import mx

pytestmark = pytest.mark.gpu
DEV = "cuda"

HALF = {0.0: 0, 0.5: 1, 1.0: 2, 1.5: 3, 2.0: 4, 3.0: 5, 4.0: 6, 6.0: 7}


def coded(v):
    return HALF[abs(v)] | (8 if v < 0 else 0)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_gates_far_below_zero(m):
    """silu(g) of gates to -88.5 is a normal fp32 number, which ups of 2^100 make plain.  Sums are exact here, so what is left is expf (2
    units in the last place), the division and a product in fp32 (2^-20 in all covers them), and the rounding to bf16 (2^-8)."""

    gates = [(-4, -1.5, 0.5), (-4, -1.5, 0), (-4, -1.5, -0.5), (-4, -1, -6), (-4, -1.5, 2), (-1, -0.5, 1), (4, 1.5, 0), (0, 0, 0)]
    gc, gs = torch.zeros((16, 64), dtype=torch.long), torch.full((16, 2), 127)
    for r in range(16):
        for at, v in zip((0, 1, 32), gates[r % 8]):
            gc[r, at] = coded(v)
    gs[:, 0] += 4                                              # the first block's values are sixteen times as large
    uc, us = torch.zeros((16, 64), dtype=torch.long), torch.full((16, 2), 227)
    uc[:, 0] = coded(1.0)
    x = torch.zeros((m, 64), dtype=torch.bfloat16, device=DEV)
    x[:, 0] = x[:, 1] = x[:, 32] = 1
    pair = lambda c, s: (mx_util.to_words(c).to(DEV), s.to(torch.uint8).to(DEV))
    y = mx.matmul_act(x, mx.pack_pair(pair(gc, gs), pair(uc, us)))
    g = torch.tensor([16 * a + 16 * b + c for a, b, c in gates * 2], dtype=torch.double)
    assert g.min() == -88.5
    ref = (g / (1 + torch.exp(-g)) * 2.0 ** 100).to(DEV).expand(m, 16)
    assert ((y.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -20) * ref.abs()).all()
    assert _lib.device_error(x) == 0
