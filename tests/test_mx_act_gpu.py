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


# (n, k): columns of both projections, inputs; K slices 2, 4, 6 and 3
SLICED = [(256, 1024), (4096, 2048), (1024, 2720), (5120, 1536)]


def pair_of(n, k, seed):
    return [mx_util.random_weight(n // 2, k, seed + i, DEV) for i in range(2)]


def pack_pair(pair):
    return mx.pack_pair(*[(mx_util.to_words(c), s.to(torch.uint8)) for c, s in pair])


@pytest.mark.parametrize("n,k", SLICED)
@pytest.mark.parametrize("act,limit", [("swiglu", 0.0), ("swiglu", 1.5), ("relu2", 0.0)])
def test_activations_of_sliced_weights(n, k, act, limit):
    """test_mx_gpu.test_matmul_act's bound, with the additions of the slices (6 at most) beside the k others; every row count's rows
    are those of one row."""

    assert _lib.lib().tf_mx_split(n, k) in (2, 3, 4, 6)
    pair = pair_of(n, k, 1)
    x = mx_util.rows(200, k, 3, DEV, std=0.3)
    e = (k + 6) * 2.0 ** -23
    if act == "swiglu":
        q = pack_pair(pair)
        (g, gt), (u, ut) = (mx_util.sums(x, *w) for w in pair)
        if limit:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        ref = g * torch.sigmoid(g) * u
        slack = e * gt * 1.1 * u.abs() + e * ut * (1.1 * g.abs() + 0.3)
    else:
        whole = [torch.cat([w[i] for w in pair]) for i in range(2)]
        q = mx.pack(mx_util.to_words(whole[0]), whole[1].to(torch.uint8))
        v, t = mx_util.sums(x, *whole)
        ref, slack = v.clamp(min=0) ** 2, e * t * 2 * (v.abs() + e * t)
    bound = (2.0 ** -8 + 2.0 ** -20) * ref.abs() + slack * 1.01 + 2.0 ** -126
    y = mx.matmul_act(x, q, act=act, limit=limit)
    assert ((y.double() - ref).abs() <= bound).all()
    for m in (1, 3, 13, 16, 17, 40, 64, 129):
        assert torch.equal(mx.matmul_act(x[:m], q, act=act, limit=limit), y[:m]), m
    assert torch.equal(mx.matmul_act(x[77:78], q, act=act, limit=limit), y[77:78]) and _lib.device_error(x) == 0


@pytest.mark.parametrize("n,k", SLICED)
@pytest.mark.parametrize("m", [1, 13, 40, 200])
def test_bad_blocks_of_sliced_weights(n, k, m):
    codes, scales = mx_util.random_weight(n, k, 4, DEV)
    scales[17, 5] = 255
    q = mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))
    x = mx_util.rows(m, k, 8, DEV)
    clean = mx.matmul(x, q)
    assert torch.isnan(clean[:, 17]).all() and torch.isfinite(clean[:, :17]).all() and torch.isfinite(clean[:, 18:]).all()
    x[m // 2, k - 1] = float("inf")                            # the last slice's last block
    y, keep = mx.matmul(x, q), torch.arange(m, device=DEV) != m // 2
    assert torch.isnan(y[m // 2]).all() and torch.equal(y[keep].nan_to_num(0.5), clean[keep].nan_to_num(0.5))
    act = mx.matmul_act(x, q, limit=1.0)                       # column 17 is an up
    assert torch.isnan(act[m // 2]).all() and torch.isnan(act[:, 1]).all()
    assert torch.isfinite(act[keep][:, 2:]).all() and torch.isfinite(act[keep][:, :1]).all()


@pytest.mark.parametrize("n,k", [(264, 1024), (1000, 2720), (4090, 2048)])
@pytest.mark.parametrize("m", [1, 5, 13, 40, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs_of_sliced_weights(n, k, m, dtype):
    """Columns that are no multiple of a block, outputs off their 16-byte boundaries; what lies beside them stays as it was."""

    assert _lib.lib().tf_mx_split(n, k) > 1
    codes, scales = mx_util.random_weight(n, k, 6, DEV)
    q = mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))
    x = mx_util.rows(m, k, 3, DEV)
    f32 = dtype == torch.float32
    want = mx.matmul(x, q, f32=f32)
    mx_util.assert_product(want, *mx_util.sums(x, codes, scales), k + 6)
    for left in (4, 8, 3):
        out = torch.full((m + 2, n + 16), 7.0, dtype=dtype, device=DEV)
        mx.matmul(x, q, f32=f32, out=out[1:m + 1, left:n + left])
        assert torch.equal(out[1:m + 1, left:n + left], want)
        out[1:m + 1, left:n + left] = 7
        assert (out == 7).all()
