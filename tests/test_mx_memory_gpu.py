"""Microscaled calls whose tensors share memory."""

import pytest
import torch

import mx_util
from tensorfold_b200.cuda import mx_experts
from tensorfold_b200.cuda.kernels import mx
from test_mx_experts_gpu import build, picks_for, plan_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def weight(n, k, seed=3):
    codes, scales = mx_util.random_weight(n, k, seed, DEV)
    return mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))


@pytest.mark.parametrize("m", [1, 5, 200])
def test_out_over_x_is_refused(m):
    q = weight(256, 256)
    flat = torch.zeros((m + 2) * 256 * 4, dtype=torch.bfloat16, device=DEV)
    x = flat[:m * 256].view(m, 256)
    x.copy_(mx_util.rows(m, 256, 1, DEV))
    want = mx.matmul(x, q)
    wide = torch.zeros((m, 1024), dtype=torch.bfloat16, device=DEV)
    side = wide[:, 256:512]
    side.copy_(x)
    for given, out in ((x, x), (x, flat[8:8 + m * 256].view(m, 256)), (x, flat[m * 256 - 8:2 * m * 256 - 8].view(m, 256)),
                       (side, wide[:, 248:504]), (side, wide[:, 504:760]), (side, side)):
        with pytest.raises(ValueError, match="shares memory"):
            mx.matmul(given, q, out=out)
        with pytest.raises(ValueError, match="shares memory"):
            mx.matmul_act(given, q, act="relu2", out=out)
    assert torch.equal(x, mx_util.rows(m, 256, 1, DEV)) and torch.equal(side, x)        # nothing was launched
    for given, out in ((x, flat[m * 256:2 * m * 256].view(m, 256)), (side, wide[:, :256]), (side, wide[:, 512:768])):
        assert torch.equal(mx.matmul(given, q, out=out), want)
    if m > 1:                                                  # rows of one pitch that begin elsewhere in the buffer
        shifted = lambda at: wide.view(-1)[at:at + 1024 * (m - 1)].view(m - 1, 1024)[:, :256]
        assert torch.equal(mx.matmul(side[:-1], q, out=shifted(600)), want[:-1])
        for given, out in ((side[:-1], shifted(1000 - 640)), (wide[:-1, :256], shifted(900))):
            with pytest.raises(ValueError, match="shares memory"):
                mx.matmul(given, q, out=out)
        if m > 2:
            with pytest.raises(ValueError, match="shares memory"):
                mx.matmul(side[:-2], q, out=wide[1:-1, 256:512])


@pytest.mark.parametrize("prefill", [False, True])
def test_experts_out_over_x_is_refused(prefill):
    ex, _, _ = build((6, 128, 128, True, 0.0), 3)
    rows, slots = 20, 2
    picks = picks_for(rows, slots, 6, 1)
    plan = plan_of(picks, 6, prefill)
    x = torch.zeros((rows * slots, 128), dtype=torch.bfloat16, device=DEV)
    x[:rows] = mx_util.rows(rows, 128, 2, DEV, std=0.5)
    act = torch.empty_like(x)
    mx_experts.gate_up(x, ex, plan, act, rows)
    for call in (lambda: mx_experts.gate_up(x, ex, plan, x, rows), lambda: mx_experts.down(act, ex, plan, act, rows)):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    want = torch.empty_like(x)
    mx_experts.layer(x, ex, plan, want, rows)
    mx_experts.layer(x, ex, plan, x, rows)                     # reads all of x first
    assert torch.equal(x, want)
