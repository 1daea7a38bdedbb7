"""Routed layers on microscaled experts: what a user of ``moe.run`` meets beside the parts that test_mx_experts_gpu holds."""

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib
from tensorfold_b200.cuda import moe, mx_experts
from test_mx_experts_gpu import build

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layer_of(seed=9, e=12, d=384, ni=128, k=3):
    """Experts whose last one is the shared expert, and a router over the others."""

    ex, _, _ = build((e, d, ni, True, 0.0), seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    router = (torch.randn((e, d), generator=g, device=DEV) * d ** -0.5).to(torch.bfloat16)
    return moe.Routed(router, ex, k)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_prompt_pairs_stay_unrounded(rows):
    """With f32 a prompt's layer rounds once: |out - sum w y| <= 2^-8 |sum w y| (half a step of bf16) + (slots + 1) 2^-24 sum |w y| (fp32
    fma chain over the slots), y being each pair's fp32 result."""

    layer = layer_of()
    x = mx_util.rows(rows, 384, 5, DEV, std=0.5)
    got = moe.run(x, layer, prefill=True, f32=True)
    buf = moe.MoEBuffers(rows, moe._Shape(layer), DEV, prefill=True, table_experts=12, f32=True)
    assert buf.y.dtype == torch.float32
    moe.select(moe.router(x, layer.router, prefill=True), buf, 3, 11)
    y = torch.zeros((rows, 4, 384), device=DEV)
    mx_experts.layer(x, layer.experts, buf.plan, y.view(-1, 384), rows)
    terms = y.double() * buf.wts.double()[..., None]
    ref = terms.sum(1)
    bound = 2.0 ** -8 * ref.abs() + 5 * 2.0 ** -24 * terms.abs().sum(1) + 2.0 ** -126
    assert ((got.double() - ref).abs() <= bound).all()
    assert torch.equal(got, moe.combine(y, buf.wts)) and torch.equal(moe.run(x[:1], layer, prefill=True, f32=True), got[:1])
    assert _lib.device_error(x) == 0
