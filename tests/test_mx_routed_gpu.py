"""Routed layers on microscaled experts: what a user of ``moe.run`` meets beside the parts that test_mx_experts_gpu holds."""

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib, synthetic
from tensorfold_b200.cuda import experts, moe, mx_experts
from tensorfold_b200.cuda.kernels import mx
from test_mx_experts_gpu import build, stored

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


def affine_layer(e=12, d=384, ni=128, k=3):
    dev = lambda i, n, kk: tuple(torch.stack([synthetic.affine_weight(n, kk, 4, 64, seed=100 * i + j)[t] for j in range(e)]).to(DEV) for t in range(3))
    ex = experts.make([dev(1, ni, d), dev(2, ni, d)], dev(3, d, ni), 64)
    return moe.Routed(layer_of(e=e, d=d, ni=ni, k=k).router, ex, k)


@pytest.mark.parametrize("kind", ["mx", "affine", "shared"])
@pytest.mark.parametrize("rows,prefill", [(5, False), (40, True)])
def test_layers_of_one_shape_run_side_by_side(kind, rows, prefill, monkeypatch):
    """A layer that is held up between its plan and its experts, while another of its shape runs from end to end on another stream or in
    a graph, still gets its own plan's pairs."""

    layer = affine_layer() if kind == "affine" else layer_of()
    if kind == "shared":
        ws = [stored(mx_util.random_weight(*shape, 40, DEV)) for shape in ((256, 384), (256, 384), (384, 256))]
        layer = moe.Routed(torch.cat([layer.router, layer.router[:1]]), layer.experts, 3, moe.SharedExpert(mx.pack_pair(*ws[:2]), mx.pack(ws[2][0], ws[2][1])))
    xs = [mx_util.rows(rows, 384, seed, DEV, std=0.5) for seed in (1, 2, 3)]
    want = [moe.run(x, layer, prefill=prefill) for x in xs]
    slow, quick = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for x in xs[1:]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = moe.run(x, layer, prefill=prefill)
        graphs.append((graph, out))
    select = moe.select

    def held_up(*args):
        select(*args)
        if torch.cuda.current_stream() == slow:
            torch.cuda._sleep(4_000_000)                       # about two milliseconds

    monkeypatch.setattr(moe, "select", held_up)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(slow):
            got = [moe.run(xs[0], layer, prefill=prefill)]
        with torch.cuda.stream(quick):
            got.append(moe.run(xs[1], layer, prefill=prefill))
            graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(graphs[1][1], want[2])
    slow_graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(slow_graph, stream=slow):
        out = moe.run(xs[0], layer, prefill=prefill)
    for _ in range(3):                                         # two graphs at once, eager calls beside them
        out.zero_(), graphs[0][1].zero_(), torch.cuda.synchronize()
        with torch.cuda.stream(slow):
            slow_graph.replay()
        with torch.cuda.stream(quick):
            graphs[0][0].replay()
            again = moe.run(xs[2], layer, prefill=prefill)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(graphs[0][1], want[1]) and torch.equal(again, want[2])
    assert _lib.device_error(xs[0]) == 0
