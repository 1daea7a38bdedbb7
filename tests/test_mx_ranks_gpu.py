"""Microscaled weights in the rank containers: each rank's share in turn on one GPU."""

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib
from tensorfold_b200.cuda import checkpoint, moe, mx_experts, tp
from test_mx_experts_gpu import build, stored

pytestmark = pytest.mark.gpu
DEV = "cuda"


def saved(tmp_path, tensors):
    from test_checkpoint import write_safetensors

    path = tmp_path / "model.safetensors"
    write_safetensors(path, tensors, pad=1)
    return checkpoint.Checkpoint([path])


@pytest.mark.parametrize("rows", [1, 13, 70])
@pytest.mark.parametrize("world", [2, 4])
def test_row_and_column_parallel(tmp_path, rows, world):
    """Row-parallel partials added in rank order in fp32: the shares' own sums, and world additions more than one product has.
    Column-parallel outputs side by side are the product's."""

    n, k = 384, 1280
    codes, scales = mx_util.random_weight(n, k, 3, DEV)
    words, bytes_ = stored((codes, scales))
    ckpt = saved(tmp_path, {"o.weight": words.cpu().view(torch.uint32), "o.scales": bytes_.cpu()})
    x = mx_util.rows(rows, k, 4, DEV)
    ref, terms = mx_util.sums(x, codes, scales)
    total, columns, share = torch.zeros((rows, n), device=DEV), [], k // world
    for rank in range(world):
        own = tp.RowParallelLinear(checkpoint.load_microscaled(ckpt, "o", DEV, rank=rank, world=world, parallel="row"))
        part = own.partial(x[:, rank * share:(rank + 1) * share])
        assert part.dtype == torch.float32
        total += part
        cols = tp.ColumnParallelLinear(checkpoint.load_microscaled(ckpt, "o", DEV, rank=rank, world=world, parallel="column"))
        columns.append(cols.forward(x))
        assert torch.equal(tp.RowParallelLinear(own.q).forward(x[:, rank * share:(rank + 1) * share]), part.to(torch.bfloat16))
    mx_util.assert_product(total, ref, terms, k + world)
    mx_util.assert_product(torch.cat(columns, 1), ref, terms, k)
    ckpt.close()


def test_segments_read_on_the_device(tmp_path):
    """A rank's share of stacked projections: a run of rows of each, joined on the device."""

    codes, scales = mx_util.random_weight(96, 256, 3, DEV)
    words, bytes_ = stored((codes, scales))
    ckpt = saved(tmp_path, {"q.weight": words.cpu().view(torch.uint32), "q.scales": bytes_.cpu()})
    for rank in range(2):
        w, s = ckpt.microscaled("q", device=DEV, rank=rank, world=2, parallel="column", segments=(64, 32))
        rows = torch.cat([torch.arange(32) + 32 * rank, torch.arange(16) + 64 + 16 * rank]).to(DEV)
        assert w.dtype == torch.int32 and torch.equal(w, words[rows]) and torch.equal(s, bytes_[rows])
        q = checkpoint.load_microscaled(ckpt, "q", DEV, rank=rank, world=2, parallel="column", segments=(64, 32))
        assert (q.n, q.k) == (48, 256)
    ckpt.close()


@pytest.mark.parametrize("rows,prefill,f32", [(1, False, False), (9, False, False), (40, True, False), (200, True, True)])
def test_expert_parallel(rows, prefill, f32):
    """A rank's partial is the sum over the pairs whose expert it owns, with those pairs' bits in the whole table."""

    e, d, ni, k, world = 12, 384, 128, 3, 3
    ex, up, down = build((e, d, ni, True, 1.0), 9)
    g = torch.Generator(device=DEV).manual_seed(9)
    router = (torch.randn((e, d), generator=g, device=DEV) * d ** -0.5).to(torch.bfloat16)
    x = mx_util.rows(rows, d, 5, DEV, std=0.5)
    whole = tp.ExpertParallelMoE(router, ex, k, 0, e)
    buf = whole.buffers(rows, DEV, prefill=prefill, f32=f32)
    together = whole.partial(x, buf)
    y, picks, wts = buf.y[:rows].clone(), buf.pick[:rows].clone(), buf.wts[:rows].clone()
    assert y.dtype == (torch.bfloat16 if prefill and not f32 else torch.float32) and torch.equal(together, moe.combine(y, wts))
    for rank in range(world):
        raw_up, raw_down, first = tp.shard_experts([stored(u) for u in up], stored(down), rank, world)
        own = tp.ExpertParallelMoE(router, mx_experts.make(raw_up, raw_down, limit=1.0), k, first, e)
        got = own.partial(x, own.buffers(rows, DEV, prefill=prefill, f32=f32))
        mine = (picks >= first) & (picks < first + e // world)
        assert torch.equal(got, moe.combine(y, torch.where(mine, wts, 0.0)))
    assert torch.equal(whole.run(x, buf), together) and _lib.device_error(x) == 0
