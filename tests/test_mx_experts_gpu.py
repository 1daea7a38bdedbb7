"""Grouped experts on microscaled weights against their definition in 64 bits: ragged groups, the two forms of plans, activations
quantised between the projections, and the routed layer they make up."""

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib
from tensorfold_b200.cuda import experts, moe, mx_experts
from tensorfold_b200.cuda.kernels import mx, qmm

pytestmark = pytest.mark.gpu
DEV = "cuda"

# experts, D, NI, SwiGLU, limit: K of both projections ends in every part of a stage; a table wider than a block of columns
CASES = [(9, 256, 96, True, 0.0), (24, 416, 160, True, 1.0), (12, 1184, 224, False, 0.0), (5, 2688, 1856, True, 0.0), (3, 32, 32, True, 0.0)]


def stored(w):
    return mx_util.to_words(w[0]), w[1].to(torch.uint8)


def build(case, seed):
    e, d, ni, gated, limit = case
    up = [mx_util.random_weight(ni, d, seed + i, DEV, lead=(e,)) for i in range(2 if gated else 1)]
    down = mx_util.random_weight(d, ni, seed + 5, DEV, lead=(e,))
    return mx_experts.make([stored(u) for u in up], stored(down), limit=limit), up, down


def picks_for(rows, slots, count, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.stack([torch.randperm(count, generator=g)[:slots] for _ in range(rows)]).to(torch.int32).to(DEV)


def plan_of(picks, count, prefill, rows=None):
    plan = experts.Plan(rows or picks.shape[0], picks.shape[1], count, DEV, prefill=prefill)
    experts.route(picks.contiguous(), plan)
    return plan


def run(x, ex, picks, prefill, dtype=torch.float32):
    plan = plan_of(picks, ex.count, prefill)
    pairs = picks.numel()
    act = torch.full((pairs, ex.width), 3.0, dtype=torch.bfloat16, device=DEV)
    y = torch.full((pairs, ex.dims), 3.0, dtype=dtype, device=DEV)
    whole = torch.full((pairs, ex.dims), 3.0, dtype=dtype, device=DEV)
    mx_experts.gate_up(x, ex, plan, act, picks.shape[0])
    mx_experts.down(act, ex, plan, y, picks.shape[0])
    mx_experts.layer(x, ex, plan, whole, picks.shape[0])
    return act, y, whole


def activation(up, expert, rows, limit):
    """float64 activations of rows for one expert, and a bound on the kernel's error before any rounding (see
    test_mx_gpu.test_matmul_act)."""

    parts = [mx_util.sums(rows, u[0][expert], u[1][expert]) for u in up]
    e = rows.shape[1] * 2.0 ** -23
    if len(up) == 1:
        (v, t), = parts
        return v.clamp(min=0) ** 2, e * t * 2 * (v.abs() + e * t)
    (g, gt), (u, ut) = parts
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    ref = g * torch.sigmoid(g) * u
    return ref, e * gt * 1.1 * u.abs() + e * ut * (1.1 * g.abs() + 0.3) + 2.0 ** -20 * ref.abs()


def requantized(a, off):
    """a rounded to the format, and how far the rounding of anything within ``off`` of a may be from that: rounding is monotone
    at a scale, and a block whose largest value may cross a power of two may move by a quarter of it."""

    codes, scales = mx_util.quantize(a)
    q = mx_util.values(codes, scales)
    x = torch.ldexp(torch.ones_like(scales, dtype=torch.double), scales - 127).repeat_interleave(32, -1)

    def at_scale(v):
        r = (v / x).clamp(-6, 6)
        step = torch.ldexp(torch.full_like(r, 0.5), (torch.frexp(r).exponent - 1).clamp(0, 2))
        return (r / step).round() * step * x

    far = torch.maximum((at_scale(a + off) - q).abs(), (at_scale(a - off) - q).abs())
    top = a.abs().unflatten(-1, (-1, 32)).amax(-1)
    room = off.unflatten(-1, (-1, 32)).amax(-1)
    crosses = torch.frexp(top + room).exponent != torch.frexp((top - room).clamp(min=0)).exponent
    return q, torch.where(crosses.repeat_interleave(32, -1), far + 2 * x, far)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("rows,prefill", [(1, False), (7, False), (40, False), (40, True), (150, True)])
def test_layer_tracks_float64(case, rows, prefill):
    e, d, ni, gated, limit = case
    ex, up, dn = build(case, 3)
    x = mx_util.rows(rows, d, 1, DEV, std=0.3)
    picks = picks_for(rows, min(4, e), e, 2)
    slots = picks.shape[1]
    act, y, whole = run(x, ex, picks, prefill)
    _, _, half = run(x, ex, picks, prefill, torch.bfloat16)
    flat = picks.flatten()
    for expert in range(e):
        pairs = (flat == expert).nonzero().flatten()
        if not pairs.numel():
            continue
        a, off = activation(up, expert, x[pairs // slots], limit)
        assert ((act[pairs].double() - a).abs() <= 2.0 ** -8 * a.abs() + off * 1.01 + 2.0 ** -126).all()
        ref, terms = mx_util.sums(act[pairs], dn[0][expert], dn[1][expert])
        mx_util.assert_product(y[pairs], ref, terms, ni)
        q, far = requantized(a, off * 1.01)
        w = mx_util.values(dn[0][expert], dn[1][expert])
        bound = far @ w.abs().T + ni * 2.0 ** -23 * (q.abs() + far) @ w.abs().T + 2.0 ** -126
        ref = q @ w.T
        assert ((whole[pairs].double() - ref).abs() <= bound + 2.0 ** -24 * ref.abs()).all()
        assert ((half[pairs].double() - ref).abs() <= bound + 2.0 ** -8 * (ref.abs() + bound)).all()
    assert _lib.device_error(x) == 0


@pytest.mark.parametrize("case", CASES)
def test_pairs_do_not_depend_on_the_window_or_the_plan(case):
    ex, _, _ = build(case, 11)
    rows = 60
    x = mx_util.rows(rows, ex.dims, 1, DEV, std=0.5)
    picks = picks_for(rows, min(4, ex.count), ex.count, 3)
    slots = picks.shape[1]
    want = run(x, ex, picks, True)
    for m, prefill in ((60, False), (1, False), (1, True), (3, False), (17, False), (33, True)):
        got = run(x[:m], ex, picks[:m], prefill)
        assert all(torch.equal(a, b[:m * slots]) for a, b in zip(got, want)), (m, prefill)


@pytest.mark.parametrize("prefill", [False, True])
def test_ragged_plans(prefill):
    """One expert with every row (items past the first), experts with none, ids outside the table left as they were."""

    case = CASES[1]
    ex, _, _ = build(case, 21)
    rows = 300
    x = mx_util.rows(rows, ex.dims, 2, DEV, std=0.5)
    picks = torch.full((rows, 3), -1, dtype=torch.int32, device=DEV)
    picks[:, 0] = 5
    picks[::7, 1] = 23
    picks[3, 2] = 0
    picks[11, 1:] = 5                                          # the same expert in all three slots of a row
    act, y, whole = run(x, ex, picks, prefill)
    out = (picks.flatten() < 0)
    assert (act[out] == 3).all() and (y[out] == 3).all() and (whole[out] == 3).all()
    for r in (0, 3, 7, 11, 299):
        alone = run(x[r:r + 1], ex, picks[r:r + 1], False)
        assert all(torch.equal(a, b[3 * r:3 * r + 3]) for a, b in zip(alone, (act, y, whole)))
    # fewer rows than the plan's buffers hold, nothing routed at all
    plan = plan_of(picks[:5], ex.count, prefill, rows=40)
    part = torch.full((40 * 3, ex.dims), 3.0, dtype=torch.float32, device=DEV)
    mx_experts.layer(x, ex, plan, part, 5)
    assert torch.equal(part[:15], whole[:15]) and (part[15:] == 3).all()
    empty = plan_of(torch.full((4, 3), -1, dtype=torch.int32, device=DEV), ex.count, prefill)
    part.fill_(3)
    mx_experts.layer(x, ex, empty, part, 4)
    assert (part == 3).all() and _lib.device_error(x) == 0


@pytest.mark.parametrize("case", [(400, 800, 416, True, 1.0), (420, 768, 800, False, 0.0), (2400, 32, 32, True, 0.0)])
def test_many_tiles(case):
    """Tables of so many tiles that blocks take them in pairs: the bits of the form for few rows, over a ragged plan, odd numbers of
    column blocks, a row of NaN and an item outside the table."""

    ex, _, _ = build(case, 31)
    rows = 150
    x = mx_util.rows(rows, ex.dims, 2, DEV, std=0.5)
    x[9, 3] = float("nan")
    picks = picks_for(rows, 4, ex.count, 3)
    picks[:140, 0] = 7                                         # two items of one expert
    picks[20:30, 1] = -1
    got = run(x, ex, picks, True)
    for lo in range(0, rows, 16):
        few = run(x[lo:lo + 16], ex, picks[lo:lo + 16], False)
        for a, b in zip(few, got):
            assert torch.equal(a.view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32),
                               b[4 * lo:4 * lo + a.shape[0]].view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32))
    assert bool(torch.isnan(got[2][36:40]).all()) and not torch.isnan(got[2][40:]).any() and _lib.device_error(x) == 0
    plan = plan_of(picks, ex.count, True)
    plan.items[1, 0] = ex.count + 3
    y = torch.full((rows * 4, ex.dims), 3.0, dtype=torch.float32, device=DEV)
    mx_experts.layer(x, ex, plan, y, rows)
    assert _lib.device_error(x) == 5
    left = (y == 3).all(1)
    unrouted = int((picks < 0).sum())
    assert int(left.sum()) == int(plan.items[1, 2]) + unrouted and torch.equal(y[~left].nan_to_num(), got[2][~left].nan_to_num())


def test_items_outside_the_table_are_reported():
    ex, _, _ = build(CASES[0], 5)
    x = mx_util.rows(8, ex.dims, 2, DEV)
    picks = picks_for(8, 2, ex.count, 3)
    for prefill in (False, True):
        plan = plan_of(picks, ex.count, prefill)
        plan.items[1, 0] = ex.count + 3
        y = torch.full((16, ex.dims), 3.0, dtype=torch.float32, device=DEV)
        mx_experts.layer(x, ex, plan, y, 8)
        assert _lib.device_error(x) == 5 and int((y == 3).all(1).sum()) == int(plan.items[1, 2])


@pytest.mark.parametrize("prefill", [False, True])
def test_tables_past_32_bits(prefill):
    """Experts that lie gigabytes apart give what they give side by side."""

    ex, _, _ = build(CASES[0], 9)

    def apart(t):
        step = 2 ** 29 + 4096
        big = torch.empty((t.shape[0] * step,), dtype=torch.uint8, device=DEV).as_strided(t.shape, (step, t.shape[2], 1))
        return big.copy_(t)

    wide = mx_experts.Experts(apart(ex.up), apart(ex.down), ex.width, ex.dims, ex.limit, ex.gated)
    assert wide.up[-1].data_ptr() - wide.up[0].data_ptr() > 2 ** 32
    x, picks = mx_util.rows(40, ex.dims, 2, DEV, std=0.5), picks_for(40, 4, ex.count, 3)
    for a, b in zip(run(x, ex, picks, prefill), run(x, wide, picks, prefill)):
        assert torch.equal(a, b)


def test_infinite_rows_stay_in_their_pairs():
    for case, prefill in ((CASES[1], False), (CASES[1], True), (CASES[2], False), (CASES[2], True)):
        ex, _, _ = build(case, 6)
        x = mx_util.rows(20, ex.dims, 2, DEV, std=0.5)
        picks = picks_for(20, 4, ex.count, 3)
        clean = run(x, ex, picks, prefill)
        bad = x.clone()
        bad[4, 9] = float("nan")
        got = run(bad, ex, picks, prefill)
        for a, b in zip(got, clean):
            assert bool(torch.isnan(a[16:20]).all()), (case, prefill)
            assert torch.equal(a[:16], b[:16]) and torch.equal(a[20:], b[20:])


@pytest.mark.parametrize("prefill", [False, True])
def test_graph_replays_follow_new_picks(prefill):
    ex, _, _ = build(CASES[1], 8)
    rows, slots = 24, 4
    x, picks = mx_util.rows(rows, ex.dims, 1, DEV, std=0.5), picks_for(rows, slots, ex.count, 1)
    plan = experts.Plan(rows, slots, ex.count, DEV, prefill=prefill)
    y = torch.zeros((rows * slots, ex.dims), dtype=torch.float32, device=DEV)

    def step():
        experts.route(picks, plan)
        mx_experts.layer(x, ex, plan, y, rows)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (4, 5, 6):
        x.copy_(mx_util.rows(rows, ex.dims, seed, DEV, std=0.5))
        picks.copy_(picks_for(rows, slots, ex.count, seed))
        graph.replay()
        assert torch.equal(y, run(x, ex, picks, prefill)[2])


def affine_pair(n, k, seed):
    from tensorfold_b200 import synthetic

    return tuple(t.to(DEV) for t in synthetic.affine_weight(n, k, 4, 64, seed=seed))


@pytest.mark.parametrize("rows,prefill", [(1, False), (16, False), (16, True), (200, True)])
@pytest.mark.parametrize("shared", [None, "mx", "affine"])
def test_routed_layer(rows, prefill, shared):
    """moe.run with microscaled experts is its parts in order: router, plan, experts, the shared expert, combine."""

    d, ni, k = 384, 128, 3
    ex, _, _ = build((12, d, ni, True, 0.0), 9)
    e = 12 if shared else 11                                   # without a dense shared expert the table's last entry is it
    g = torch.Generator(device=DEV).manual_seed(4)
    router = (torch.randn((e + 1, d), generator=g, device=DEV) * d ** -0.5).to(torch.bfloat16)
    x = mx_util.rows(rows, d, 5, DEV, std=0.5)
    extra = None
    if shared == "mx":
        ws = [stored(mx_util.random_weight(256, d, 40 + i, DEV)) for i in range(2)]
        extra = moe.SharedExpert(mx.pack_pair(*ws), mx.pack(*stored(mx_util.random_weight(d, 256, 42, DEV))), limit=2.0)
    elif shared == "affine":
        extra = moe.SharedExpert(qmm.pack_pair(affine_pair(256, d, 1), affine_pair(256, d, 2), 64), qmm.pack(*affine_pair(d, 256, 3), 64))
    layer = moe.Routed(router, ex, k, extra)
    got = moe.run(x, layer, prefill=prefill)

    dtype = torch.bfloat16 if prefill else torch.float32
    logits = moe.router(x, router, prefill=prefill)
    buf = moe.MoEBuffers(rows, moe._Shape(layer), DEV, prefill=prefill, table_experts=ex.count)
    moe.select(logits, buf, k, e)
    y = torch.zeros((rows, k + 1, d), dtype=dtype, device=DEV)
    mx_experts.layer(x, ex, buf.plan, y.view(-1, d), rows)
    if shared == "mx":
        y[:, k] = mx.matmul(mx.matmul_act(x, extra.up, limit=2.0), extra.down, f32=not prefill)
    elif shared == "affine":
        act = qmm.matmul_act(x, extra.up, prefill=prefill)
        y[:, k] = (qmm.prefill_matmul if prefill else qmm.matmul)(act, extra.down, f32=not prefill)
    assert torch.equal(got, moe.combine(y, buf.wts))
    assert torch.equal(moe.run(x[:1], layer, prefill=prefill), got[:1])


def test_refusals():
    ex, up, dn = build(CASES[0], 3)
    x = mx_util.rows(4, ex.dims, 1, DEV)
    plan = plan_of(picks_for(4, 2, ex.count, 1), ex.count, False)
    y = torch.empty((8, ex.dims), device=DEV)
    for call in (lambda: mx_experts.layer(x, ex, plan, y, 5), lambda: mx_experts.layer(x[:3], ex, plan, y, 4),
                 lambda: mx_experts.layer(x, ex, plan, y[:7], 4), lambda: mx_experts.layer(x, ex, plan, y.half(), 4),
                 lambda: mx_experts.layer(x.float(), ex, plan, y, 4), lambda: mx_experts.layer(x, ex, plan, y.T, 4),
                 lambda: mx_experts.layer(x, ex, plan, y, 0), lambda: mx_experts.gate_up(x, ex, plan, y, 4),
                 lambda: mx_experts.down(x, ex, plan, y, 4),
                 lambda: mx_experts.layer(x, ex, plan_of(picks_for(4, 2, 5, 1), ex.count + 1, False), y, 4),
                 lambda: mx_experts.make([stored(up[0])], stored(up[0])),
                 lambda: mx_experts.layer(x, mx_experts.Experts(ex.up, ex.up, ex.width, ex.dims), plan, y, 4),
                 lambda: mx_experts.layer(x, mx_experts.Experts(ex.up.cpu(), ex.down, ex.width, ex.dims), plan, y, 4)):
        with pytest.raises(ValueError):
            call()


def test_checkpoint_to_layer(tmp_path):
    """A projection and a routed layer read from safetensors are those packed from the whole tensors."""

    from tensorfold_b200.cuda import checkpoint
    from test_checkpoint import write_safetensors

    host = lambda w: {"weight": stored(w)[0].cpu().view(torch.uint32), "scales": stored(w)[1].cpu()}
    parts = {"gate_proj": mx_util.random_weight(64, 128, 1, DEV, lead=(4,)), "up_proj": mx_util.random_weight(64, 128, 2, DEV, lead=(4,)),
             "down_proj": mx_util.random_weight(128, 64, 3, DEV, lead=(4,))}
    dense = mx_util.random_weight(200, 128, 4, DEV)
    path = tmp_path / "model.safetensors"
    tensors = {f"moe.{name}.{key}": t for name, w in parts.items() for key, t in host(w).items()}
    write_safetensors(path, {**tensors, **{f"o.{key}": t for key, t in host(dense).items()}}, pad=3)
    ckpt = checkpoint.Checkpoint([path])
    q = checkpoint.load_microscaled(ckpt, "o", DEV)
    assert (q.n, q.k) == (200, 128) and torch.equal(q.weight, mx.pack(*stored(dense)).weight)
    ex, first = checkpoint.load_microscaled_experts(ckpt, "moe", DEV, rank=1, world=2, limit=3.0)
    cut = {name: tuple(t[2:] for t in stored(w)) for name, w in parts.items()}
    want = mx_experts.make([cut["gate_proj"], cut["up_proj"]], cut["down_proj"], limit=3.0)
    assert first == 2 and ex.limit == 3.0 and torch.equal(ex.up, want.up) and torch.equal(ex.down, want.down)
    ckpt.close()
