"""Microscaled 4-bit floating point on the GPU against its definition in 64 bits (``mx_util``): quantising and reading back, packing, and
the product from one row to several hundred."""

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib
from tensorfold_b200.cuda.kernels import mx, qmm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def weight(n, k, seed, **kw):
    codes, scales = mx_util.random_weight(n, k, seed, DEV, **kw)
    return codes, scales, mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))


def special_rows(dtype):
    """Blocks that try the rounding: ties, the type's ends, zeros, infinities and NaN."""

    info = torch.finfo(dtype)
    grid = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.5, 7, 7.5, 7.9375], dtype=torch.double)
    ties = torch.cat([grid, -grid])[:32]
    rows = [ties * 2.0 ** e for e in (0, -3, 5)]
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), info.max), torch.full((32,), info.tiny),
             torch.full((32,), info.smallest_normal / 4), torch.linspace(-1, 1, 32) * info.tiny]
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.linspace(-3, 3, 32)
        r[7] = bad
        rows.append(r)
    return torch.stack([r.double() for r in rows]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_special_values(dtype):
    x = special_rows(dtype).to(DEV)
    x = torch.cat([x, x.flip(0)], 1).contiguous()              # two blocks a row: a bad one leaves its neighbour alone
    words, scales = mx.quantize(x)
    codes, want = mx_util.quantize(x)
    assert torch.equal(scales.long(), want)
    assert torch.equal(words, mx_util.to_words(codes))


@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (391, 2720), (2, 5, 64), (16, 5120), (32,)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_and_back(shape, dtype):
    g = torch.Generator(device=DEV).manual_seed(7)
    x = (torch.randn(shape, generator=g, device=DEV) * torch.exp2(torch.randint(-9, 9, shape, generator=g, device=DEV))).to(dtype)
    words, scales = mx.quantize(x)
    codes, want = mx_util.quantize(x)
    assert words.shape == (*shape[:-1], shape[-1] // 8) and scales.shape == (*shape[:-1], shape[-1] // 32)
    assert torch.equal(words, mx_util.to_words(codes)) and torch.equal(scales.long(), want)
    for out in (torch.bfloat16, torch.float32):
        assert torch.equal(mx.dequantize(words, scales, out).double(), mx_util.values(codes, want))


def test_quantize_takes_views():
    x = mx_util.rows(40, 512, 3, DEV)
    for view in (x[::2], x[:, 128:256], x[:, 32:].T.contiguous().T, x[3:4], x[:, 8:264], x.view(4, 10, 512)[:, 3]):
        got, want = mx.quantize(view), mx.quantize(view.contiguous())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    empty = mx.quantize(x[:0])
    assert empty[0].shape == (0, 64) and mx.dequantize(*empty).shape == (0, 512)


def test_dequantize_every_code_and_scale():
    scales = torch.arange(256, device=DEV).repeat_interleave(2).view(256, 2)
    codes = torch.arange(16, device=DEV).repeat(256, 4)
    want = mx_util.values(codes, scales)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        got = mx.dequantize(mx_util.to_words(codes), scales.to(torch.uint8), dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.5), want.to(dtype).nan_to_num(0.5))


@pytest.mark.parametrize("n,k", [(1, 32), (129, 64), (48, 96), (300, 288), (128, 256), (257, 320), (64, 448), (1000, 992)])
def test_pack_round_trip(n, k):
    codes, scales = mx_util.random_weight(n, k, n + k, DEV)
    words, s8 = mx_util.to_words(codes), scales.to(torch.uint8)
    back = mx.unpack(mx.pack(words, s8))
    assert torch.equal(back[0], words) and torch.equal(back[1], s8)


# one K slice and several, K that ends in every part of a stage (whole, one to three steps, half a step), columns past a block
SHAPES = [(128, 256), (128, 64), (1, 32), (130, 96), (257, 160), (256, 1024), (1024, 5120), (384, 2720), (200, 4384), (2500, 736)]
ROWS = (1, 2, 7, 8, 9, 16, 17, 48, 64, 65, 128, 129, 256, 257, 391)


@pytest.mark.parametrize("n,k", SHAPES)
def test_matmul_tracks_float64(n, k):
    codes, scales, q = weight(n, k, n + k)
    x = mx_util.rows(max(ROWS), k, 5, DEV)
    ref, terms = mx_util.sums(x, codes, scales)
    for m in ROWS:
        for f32 in (False, True):
            y = mx.matmul(x[:m], q, f32=f32)
            mx_util.assert_product(y, ref[:m], terms[:m], k, f"m {m} f32 {f32}")
    assert _lib.device_error(x) == 0


# wide weights on prompts: two blocks share a tile, with an odd number of column blocks and K that ends in every part of a stage
@pytest.mark.parametrize("n,k", [(9500, 2080), (9728, 2048), (9601, 2176), (9856, 2240)])
def test_prompts_on_wide_weights(n, k):
    codes, scales, q = weight(n, k, n + k)
    x = mx_util.rows(391, k, 5, DEV)
    x[300, 7] = float("nan")
    y = mx.matmul(x, q, f32=True)
    good = torch.arange(391, device=DEV) != 300
    ref, terms = mx_util.sums(x[good], codes, scales)
    mx_util.assert_product(y[good], ref, terms, k)
    assert bool(torch.isnan(y[300]).all())
    want = y.to(torch.bfloat16).nan_to_num(0.5)
    out = torch.full((393, n + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    mx.matmul(x, q, out=out[1:392, 8:])
    assert torch.equal(out[1:392, 8:].nan_to_num(0.5), want) and (out[0] == 7).all() and (out[392] == 7).all() and (out[:, :8] == 7).all()
    for m in (1, 16, 40, 129, 300):                            # the other forms, and pairs with other tiles
        assert torch.equal(mx.matmul(x[:m], q, f32=True), y[:m]), m
    if n % 32 == 0:
        act = mx.matmul_act(x[good], q, limit=3.0)             # (any weight of whole tiles is a pair of something)
        assert torch.equal(mx.matmul_act(x[:9], q, limit=3.0), act[:9]) and bool(torch.isfinite(act).all())
    assert _lib.device_error(x) == 0


@pytest.mark.parametrize("n,k", [(257, 160), (1024, 5120), (2500, 736)])
def test_whole_numbers_are_exact(n, k):
    """Scales of one and whole values: every partial sum is a whole number of quarters below 2^24, so any order is exact."""

    codes, scales = mx_util.random_weight(n, k, 9, DEV)
    scales = torch.full_like(scales, 127)
    q = mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randint(-4, 5, (300, k), generator=g, device=DEV).to(torch.bfloat16)
    x[:, ::32] = 4                                             # every block's scale is one
    ref = mx_util.rounded(x) @ mx_util.values(codes, scales).T
    for m in (1, 16, 40, 100, 300):
        assert torch.equal(mx.matmul(x[:m], q, f32=True).double(), ref[:m]), m


@pytest.mark.parametrize("n,k", SHAPES)
def test_rows_do_not_depend_on_the_window(n, k):
    _, _, q = weight(n, k, n + k)
    x = mx_util.rows(300, k, 6, DEV)
    y = mx.matmul(x, q, f32=True)
    for m in (1, 2, 9, 16, 17, 33, 64, 100, 129, 256):
        assert torch.equal(mx.matmul(x[300 - m:], q, f32=True), y[300 - m:]), m
    perm = torch.randperm(300, generator=torch.Generator().manual_seed(2)).to(DEV)
    assert torch.equal(mx.matmul(x[perm], q, f32=True), y[perm])


@pytest.mark.parametrize("m", [1, 13, 40, 200])
def test_bad_blocks_stay_in_their_row_and_column(m):
    n, k = 300, 416
    codes, scales, _ = weight(n, k, 4)
    scales[17, 5] = 255
    q = mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))
    x = mx_util.rows(m, k, 8, DEV)
    clean = mx.matmul(x, q)
    assert torch.isnan(clean[:, 17]).all() and torch.isfinite(clean[:, :17]).all() and torch.isfinite(clean[:, 18:]).all()
    x[m // 2, 100] = float("inf")
    y = mx.matmul(x, q)
    keep = torch.arange(m, device=DEV) != m // 2
    assert torch.isnan(y[m // 2]).all()
    assert torch.equal(y[keep].nan_to_num(0.5), clean[keep].nan_to_num(0.5))


@pytest.mark.parametrize("m", [1, 16, 50, 300])
def test_scales_at_the_ends(m):
    """Zero rows, rows and weights far below and above one: products stay within fp32's normal range."""

    n, k = 160, 512
    codes, scales, _ = weight(n, k, 4)
    for e in (-100, 0, 100):
        q = mx.pack(mx_util.to_words(codes), (scales - e).to(torch.uint8))
        x = (mx_util.rows(m, k, 8, DEV).float() * 2.0 ** e).to(torch.bfloat16)
        x[0, :256] = 0
        ref, terms = mx_util.sums(x, codes, scales - e)
        mx_util.assert_product(mx.matmul(x, q, f32=True), ref, terms, k, f"2^{e}")
    q = mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))
    assert torch.equal(mx.matmul(torch.zeros((m, k), dtype=torch.bfloat16, device=DEV), q), torch.zeros((m, n), dtype=torch.bfloat16, device=DEV))


@pytest.mark.parametrize("m", [1, 5, 16, 70, 260])
def test_views_and_outputs(m):
    """Strided and misaligned rows give the same bits; rows and columns beside the output stay as they were."""

    n, k = 272, 608
    _, _, q = weight(n, k, 12)
    x = mx_util.rows(m, k, 3, DEV)
    want = mx.matmul(x, q)
    wide = torch.zeros((m, k + 24), dtype=torch.bfloat16, device=DEV)
    for at in (0, 8, 3):
        wide[:, at:at + k] = x
        assert torch.equal(mx.matmul(wide[:, at:at + k], q), want)
    assert torch.equal(mx.matmul(x.T.contiguous().T, q), want)
    out = torch.full((m + 2, n + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    got = mx.matmul(x, q, out=out[1:m + 1, 4:n + 4])
    assert torch.equal(got, want) and torch.equal(out[1:m + 1, 4:n + 4], want)
    out[1:m + 1, 4:n + 4] = 7
    assert (out == 7).all()


@pytest.mark.parametrize("m", [1, 12, 48, 200])
@pytest.mark.parametrize("act,limit", [("swiglu", 0.0), ("swiglu", 1.5), ("relu2", 0.0)])
def test_matmul_act(m, act, limit):
    """|y - f(ref)| <= rounding + the sums' error through the activation, whose slopes are below 1.1 |u| and 1.1 |g| + 0.3 (SwiGLU:
    silu' is at most 1.0999, |silu(g)| <= |g|) and 2 |v| (relu^2), plus 2^-20 of the value for exp and the divide."""

    n, k = 176, 480
    (gc, gs), (uc, us) = mx_util.random_weight(n, k, 1, DEV), mx_util.random_weight(n, k, 2, DEV)
    x = mx_util.rows(m, k, 3, DEV, std=0.3)
    pair = lambda c, s: (mx_util.to_words(c), s.to(torch.uint8))
    (g, gt), (u, ut) = mx_util.sums(x, gc, gs), mx_util.sums(x, uc, us)
    e = k * 2.0 ** -23
    if act == "swiglu":
        y = mx.matmul_act(x, mx.pack_pair(pair(gc, gs), pair(uc, us)), limit=limit)
        if limit:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        ref = g * torch.sigmoid(g) * u
        slack = e * gt * 1.1 * u.abs() + e * ut * (1.1 * g.abs() + 0.3)
    else:
        y = mx.matmul_act(x, mx.pack(*pair(gc, gs)), act=act)
        ref = g.clamp(min=0) ** 2
        slack = e * gt * 2 * (g.abs() + e * gt)
    bound = (2.0 ** -8 + 2.0 ** -20) * ref.abs() + slack * 1.01 + 2.0 ** -126
    assert ((y.double() - ref).abs() <= bound).all()
    assert torch.equal(mx.matmul_act(x[:1], mx.pack_pair(pair(gc, gs), pair(uc, us)) if act == "swiglu" else mx.pack(*pair(gc, gs)), act=act,
                                     limit=limit), y[:1])


@pytest.mark.parametrize("m,wide", [(4, False), (40, False), (300, False), (391, True)])
def test_graphs_and_streams(m, wide):
    """Two calls captured in one graph and replayed on new rows, and calls on three streams at once."""

    _, _, qa = weight(9600 if wide else 1024, 2048 if wide else 1184, 5)
    _, _, qb = weight(512, qa.n, 6)
    x = mx_util.rows(m, qa.k, 1, DEV)
    want = []
    for seed in (1, 2, 3):
        h = mx.matmul(mx_util.rows(m, qa.k, seed, DEV), qa)
        want.append((h, mx.matmul(h, qb)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = mx.matmul(x, qa, pdl=True)
        y = mx.matmul(h, qb, pdl=True)
    for i, seed in enumerate((1, 2, 3)):
        x.copy_(mx_util.rows(m, qa.k, seed, DEV))
        graph.replay()
        assert torch.equal(h, want[i][0]) and torch.equal(y, want[i][1])
    streams = [torch.cuda.Stream() for _ in range(3)]
    inputs = [mx_util.rows(m, qa.k, seed, DEV) for seed in (1, 2, 3)]
    torch.cuda.synchronize()
    got = [[] for _ in streams]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mx.matmul(mx.matmul(inputs[i], qa), qb))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i][1]) for i in range(3) for y in got[i])


def test_offsets_past_32_bits():
    """Inputs and outputs of more than 2^31 values: the first and last rows are what they are in small calls."""

    x = torch.zeros((65552, 32768), dtype=torch.bfloat16, device=DEV)
    ends = mx_util.rows(4, 32768, 1, DEV)
    x[:2], x[-2:] = ends[:2], ends[2:]
    words, scales = mx.quantize(x)
    few = mx.quantize(ends)
    assert torch.equal(words[[0, 1, -2, -1]], few[0]) and torch.equal(scales[[0, 1, -2, -1]], few[1]) and not words[2:-2].any()
    del x
    back = mx.dequantize(words, scales)
    assert torch.equal(back[[0, 1, -2, -1]], mx.dequantize(*few)) and not back[2:-2].any()
    del back, words, scales
    _, _, q = weight(11000, 96, 3)
    rows = mx_util.rows(64, 96, 2, DEV)
    y = mx.matmul(rows.repeat(3200, 1), q)
    assert y.numel() > 2 ** 31
    want = mx.matmul(rows, q)
    assert all(torch.equal(y[i:i + 64], want) for i in (0, 64 * 1600, 64 * 3050, 64 * 3199))


def test_beside_other_products():
    """Affine and microscaled products in turn on one stream with early launches, and both kinds at once on two streams: they share
    tensor memory and shared memory of the SMs."""

    _, _, q = weight(4096, 1024, 7)
    g = torch.Generator(device=DEV).manual_seed(8)
    w = torch.randint(-2 ** 31, 2 ** 31, (1024, 4096 // 8), generator=g, device=DEV).to(torch.int32)
    s = (torch.rand((1024, 4096 // 64), generator=g, device=DEV) * .01).bfloat16()
    affine = qmm.pack(w, s, -8 * s, 64)
    for m in (1, 16, 300):
        x = mx_util.rows(m, 1024, m, DEV)
        h0 = mx.matmul(x, q)
        y0 = qmm.matmul(h0, affine)
        for _ in range(4):
            h = mx.matmul(x, q, pdl=True)
            assert torch.equal(h, h0) and torch.equal(qmm.matmul(h, affine), y0)
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        got = [], []
        for _ in range(8):
            with torch.cuda.stream(a):
                got[0].append(mx.matmul(x, q, pdl=True))
            with torch.cuda.stream(b):
                got[1].append(qmm.matmul(h0, affine))
        torch.cuda.synchronize()
        assert all(torch.equal(t, h0) for t in got[0]) and all(torch.equal(t, y0) for t in got[1])


def test_refusals_on_the_device():
    _, _, q = weight(64, 128, 1)
    x = mx_util.rows(4, 128, 1, DEV)
    for bad in (x.float(), x[:, :64], x[:0], x[0]):
        with pytest.raises(ValueError):
            mx.matmul(bad, q)
    for out in (torch.empty((4, 64), device=DEV), torch.empty((4, 65), dtype=torch.bfloat16, device=DEV),
                torch.empty((4, 64), dtype=torch.bfloat16), torch.empty((64, 4), dtype=torch.bfloat16, device=DEV).T):
        with pytest.raises(ValueError):
            mx.matmul(x, q, out=out)
    with pytest.raises(ValueError):
        mx.matmul(x, mx.MX4(q.weight, 200, 128))               # super-blocks of another shape
    with pytest.raises(ValueError):
        mx.matmul(x, mx.MX4(q.weight.cpu(), 64, 128))
    with pytest.raises(ValueError):
        mx.matmul_act(x, weight(48, 128, 1)[2])                # no whole pairs of tiles
    with pytest.raises(ValueError):
        mx.quantize(x[:, :40])
    with pytest.raises(ValueError):
        mx.quantize(x.long())
    words, scales = mx.quantize(x)
    with pytest.raises(ValueError):
        mx.dequantize(words, scales[:, :2])
    with pytest.raises(ValueError):
        mx.pack(words, scales.float())
