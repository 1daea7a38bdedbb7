"""The microscaled format written out in 64 bits: what the tests hold the kernels to."""

import torch

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(x):
    """[.., k] of any float type -> (codes [.., k] int64, scales [.., k / 32] int64) by the definition: the nearest of the eight
    magnitudes, ties to the even code."""

    v = x.double().unflatten(-1, (-1, BLOCK))
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], 0.0, v)
    top = v.abs().amax(-1)
    scale = (torch.frexp(top).exponent.long() - 1 - 2 + 127).clamp(min=0)
    scale = torch.where(top == 0, 0, scale)
    r = v.abs() * torch.ldexp(torch.ones_like(top), 127 - scale)[..., None]
    grid = torch.tensor(GRID, dtype=torch.double, device=x.device)
    gap = (r[..., None] - grid).abs()
    # ties: an even code wins over an odd one at the same distance (above 6 only 6 is nearest)
    order = gap + torch.tensor([0, 1] * 4, device=x.device) * 1e-9
    codes = torch.where(r > 6, 7, order.argmin(-1)) | (torch.signbit(v).long() << 3)
    return torch.where(bad[..., None], 0, codes).flatten(-2), torch.where(bad, 255, scale)


def values(codes, scales):
    """float64 values of codes [.., k] and scale codes [.., k / 32]."""

    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.double, device=codes.device)
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.double), scales - 127)
    s = torch.where(scales == 255, float("nan"), s)
    return (grid[codes].unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def to_words(codes):
    """Codes [.., k] -> int32 words [.., k / 8], the first code in the low bits."""

    shifts = torch.arange(0, 32, 4, device=codes.device)
    w = (codes.unflatten(-1, (-1, 8)) << shifts).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def to_codes(words):
    shifts = torch.arange(0, 32, 4, device=words.device)
    return ((words.long()[..., None] >> shifts) & 15).flatten(-2)


def rounded(x):
    """x with every block rounded to the format, float64."""

    return values(*quantize(x))


def random_weight(n, k, seed, device, lead=(), spread=6):
    """Codes and scales of a stored weight: every code, scales over 2^spread around 2^-7.  (codes, scale codes) int64."""

    g = torch.Generator(device=device).manual_seed(seed)
    codes = torch.randint(0, 16, (*lead, n, k), generator=g, device=device)
    scales = torch.randint(120 - spread // 2, 121 + spread // 2, (*lead, n, k // BLOCK), generator=g, device=device)
    return codes, scales


def rows(m, k, seed, device, std=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn((m, k), generator=g, device=device) * std
    x[:, ::37] *= 8
    return x.to(torch.bfloat16)


def sums(x, codes, scales):
    """float64 products of rounded rows with a stored weight, and the sums of their terms' magnitudes."""

    a, w = rounded(x), values(codes, scales)
    return a @ w.T, a.abs() @ w.abs().T


def assert_product(y, ref, terms, k, what=""):
    """|y - ref| <= (rounding of the result) + k 2^-23 (sum of the terms' magnitudes): products are exact, and k additions in
    fp32, in any order and even truncated, lose 2^-23 of a partial sum each, which the magnitudes' sum bounds."""

    half = torch.finfo(y.dtype).eps / 2
    bound = half * ref.abs() + k * 2.0 ** -23 * terms + 2.0 ** -126
    off = (y.double() - ref).abs()
    assert torch.isfinite(y).all(), f"{what}: not finite"
    worst = (off / bound).max()
    assert worst <= 1, f"{what}: {float(worst):.3f} times the bound"
