"""Microscaled 4-bit floating point as this library's users meet it, as cases that can be timed: rows and weights quantised
and read back, products of quantised rows with quantised weights from one row to a prompt chunk, and the routed experts of
a mixture layer with ragged numbers of rows.

A block is 32 neighbouring inputs.  Its scale is the power of two 2^(floor(log2 amax) - 2), stored as a biased exponent of
eight bits (255 stands for NaN); its values are e2m1 numbers: a sign and 0, 0.5, 1, 1.5, 2, 3, 4 or 6, rounded to nearest
even and saturated.  Eight codes a 32-bit word, the first in the low bits.

Weights are N(0, 0.02) and activations N(0, 1) with one channel in 64 eight times as large, as layers of language models
have them.  Everything is drawn on the GPU from the seed."""

from __future__ import annotations

import torch

own = False

DEV = "cuda"
BLOCK = 32
ROUTED_DECODE_ROWS = 128  # routed layers take the prompt form past this


def listed() -> list[dict]:
    return [
        # the rows of a verify window, quantised and read back: the smallest call, all latency
        {"name": "quantize 16x5120", "kind": "quantize", "rows": 16, "k": 5120},
        # a projection of a checkpoint brought to four bits, and the values it then stands for
        {"name": "quantize 17408x5120", "kind": "quantize", "rows": 17408, "k": 5120},
        # plain decoding of one stream: the wide projection of a dense layer
        {"name": "matmul 17408x5120 m1", "kind": "matmul", "n": 17408, "k": 5120, "rows": 1, "f32": False},
        # a verify window on the narrow key projection: few columns, an odd number of rows
        {"name": "matmul 1024x5120 m13", "kind": "matmul", "n": 1024, "k": 5120, "rows": 13, "f32": False},
        # a verify window on the down projection, whose unrounded sums a row-parallel layer adds over its ranks
        {"name": "matmul 5120x17408 m16 f32", "kind": "matmul", "n": 5120, "k": 17408, "rows": 16, "f32": True},
        # four streams' twelve-row windows in one batch
        {"name": "matmul 6144x5120 m48", "kind": "matmul", "n": 6144, "k": 5120, "rows": 48, "f32": False},
        # the ragged last chunk of a prompt
        {"name": "matmul 17408x5120 m391", "kind": "matmul", "n": 17408, "k": 5120, "rows": 391, "f32": False},
        # a whole prompt chunk
        {"name": "matmul 17408x5120 m2048", "kind": "matmul", "n": 17408, "k": 5120, "rows": 2048, "f32": False},
        # the logits of one token over the whole vocabulary
        {"name": "matmul 248320x5120 m1", "kind": "matmul", "n": 248320, "k": 5120, "rows": 1, "f32": False},
        # the routed experts of a layer (128 experts, top 6): plain decoding, a verify window and a prompt chunk
        {"name": "experts m1", "kind": "experts", "hidden": 2688, "width": 1856, "experts": 128, "top_k": 6, "rows": 1},
        {"name": "experts m16", "kind": "experts", "hidden": 2688, "width": 1856, "experts": 128, "top_k": 6, "rows": 16},
        {"name": "experts m2048", "kind": "experts", "hidden": 2688, "width": 1856, "experts": 128, "top_k": 6, "rows": 2048},
    ]


def _log(rng, lo: int, hi: int, step: int = 1) -> int:
    """An integer of [lo, hi], spread evenly over its logarithm, a multiple of ``step``."""

    v = lo * (hi / lo) ** rng.random()
    return max(lo, min(hi, round(v / step) * step))


def _rows(rng) -> int:
    """Rows of a call: windows, batches of windows and prompt chunks alike."""

    return rng.choice([rng.randint(1, 16), _log(rng, 17, 256), _log(rng, 257, 2048)])


def draw(rng) -> dict:
    kind = rng.choice(["quantize", "matmul", "matmul", "matmul", "experts", "experts"])
    if kind == "quantize":
        return {"kind": kind, "rows": _log(rng, 1, 17408), "k": _log(rng, 256, 5120, BLOCK)}
    if kind == "matmul":
        return {"kind": kind, "n": _log(rng, 256, 17408, rng.choice([1, 16, 128])), "k": _log(rng, 512, 17408, BLOCK),
                "rows": min(_rows(rng), 640) if rng.random() < 0.5 else rng.randint(1, 16), "f32": rng.random() < 0.25}
    return {"kind": kind, "hidden": _log(rng, 1024, 2688, 64), "width": _log(rng, 512, 1856, 64),
            "experts": rng.choice([32, 64, 96, 128]), "top_k": rng.randint(2, 6), "rows": _rows(rng)}


# ---------------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------------

def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[.., k] -> words [.., k / 8] int32 and scales [.., k / 32] uint8."""

    v = x.float().unflatten(-1, (-1, BLOCK))
    top = v.abs().amax(-1).view(torch.int32) >> 23                       # the largest value's biased exponent
    code = torch.where(top == 255, 255, (top - 2).clamp(min=0))          # an infinity or a NaN makes the scale a NaN
    inverse = ((254 - code).clamp(min=0) << 23).view(torch.float32)      # 2^(127 - code)
    v = torch.where((code == 255).unsqueeze(-1), 0.0, v * inverse.unsqueeze(-1))
    m = v.abs()
    q = (m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int()      # ties go to the even code
    q = q + (m > 2.5).int() + (m >= 3.5).int() + (m > 5.0).int()
    q = (q | (torch.signbit(v).int() << 3)).flatten(-2).unflatten(-1, (-1, 8))
    shifts = torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)
    return (q << shifts).sum(-1, dtype=torch.int32), code.to(torch.uint8)


def _dequantize(words: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values that words [.., k / 8] and scales [.., k / 32] stand for."""

    shifts = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=words.device)
    v = values[(words.unsqueeze(-1) >> shifts) & 15].flatten(-2).unflatten(-1, (-1, BLOCK))
    code = scales.int()
    scale = torch.where(code == 0, 0x00400000, torch.where(code == 255, 0x7FC00000, code << 23)).view(torch.float32)
    return (v * scale.unsqueeze(-1)).flatten(-2)


def _matmul(x: torch.Tensor, words: torch.Tensor, scales: torch.Tensor, f32: bool) -> torch.Tensor:
    y = _dequantize(*_quantize(x)) @ _dequantize(words, scales).T
    return y if f32 else y.to(torch.bfloat16)


def _experts(s) -> torch.Tensor:
    """Pairs sorted by expert, each expert's rows in a slot of ``most`` rows, batched products over all experts."""

    x, picks, wts, most = s["x"], s["picks"], s["wts"], s["most"]
    rows, slots = picks.shape
    count = s["gate"][0].shape[0]
    flat = picks.flatten().long()
    order = torch.argsort(flat, stable=True)
    expert = flat[order]
    first = torch.searchsorted(expert, torch.arange(count, device=DEV))
    place = torch.arange(rows * slots, device=DEV) - first[expert]
    xq = _dequantize(*_quantize(x))
    a = torch.zeros((count, most, x.shape[1]), device=DEV)
    a[expert, place] = xq[order // slots]
    g = torch.bmm(a, _dequantize(*s["gate"]).transpose(1, 2))
    u = torch.bmm(a, _dequantize(*s["up"]).transpose(1, 2))
    act = _dequantize(*_quantize(g / (1 + torch.exp(-g)) * u))
    y = torch.bmm(act, _dequantize(*s["down"]).transpose(1, 2))
    pairs = torch.empty((rows * slots, x.shape[1]), device=DEV)
    pairs[order] = y[expert, place]
    return (pairs.view(rows, slots, -1) * wts.unsqueeze(-1)).sum(1).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------------------------------------------------

class _Make:
    def __init__(self, seed: int) -> None:
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape: int, std: float = 1.0) -> torch.Tensor:
        return torch.randn(shape, generator=self.g, device=DEV) * std

    def rows(self, m: int, k: int) -> torch.Tensor:
        channel = torch.where(torch.rand(k, generator=self.g, device=DEV) < 1 / 64, 8.0, 1.0)
        return (self.normal(m, k) * channel).to(torch.bfloat16)

    def weight(self, *shape: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Stored words and scales of N(0, 0.02) weights, made in pieces."""

        *lead, n, k = shape
        flat = n * (lead[0] if lead else 1)
        parts = [_quantize(self.normal(min(16384, flat - at), k, std=0.02)) for at in range(0, flat, 16384)]
        words, scales = (torch.cat(p).view(*lead, n, -1) for p in zip(*parts))
        return words, scales


def _plan(c, make):
    """Which experts each row takes and with what weight, as a router hands them on."""

    rows, slots, count = c["rows"], c["top_k"], c["experts"]
    popular = make.normal(count, std=0.5)
    logits = make.normal(rows, count) + popular
    wts, picks = logits.topk(slots, dim=1)
    most = int(torch.bincount(picks.flatten(), minlength=count).max())
    return picks.int().contiguous(), torch.softmax(wts, 1).contiguous(), most


def prepare(case: dict, seed: int) -> dict:
    c, make = case, _Make(seed)
    kind = c["kind"]
    if kind == "quantize":
        std = 0.02 if c["rows"] > 2048 else 1.0
        return {"case": c, "x": (make.rows(c["rows"], c["k"]).float() * std).to(torch.bfloat16)}
    if kind == "matmul":
        s = {"case": c, "x": make.rows(c["rows"], c["k"]), "weight": make.weight(c["n"], c["k"])}
        if own:
            from tensorfold_b200.cuda.kernels import mx

            s["q"] = mx.pack(*s["weight"])
        return s
    e, d, w = c["experts"], c["hidden"], c["width"]
    s = {"case": c, "x": make.rows(c["rows"], d), "gate": make.weight(e, w, d), "up": make.weight(e, w, d), "down": make.weight(e, d, w)}
    s["picks"], s["wts"], s["most"] = _plan(c, make)
    if own:
        from tensorfold_b200.cuda import experts, mx_experts

        prompt = c["rows"] > ROUTED_DECODE_ROWS
        s["table"] = mx_experts.make([s["gate"], s["up"]], s["down"])
        s["plan"] = experts.Plan(c["rows"], c["top_k"], e, DEV, prefill=prompt)
        s["y"] = torch.empty((c["rows"] * c["top_k"], d), dtype=torch.float32, device=DEV)   # rounded once, after the slots are added
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------

def run(state: dict):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind == "quantize":
            return _dequantize(*_quantize(s["x"])).to(torch.bfloat16)
        if kind == "matmul":
            return _matmul(s["x"], *s["weight"], c["f32"])
        return _experts(s)
    from tensorfold_b200.cuda import experts, moe, mx_experts
    from tensorfold_b200.cuda.kernels import mx

    if kind == "quantize":
        return mx.dequantize(*mx.quantize(s["x"]))
    if kind == "matmul":
        return mx.matmul(s["x"], s["q"], f32=c["f32"])
    experts.route(s["picks"], s["plan"])
    mx_experts.layer(s["x"], s["table"], s["plan"], s["y"], c["rows"])
    return moe.combine(s["y"].view(c["rows"], c["top_k"], -1), s["wts"])


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, and what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def _values64(x: torch.Tensor) -> torch.Tensor:
    """What the blocks of ``x`` are rounded to, from the definition: steps of a quarter, half or whole power of two."""

    v = x.double().reshape(-1, BLOCK)
    top = v.abs().amax(1, keepdim=True)
    scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top).exponent - 3).clamp(min=-127))
    scale = torch.where(top == 0, 2.0 ** -127, scale)
    r = v / scale
    step = torch.ldexp(torch.full_like(r, 0.5), (torch.frexp(r).exponent - 1).clamp(0, 2))
    return ((r / step).round() * step).clamp(-6, 6).mul(scale).reshape(x.shape)


def _stored64(words: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Stored codes by the meaning of their bits: sign, two bits of exponent, one of fraction."""

    bits = torch.stack([(words >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2)
    e, f = (bits >> 1) & 3, (bits & 1).double()
    v = torch.where(e == 0, f / 2, torch.ldexp(1 + f / 2, e - 1)) * torch.where(bits > 7, -1.0, 1.0)
    return v * torch.ldexp(torch.ones_like(scales, dtype=torch.double), scales.int() - 127).repeat_interleave(BLOCK, -1)


def exact(case: dict, seed: int):
    s, c = prepare(case, seed), case
    if c["kind"] == "quantize":
        return _values64(s["x"])
    if c["kind"] == "matmul":
        x, step = _values64(s["x"]), 32768
        words, scales = s["weight"]
        return torch.cat([x @ _stored64(words[i:i + step], scales[i:i + step]).T for i in range(0, c["n"], step)], 1)
    x = _values64(s["x"])
    out = torch.zeros_like(x)
    for e in range(c["experts"]):
        row, slot = (s["picks"] == e).nonzero(as_tuple=True)
        if row.numel():
            g, u = (x[row] @ _stored64(s[name][0][e], s[name][1][e]).T for name in ("gate", "up"))
            act = _values64(g * torch.sigmoid(g) * u)
            y = act @ _stored64(s["down"][0][e], s["down"][1][e]).T
            out.index_add_(0, row, y * s["wts"][row, slot].double().unsqueeze(1))
    return out


def _weight_bytes(n: int, k: int) -> float:
    return n * k * (0.5 + 1 / BLOCK)


def work(case: dict) -> dict:
    c, m = case, case["rows"]
    if c["kind"] == "quantize":
        return {"bytes": 4 * m * c["k"], "flops": 0}                     # the values in, the values they are rounded to out
    if c["kind"] == "matmul":
        n, k = c["n"], c["k"]
        return {"bytes": _weight_bytes(n, k) + 2 * m * k + (4 if c["f32"] else 2) * m * n, "flops": 2 * m * n * k}
    e, d, w, t = c["experts"], c["hidden"], c["width"], c["top_k"]
    touched = e * (1 - (1 - t / e) ** m)                                 # experts that see a row, in expectation
    return {"bytes": touched * 3 * _weight_bytes(w, d) + 4 * m * d + 8 * m * t, "flops": 2 * m * t * 3 * w * d}
