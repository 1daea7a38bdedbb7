"""Microscaled 4-bit floating point (MXFP4): blocks of 32 inputs with e2m1 codes and one power-of-two scale, quantisation and the
product of quantised rows with quantised weights on the block-scaled tensor cores.

Beside ``qmm`` (affine integers): a checkpoint's words [n, k / 8] and scale bytes [n, k / 32] become an ``MX4`` with ``pack``, and
``matmul`` takes any number of rows.  Rows of x are quantised to the same format inside the call, so both operands of a product
have four bits; sums are fp32.  A row's bits never depend on the row count.  Rounding N(0, 1) rows moves a product by 0.11 of its norm,
as much as rounding N(0, 0.02) weights does; rows with one channel in 64 eight times as large by 0.15.
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from ... import _lib

BLOCK = 32                                       # inputs that share a scale
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_EPILOGUES = {"relu2": 1, "swiglu": 2}


@dataclass
class MX4:
    """A packed (n, k) weight: uint8 super-blocks [ceil(n / 128), bytes] of 128 output columns, codes and scales inside."""

    weight: torch.Tensor
    n: int
    k: int

    def nbytes(self) -> int:
        return self.weight.numel()


def _check_stored(words: torch.Tensor, scales: torch.Tensor, who: str) -> int:
    """K of stored words [.., k / 8] and scales [.., k / 32]."""

    if words.dtype not in (torch.int32, torch.uint32) or scales.dtype != torch.uint8:
        raise ValueError(f"{who}: words must be int32 or uint32, scales uint8")
    if words.dim() < 1 or words.dim() != scales.dim() or words.shape[:-1] != scales.shape[:-1] or words.shape[-1] != 4 * scales.shape[-1]:
        raise ValueError(f"{who}: words {tuple(words.shape)} do not match scales {tuple(scales.shape)} of blocks of {BLOCK}")
    if words.device != scales.device:
        raise ValueError(f"{who}: words and scales must share a device")
    return 8 * words.shape[-1]


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[.., k] bf16, fp16 or fp32 -> (words [.., k / 8] int32, scales [.., k / 32] uint8).  A block's scale is
    2^(floor(log2 of its largest magnitude) - 2), values are rounded to nearest even and saturated at 6 times the scale; a block
    that holds an infinity or a NaN gets the scale NaN (255)."""

    return _lib.native().mx_quantize(x)


def dequantize(words: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``quantize``'s words and scales stand for (exact in fp32, and in bf16 below 2^128)."""

    if dtype not in _TYPES:
        raise ValueError("dequantize: bf16, fp16 or fp32")
    return _lib.native().mx_dequantize(words, scales, _TYPES[dtype])


@lru_cache(maxsize=None)
def super_block_bytes(k: int) -> int:
    return _lib.lib().tf_mx_tiled_bytes(128, k)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def pack_experts(words, scales, up=None) -> torch.Tensor:
    """Stored words [E, n, k / 8] and scales -> super-blocks [E, ceil(n / 128), bytes]; with ``up`` (words, scales of the same
    shape) 2 n rows, gate and up interleaved in tiles of 16."""

    k = _check_stored(words, scales, "pack")
    if words.dim() != 3 or 0 in words.shape:
        raise ValueError("pack: words of n rows and at least one block are wanted")
    e, n, _ = words.shape
    if up is not None:
        if _check_stored(*up, "pack_pair") != k or up[0].shape != words.shape or up[0].device != words.device:
            raise ValueError("pack_pair: gate and up must have the same shapes")
        if n % 16:
            raise ValueError("pack_pair: rows in whole 16-row tiles")
        n *= 2
    stream = _lib.stream_of(words)
    ts = [_aligned(words), _aligned(scales)] + ([_aligned(up[0]), _aligned(up[1])] if up is not None else [None, None])
    out = torch.empty((e, -(-n // 128), super_block_bytes(k)), dtype=torch.uint8, device=words.device)
    _lib.native().tf_mx_pack("pack", *ts, e, n, k, out, stream)
    return out


def pack(words: torch.Tensor, scales: torch.Tensor) -> MX4:
    """Stored (n, k / 8) words and (n, k / 32) scale bytes -> ``MX4``."""

    if words.dim() != 2 or scales.dim() != 2:
        raise ValueError("pack: words and scales must be 2-D")
    return MX4(pack_experts(words[None], scales[None])[0], words.shape[0], words.shape[1] * 8)


def pack_pair(gate: tuple, up: tuple) -> MX4:
    """Gate and up projections (each stored words and scales of n rows) as one weight of 2 n rows for ``matmul_act``."""

    if gate[0].dim() != 2 or gate[1].dim() != 2 or up[0].dim() != 2 or up[1].dim() != 2:
        raise ValueError("pack_pair: words and scales must be 2-D")
    return MX4(pack_experts(gate[0][None], gate[1][None], (up[0][None], up[1][None]))[0], 2 * gate[0].shape[0], gate[0].shape[1] * 8)


def unpack(q: MX4) -> tuple[torch.Tensor, torch.Tensor]:
    """The stored layout again: (n, k / 8) int32 words and (n, k / 32) scale bytes."""

    stream = _lib.stream_of(q.weight)
    words = torch.empty((q.n, q.k // 8), dtype=torch.int32, device=q.weight.device)
    scales = torch.empty((q.n, q.k // BLOCK), dtype=torch.uint8, device=q.weight.device)
    _lib.native().tf_mx_unpack("unpack", _packed(q, "unpack"), q.n, q.k, words, scales, stream)
    return words, scales


def _packed(q: MX4, who: str) -> torch.Tensor:
    w = q.weight
    if w.dtype != torch.uint8 or w.shape != (-(-q.n // 128), super_block_bytes(q.k)) or not w.is_contiguous():
        raise ValueError(f"{who}: the packed weight does not have the super-blocks of its shape")
    return w


def matmul(x: torch.Tensor, q: MX4, *, f32: bool = False, out: torch.Tensor | None = None, pdl: bool = False) -> torch.Tensor:
    """x (M, k) bf16, quantised as by ``quantize``, times q.T as (M, n) bf16, or unrounded fp32 with ``f32``.  ``out`` may not share
    memory with x.

    ``pdl`` launches with programmatic stream serialisation so that the weights' first bytes overlap the end of the previous
    kernel in the stream: they must not be what a kernel still in flight writes."""

    return _lib.native().mx_matmul(x, q, 0, 0.0, f32, out, pdl)


def matmul_act(x: torch.Tensor, q: MX4, *, act: str = "swiglu", limit: float = 0.0, out: torch.Tensor | None = None,
               pdl: bool = False) -> torch.Tensor:
    """``matmul`` with an activation of its fp32 sums: "swiglu" on a ``pack_pair`` weight gives bf16(silu(gate) up) as (M, n / 2),
    clipped first with ``limit``; "relu2" gives bf16(relu(v)^2) as (M, n)."""

    if act not in ("swiglu", "relu2"):
        raise ValueError("matmul_act: act is 'swiglu' or 'relu2'")
    return _lib.native().mx_matmul(x, q, _EPILOGUES[act], limit, False, out, pdl)
