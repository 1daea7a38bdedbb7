"""Microscaled 4-bit floating point without a GPU: the operand layout, sizes, and refused arguments (nothing is launched)."""

import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib
from tensorfold_b200.cuda import mx_experts
from tensorfold_b200.cuda.kernels import mx

ROOT = Path(__file__).resolve().parents[1]


def test_layout_header_is_self_consistent(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("needs a C++ compiler")
    exe = tmp_path / "mx_layout_check"
    subprocess.run([cxx, "-std=c++17", "-O1", str(ROOT / "tests" / "mx_layout_check.cpp"), "-o", str(exe)], check=True, capture_output=True,
                   timeout=120)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.strip().endswith("OK"), done.stdout


def test_sizes():
    lib = _lib.lib()
    assert lib.tf_mx_tiled_bytes(128, 256) == 128 * 256 * 17 // 32
    assert lib.tf_mx_tiled_bytes(17408, 5120) == 17408 * 5120 * 17 // 32            # nothing padded
    assert lib.tf_mx_tiled_bytes(1, 32) == 128 * 32 + 512 and lib.tf_mx_tiled_bytes(129, 64) == 2 * (128 * 32 + 512)
    assert lib.tf_mx_tiled_bytes(0, 32) < 0 and lib.tf_mx_tiled_bytes(8, 48) < 0 and lib.tf_mx_tiled_bytes(8, 0) < 0
    for n, k in ((1, 32), (1024, 5120), (5120, 17408), (17408, 5120), (248320, 5120), (128, 100000)):
        sk = lib.tf_mx_split(n, k)
        assert 1 <= sk <= 6 and sk <= max(1, k // 512)
        assert lib.tf_mx_matmul_bytes(17, n, k) > 0 and lib.tf_mx_matmul_bytes(1, n, k) >= 0
    assert lib.tf_mx_matmul_bytes(1, 17408, 5120) == 0                               # windows need no scratch
    assert lib.tf_mx_split(4, 40) < 0 and lib.tf_mx_matmul_bytes(0, 128, 64) < 0 and lib.tf_mx_experts_bytes(64, 7, 1) < 0


def test_the_oracle_rounds_as_defined():
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 4, [0.0] * 32, [7.9] * 32])
    codes, scales = mx_util.quantize(x)
    assert scales.flatten().tolist() == [127, 0, 127]
    assert mx_util.values(codes, scales)[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 4.0]
    assert mx_util.values(codes, scales)[2, 0] == 6.0
    assert torch.equal(mx_util.to_codes(mx_util.to_words(codes)), codes)


def test_refused_arguments_raise_before_any_launch():
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    words, scales = torch.zeros((64, 16), dtype=torch.int32), torch.zeros((64, 4), dtype=torch.uint8)
    q = mx.MX4(torch.zeros((1, mx.super_block_bytes(128)), dtype=torch.uint8), 64, 128)
    refused = [lambda: mx.quantize(x), lambda: mx.quantize(x.int()), lambda: mx.quantize(x[:, :100]),               # CPU; type; blocks
               lambda: mx.dequantize(words, scales), lambda: mx.dequantize(words, scales[:, :3]), lambda: mx.dequantize(words, scales, torch.int8),
               lambda: mx.pack(words, scales), lambda: mx.pack(words[0], scales[0]), lambda: mx.pack(words.float(), scales),
               lambda: mx.pack_pair((words[:8], scales[:8]), (words[:8], scales[:8])),                                # half a tile
               lambda: mx.pack_pair((words, scales), (words[:32], scales[:32])),
               lambda: mx.matmul(x, q), lambda: mx.matmul(x.float(), q), lambda: mx.matmul(x[:, :64], q), lambda: mx.matmul(x[:0], q),
               lambda: mx.matmul_act(x, q, act="gelu"), lambda: mx.unpack(q),
               lambda: mx_experts.make([(words[None], scales[None])] * 3, (words[None], scales[None])),
               lambda: mx_experts.make([(words[None], scales[None])], (words[None], scales[None]))]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_c_abi_refuses_before_launching():
    """Made-up addresses: every call must be refused, or stop at the missing set-up, before any of them is touched."""

    lib = _lib.lib()
    x, w, out, work = 0x10000, 0x20000, 0x30000, 0x40000

    def call(**kw):
        a = dict(x=x, ldx=128, m=4, w=w, n=64, k=128, out=out, ldo=64, f32=0, epi=0, limit=0.0, work=None, bytes=0, pdl=0)
        a.update(kw)
        return lib.tf_mx_matmul(*a.values(), None)

    for kw in (dict(x=None), dict(w=None), dict(out=None), dict(k=40), dict(k=0), dict(n=0), dict(m=0), dict(ldx=64), dict(ldo=32), dict(epi=3),
               dict(epi=2, n=48), dict(epi=1, f32=1), dict(x=x + 8), dict(ldx=132), dict(w=w + 4), dict(out=out + 1), dict(m=40),
               dict(m=40, work=work, bytes=16)):
        assert call(**kw) < 0, kw
    assert call() != 0 and call(m=40, work=work, bytes=1 << 20) != 0

    def experts(**kw):
        a = dict(x=x, ldx=128, slots=2, w=w, stride=1 << 16, experts=4, n=64, k=128, items=work, counts=work, members=work, pairs=8, max_items=8,
                 tile=16, out=out, ldo=64, f32=0, operands=None, epi=0, limit=0.0, work=None, bytes=0, pdl=0)
        a.update(kw)
        return lib.tf_mx_experts(*a.values(), None)

    for kw in (dict(experts=0), dict(k=40), dict(pairs=0), dict(max_items=0), dict(tile=12), dict(tile=256), dict(out=None),
               dict(operands=work), dict(out=None, operands=work, n=48), dict(items=None), dict(counts=None), dict(members=None), dict(w=None),
               dict(ldx=132), dict(stride=8), dict(ldo=32), dict(tile=128), dict(x=None), dict(epi=2, f32=1), dict(slots=-1)):
        assert experts(**kw) < 0, kw
    assert experts() != 0


def test_sizes_at_the_end_of_an_int_are_refused():
    lib, end = _lib.lib(), 2 ** 31 - 1
    assert lib.tf_mx_matmul_bytes(end, 64, 128) < 0 and lib.tf_mx_matmul_bytes(4, end, 128) < 0 and lib.tf_mx_matmul_bytes(4, 64, end - 31) < 0
    assert lib.tf_mx_tiled_bytes(end, 128) < 0 and lib.tf_mx_tiled_bytes(64, end - 31) < 0 and lib.tf_mx_split(end, 128) < 0
    assert lib.tf_mx_matmul_bytes(1 << 30, 64, 128) > (1 << 30) * 64
    assert lib.tf_mx_matmul_bytes(1, 1, 1 << 30) > 0 and lib.tf_mx_experts_bytes(1 << 30, 16, 4) > 0    # rows too long to be held by a block


def stored(n, k, seed, lead=()):
    codes, scales = mx_util.random_weight(n, k, seed, "cpu", lead=lead)
    return {"weight": mx_util.to_words(codes).view(torch.uint32), "scales": scales.to(torch.uint8)}


def test_checkpoint_shards(tmp_path):
    """Words and scale bytes of a microscaled projection as each rank reads them."""

    from tensorfold_b200.cuda import checkpoint
    from test_checkpoint import write_safetensors

    path = tmp_path / "model.safetensors"
    src, table = stored(96, 256, 1), stored(32, 64, 2, lead=(4,))
    write_safetensors(path, {**{f"q.{k}": v for k, v in src.items()}, **{f"moe.up_proj.{k}": v for k, v in table.items()},
                             "bad.weight": src["weight"], "bad.scales": src["scales"][:, :4].contiguous()}, pad=2)
    ckpt = checkpoint.Checkpoint([path])
    words, scales = src["weight"].view(torch.int32), src["scales"]
    whole = ckpt.microscaled("q")
    assert torch.equal(whole[0], words) and torch.equal(whole[1], scales) and whole[0].dtype == torch.int32
    for rank in range(2):
        w, s = ckpt.microscaled("q", rank=rank, world=2, parallel="column", segments=(64, 32))
        rows = torch.cat([torch.arange(32) + 32 * rank, torch.arange(16) + 64 + 16 * rank])
        assert torch.equal(w, words[rows]) and torch.equal(s, scales[rows])
        w, s = ckpt.microscaled("q", rank=rank, world=2, parallel="row")
        assert torch.equal(w, words[:, 16 * rank:16 * rank + 16]) and torch.equal(s, scales[:, 4 * rank:4 * rank + 4])
        tables, first = checkpoint.expert_tables(ckpt, "moe", ("up_proj",), rank=rank, world=2, parts=("weight", "scales"))
        assert first == 2 * rank and torch.equal(tables["up_proj"][0], table["weight"].view(torch.int32)[first:first + 2])
        assert torch.equal(tables["up_proj"][1], table["scales"][first:first + 2])
    for kw in (dict(world=3, parallel="row"), dict(world=2, parallel="column", segments=(95, 1)), dict(rank=2, world=2), dict(parallel="diagonal")):
        with pytest.raises(ValueError):
            ckpt.microscaled("q", **kw)
    with pytest.raises(ValueError):
        ckpt.microscaled("bad")
    with pytest.raises(KeyError):
        ckpt.microscaled("none")
    ckpt.close()
