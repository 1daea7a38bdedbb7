"""Which buffers a call of ``moe.run`` uses (no GPU: nothing is launched)."""

import pytest
import torch

from tensorfold_b200.cuda import moe


class Cfg:
    num_experts_per_tok, num_experts = 2, 8
    moe_intermediate_size, hidden_size = 64, 32


def test_streams_and_captures_have_buffers_of_their_own(monkeypatch):
    monkeypatch.setattr(moe, "_scratch", {})
    monkeypatch.setattr(moe, "_captured", {})
    made = []

    def make(cleared):
        made.append(cleared)
        return moe.MoEBuffers(4, Cfg, "cpu", cleared=cleared)

    a = moe._kept(("shape",), 1, None, make)
    assert moe._kept(("shape",), 1, None, make) is a and made == [True]
    b = moe._kept(("shape",), 2, None, make)                    # another stream may run beside the first
    assert b is not a and moe._kept(("other",), 1, None, make) not in (a, b)
    first = moe._kept(("shape",), 1, 7, make)                   # a graph may be replayed beside eager calls and other graphs
    assert first not in (a, b) and moe._kept(("shape",), 1, 7, make) is first and not made[-1]
    assert moe._kept(("shape",), 2, 7, make) is not first       # another branch of the same capture
    second = moe._kept(("shape",), 1, 8, make)
    assert second not in (a, b, first)
    assert moe._kept(("shape",), 1, None, make) is a            # eager calls never take what a graph owns
    assert not any(buf is second for _, buf in moe._captured.values())


def test_what_buffers_hold():
    assert moe.MoEBuffers(4, Cfg, "cpu", microscaled=True).act is None and moe.MoEBuffers(4, Cfg, "cpu").act.shape == (4, 3, 64)
    with pytest.raises(ValueError):
        moe.run_experts(None, None, moe.MoEBuffers(4, Cfg, "cpu", microscaled=True), 4)
    for prefill, f32, dtype in ((False, False, torch.float32), (True, False, torch.bfloat16), (True, True, torch.float32)):
        assert moe.MoEBuffers(4, Cfg, "cpu", prefill=prefill, f32=f32).y.dtype == dtype
