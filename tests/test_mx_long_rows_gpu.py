"""Microscaled experts whose inputs are so long that a decode block holds one item's rows at a time (from 6500 inputs or so), or none,
so that a kernel of their own quantises them (past 12288)."""

import pytest
import torch

import mx_util
import test_mx_experts_gpu as base
from tensorfold_b200 import _lib

pytestmark = pytest.mark.gpu

# experts, D, NI, SwiGLU, limit
LONG = [(5, 7168, 64, True, 0.0), (4, 12288, 32, False, 0.0), (3, 12800, 32, True, 1.0), (3, 12320, 64, False, 0.0)]


@pytest.mark.parametrize("case", LONG)
def test_work_of_decode_items(case):
    need = _lib.lib().tf_mx_experts_bytes(case[1], 16, 4)
    assert (need == 0) == (case[1] <= 12288)


@pytest.mark.parametrize("case", LONG)
@pytest.mark.parametrize("rows,prefill", [(1, False), (7, False), (40, False), (40, True)])
def test_long_rows_track_float64(case, rows, prefill):
    base.test_layer_tracks_float64(case, rows, prefill)


@pytest.mark.parametrize("case", LONG)
def test_long_rows_do_not_depend_on_the_window_or_the_plan(case):
    ex, _, _ = base.build(case, 11)
    rows = 60
    x = mx_util.rows(rows, ex.dims, 1, base.DEV, std=0.5)
    x[20, 5] = float("nan")
    picks = base.picks_for(rows, 3, ex.count, 3)
    same = lambda a, b: torch.equal(a.nan_to_num(0.5), b.nan_to_num(0.5)) and torch.equal(torch.isnan(a), torch.isnan(b))
    want = base.run(x, ex, picks, True)
    for m, prefill in ((60, False), (1, False), (3, False), (17, False), (33, True)):
        got = base.run(x[:m], ex, picks[:m], prefill)
        assert all(same(a, b[:m * 3]) for a, b in zip(got, want)), (m, prefill)
    assert bool(torch.isnan(want[2][60:63]).all()) and int(torch.isnan(want[2]).any(1).sum()) == 3 and _lib.device_error(x) == 0
