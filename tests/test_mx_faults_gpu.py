"""Lost waits of the microscaled product come back as error codes: no GPU fault, no block that is stored to after it has left."""

import pytest
import torch

import mx_util
from tensorfold_b200 import _lib
from tensorfold_b200.cuda.kernels import mx

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n,k", [(256, 1024), (256, 2048), (4096, 4096)])
def test_a_lost_slice_leaves_the_context_usable(n, k):
    """One block of a cluster gives up, the others run out of their limit: error 1, and the next product is right."""

    lib = _lib.lib()
    codes, scales = mx_util.random_weight(n, k, 3, DEV)
    q = mx.pack(mx_util.to_words(codes), scales.to(torch.uint8))
    x = mx_util.rows(1, k, 4, DEV)
    want = mx.matmul(x, q, f32=True)
    sk = lib.tf_mx_split(n, k)
    assert sk > 1 and _lib.device_error(x) == 0
    out = torch.empty((1, n), device=DEV)
    for slice in {0, sk - 1}:
        _lib.check(lib.tf_mx_selftest_lost_slice(slice, x.data_ptr(), q.weight.data_ptr(), n, k, out.data_ptr(), _lib.stream_of(x)), "self-test")
        assert _lib.device_error(x) == 1 and _lib.device_error(x) == 0
        assert torch.equal(mx.matmul(x, q, f32=True), want) and _lib.device_error(x) == 0
    assert lib.tf_mx_selftest_lost_slice(sk, x.data_ptr(), q.weight.data_ptr(), n, k, out.data_ptr(), _lib.stream_of(x)) < 0
    assert lib.tf_mx_selftest_lost_slice(0, x.data_ptr(), q.weight.data_ptr(), 17408, 5120, out.data_ptr(), _lib.stream_of(x)) < 0
