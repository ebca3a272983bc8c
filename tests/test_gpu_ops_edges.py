"""The dense operators at their edges: waits that run out, errors and what follows them, threads, streams, far offsets, every
kernel form of the matrix product.  Helpers and the way tolerances are derived are those of test_gpu_ops."""
import pytest

torch = pytest.importorskip("torch")

from flyvec_b200 import ops  # noqa: E402
from tests.test_gpu_ops import made  # noqa: E402

pytestmark = pytest.mark.gpu


def norm_call(rows, cols, dtype):
    x = made((rows, cols), dtype, 1)
    return lambda: (ops.layer_norm(x),)


def norm_grad_call(rows, cols, dtype):
    x, dy, w = made((rows, cols), dtype, 1), made((rows, cols), dtype, 2), made((cols,), dtype, 3)
    _, mean, rstd = ops.layer_norm(x, return_stats=True)
    return lambda: ops.layer_norm_backward(dy, x, mean, rstd, w)


def linear_call(rows, inner, outer, dtype):
    x, w = made((rows, inner), dtype, 1), made((outer, inner), dtype, 2)
    return lambda: (ops.linear(x, w, activation="gelu"),)


# a warp a row, a block a row, aligned and not; the product by single blocks, by clusters that split the sums, by pairs
@pytest.mark.parametrize("make,sizes", [(norm_call, (3000, 200, "bfloat16")), (norm_call, (300, 4096, "float32")), (norm_call, (300, 4097, "float16")),
                                        (norm_grad_call, (3000, 200, "float32")), (norm_grad_call, (300, 4097, "bfloat16")),
                                        (linear_call, (40, 64, 200, "bfloat16")), (linear_call, (100, 4096, 128, "float16")),
                                        (linear_call, (4100, 1000, 4104, "bfloat16"))])
def test_waits_that_run_out(built_lib, make, sizes):
    """The kernel returns, the status says so once, and the next call is right."""
    call = make(*sizes)
    want = call()
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    try:
        assert built_lib.fv_ops_wait_limit(0) == 0  # gives up at once, with copies in flight
        call()
        torch.cuda.synchronize()
        assert ops.device_status() == 1 and ops.device_status() == 0
        assert built_lib.fv_ops_wait_limit(1) == 0  # gives up somewhere on the way, if a wait takes longer than one look
        got = call()
        torch.cuda.synchronize()
        assert ops.device_status() == 1 or all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        assert built_lib.fv_ops_wait_limit(-1) == 0
    got = call()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert ops.device_status() == 0
