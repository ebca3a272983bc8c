"""The dense operators at their edges, as far as no GPU is needed."""
import ctypes as C
import math
import os
import subprocess
from pathlib import Path

import pytest

from flyvec_b200 import ops
from tests import product_shapes
from tests.test_ops_refusals import Fake

ROOT = Path(__file__).resolve().parent.parent


def test_wait_limit_refuses(built_lib):
    assert built_lib.fv_ops_wait_limit(-2) == 1 and b"cycles" in built_lib.fv_last_error()
    assert built_lib.fv_ops_wait_limit(-1) == 0


def test_threads_that_ask_for_different_shared_memory(tmp_path):
    """Whichever thread sets a kernel's limit last, every size that was ever allowed stays allowed."""
    exe = tmp_path / "smem_limit_threads"
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-pthread", f"-I{cuda}/include", f"-I{ROOT}/flyvec_b200/csrc", str(ROOT / "tests" / "smem_limit_threads.cpp"),
                    "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout


def test_row_vectors_of_another_shape_are_refused(built_lib):
    """As many elements in another order: [T, B] for rows [B, T].  One axis for all rows has the rows' order."""
    rows, flat = Fake((2, 3)), Fake((6,))
    x, t, w = Fake((2, 3, 8)), Fake((2, 3), "int64"), Fake((8,))
    for wrong in (Fake((3, 2)), Fake((1, 6)), Fake((2, 3, 1))):
        for args, kw, what in [((x, x, wrong, rows, w), {}, "mean"), ((x, x, rows, wrong, w), {}, "rstd"), ((x, x, rows, wrong), {}, "rstd")]:
            with pytest.raises(ValueError, match=what + " must have shape"):
                ops.layer_norm_backward(*args, **kw)
        with pytest.raises(ValueError, match="targets must have shape"):
            ops.token_log_probs(x, Fake(wrong.shape, "int32"))
        for args, kw, what in [((wrong, x, t, rows, rows), {}, "grad_log_prob"), ((rows, x, t, wrong, rows), {}, "row_max"),
                               ((rows, x, Fake(wrong.shape, "int64"), rows, rows), {}, "targets"), ((rows, x, t, rows, wrong), {}, "log_z"),
                               ((rows, x, t, rows, rows, wrong), {"grad_entropy": rows}, "entropy"),
                               ((rows, x, t, rows, rows, rows), {"grad_entropy": wrong}, "grad_entropy")]:
            with pytest.raises(ValueError, match=what + " must have shape"):
                ops.token_log_probs_backward(*args, **kw)
    for call in (lambda: ops.layer_norm_backward(x, x, flat, flat, w), lambda: ops.token_log_probs_backward(flat, x, t, flat, flat)):
        with pytest.raises(AssertionError, match="too late"):  # it got past the checks
            call()


def test_forward_mode_tensors_are_refused(built_lib):
    """A dual tensor does not require a gradient, yet its tangent would be lost."""
    torch = pytest.importorskip("torch")
    ad = torch.autograd.forward_ad

    class OnGpu(torch.Tensor):
        """A tensor that says it lies on a GPU; nothing may ask where."""

        is_cuda = True

        def get_device(self):
            return 0

        def data_ptr(self):
            raise AssertionError("the refusal came too late")

    made = lambda *shape: torch.randn(*shape).as_subclass(OnGpu)  # noqa: E731
    with ad.dual_level():
        dual = lambda *shape: ad.make_dual(made(*shape), made(*shape))  # noqa: E731
        t = torch.zeros(3, dtype=torch.int64).as_subclass(OnGpu)
        half = lambda x: x.bfloat16()  # noqa: E731
        for call, what in [(lambda: ops.layer_norm(dual(3, 8)), "x"), (lambda: ops.layer_norm(made(3, 8), dual(8)), "weight"),
                           (lambda: ops.layer_norm_backward(dual(3, 8), made(3, 8), made(3), made(3)), "dy"),
                           (lambda: ops.linear(half(dual(3, 8)), half(made(5, 8))), "x"), (lambda: ops.linear(half(made(3, 8)), half(dual(5, 8))), "weight"),
                           (lambda: ops.token_log_probs(dual(3, 8), t), "logits"),
                           (lambda: ops.token_log_probs_backward(dual(3), made(3, 8), t, made(3), made(3)), "grad_log_prob")]:
            with pytest.raises(ValueError, match=f"{what} has a forward-mode tangent"):
                call()


def test_numbers_that_no_float_holds_are_refused(built_lib):
    """Python's floats reach further than the kernels': a beta that becomes 0, or infinite with log2(e), and an infinite eps."""
    x, t, f = Fake((3, 50)), Fake((3,), "int64"), Fake((3,))
    for beta in (3e38, 1e39, 1e-46, 0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="beta"):
            ops.token_log_probs(x, t, beta=beta)
        with pytest.raises(ValueError, match="beta"):
            ops.token_log_probs_backward(f, x, t, f, f, beta=beta)
    for eps in (1e39, math.inf, -1e-5, math.nan):
        with pytest.raises(ValueError, match="eps"):
            ops.layer_norm(x, eps=eps)
    lib, p = built_lib, C.c_void_p(4096)
    assert lib.fv_token_log_probs(0, None, p, 50, 3, 50, 0, p, 1, 3e38, 0, p, p, p, p, None, None) == 1 and b"beta" in lib.fv_last_error()
    assert lib.fv_token_log_probs_backward(0, None, p, None, p, 50, 3, 50, 0, p, 1, p, p, None, 3e38, p) == 1 and b"beta" in lib.fv_last_error()
    assert lib.fv_layer_norm(0, None, p, 8, 3, 8, 0, None, None, math.inf, p, 0, None, None) == 1 and b"eps" in lib.fv_last_error()


def test_similar_words_refuses(tmp_path):
    """Before anything is loaded, with the number the caller gave."""
    from flyvec_b200 import FlyVec

    (tmp_path / "vocab.txt").write_text("<UNK>\nw1\nw2")
    m = FlyVec(tmp_path / "nothing.npy", tmp_path / "vocab.txt")
    for top in (64, 65, 1000, -1, -2):
        with pytest.raises(ValueError, match=f"between 0 and 63, got {top}"):
            m.similar_words("w1", top=top)
    assert m.similar_words("w1", top=0) == [] and m.similar_words("nothere") == []


def test_the_products_sizes_reach_every_form(built_lib):
    """The sizes at which the products are compared with 64 bits take the forms they are listed for."""
    for size, want in product_shapes.FORWARD.items():
        assert product_shapes.shapes(built_lib, product_shapes.SMS, size, False) == [want], size
    for size, want in product_shapes.BACKWARD.items():
        assert product_shapes.shapes(built_lib, product_shapes.SMS, size, True) == want, size
    bad = (C.c_int32 * 7)()
    assert built_lib.fv_linear_shapes(148, 0, 8, 8, 0, bad) == 1 and built_lib.fv_linear_shapes(1, 8, 8, 8, 0, bad) == 1
    assert built_lib.fv_linear_shapes(148, 8, 8, 8, 0, None) == 1
