"""What the dense operators refuse, before anything reaches a GPU: arguments of the Python functions (stand-ins for
arrays are enough) and of the C entry points."""
import ctypes as C
import math

import numpy as np
import pytest

from flyvec_b200 import _lib, ops
from flyvec_b200.engine import DeviceArray


class Fake(DeviceArray):
    """A device array without memory: a shape, a type, strides."""

    def __init__(self, shape, dtype="float32", stride=None, device=0):
        self.shape, self.dtype, self.device, self.ptr = tuple(shape), dtype, device, None
        self.size = math.prod(self.shape)
        self._stride = stride

    def stride(self):
        return self._stride or super().stride()

    def data_ptr(self):
        raise AssertionError("the refusal came too late")

    def new_empty(self, shape, dtype):
        raise AssertionError("the refusal came too late")


def test_layer_norm_refuses(built_lib):
    x, w = Fake((3, 8)), Fake((8,))
    for args, kw, error, text in [
        ((np.zeros((3, 8), np.float32),), {}, TypeError, "DeviceArray or a CUDA tensor"),
        ((Fake((3, 8), "int32"),), {}, TypeError, "types"),
        ((Fake((3, 0)),), {}, ValueError, "no columns"),
        ((Fake(()),), {}, ValueError, "at least one axis"),
        ((Fake((3, 8), stride=(1, 3)),), {}, ValueError, "contiguous"),
        ((Fake((2, 3, 8), stride=(100, 8, 1)),), {}, ValueError, "common distance"),
        ((x, None, w), {}, ValueError, "a bias needs a weight"),
        ((x, Fake((7,))), {}, ValueError, "8 elements"),
        ((x, Fake((8,), "bfloat16")), {}, TypeError, "weight"),
        ((x, Fake((8,), device=1)), {}, ValueError, "device 1"),
        ((x, w), {"eps": -1e-5}, ValueError, "eps"),
        ((x, w), {"eps": math.nan}, ValueError, "eps"),
        ((x, w), {"out_dtype": "float64"}, TypeError, "out_dtype"),
    ]:
        with pytest.raises(error, match=text):
            ops.layer_norm(*args, **kw)
    s = Fake((3,))
    for args, error, text in [
        ((Fake((3, 7)), x, s, s, w), ValueError, "dy must have shape"),
        ((Fake((3, 8), "float16"), x, s, s, w), TypeError, "dy"),
        ((x, x, Fake((4,)), s, w), ValueError, "mean must have 3"),
        ((x, x, s, Fake((3,), "float16"), w), TypeError, "rstd"),
        ((x, Fake((3, 0)), s, s), ValueError, "no columns"),
    ]:
        with pytest.raises(error, match=text):
            ops.layer_norm_backward(*args)


def test_linear_refuses(built_lib):
    b = "bfloat16"
    x, w = Fake((3, 8), b), Fake((5, 8), b)
    for args, kw, error, text in [
        ((Fake((3, 8)), w), {}, TypeError, "x must have one of the types"),
        ((x, Fake((5, 8), "float16")), {}, TypeError, "weight"),
        ((x, Fake((5, 7), b)), {}, ValueError, "8 columns, the weight 7"),
        ((x, Fake((5, 8, 1), b)), {}, ValueError, r"\[outer, inner\]"),
        ((x, Fake((0, 8), b)), {}, ValueError, "empty"),
        ((Fake((3, 0), b), Fake((5, 0), b)), {}, ValueError, "empty"),
        ((Fake((3, 8), b, stride=(16, 2)), w), {}, ValueError, "contiguous"),
        ((x, w, Fake((4,), b)), {}, ValueError, "5 elements"),
        ((x, w, Fake((5,))), {}, TypeError, "bias"),
        ((x, w), {"activation": "swish"}, ValueError, "activation"),
        ((x, w), {"out_dtype": "float16"}, TypeError, "out_dtype"),
        ((x, w), {"residual": Fake((3, 8), b)}, ValueError, "residual must have shape"),
        ((x, w), {"residual": Fake((3, 5), b, stride=(1, 3))}, ValueError, "residual must be contiguous"),
    ]:
        with pytest.raises(error, match=text):
            ops.linear(*args, **kw)
    dy = Fake((3, 5), b)
    for args, kw, error, text in [
        ((Fake((3, 6), b), x, w), {}, ValueError, "dy must have shape"),
        ((Fake((3, 5), b, stride=(0, 0)), x, w), {}, ValueError, "dy must be contiguous"),
        ((dy, x, w), {"activation": "gelu"}, ValueError, "needs the pre-activation"),
        ((dy, x, w), {"activation": "gelu", "preactivation": Fake((3, 4), b)}, ValueError, "preactivation must have shape"),
        ((dy, x, w), {"activation": "gelu", "preactivation": Fake((3, 5))}, TypeError, "preactivation"),
    ]:
        with pytest.raises(error, match=text):
            ops.linear_backward(*args, **kw)


def test_token_log_probs_refuses(built_lib):
    x, t = Fake((3, 50)), Fake((3,), "int64")
    for args, kw, error, text in [
        ((Fake((3, 50), "int32"), t), {}, TypeError, "logits"),
        ((Fake((3, 0)), t), {}, ValueError, "empty"),
        ((x, Fake((4,), "int64")), {}, ValueError, "3 elements"),
        ((x, Fake((3, 1), "int64")), {}, ValueError, "targets must have shape"),
        ((x, Fake((3,))), {}, TypeError, "targets"),
        ((x, t), {"beta": 0.0}, ValueError, "beta"),
        ((x, t), {"beta": math.inf}, ValueError, "beta"),
        ((x, t), {"beta": math.nan}, ValueError, "beta"),
        ((x, t), {"top": 51}, ValueError, "top"),
        ((x, t), {"top": -1}, ValueError, "top"),
        ((Fake((3, 500)), t), {"top": 65}, ValueError, "top"),
    ]:
        with pytest.raises(error, match=text):
            ops.token_log_probs(*args, **kw)
    f = Fake((3,))
    for args, kw, error, text in [
        ((Fake((2,)), x, t, f, f), {}, ValueError, "grad_log_prob must have 3"),
        ((Fake((3,), "bfloat16"), x, t, f, f), {}, TypeError, "grad_log_prob"),
        ((f, x, t, f, f), {"grad_entropy": f}, ValueError, "needs the entropy"),
        ((f, x, t, f, f), {"beta": -1.0}, ValueError, "beta"),
    ]:
        with pytest.raises(error, match=text):
            ops.token_log_probs_backward(*args, **kw)


def test_tensors_off_the_gpu_and_with_gradients(built_lib):
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="on a GPU"):
        ops.layer_norm(torch.zeros(3, 8))
    with pytest.raises(ValueError, match="on a GPU"):
        ops.token_log_probs(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64))


def test_c_entry_points_refuse(built_lib):
    """Bad arguments come back as FV_ERR_INVALID with a message, before a device is looked for."""
    lib, p = built_lib, C.c_void_p(4096)

    def refused(status, text):
        assert status == 1 and text in lib.fv_last_error().decode(), (status, lib.fv_last_error())

    refused(lib.fv_layer_norm(0, None, p, 8, 3, 0, 0, None, None, 1e-5, p, 0, None, None), "shape")
    refused(lib.fv_layer_norm(0, None, p, -8, 3, 8, 0, None, None, 1e-5, p, 0, None, None), "stride")
    refused(lib.fv_layer_norm(0, None, p, 8, 3, 8, 7, None, None, 1e-5, p, 0, None, None), "element type")
    refused(lib.fv_layer_norm(0, None, p, 8, 3, 8, 0, None, p, 1e-5, p, 0, None, None), "bias needs a weight")
    refused(lib.fv_layer_norm(0, None, p, 8, 3, 8, 0, None, None, -1.0, p, 0, None, None), "eps")
    refused(lib.fv_layer_norm(0, None, None, 8, 3, 8, 0, None, None, 1e-5, p, 0, None, None), "NULL")
    refused(lib.fv_layer_norm_backward(0, None, p, 8, p, 8, 3, 8, 0, p, p, p, p, None, None, None, 0), "go with a weight")
    refused(lib.fv_layer_norm_backward(0, None, p, 8, p, 8, 3, 8, 0, None, p, None, p, None, None, None, 0), "NULL")
    n = C.c_size_t(7)
    refused(lib.fv_layer_norm_backward_workspace(0, -1, 8, 0, C.byref(n)), "bad argument")
    refused(lib.fv_linear(0, None, p, 8, 1, p, 8, 1, 3, 8, 5, 0, None, 0, None, 0, p, 0, None, None, 0), "bfloat16 or float16")
    refused(lib.fv_linear(0, None, p, 8, 1, p, 8, 1, 3, 8, 5, 1, None, 0, None, 0, p, 2, None, None, 0), "output")
    refused(lib.fv_linear(0, None, p, 8, 1, p, 8, 1, 3, 8, 5, 1, None, 9, None, 0, p, 1, None, None, 0), "activation")
    refused(lib.fv_linear(0, None, p, 8, 2, p, 8, 1, 3, 8, 5, 1, None, 0, None, 0, p, 1, None, None, 0), "contiguous")
    refused(lib.fv_linear(0, None, p, 8, 1, p, 8, 1, 3, 0, 5, 1, None, 0, None, 0, p, 1, None, None, 0), "shape")
    refused(lib.fv_linear(0, None, p, 8, 1, p, 8, 1, 3, 8, 5, 1, None, 0, None, 0, None, 1, None, None, 0), "NULL")
    refused(lib.fv_linear(0, None, p, 8, 1, p, 8, 1, 3, 8, 5, 1, None, 0, None, 0, p, 1, None, C.c_void_p(4100), 64), "aligned")
    refused(lib.fv_linear_workspace(3, 8, 5, p, 8, 2, p, 8, 1, C.byref(n)), "contiguous")
    refused(lib.fv_linear_backward(0, None, p, 5, p, 8, 1, p, 8, 1, 3, 8, 5, 1, None, 0, 2, p, None, p, None, 0), "NULL")
    refused(lib.fv_token_log_probs(0, None, p, 50, 3, 50, 0, p, 1, 1.0, 65, p, p, p, p, p, p), "top")
    refused(lib.fv_token_log_probs(0, None, p, 50, 3, 50, 0, p, 1, 0.0, 0, p, p, p, p, None, None), "beta")
    refused(lib.fv_token_log_probs(0, None, p, 50, 3, 50, 0, p, 1, 1.0, 5, p, p, p, p, None, None), "NULL")
    refused(lib.fv_token_log_probs_backward(0, None, p, p, p, 50, 3, 50, 0, p, 1, p, p, None, 1.0, p), "NULL")
    refused(lib.fv_ops_status(0, None), "NULL")
    # nothing to do is no error
    assert lib.fv_layer_norm(0, None, None, 8, 0, 8, 0, None, None, 1e-5, None, 0, None, None) == 0
    assert lib.fv_token_log_probs(0, None, None, 50, 0, 50, 0, None, 1, 1.0, 0, None, None, None, None, None, None) == 0


def test_workspace_sizes(built_lib):
    """Operands whose rows start on 16-byte boundaries need none; others are copied with rows of a multiple of 8."""
    lib, n = built_lib, C.c_size_t(99)

    def size(rows, inner, outer, x, xr, w, wr):
        assert lib.fv_linear_workspace(rows, inner, outer, C.c_void_p(x), xr, 1, C.c_void_p(w), wr, 1, C.byref(n)) == 0
        return n.value

    up = lambda b: (b + 255) // 256 * 256  # noqa: E731
    assert size(100, 64, 32, 0, 64, 0, 64) == 0
    assert size(100, 63, 32, 0, 63, 0, 63) == up(100 * 64 * 2) + up(32 * 64 * 2)
    assert size(100, 64, 32, 2, 64, 0, 64) == up(100 * 64 * 2)
    assert size(100, 64, 32, 0, 67, 0, 64) == up(100 * 64 * 2)
    assert size(100, 64, 32, 0, 0, 0, 64) == up(100 * 64 * 2)  # a broadcast row
    assert size(2, 63, 32, 0, 63, 0, 63) == 0  # few rows: plain loads
    assert size(0, 63, 32, 0, 63, 0, 63) == 0
