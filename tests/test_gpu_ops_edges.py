"""The dense operators at their edges: waits that run out, errors and what follows them, threads, streams, far offsets, every
kernel form of the matrix product.  Helpers and the way tolerances are derived are those of test_gpu_ops."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from flyvec_b200 import ops  # noqa: E402
from tests import product_shapes  # noqa: E402
from tests import test_gpu_ops as base  # noqa: E402
from tests.test_gpu_ops import made  # noqa: E402

pytestmark = pytest.mark.gpu


def word_model(path, K, V, weights=None):
    """A model of V words w1, w2, ... in K neurons."""
    from flyvec_b200 import FlyVec, synth

    np.save(path / "syn.npy", synth.make_weights(K, 2 * V, seed=2) if weights is None else weights)
    (path / "vocab.txt").write_text("\n".join(["<UNK>"] + [f"w{i}" for i in range(1, V)]))
    (path / "config.yaml").write_text("synapses: syn.npy\ntokenizer: vocab.txt\n")
    return FlyVec.from_config(path / "config.yaml")


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


FIRST_MEETING = """
import threading
import numpy as np
from flyvec_b200 import ops
from flyvec_b200.engine import DeviceArray

# two widths that one layer-norm kernel takes with different amounts of shared memory, both beyond 48 KB
for dtype, widths in (("bfloat16", (16384, 9000)), ("float16", (16384, 9000)), ("float32", (16384, 9000)), ("bfloat16", (16373, 9001)),
                      ("float16", (16373, 9001)), ("float32", (16381, 9001)), ("float32", (8192, 6000)), ("float32", (8191, 6001))):
    rng = np.random.default_rng(1)
    x = [DeviceArray.from_numpy(rng.standard_normal((4, n)), dtype) for n in widths]
    w = [DeviceArray.from_numpy(np.ones(n), dtype) for n in widths]
    m = DeviceArray.from_numpy(np.zeros(4, np.float32)), DeviceArray.from_numpy(np.ones(4, np.float32))
    gate, got, errors = threading.Barrier(2), {}, []

    def both(k):
        return [a.numpy() for a in (ops.layer_norm(x[k]), *ops.layer_norm_backward(x[k], x[k], *m, w[k]))]

    def work(k):
        gate.wait()
        try:
            got[k] = both(k)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, (dtype, widths, errors)
    for k in (0, 1):
        for a, b in zip(got[k], both(k)):
            np.testing.assert_array_equal(a, b)
assert ops.device_status() == 0
"""


def test_threads_that_meet_a_kernel_first_with_different_widths(built_lib):
    done = subprocess.run([sys.executable, "-c", FIRST_MEETING], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_the_status_waits_for_side_streams(built_lib):
    """PyTorch's streams are non-blocking: the default stream does not wait for them."""
    big = torch.randn(8192, 8192, device="cuda")
    side, end = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = (big @ big) * 1e-4
        end.record()
    assert ops.device_status() == 0
    assert end.query()


def test_word_scores_of_a_wait_that_ran_out_are_an_error(built_lib, tmp_path):
    from flyvec_b200 import _lib

    m = word_model(tmp_path, 64, 500)
    idx, words = np.arange(12, dtype=np.int32).reshape(3, 4), [1, 2, 3]
    m.hasher  # noqa: B018  made beforehand: the waits of the operators alone run out
    try:
        assert built_lib.fv_ops_wait_limit(0) == 0
        with pytest.raises(_lib.FlyvecError, match="FV_ERR_TIMEOUT"):
            m.word_log_probs(idx, words)
    finally:
        assert built_lib.fv_ops_wait_limit(-1) == 0
    again = word_model(tmp_path, 64, 500)
    np.testing.assert_array_equal(m.word_log_probs(idx, words).log_prob, again.word_log_probs(idx, words).log_prob)


def test_word_scores_do_not_depend_on_the_scale_of_the_synapses(built_lib, tmp_path):
    """Correlations: normalised synapses (elements of 1e-2 and less) answer like large ones, a power of two changes no bit."""
    from flyvec_b200 import synth

    K, V = 64, 500
    W = synth.make_weights(K, 2 * V, seed=2)
    W /= np.linalg.norm(W, axis=1, keepdims=True)
    rng = np.random.default_rng(5)
    idx, words = rng.integers(0, V, (40, 4)).astype(np.int32), rng.integers(0, V, 40)
    W[:, idx[7]] = 0.25  # a context without variance
    z = lambda a: (a - a.mean(1, keepdims=True)) / np.maximum(a.std(1, keepdims=True), 1e-12)  # noqa: E731
    s = 12.0 * z(W[:, idx].sum(-1).T.astype(np.float64)) @ z(W[:, V:].T.astype(np.float64)).T / K
    want = s[np.arange(40), words] - np.log(np.exp(s).sum(1))
    # as for the test of the words' log probabilities: a standardised value is rounded to bfloat16
    tol = 2 * 12.0 * 2.0 ** -8 * 1.01
    answers = []
    for k, scale in enumerate((1.0, 2.0 ** -14, 2.0 ** 10)):
        (tmp_path / str(k)).mkdir()
        r = word_model(tmp_path / str(k), K, V, (W * scale).astype(np.float32)).word_log_probs(idx, words, beta=12.0, top=5)
        assert np.abs(r.log_prob - want).max() < tol
        assert abs(r.log_prob[7] + np.log(V)) < 1e-5
        answers.append(r)
    for r in answers[1:]:
        for a, b in zip(r, answers[0]):
            np.testing.assert_array_equal(a, b)


def test_row_vectors_on_one_axis(built_lib):
    """[B, T] rows and their values flat; as many values in [T, B] are refused."""
    x, t = made((2, 3, 500), "float32", 1), torch.randint(0, 500, (2, 3), device="cuda")
    g = made((2, 3), "float32", 2)
    r = ops.token_log_probs(x, t)
    want = ops.token_log_probs_backward(g, x, t, r.row_max, r.log_z)
    assert torch.equal(ops.token_log_probs_backward(g.reshape(-1), x, t, r.row_max.reshape(-1), r.log_z), want)
    with pytest.raises(ValueError, match="grad_log_prob must have shape"):
        ops.token_log_probs_backward(g.t(), x, t, r.row_max, r.log_z)
    _, mean, rstd = ops.layer_norm(x, return_stats=True)
    want = ops.layer_norm_backward(x, x, mean, rstd)[0]
    assert torch.equal(ops.layer_norm_backward(x, x, mean.reshape(-1), rstd)[0], want)
    with pytest.raises(ValueError, match="rstd must have shape"):
        ops.layer_norm_backward(x, x, mean, rstd.t())


def test_forward_mode_tensors(built_lib):
    ad = torch.autograd.forward_ad
    x = made((3, 8), "float32", 1)
    with ad.dual_level():
        with pytest.raises(ValueError, match="x has a forward-mode tangent"):
            ops.layer_norm(ad.make_dual(x, x))
        plain = ops.layer_norm(ad.make_dual(x, x).detach())
    assert torch.equal(plain, ops.layer_norm(x))


def test_calls_after_a_failed_one(built_lib):
    """The runtime's record of a failure reported here does not fail the next launch, neither here nor in PyTorch."""
    from flyvec_b200 import _lib
    from flyvec_b200.engine import DeviceArray

    x = made((4, 8), "float32", 1)
    want, y = ops.layer_norm(x), torch.empty_like(x)

    def call(device):
        return built_lib.fv_layer_norm(device, None, x.data_ptr(), 8, 4, 8, 0, None, None, 1e-5, y.data_ptr(), 0, None, None)

    assert call(99) == 2 and b"device 99" in built_lib.fv_last_error()
    assert call(0) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    assert call(99) == 2
    assert (x + 1).sum().item() == pytest.approx((x.cpu() + 1).sum().item(), rel=1e-4)
    with pytest.raises(_lib.FlyvecError, match="memory"):
        DeviceArray((1 << 40,), "float32")
    assert torch.equal(ops.layer_norm(x), want)
    with pytest.raises(_lib.FlyvecError, match="memory"):
        DeviceArray((1 << 40,), "float32")
    assert torch.equal((x + 1).cpu(), x.cpu() + 1)


def test_log_probs_at_the_ends_of_beta(built_lib):
    """As a maximum (the largest beta) and as an average (the smallest)."""
    x = made((4, 3000), "float32", 1)
    x[1, 7] = x[1].max()
    t = x.argmax(1)
    for v in (x, x[:, :700].contiguous()):
        t = v.argmax(1)
        r = ops.token_log_probs(v, t, beta=2.0 ** 127, top=3)
        ties = (v == v.amax(1, keepdim=True)).sum(1).float()
        assert torch.allclose(r.log_prob, -ties.log(), atol=1e-6) and torch.allclose(r.entropy, ties.log(), atol=1e-6)
        r = ops.token_log_probs(v, t, beta=2.0 ** -149, top=3)
        n = torch.full((4,), float(v.shape[1]), device="cuda").log()
        assert torch.allclose(r.log_prob, -n, atol=1e-5) and torch.allclose(r.entropy, n, atol=1e-5)


def test_similar_words_counts(built_lib, tmp_path):
    m = word_model(tmp_path, 64, 500)
    most = m.similar_words("w7", top=63)
    assert len(most) == 63 and "w7" not in dict(most) and m.similar_words("w7", top=5) == most[:5]
    for top in (65, -1):
        with pytest.raises(ValueError, match=f"got {top}"):
            m.word_log_probs([[1]], [2], top=top)
    (tmp_path / "few").mkdir()
    few = word_model(tmp_path / "few", 64, 12)
    assert len(few.similar_words("w7", top=63)) == 11


@pytest.mark.parametrize("rows,inner,outer", [(1, 501, 1000), (16, 63, 1021), (64, 1001, 777), (3, 4001, 63), (200, 501, 1003)])
def test_linear_backward_of_few_rows_and_large_copies(built_lib, rows, inner, outer):
    """x and the weight are copied to aligned rows in the launch that forms dz, by blocks that go by their own rows."""
    base.test_linear_backward(built_lib, rows, inner, outer, "bfloat16")


def graph_time(call):
    """Microseconds of a call, the least of several replays of twenty."""
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(20):
            call()
    best = float("inf")
    for _ in range(10):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / 20 * 1e3)
    return best


def test_copies_do_not_go_by_the_rows_of_the_gradient(built_lib):
    """16 rows copy the same weight as 777: 13 and 16 us; 41 us when as few blocks copied as 16 rows of dy need."""
    def call(rows):
        x, w, dy = made((rows, 501), "bfloat16", 1), made((1000, 501), "bfloat16", 2), made((rows, 1000), "bfloat16", 3)
        return lambda: ops.linear_backward(dy, x, w)

    assert graph_time(call(16)) < 1.5 * graph_time(call(777))


# ---- every form of the product kernel --------------------------------------------------------------------
@pytest.mark.parametrize("size", list(product_shapes.FORWARD), ids=lambda s: "x".join(map(str, s)))
def test_linear_in_every_form(built_lib, size):
    """With bias, activation, residual and pre-activation, in both types of result; the sums in the order of each form."""
    base.test_linear(built_lib, *size, "float16" if size[0] % 3 == 0 else "bfloat16")


@pytest.mark.parametrize("size", list(product_shapes.BACKWARD), ids=lambda s: "x".join(map(str, s)))
def test_linear_backward_in_every_form(built_lib, size):
    base.test_linear_backward(built_lib, *size, "float16" if size[0] % 3 == 0 else "bfloat16")


def test_the_forms_on_this_gpu(built_lib):
    """With another number of multiprocessors than the sizes were chosen for, some forms may not have run."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    got = {f for size in product_shapes.FORWARD for f in product_shapes.shapes(built_lib, sms, size, False)}
    if sms != product_shapes.SMS:
        pytest.skip(f"{sms} multiprocessors: forms {sorted(got)}")
    assert got == set(product_shapes.FORWARD.values())


# ---- offsets past 2^31 elements --------------------------------------------------------------------------
def far_rows(n, at):
    """Rows at the front, around the one in which element 2^31 lies, at the end."""
    return [slice(0, 700), slice(at - 350, at + 350), slice(n - 700, n)]


def test_layer_norm_of_far_rows(built_lib):
    """A row's result is the same wherever the row lies; 700 rows take the form of all."""
    n, d = 560000, 4096
    x = made((n, d), "bfloat16", 1)
    w = made((d,), "bfloat16", 2, 0, 0.2, 1.0)
    y, mean, rstd = ops.layer_norm(x, w, return_stats=True)
    dx, dw, db = ops.layer_norm_backward(x, y, mean, rstd, w)
    want_b = torch.zeros(d, dtype=torch.float64, device="cuda")
    for a in range(0, n, 40000):
        want_b += x[a:a + 40000].double().sum(0)
    for s in far_rows(n, 2 ** 31 // d):
        part = ops.layer_norm(x[s].clone(), w, return_stats=True)
        assert torch.equal(y[s], part[0]) and torch.equal(mean[s], part[1]) and torch.equal(rstd[s], part[2])
        assert torch.equal(dx[s], ops.layer_norm_backward(x[s].clone(), y[s].clone(), part[1], part[2], w)[0])
    # sums of n normal values (of size sqrt(n)): a block's n / 296 rows one after the other, then a tree, each addition off by
    # 2^-24 of a partial sum of the size of the whole at most, and the rounding to bfloat16
    tol = (n / 296 + 20) * base.U * 4 * n ** 0.5 + want_b.abs() * base.half_step("bfloat16")
    assert ((db.double() - want_b).abs() <= tol).all()


def test_linear_of_far_rows(built_lib):
    def check(x, w, rows):
        y = ops.linear(x, w)
        for s in rows:
            want = x[s].double() @ w.double().t()
            base.close(y[s], want, base.rounded(want, "bfloat16", base.product_slack(x[s], w.t(), x.shape[1])))
        return y

    x, w = made((560000, 4096), "bfloat16", 1), base.weight(72, 4096, "bfloat16", 2, False)
    check(x, w, far_rows(560000, 2 ** 31 // 4096))
    x, w = x[:120000, :64], base.weight(20000, 64, "bfloat16", 3, False)
    y = check(x, w, far_rows(120000, 2 ** 31 // 20000))
    dx, dw, db = ops.linear_backward(y, x, w)
    for s in far_rows(120000, 2 ** 31 // 20000):
        want = y[s].double() @ w.double()
        base.close(dx[s], want, base.rounded(want, "bfloat16", base.product_slack(y[s], w, 20000)))
    del y, dx
    wide = torch.zeros(60, 40_000_000, device="cuda", dtype=torch.bfloat16)  # rows far apart
    wide[:, :136] = made((60, 136), "bfloat16", 4)
    for k in (0, 1):  # read where they lie, and copied
        x = wide[:, k:k + 128]
        for rows in (2, 60):
            for w in (base.weight(72, 128, "bfloat16", 5, False), x):
                assert torch.equal(ops.linear(x[:rows], w), ops.linear(x[:rows].contiguous(), w.contiguous()))


def test_token_log_probs_of_far_rows(built_lib):
    n, v = 120000, 20000
    x = made((n, v), "bfloat16", 1)
    t = torch.arange(n, device="cuda") * 7 % v
    g = made((n,), "float32", 2)
    r = ops.token_log_probs(x, t, top=5)
    d = ops.token_log_probs_backward(g, x, t, r.row_max, r.log_z)
    for s in far_rows(n, 2 ** 31 // v):
        part = ops.token_log_probs(x[s].clone(), t[s], top=5)
        for a, b in zip(r, part):
            assert torch.equal(a[s], b)
        assert torch.equal(d[s], ops.token_log_probs_backward(g[s], x[s].clone(), t[s], part.row_max, part.log_z))
