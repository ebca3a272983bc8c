"""The dense operators against plain implementations in 64 bits.

Tolerances count roundings.  A result rounded once to type t is off by at most finfo(t).eps / 2 of its value;
a float sum of n terms, each thread adding e of them in turn before a tree of at most 16 levels, by at most
(e + 16) * 2^-24 of the sum of the terms' magnitudes; one float operation by 2^-24 of its result."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from flyvec_b200 import ops  # noqa: E402
from flyvec_b200.engine import DeviceArray  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def half_step(t):
    return torch.finfo(TYPES[t] if isinstance(t, str) else t).eps / 2


# below the normal range a float16 is off by half its smallest step instead of half a relative one
def floor_step(t):
    f = torch.finfo(TYPES[t] if isinstance(t, str) else t)
    return f.smallest_normal * f.eps / 2


def made(shape, dtype, seed, pad=0, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    wide = torch.randn(*shape[:-1], shape[-1] + pad, generator=g, device="cuda") * scale + shift
    return wide.to(TYPES[dtype])[..., : shape[-1]]


def close(got, want, tol):
    """|got - want| <= tol element by element; infinities and NaN in the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), "NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), "infinities in other places"
    fine = ~(inf | want.isnan())
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"off by {over.max().item():.3e} more than allowed"


def rounded(want, dtype, slack):
    """Tolerance of a value known to `slack` before it is rounded to dtype."""
    return slack * (1 + half_step(dtype)) + want.abs() * half_step(dtype) + floor_step(dtype)


# ---- layer norm ------------------------------------------------------------------------------------
def norm_reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = ((c * c).mean(-1, keepdim=True) + eps).rsqrt()
    h = c * rstd
    y = h
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean[..., 0], rstd[..., 0], h


def norm_slack(x, w, b, eps):
    """How far y, mean and rstd may be off before the last rounding."""
    d = x.shape[-1]
    e = max(32, math.ceil(d / 512)) + 16
    x64 = x.double()
    y, mean, rstd, h = norm_reference(x, w, b, eps)
    mean_off = (e + 2) * U * x64.abs().mean(-1)
    # (x - mean): its own rounding and the mean's error.  The variance is Q / n - m^2 with Q and m summed about a pivot no more
    # than a standard deviation from the mean: Q / n <= 2 var off by e + 4 roundings, m^2 <= var by twice m's e + 1 roundings of
    # up to sqrt(2 var): (2 (e + 4) + 3 (e + 1) + 9) U together, halved by the root
    var = 1 / rstd ** 2
    rstd_rel = ((5 * e + 20) * U + (mean_off ** 2 + 4 * U * mean_off * x64.abs().amax(-1)) / var) / 2 + 4 * U
    ww = w.double().abs() if w is not None else 1.0
    slack = (mean_off * rstd)[..., None] * ww + (x64.abs() * rstd[..., None] * ww) * U + (h * ww).abs() * (rstd_rel[..., None] + 3 * U)
    if b is not None:
        slack = slack + y.abs() * U
    return slack, mean_off, rstd_rel


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 400), (5, 7), (3, 256), (2, 257), (700, 1000), (700, 1024), (129, 1001), (601, 513), (4, 4096),
                                       (3, 4097), (2, 8200), (3, 16384), (2, 20001)])
def test_layer_norm(built_lib, rows, cols, dtype):
    for pad, affine, shift in ((0, True, 0.3), (8, True, 30.0), (3, False, 0.0)):
        x = made((rows, cols), dtype, rows + cols, pad, 1.5, shift)
        w = made((cols,), dtype, 2, 0, 0.2, 1.0) if affine else None
        b = made((cols,), dtype, 3) if affine else None
        y, mean, rstd = ops.layer_norm(x, w, b, eps=1e-5, return_stats=True)
        want, m, r, _ = norm_reference(x, w, b, 1e-5)
        slack, mo, rr = norm_slack(x, w, b, 1e-5)
        assert y.dtype == x.dtype and y.is_contiguous()
        close(y, want, rounded(want, dtype, slack))
        close(mean, m, mo + m.abs() * U)
        close(rstd, r, r * (rr + U))
        assert torch.equal(ops.layer_norm(x, w, b, eps=1e-5), y)
        for out in TYPES:
            got = ops.layer_norm(x, w, b, eps=1e-5, out_dtype=out)
            assert got.dtype == TYPES[out]
            close(got, want, rounded(want, out, slack))


def test_layer_norm_shapes_and_weights(built_lib):
    x = made((2, 3, 5, 64), "bfloat16", 1)
    w = made((64,), "bfloat16", 2)
    y, mean, rstd = ops.layer_norm(x, w, return_stats=True)
    assert y.shape == x.shape and mean.shape == rstd.shape == (2, 3, 5)
    assert torch.equal(y.reshape(-1, 64), ops.layer_norm(x.reshape(-1, 64), w))
    assert ops.layer_norm(x[:0], w).shape == (0, 3, 5, 64)
    one = ops.layer_norm(x[0, 0, 0], w)
    assert one.shape == (64,) and torch.equal(one, y[0, 0, 0])
    same = x[0, 0, :1].expand(7, 64)  # rows at distance 0
    assert torch.equal(ops.layer_norm(same, w), y[0, 0, :1].expand(7, 64))
    bad = x[0, 0].clone()
    bad[1, 5], bad[2, 6] = math.nan, math.inf
    got = ops.layer_norm(bad, w)
    assert got[1].isnan().all() and got[2].isnan().any() and torch.equal(got[0], y[0, 0, 0]) and torch.equal(got[3], y[0, 0, 3])
    flat = torch.full((3, 64), 7.0, device="cuda")  # no variance: eps alone
    assert (ops.layer_norm(flat) == 0).all()
    for n in (64, 1000, 4096, 4097):  # elements far out where the pivot is taken, or everywhere but there
        for lo, hi in ((0, 8), (0, 16), (16, n)):
            far = torch.randn(2, n, device="cuda")
            far[:, lo:hi] += 1000.0
            w2, s2 = norm_reference(far, None, None, 1e-5)[0], norm_slack(far, None, None, 1e-5)[0]
            close(ops.layer_norm(far), w2, rounded(w2, "float32", s2))
    # rows off the 16-byte boundary are read element by element: the sums associate differently, each within the bound
    wide = torch.randn(9, 1000 + 1, device="cuda")[:, 1:]
    want, slack = norm_reference(wide, None, None, 1e-5)[0], norm_slack(wide, None, None, 1e-5)[0]
    close(ops.layer_norm(wide), want, rounded(want, "float32", slack))
    close(ops.layer_norm(wide.contiguous()), want, rounded(want, "float32", slack))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 400), (5, 7), (1237, 1001), (3000, 256), (2000, 1024), (37, 4096), (900, 2048), (5, 9000),
                                       (3, 16384), (70, 20001)])
def test_layer_norm_backward(built_lib, rows, cols, dtype):
    for pad, affine in ((0, True), (3, True), (8, False)):
        x, dy = made((rows, cols), dtype, rows + cols, pad, 1.5, 0.3), made((rows, cols), dtype, 5, pad)
        w = made((cols,), dtype, 2, 0, 0.2, 1.0) if affine else None
        _, mean, rstd, _ = norm_reference(x, None, None, 1e-5)
        mean, rstd = mean.float(), rstd.float()
        dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
        g, m, r = dy.double(), mean.double()[:, None], rstd.double()[:, None]
        h = (x.double() - m) * r
        u = g * w.double() if affine else g
        a, q = u.mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
        want = r * (u - a - h * q)
        e = max(32, math.ceil(cols / 512)) + 20
        h_off = U * (x.double().abs() + m.abs()) * r + 2 * U * h.abs()
        a_off = e * U * u.abs().mean(1, keepdim=True)
        q_off = e * U * (u * h).abs().mean(1, keepdim=True) + (u.abs() * h_off).mean(1, keepdim=True)
        slack = r * (a_off + h.abs() * q_off + q.abs() * h_off + 5 * U * (u.abs() + a.abs() + (h * q).abs()))
        close(dx, want, rounded(want, dtype, slack))
        if not affine:
            assert dw is None and db is None
            continue
        n = rows + 24  # no more additions than that follow one another
        close(db, g.sum(0), rounded(g.sum(0), dtype, n * U * g.abs().sum(0)))
        close(dw, (g * h).sum(0), rounded((g * h).sum(0), dtype, n * U * (g * h).abs().sum(0) + (g.abs() * h_off).sum(0)))
        again = ops.layer_norm_backward(dy, x, mean, rstd, w)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw) and torch.equal(again[2], db)


def test_layer_norm_backward_against_differences(built_lib):
    """The formula itself: central differences of the forward definition in 64 bits."""
    x, dy, w = made((3, 12), "float32", 1), made((3, 12), "float32", 2), made((12,), "float32", 3)
    b = torch.zeros(12, device="cuda")
    _, mean, rstd = ops.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    f = lambda xx, ww, bb: (norm_reference(xx, ww, bb, 1e-5)[0] * dy.double()).sum()  # noqa: E731
    for k, (arg, grad) in enumerate(((x, dx), (w, dw), (b, db))):
        num = torch.zeros(arg.numel(), dtype=torch.float64, device="cuda")
        for i in range(arg.numel()):
            d = torch.zeros(arg.numel(), dtype=torch.float64, device="cuda")
            d[i] = 1e-5
            args = [x.double(), w.double(), b.double()]
            args[k] = args[k] + d.reshape(arg.shape)
            up = f(*args)
            args[k] = args[k] - 2 * d.reshape(arg.shape)
            num[i] = (up - f(*args)) / 2e-5
        # differences: h^2 times a third derivative of order 10, and float roundings of the kernel
        assert (grad.double().reshape(-1) - num).abs().max() < 1e-5


def test_layer_norm_backward_empty(built_lib):
    x = torch.empty(0, 5, device="cuda")
    s = torch.empty(0, device="cuda")
    dx, dw, db = ops.layer_norm_backward(x, x, s, s, torch.ones(5, device="cuda"))
    assert dx.shape == (0, 5) and (dw == 0).all() and (db == 0).all()


# ---- log probabilities -----------------------------------------------------------------------------
def lp_reference(logits, targets, beta, top):
    s = beta * logits.double()
    bad = (logits.isnan() | (logits == math.inf)).any(-1)
    empty = (logits == -math.inf).all(-1)
    m = logits.double().amax(-1)
    d = torch.where(empty[:, None], s, s - beta * m[:, None])
    # the largest element's 1 apart from the rest: 1 + 1e-25 would be 1 in 64 bits too
    rest = d.exp().scatter(1, d.max(-1, keepdim=True)[1], 0.0).sum(-1)
    lz = torch.where(empty, torch.full_like(m, -math.inf), torch.log1p(rest))
    lp = torch.where(empty[:, None], s, d - lz[:, None])
    h = lz - torch.where(d > -700, d.exp() * d, torch.zeros_like(d)).sum(-1) / (1 + rest)
    h = torch.where(empty, torch.zeros_like(h), h)
    V = logits.shape[1]
    t = targets.long()
    lt = lp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
    lt = torch.where(t == -1, torch.zeros_like(lt), torch.where((t < 0) | (t >= V), torch.full_like(lt, math.nan), lt))
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top]
    nan = torch.full_like(m, math.nan)
    fix = lambda v: torch.where(bad if v.dim() == 1 else bad[:, None], nan if v.dim() == 1 else nan[:, None], v)  # noqa: E731
    return dict(log_prob=torch.where(t == -1, torch.zeros_like(lt), fix(lt)), entropy=fix(h), row_max=fix(m), log_z=fix(lz), top_ids=ids,
                top_log_prob=fix(lp.gather(1, ids)))


def lp_check(logits, targets, beta=1.0, top=0):
    V = logits.shape[1]
    r = ops.token_log_probs(logits, targets, beta=beta, top=top)
    w = lp_reference(logits, targets, beta, top)
    # exp of an argument d: ex2 is good to 2^-22, its argument to 2 |d| U; the largest |d| that counts is below 90; sums as
    # above with V / 256 elements a thread (its rescalings add one operation each), log1p to 4 U
    e = (max(32, V / 256) + 30) * U + 2 ** -22
    lz = w["log_z"].nan_to_num(0, 0, 0)
    # An exponent d carries four roundings (log2(e), beta log2(e), x - max, their product), which move exp(d) by 4 U |d|: R, the sum
    # without the largest element, by 4 U R times the mean of |d| over that sum.  H = log(1 + R) + R mean|d| / (1 + R) gives
    # the mean; in a nearly certain row (R = 2e-25 from d = -57) it is 57 however small H is.
    rest = torch.expm1(lz)
    mean_d = torch.where(rest > 0, (w["entropy"].nan_to_num(0) - lz) * (1 + rest) / rest.clamp_min(1e-300), torch.zeros_like(lz))
    typical = e + 4 * U * mean_d.clamp_min(1)
    lz_off = typical * -torch.expm1(-lz) + 4 * U * lz.abs()
    close(r.row_max, w["row_max"], 0.0)
    close(r.log_z, w["log_z"], lz_off)
    h = w["entropy"].nan_to_num(0)
    close(r.entropy, w["entropy"], 4 * lz_off + (2 * typical + 8 * U) * h)
    lp = w["log_prob"].nan_to_num(0, 0, 0)
    close(r.log_prob, w["log_prob"], lz_off + 4 * U * (lp.abs() + lz))
    if top:
        assert r.top_ids.dtype == torch.int32
        assert torch.equal(r.top_ids.long(), w["top_ids"])
        tl = w["top_log_prob"].nan_to_num(0, 0, 0)
        close(r.top_log_prob, w["top_log_prob"], lz_off[:, None] + 4 * U * (tl.abs() + lz[:, None]))
    else:
        assert r.top_ids is None and r.top_log_prob is None
    again = ops.token_log_probs(logits, targets, beta=beta, top=top)
    for a, b in zip(r, again):
        assert a is None or torch.equal(a.nan_to_num(1e30), b.nan_to_num(1e30))
    return r


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (6, 31), (5, 128), (4, 129), (9, 512), (300, 1000), (2, 1024), (7, 1025), (3, 2047), (1, 4099), (1, 20000),
                                    (40, 20001), (300, 8192), (2, 50001), (1, 131072)])
def test_token_log_probs(built_lib, rows, V, dtype):
    for pad, beta, top in ((0, 1.0, min(V, 20)), (3, 0.7, 0), (8, 2.5, min(V, 64)), (1, 1.0, 1)):
        x = made((rows, V), dtype, rows + V + top, pad, 2.0)
        g = torch.Generator(device="cuda")
        g.manual_seed(V)
        t = torch.randint(0, V, (rows,), generator=g, device="cuda")
        if rows > 3:
            t[1], t[2], t[3] = -1, V, -7
        lp_check(x, t if top % 2 else t.int(), beta, top)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [5, 700, 1500, 20000, 50001])
def test_token_log_probs_masks_and_ties(built_lib, V, dtype):
    lowest = torch.finfo(TYPES[dtype]).min
    x = made((16, V), dtype, V, 0, 2.0)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    hide = torch.rand(16, V, generator=g, device="cuda") < 0.95
    x[0] = -math.inf                      # nothing left
    x[1] = -math.inf
    x[1, V // 2] = 1.5                    # one word left
    x[2].masked_fill_(hide[2], -math.inf)
    x[3].masked_fill_(hide[3], lowest)    # masked by the type's lowest value
    x[4] = lowest
    x[5] = 0.25                           # all equal
    x[6] = torch.arange(V, device="cuda") * (100.0 / V)   # ascending
    x[7] = -x[6]
    x[8, 1:3] = math.nan
    x[9, V - 1] = math.inf
    x[10] = (x[10] * 2).round() / 2       # many ties
    x[11] = -math.inf
    x[11, : V // 3] = 3.0                 # a masked tail, the rest equal
    x[12, ::2], x[12, 1::2] = 0.0, -0.0   # equal to each other
    x[13] = math.nan
    x[14] = x[14] * 0 - 1e4
    x[14, 0] = 1e4                        # certain
    x[15, 2] = 60.0                       # nearly certain
    t = torch.randint(0, V, (16,), generator=g, device="cuda")
    t[1] = V // 2
    t[15] = 2
    lp_check(x, t, 1.0, min(V, 20))
    lp_check(x, t, 0.5, min(V, 64))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_token_log_probs_crowded_threads(built_lib, dtype):
    """More candidates than a block holds: large elements sit where few threads read, distinct and all equal."""
    V, vec = 70000, 128 // torch.finfo(TYPES[dtype]).bits
    rows = torch.zeros(4, V, device="cuda")
    rows += torch.randn(4, V, device="cuda")
    slot = (torch.arange(V, device="cuda") // vec) % 256
    few = slot < 20
    n = int(few.sum())
    assert n > 1024
    rows[0, few] = 50 + torch.arange(n, device="cuda") * (50.0 / n)
    rows[1, few] = 77.0
    rows[2, few] = 100 - torch.arange(n, device="cuda") * (50.0 / n)
    rows[3, few] = math.nan
    x = rows.to(TYPES[dtype])
    t = torch.tensor([0, 1, V - 1, 5], device="cuda")
    many = x.repeat(80, 1)  # rows enough for one block each
    for top in (1, 20, 64):
        lp_check(x[:3], t[:3], 1.0, top)
        lp_check(many, t.repeat(80), 1.0, top)


def lp_grad_reference(x, t, beta, r, g, gh):
    V = x.shape[1]
    empty = r.log_z == -math.inf
    lp = beta * (x.double() - r.row_max.double()[:, None]) - r.log_z.double()[:, None]
    lp = torch.where(empty[:, None], torch.full_like(lp, -math.inf), lp)
    p = lp.exp()
    one = torch.zeros_like(p)
    one.scatter_(1, t.long().clamp(0, V - 1)[:, None], 1.0)
    gg = torch.where((t == -1) | empty, torch.zeros_like(g), g).double()
    d = gg[:, None] * (one - p)
    size = gg.abs()[:, None] * torch.where(one > 0, (one - p).abs(), p)
    if gh is not None:
        ent = torch.special.xlogy(p, p) + p * r.entropy.double()[:, None]
        d = d - gh.double()[:, None] * ent
        size = size + gh.double().abs()[:, None] * (torch.special.xlogy(p, p).abs() + p * r.entropy.double()[:, None].abs())
    return beta * d, beta * size


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (9, 33), (300, 1000), (2, 1024), (7, 1025), (3, 9001), (37, 20000), (5, 50001), (1, 131072)])
def test_token_log_probs_backward(built_lib, rows, V, dtype):
    for pad, beta, entropy in ((0, 1.0, True), (3, 0.7, False), (8, 2.5, True)):
        x = made((rows, V), dtype, rows + V, pad, 2.0)
        g = torch.Generator(device="cuda")
        g.manual_seed(V)
        t = torch.randint(0, V, (rows,), generator=g, device="cuda")
        if rows > 4:
            x[1] = -math.inf
            x[2, ::2] = -math.inf
            x[3] = torch.finfo(TYPES[dtype]).min
            x[4, 0], t[4] = 200.0, 0  # certain: the token's own 1 - p
            t[0] = -1
        r = ops.token_log_probs(x, t, beta=beta)
        gl = torch.randn(rows, generator=g, device="cuda")
        gh = torch.randn(rows, generator=g, device="cuda") if entropy else None
        got = ops.token_log_probs_backward(gl, x, t, r.row_max, r.log_z, r.entropy, grad_entropy=gh, beta=beta)
        assert got.dtype == x.dtype and got.is_contiguous()
        want, size = lp_grad_reference(x, t, beta, r, gl, gh)
        # p: its exponent is good to 4 U of |lp| + log_z (below 110 where p counts), ex2 to 2^-22; then ten operations.  Where
        # 1 - p is small its error is that of the exponent, relative to it
        lp = (beta * (x.double() - r.row_max.double()[:, None])).abs().clamp_max(110).nan_to_num(110)
        rel = 4 * U * (lp + r.log_z.double().abs().nan_to_num(0, 0, 0)[:, None]) + 2.0 ** -22 + 12 * U
        extra = 4 * U * beta * gl.double().abs()[:, None] * (torch.arange(V, device="cuda")[None] == t[:, None]) * \
            r.log_z.double().abs().nan_to_num(0, 0, 0)[:, None]
        # p below 2^-126 counts as 0
        close(got, want, rounded(want, dtype, rel * size + extra + 2.0 ** -119 * (1 + gl.abs().double()[:, None])))
        if entropy:
            t2 = torch.full_like(t, -1)
            none = ops.token_log_probs_backward(gl, x, t2, r.row_max, r.log_z, beta=beta)
            assert (none == 0).all()


def test_token_log_probs_backward_bad_rows(built_lib):
    x = made((4, 1500), "float32", 1)
    x[1, 3] = math.nan
    t = torch.tensor([2, 2, 1500, -3], device="cuda")
    r = ops.token_log_probs(x, t)
    d = ops.token_log_probs_backward(torch.ones(4, device="cuda"), x, t, r.row_max, r.log_z)
    assert not d[0].isnan().any() and d[1:].isnan().all()


def test_token_log_probs_backward_against_differences(built_lib):
    x = made((3, 10), "float32", 7)
    t = torch.tensor([1, 9, 4], device="cuda")
    gl, gh = torch.tensor([0.5, -1.0, 2.0], device="cuda"), torch.tensor([1.0, 0.3, -0.7], device="cuda")
    r = ops.token_log_probs(x, t, beta=0.8)
    got = ops.token_log_probs_backward(gl, x, t, r.row_max, r.log_z, r.entropy, grad_entropy=gh, beta=0.8)

    def f(v):
        w = lp_reference(v, t, 0.8, 1)
        return (w["log_prob"] * gl.double()).sum() + (w["entropy"] * gh.double()).sum()

    num = torch.zeros(30, dtype=torch.float64, device="cuda")
    for i in range(30):
        d = torch.zeros(30, dtype=torch.float64, device="cuda")
        d[i] = 1e-5
        num[i] = (f(x.double() + d.view(3, 10)) - f(x.double() - d.view(3, 10))) / 2e-5
    assert (got.double().reshape(-1) - num).abs().max() < 1e-5


def test_token_log_probs_shapes(built_lib):
    x = made((2, 3, 2000), "bfloat16", 1)
    t = torch.randint(0, 2000, (2, 3), device="cuda")
    r = ops.token_log_probs(x, t, top=5)
    assert r.log_prob.shape == r.entropy.shape == (2, 3) and r.top_ids.shape == r.top_log_prob.shape == (2, 3, 5)
    shifted = torch.randint(0, 2000, (2, 4), device="cuda")[:, 1:]  # not contiguous
    lp = ops.token_log_probs(x, shifted).log_prob
    assert torch.equal(lp, ops.token_log_probs(x, shifted.contiguous()).log_prob)
    none = ops.token_log_probs(x[:0], t[:0], top=5)
    assert none.log_prob.shape == (0, 3) and none.top_ids.shape == (0, 3, 5)
    d = ops.token_log_probs_backward(none.log_prob, x[:0], t[:0], none.row_max, none.log_z)
    assert d.shape == (0, 3, 2000)


# ---- matrix product --------------------------------------------------------------------------------
ACTS = {"none": lambda z: z, "relu": torch.relu, "gelu": lambda z: 0.5 * z * torch.erfc(-z / math.sqrt(2)), "silu": lambda z: z * torch.sigmoid(z),
        "gelu_tanh": lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}


def weight(outer, inner, dtype, seed, flip):
    w = made((inner, outer) if flip else (outer, inner), dtype, seed, 0, inner ** -0.5)
    return w.t() if flip else w


def product_slack(a, b, depth):
    """Float accumulation of exact products: a step of 16 terms (one for the scalar form: counted alike) adds to the running sum
    with at most 2^-22 of the magnitudes gathered so far; partial sums of up to 8 blocks are added after that."""
    return (depth / 16 + 12) * 2.0 ** -22 * (a.double().abs() @ b.double().abs())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,inner,outer", [(1, 400, 1000), (1, 7, 3), (2, 64, 130), (3, 4097, 65), (4, 5000, 257), (4, 9000, 40), (3, 2048, 1000), (4, 4096, 512), (4, 1032, 90), (1, 400, 20000), (5, 64, 128),
                                              (5, 1, 1), (17, 130, 300), (33, 501, 127), (64, 400, 4000), (64, 2048, 264), (65, 64, 64), (127, 65, 129),
                                              (128, 128, 256), (129, 1000, 257), (300, 63, 1003), (777, 501, 1003), (1000, 2048, 512), (2500, 136, 1600)])
def test_linear(built_lib, rows, inner, outer, dtype):
    for k, (act, bias, residual, out, pad, flip) in enumerate((("none", False, False, dtype, 0, False), ("gelu", True, True, dtype, 3, False),
                                                               ("silu", True, False, "float32", 8, True), ("relu", False, True, "float32", 0, True),
                                                               ("gelu_tanh", True, True, dtype, 0, False))):
        x, w = made((rows, inner), dtype, 1 + k, pad), weight(outer, inner, dtype, 7 + k, flip)
        b = made((outer,), dtype, 3, 0, 0.5) if bias else None
        r = made((rows, outer), dtype, 4, pad) if residual else None
        got, z = ops.linear(x, w, b, activation=act, residual=r, out_dtype=out, return_preactivation=True)
        assert got.dtype == TYPES[out] and got.shape == (rows, outer) and z.dtype == x.dtype
        want = x.double() @ w.double().t()
        slack = product_slack(x, w.t(), inner)
        if bias:
            want = want + b.double()
            slack = slack + want.abs() * U
        close(z, want, rounded(want, dtype, slack))
        y = ACTS[act](want)
        # slopes are below 1.13; the activation itself: an exp and a quotient, 2^-20 of its value with arguments below 32, and
        # for the gelu the published bound of its erf, 1.5e-7, times z / 2
        s = 1.13 * slack + y.abs() * 2.0 ** -20 * (act != "none") + want.abs() * 7.5e-8 * (act == "gelu")
        if residual:
            y = y + r.double()
            s = s + y.abs() * U
        close(got, y, rounded(y, out, s))
        assert torch.equal(ops.linear(x, w, b, activation=act, residual=r, out_dtype=out), got)
    assert ops.device_status() == 0


def test_linear_special_values_and_shapes(built_lib):
    x, w = made((200, 72), "bfloat16", 1), made((136, 72), "bfloat16", 2)
    x[3, 5], x[7, 9] = math.nan, math.inf
    got = ops.linear(x, w)
    want = x.double() @ w.double().t()
    assert torch.equal(got.isnan(), want.isnan()) and got[3].isnan().all()
    assert ops.linear(x, w, activation="relu")[3].isnan().all()
    x3 = made((2, 5, 3, 72), "bfloat16", 3)
    assert torch.equal(ops.linear(x3, w).reshape(-1, 136), ops.linear(x3.reshape(-1, 72), w))
    assert ops.linear(x3[:0], w).shape == (0, 5, 3, 136)
    v = ops.linear(x3[0, 0, 0], w)
    assert v.shape == (136,)
    xt = made((72, 200), "bfloat16", 4).t()  # x stored the other way round
    for n in (2, 40, 200):
        assert torch.equal(ops.linear(xt[:n], w), ops.linear(xt[:n].contiguous(), w)) or n <= 4
        close(ops.linear(xt[:n], w), xt[:n].double() @ w.double().t(),
              rounded(xt[:n].double() @ w.double().t(), "bfloat16", product_slack(xt[:n], w.t(), 72)))
    row = made((1, 72), "bfloat16", 5).expand(90, 72)  # a broadcast row
    got = ops.linear(row, w)
    assert torch.equal(got, got[:1].expand(90, 136))
    res = made((1, 136), "bfloat16", 6)
    assert torch.equal(ops.linear(x3[0, 0], w, residual=res.expand(3, 136)), ops.linear(x3[0, 0], w, residual=res.repeat(3, 1)))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,inner,outer", [(1, 16, 16), (1, 401, 33), (3, 64, 200), (50, 136, 72), (128, 64, 64), (129, 257, 131), (777, 501, 1003),
                                              (2000, 400, 1000), (5000, 72, 264)])
def test_linear_backward(built_lib, rows, inner, outer, dtype):
    for k, (act, pad, flip) in enumerate((("none", 0, False), ("gelu", 0, False), ("silu", 3, True), ("gelu_tanh", 8, False), ("relu", 0, True), ("none", 3, False))):
        x, w = made((rows, inner), dtype, 1 + k, pad), weight(outer, inner, dtype, 7 + k, flip)
        dy = made((rows, outer), dtype, 5, pad)
        z = made((rows, outer), dtype, 6, pad, 2.0) if act != "none" else None
        dx, dw, db = ops.linear_backward(dy, x, w, preactivation=z, activation=act)
        dz = dy.double()
        off = torch.zeros_like(dz)
        if act != "none":
            zz = z.double().requires_grad_()
            dz, = torch.autograd.grad(ACTS[act](zz), zz, dy.double())
            # the slope: sums of terms up to 1.13 + |z| / 2 in magnitude, each good to 2^-20 (erf: 1.5e-7 / 2)
            off = dy.double().abs() * 2.0 ** -20 * (2 + z.double().abs())
        dz16 = off + dz.abs() * half_step(dtype) + floor_step(dtype) if act != "none" else off  # as the products see it
        want = dz @ w.double()
        close(dx, want, rounded(want, dtype, dz16 @ w.double().abs() + product_slack(dz.abs() + dz16, w, outer)))
        want = dz.t() @ x.double()
        close(dw, want, rounded(want, dtype, dz16.t() @ x.double().abs() + product_slack((dz.abs() + dz16).t(), x, rows)))
        want = dz.sum(0)
        close(db, want, rounded(want, dtype, off.sum(0) + (rows / 8 + 40) * U * dz.abs().sum(0)))
        again = ops.linear_backward(dy, x, w, preactivation=z, activation=act)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw) and torch.equal(again[2], db)
    assert ops.device_status() == 0


def test_linear_backward_empty(built_lib):
    x, w = torch.empty(0, 24, device="cuda", dtype=torch.bfloat16), made((40, 24), "bfloat16", 1)
    dx, dw, db = ops.linear_backward(torch.empty(0, 40, device="cuda", dtype=torch.bfloat16), x, w)
    assert dx.shape == (0, 24) and (dw == 0).all() and (db == 0).all()


# ---- how the operators are used ------------------------------------------------------------------------
def test_arrays_without_pytorch(built_lib):
    """The same calls on DeviceArray."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((37, 400)).astype(np.float32)
    a = DeviceArray.from_numpy(x)
    y, mean, rstd = ops.layer_norm(a, return_stats=True)
    t = torch.from_numpy(x).cuda()
    ty, tm, tr = ops.layer_norm(t, return_stats=True)
    assert isinstance(y, DeviceArray) and y.shape == (37, 400)
    np.testing.assert_array_equal(y.numpy(), ty.cpu().numpy())
    np.testing.assert_array_equal(rstd.numpy(), tr.cpu().numpy())
    w = rng.standard_normal((90, 400)).astype(np.float32)
    xb, wb = DeviceArray.from_numpy(x, "bfloat16"), DeviceArray.from_numpy(w, "bfloat16")
    np.testing.assert_array_equal(xb.numpy(), t.bfloat16().float().cpu().numpy())  # rounded to nearest even
    tw = torch.from_numpy(w).cuda().bfloat16()
    s, ts = ops.linear(xb, wb, out_dtype="float32"), ops.linear(t.bfloat16(), tw, out_dtype="float32")
    np.testing.assert_array_equal(s.numpy(), ts.cpu().numpy())
    dy = DeviceArray.from_numpy(rng.standard_normal((37, 90)), "bfloat16")
    for got, want in zip(ops.linear_backward(dy, xb, wb), ops.linear_backward(torch.from_numpy(dy.numpy()).cuda().bfloat16(), t.bfloat16(), tw)):
        np.testing.assert_array_equal(got.numpy(), want.float().cpu().numpy())
    ids = rng.integers(0, 90, 37)
    r, tr_ = ops.token_log_probs(s, DeviceArray.from_numpy(ids), top=5), ops.token_log_probs(ts, torch.from_numpy(ids).cuda(), top=5)
    for got, want in zip(r, tr_):
        np.testing.assert_array_equal(got.numpy(), want.cpu().numpy())
    one = DeviceArray.from_numpy(np.ones(37, np.float32))
    d = ops.token_log_probs_backward(one, s, DeviceArray.from_numpy(ids), r.row_max, r.log_z, r.entropy, grad_entropy=one)
    td = ops.token_log_probs_backward(torch.ones(37, device="cuda"), ts, torch.from_numpy(ids).cuda(), tr_.row_max, tr_.log_z, tr_.entropy,
                                      grad_entropy=torch.ones(37, device="cuda"))
    np.testing.assert_array_equal(d.numpy(), td.cpu().numpy())
    with pytest.raises(TypeError, match="first argument"):
        ops.layer_norm(a, torch.ones(400, device="cuda"))
    half = DeviceArray.from_numpy(np.array([1.5, np.nan, -np.inf], np.float32), "float16").numpy()
    assert half.dtype == np.float16 and half[0] == 1.5 and np.isnan(half[1]) and half[2] == -np.inf


def head_forward(p, x, t):
    """A readout: norm, hidden layer with a residual around it, norm, vocabulary, the token's log probability."""
    h0, m0, r0 = ops.layer_norm(x, p["g0"], p["b0"], return_stats=True)
    h1, z1 = ops.linear(h0, p["w1"], p["c1"], activation="gelu", residual=x, return_preactivation=True)
    h2, m2, r2 = ops.layer_norm(h1, p["g2"], p["b2"], return_stats=True)
    s = ops.linear(h2, p["w3"], p["c3"])
    return ops.token_log_probs(s, t, top=3), (h0, m0, r0, h1, z1, h2, m2, r2, s)


def head_backward(p, x, t, r, saved, g):
    h0, m0, r0, h1, z1, h2, m2, r2, s = saved
    ds = ops.token_log_probs_backward(g, s, t, r.row_max, r.log_z)
    d = {}
    dh2, d["w3"], d["c3"] = ops.linear_backward(ds, h2, p["w3"])
    dh1, d["g2"], d["b2"] = ops.layer_norm_backward(dh2, h1, m2, r2, p["g2"])
    dh0, d["w1"], d["c1"] = ops.linear_backward(dh1, h0, p["w1"], preactivation=z1, activation="gelu")
    dx, d["g0"], d["b0"] = ops.layer_norm_backward(dh0, x, m0, r0, p["g0"])
    return dx + dh1, d


def head_problem(n=300, K=136, V=1003, seed=1):
    p = {"g0": made((K,), "bfloat16", seed, 0, 0.2, 1.0), "b0": made((K,), "bfloat16", seed + 1, 0, 0.2), "w1": made((K, K), "bfloat16", seed + 2, 0, K ** -0.5),
         "c1": made((K,), "bfloat16", seed + 3, 0, 0.2), "g2": made((K,), "bfloat16", seed + 4, 0, 0.2, 1.0), "b2": made((K,), "bfloat16", seed + 5, 0, 0.2),
         "w3": made((V, K), "bfloat16", seed + 6, 0, K ** -0.5), "c3": made((V,), "bfloat16", seed + 7, 0, 0.2)}
    x = made((n, K), "bfloat16", seed + 8)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = torch.randint(0, V, (n,), generator=g, device="cuda")
    t[::17] = -1
    return p, x, t


def test_a_run_of_them_together(built_lib):
    p, x, t = head_problem()
    r, saved = head_forward(p, x, t)
    up = torch.full((300,), 1.0 / 300, device="cuda")
    dx, d = head_backward(p, x, t, r, saved, up)
    # the same in 64 bits with automatic differentiation
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    x64 = x.double().requires_grad_()
    F = torch.nn.functional
    h = F.layer_norm(x64, (136,), q["g0"], q["b0"])
    h = ACTS["gelu"](h @ q["w1"].t() + q["c1"]) + x64
    h = F.layer_norm(h, (136,), q["g2"], q["b2"])
    lp = F.log_softmax(h @ q["w3"].t() + q["c3"], -1)
    want = lp.gather(1, t.clamp_min(0)[:, None])[:, 0].masked_fill(t < 0, 0.0)
    want.mean().backward()
    # a chain of bfloat16 values: each of the 5 tensors between the operators is off by 2^-9 of its size, a logit of size about 3 by
    # a few of these together
    assert (r.log_prob.double() - want).abs().max() < 10 * 3 * 2.0 ** -8
    for k, v in list(d.items()) + [("x", dx)]:
        g = x64.grad if k == "x" else q[k].grad
        rel = ((v.double() - g).norm() / g.norm()).item()
        assert rel < 10 * 2.0 ** -8, (k, rel)


def test_captured_and_replayed(built_lib):
    """A training step captured once and replayed on new inputs gives what the calls give; two graphs share nothing."""
    p, x, t = head_problem()
    p2, x2, t2 = head_problem(n=300, seed=50)
    up = torch.full((300,), 1.0 / 300, device="cuda")
    run = lambda pp, xx, tt: (lambda r, s: (r.log_prob, *head_backward(pp, xx, tt, r, s, up)[1].values()))(*head_forward(pp, xx, tt))  # noqa: E731
    want1, want2 = run(p, x, t), run(p2, x2, t2)
    sx, st = x.clone(), t.clone()
    sx2, st2 = x2.clone(), t2.clone()
    run(p, sx, st)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = run(p, sx, st)
    with torch.cuda.graph(g2):
        out2 = run(p2, sx2, st2)
    for _ in range(2):
        g1.replay()
        g2.replay()
    g1.replay()
    torch.cuda.synchronize()
    for a, b in list(zip(out1, want1)) + list(zip(out2, want2)):
        assert torch.equal(a, b)
    x3 = made((300, 136), "bfloat16", 99)
    sx.copy_(x3)
    g1.replay()
    torch.cuda.synchronize()
    for a, b in zip(out1, run(p, x3, t)):
        assert torch.equal(a, b)


def test_streams(built_lib):
    """Work goes to the current stream; calls on two streams at once do not disturb each other."""
    p, x, t = head_problem(n=2000)
    p2, x2, t2 = head_problem(n=2000, seed=50)
    want, want2 = head_forward(p, x, t)[0], head_forward(p2, x2, t2)[0]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(5):
        with torch.cuda.stream(a):
            outs.append((head_forward(p, x, t)[0], want))
        with torch.cuda.stream(b):
            outs.append((head_forward(p2, x2, t2)[0], want2))
    torch.cuda.synchronize()
    for r, w in outs:
        for u, v in zip(r, w):
            assert torch.equal(u, v)
    # a slow producer on a side stream: the call waits for it because it runs on the same stream
    with torch.cuda.stream(a):
        big = torch.zeros(4000, 4000, device="cuda")
        for _ in range(20):
            big = big @ big
        z = x * 2 + big[0, 0].bfloat16()
        got = ops.layer_norm(z)
    torch.cuda.synchronize()
    assert torch.equal(got, ops.layer_norm(x * 2))


def test_rows_behind_the_last_stay_as_they_were(built_lib):
    """Outputs lie in larger buffers where the allocator puts them: nothing beyond their ends is written."""
    import ctypes as C

    from flyvec_b200 import _lib

    lib = _lib.lib()
    for rows, inner, outer in ((129, 64, 96), (130, 64, 103), (5, 64, 200), (2, 64, 30), (300, 4096, 300)):
        x, w = made((rows, inner), "bfloat16", 1), made((outer, inner), "bfloat16", 2)
        buf = torch.full((rows * outer + 512,), 7.0, device="cuda", dtype=torch.bfloat16)
        st = torch.cuda.current_stream().cuda_stream
        assert lib.fv_linear(0, st, x.data_ptr(), inner, 1, w.data_ptr(), inner, 1, rows, inner, outer, 1, None, 0, None, 0, buf.data_ptr(), 1, None,
                             None, 0) == 0
        assert (buf[rows * outer:] == 7).all()
        assert torch.equal(buf[: rows * outer].view(rows, outer), ops.linear(x, w))
    for cols in (400, 1001, 4097):
        x = made((9, cols), "bfloat16", 3)
        buf = torch.full((9 * cols + 512,), 7.0, device="cuda", dtype=torch.bfloat16)
        assert lib.fv_layer_norm(0, torch.cuda.current_stream().cuda_stream, x.data_ptr(), cols, 9, cols, 1, None, None, 1e-5, buf.data_ptr(), 1,
                                 None, None) == 0
        assert (buf[9 * cols:] == 7).all() and torch.equal(buf[: 9 * cols].view(9, cols), ops.layer_norm(x))


def test_tensors_that_need_gradients(built_lib):
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="detach"):
        ops.layer_norm(x)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x), ops.layer_norm(x.detach()))
    par = torch.nn.Parameter(torch.ones(8, device="cuda"), requires_grad=False)
    assert torch.equal(ops.layer_norm(x.detach(), par), ops.layer_norm(x.detach()))
    neg = torch.view_as_complex(torch.randn(3, 8, 2, device="cuda")).conj().imag
    assert neg.is_neg()
    with pytest.raises(ValueError, match="negated|contiguous"):
        ops.layer_norm(neg)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(built_lib):
    p, x, t = head_problem()
    want = head_forward(p, x, t)[0]
    got = head_forward({k: v.to("cuda:1") for k, v in p.items()}, x.to("cuda:1"), t.to("cuda:1"))[0]
    for a, b in zip(got, want):
        assert a.device.index == 1 and torch.equal(a.cpu(), b.cpu())


# ---- words by their dense embeddings ---------------------------------------------------------------------
def test_window_activations(built_lib):
    from flyvec_b200 import _lib, synth
    from flyvec_b200.engine import Hasher

    W = synth.make_weights(70, 2 * 90, seed=3)
    h = Hasher(W)
    rng = np.random.default_rng(1)
    idx = rng.integers(-1, 180, (50, 7)).astype(np.int32)
    ext = np.concatenate([W.astype(np.float64), np.zeros((70, 1))], 1)  # -1 is padding
    np.testing.assert_array_equal(h.activations(idx).numpy(), ext[:, idx].sum(-1).T.astype(np.float32))
    assert h.activations(np.zeros((0, 3), np.int32)).shape == (0, 70)
    with pytest.raises(_lib.FlyvecError, match="out of range"):
        h.activations(np.array([[180]]))
    with pytest.raises(ValueError):
        h.activations(np.zeros(3, np.int32))
    h.close()


def test_word_log_probs_and_similar_words(built_lib, tmp_path):
    from flyvec_b200 import FlyVec, synth

    K, V = 64, 500
    W = synth.make_weights(K, 2 * V, seed=2)
    W[:, V + 8] = W[:, V + 7] + 0.1 * W[:, V + 9]  # a near twin of word 7
    np.save(tmp_path / "syn.npy", W)
    (tmp_path / "vocab.txt").write_text("\n".join(["<UNK>"] + [f"w{i}" for i in range(1, V)]))
    (tmp_path / "config.yaml").write_text("synapses: syn.npy\ntokenizer: vocab.txt\n")
    m = FlyVec.from_config(tmp_path / "config.yaml")
    rng = np.random.default_rng(5)
    idx = rng.integers(0, V, (40, 4)).astype(np.int32)
    words = rng.integers(0, V, 40)
    words[3] = -1
    r = m.word_log_probs(idx, words, beta=12.0, top=5)
    z = lambda a: (a - a.mean(1, keepdims=True)) / a.std(1, keepdims=True)  # noqa: E731
    corr = z(W[:, idx].sum(-1).T.astype(np.float64)) @ z(W[:, V:].T.astype(np.float64)).T / K
    s = 12.0 * corr
    lse = np.log(np.exp(s - s.max(1, keepdims=True)).sum(1)) + s.max(1)
    want = np.where(words < 0, 0.0, s[np.arange(40), words] - lse)
    # standardised values are rounded to bfloat16: a product of two is off by 2^-8 of its size at most, their sum of K such by
    # 2^-8 of the sum of their magnitudes, at most 1 in units of the correlation (Cauchy and Schwarz); the maximum may move as much
    tol = 2 * 12.0 * 2.0 ** -8 * 1.01
    assert np.abs(r.log_prob - want).max() < tol
    assert r.top_ids.shape == (40, 5)
    best = np.take_along_axis(s, r.top_ids.astype(np.int64), 1)
    assert (best[:, -1] >= np.sort(s, 1)[:, -5] - tol).all()
    near = m.similar_words("w7", top=4)
    assert len(near) == 4 and near[0][0] == "w8" and all(a[1] >= b[1] for a, b in zip(near, near[1:])) and "w7" not in dict(near)
    assert m.similar_words("nothere") == []
    with pytest.raises(ValueError):
        m.word_log_probs(idx, words[:3])


def test_two_host_threads(built_lib):
    """Calls from two threads at once, each on its own stream."""
    import threading

    problems = [head_problem(n=500, seed=s) for s in (1, 70)]
    want = [head_forward(*p)[0] for p in problems]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k].append(head_forward(*problems[k])[0])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001  reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))


def test_small_workspaces_are_refused(built_lib):
    """A workspace that does not hold what the size function answers ends the call before anything is launched."""
    import ctypes as C

    lib, n = built_lib, C.c_size_t(0)
    x, w = made((300, 63), "bfloat16", 1), made((40, 63), "bfloat16", 2)
    y = torch.zeros(300, 40, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(1 << 20, device="cuda", dtype=torch.uint8)
    st = torch.cuda.current_stream().cuda_stream
    assert lib.fv_linear_workspace(300, 63, 40, x.data_ptr(), 63, 1, w.data_ptr(), 63, 1, C.byref(n)) == 0 and n.value > 0
    args = (0, st, x.data_ptr(), 63, 1, w.data_ptr(), 63, 1, 300, 63, 40, 1, None, 0, None, 0, y.data_ptr(), 1, None)
    assert lib.fv_linear(*args, ws.data_ptr(), n.value - 256) == 1 and b"workspace" in lib.fv_last_error()
    assert lib.fv_linear(*args, None, 0) == 1
    assert (y == 0).all()
    assert lib.fv_linear(*args, ws.data_ptr(), n.value) == 0 and torch.equal(y, ops.linear(x, w))
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(40, device="cuda", dtype=torch.bfloat16)
    assert lib.fv_linear_backward_workspace(0, 300, 63, 40, y.data_ptr(), 40, x.data_ptr(), 63, 1, w.data_ptr(), 63, 1, 0, C.byref(n)) == 0
    back = (0, st, y.data_ptr(), 40, x.data_ptr(), 63, 1, w.data_ptr(), 63, 1, 300, 63, 40, 1, None, 0, 0, dx.data_ptr(), dw.data_ptr(), db.data_ptr())
    assert lib.fv_linear_backward(*back, ws.data_ptr(), n.value - 1) == 1 and b"workspace" in lib.fv_last_error()
    assert lib.fv_linear_backward(*back, ws.data_ptr(), n.value) == 0
    s = torch.zeros(300, device="cuda")
    g = torch.ones(63, device="cuda", dtype=torch.bfloat16)
    assert lib.fv_layer_norm_backward_workspace(0, 300, 63, 1, C.byref(n)) == 0
    norm = (0, st, x.data_ptr(), 63, x.data_ptr(), 63, 300, 63, 1, s.data_ptr(), s.data_ptr(), g.data_ptr(), dx.data_ptr(), g.data_ptr(), g.data_ptr())
    assert lib.fv_layer_norm_backward(*norm, ws.data_ptr(), n.value - 4) == 1 and b"workspace" in lib.fv_last_error()
