"""The score-matrix operators where single rows, columns or sizes lie far from the others: finite masks, masses of zero,
infinite starting potentials, far scores and small temperatures. Against 64-bit formulas, as in test_gpu_scores.py, but with
a tolerance per row and column from that row's or column's own size."""

import math

import pytest
import torch

from trnopt import scores
from test_gpu_scores import GAMMA, INF, TYPES, U, check_gradient, check_log_probs, close, gen, lp_reference, make

pytestmark = pytest.mark.gpu


# balance -------------------------------------------------------------------------------------------------------------

def reference(s, eps, iters, a, b, g):
    """The half-steps in 64 bits. A constant added to a row only moves its f by the same amount back, so each row's largest
    finite score is taken off first; a row or column without terms has potential 0."""
    s = s.double()
    n, e = s.shape
    top = torch.where(torch.isfinite(s), s, -INF).amax(1)
    top = torch.where(top == -INF, 0.0, top)
    s = s - top[:, None]
    la = torch.full((n,), -math.log(n), dtype=torch.float64, device="cuda") if a is None else a.double().log()
    lb = torch.full((e,), -math.log(e), dtype=torch.float64, device="cuda") if b is None else b.double().log()
    g = torch.zeros(e, dtype=torch.float64, device="cuda") if g is None else g.double()
    for _ in range(iters):
        f = -eps * torch.logsumexp(lb + (g + s) / eps, 1)
        f = torch.where(torch.isinf(f), top, f)                  # (0 once the row's constant is back)
        g = -eps * torch.logsumexp(la[:, None] + (f[:, None] + s) / eps, 0)
        g = torch.where(torch.isinf(g), 0.0, g)
    return f - top, g, s


def check(s, eps, iters, a=None, b=None, g=None, far=()):
    """`far`: columns whose scores or potentials lie far from the others'. As in test_gpu_scores.py each of the 2 iters
    half-steps adds the roundings of terms of size z (now over the ordinary columns, relative to each row's largest score)
    and of a sum's chain; a potential itself rounds to float32, and a far column's terms round by their own size."""
    r = scores.balance(s, eps=eps, iters=iters, a=a, b=b, g=g)
    f, w, rest = reference(s, eps, iters, a, b, g)
    near = torch.ones(s.shape[1], dtype=torch.bool, device="cuda")
    near[list(far)] = False
    rest = rest[:, near]
    top = lambda t: torch.where(torch.isfinite(t), t, 0.0).abs().max().item()
    base = rest + f[:, None] * 0
    size = (top(base) + top(w[near]) + (0 if g is None else top(g.double()[near]))) / eps + 16
    tol = U * eps * 2 * iters * (4 * size + GAMMA + max(s.shape) / 32)
    fin = lambda t: torch.where(torch.isfinite(t), t, 0.0).abs()
    close(r.f, f, tol + 8 * U * fin(f), "f")
    close(r.g[near], w[near], tol + 8 * U * fin(w[near]), "g")
    close(r.g[~near], w[~near], tol + 8 * U * fin(w[~near]) + 8 * U * (0 if g is None else fin(g.double()[~near])), "far g")
    return r


SHAPES = [(400, 16), (1000, 24), (20000, 16), (3000, 64), (6000, 200)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("column", [0, 5, -1])
@pytest.mark.parametrize("value,eps,dtype", [(-1e4, 0.1, "f32"), (-65504.0, 0.1, "f16"), (-65504.0, 0.02, "f32"),
                                             (-3.3895e38, 2.0, "bf16")])
def test_balance_masked_column_without_mass(rows, cols, column, value, eps, dtype):
    """A column of mass 0 closed by a large finite score."""
    s = make(rows, cols, TYPES[dtype], seed=rows, scale=1.0)
    s[:, column] = value
    b = torch.full((cols,), 1 / (cols - 1), device="cuda")
    b[column] = 0
    for iters in (1, 2, 8):
        check(s, eps, iters, None, b, far=[column])


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("column", [0, 5])
@pytest.mark.parametrize("value,eps,dtype", [(-1e4, 0.1, "f32"), (-65504.0, 0.1, "bf16"), (3e4, 0.5, "f16")])
def test_balance_far_column_with_mass(rows, cols, column, value, eps, dtype):
    """Its potential makes up for the scores; the others' keep their accuracy."""
    s = make(rows, cols, TYPES[dtype], seed=rows, scale=1.0)
    s[:, column] = value
    for iters in (1, 2, 8):
        check(s, eps, iters, far=[column])
    check(s, eps, 3, g=torch.where(torch.arange(cols, device="cuda") == column, -value, 0.5), far=[column])


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_balance_far_rows(rows, cols, dtype):
    """Rows of nothing but the lowest value or -65504, and rows far above: a row's constant does not move the columns."""
    s = make(rows, cols, TYPES[dtype], seed=rows, scale=1.0)
    s[3::50] = -65504.0
    s[7::50] = torch.finfo(s.dtype).min
    s[9::50] += 30000.0
    s[11::50, 1::2] = torch.finfo(s.dtype).min
    for iters in (1, 2, 8):
        check(s, 0.1, iters)


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_balance_scores_below_the_range_close_a_column(rows, cols):
    """Scores whose multiple by log2(e) / eps passes float32's range are as good as -inf."""
    s = make(rows, cols, torch.bfloat16, seed=rows, scale=1.0)
    b = torch.rand(cols, generator=gen(1), device="cuda") + 0.5
    b[0] = 0
    for column in (0, 5):
        x, y = s.clone(), s.clone()
        x[:, column], y[:, column] = torch.finfo(torch.bfloat16).min, -INF
        for iters in (1, 3):
            u, v = (scores.balance(z, eps=0.1, iters=iters, b=b / b.sum()) for z in (x, y))
            assert torch.equal(u.f, v.f) and torch.equal(u.g, v.g) and u.g[column] == 0


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("iters", [1, 2, 3, 9])
@pytest.mark.parametrize("low", [-25.0, -400.0, 25.0])
def test_balance_zero_masses_far_apart(rows, cols, iters, low):
    """Rows of mass 0 send nothing, however far a column of mass 0 lies above their others; it still gets its potential."""
    s = make(rows, cols, torch.float32, seed=rows, scale=1.0)
    a, b = torch.ones(rows, device="cuda"), torch.ones(cols, device="cuda")
    a[1::7] = 0
    b[[5, cols - 2]] = 0
    s[1::7] += low
    s[1::7, 5] -= low
    check(s, 0.25, iters, a / a.sum(), b / b.sum())


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("start", [-6.0, 0.0, 6.0])
@pytest.mark.parametrize("iters", [1, 2, 7])
def test_balance_rows_open_to_columns_without_mass(rows, cols, start, iters):
    """Rows whose only scores are on columns of mass 0 have potential 0, and their terms reach those columns, whether the
    others' potentials lie far above or below."""
    s = make(rows, cols, torch.float32, seed=rows, scale=0.5)
    b = torch.ones(cols, device="cuda")
    b[[2, 6]] = 0
    shut = torch.ones(cols, dtype=torch.bool, device="cuda")
    shut[[2, 6]] = False
    for row in (4, 5, rows - 1):
        s[row, shut] = -INF
    s[11] = -INF
    check(s, 0.05, iters, None, b / b.sum(), torch.full((cols,), start, device="cuda"), far=[2, 6])


def test_balance_tiny_masses():
    s = make(900, 12, torch.float32, scale=1.0)
    a, b = torch.rand(900, generator=gen(1), device="cuda"), torch.ones(12, device="cuda")
    a[5::9] *= 1e-36
    b[3] = 0
    s[5::9, 3] += 20.0
    check(s, 0.3, 6, a / a.sum(), b / b.sum())


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("iters", [1, 2, 6])
@pytest.mark.parametrize("mass", [True, False])
def test_balance_start_of_minus_infinity(rows, cols, iters, mass):
    """g = -inf leaves a column out of the first row sums only."""
    s = make(rows, cols, torch.bfloat16, seed=rows, scale=1.0)
    g = 0.3 * make(1, cols, torch.float32, seed=2)[0]
    g[[0, 7]] = -INF
    b = torch.rand(cols, generator=gen(3), device="cuda") + 0.5
    if not mass:
        b[7] = 0
    check(s, 0.2, iters, None, b / b.sum(), g)


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("value", [-1e4, 2e4])
def test_balance_start_of_minus_infinity_on_a_far_column(rows, cols, value):
    """Its first terms are its own size, which the later row sums must not see."""
    s = make(rows, cols, torch.float32, seed=rows, scale=1.0)
    s[:, 3] += value
    s[5, torch.arange(cols, device="cuda") != 3] = -INF
    g = torch.zeros(cols, device="cuda")
    g[3] = -INF
    for iters in (1, 2, 6):
        check(s, 0.15, iters, g=g, far=[3])


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_balance_start_of_minus_infinity_beside_scores_below_the_range(rows, cols):
    """Rows whose only normal score is on the column that starts from -inf: the lowest values beside it are as good as -inf,
    also where other rows, of nothing but the lowest value, have their terms formed from pairs of float32."""
    s = make(rows, cols, torch.bfloat16, seed=rows, scale=1.0)
    low, g = torch.finfo(torch.bfloat16).min, torch.zeros(cols, device="cuda")
    g[2] = -INF
    s[4::9, torch.arange(cols, device="cuda") != 2] = low
    want = torch.where(s == low, -INF, s)
    s[3::9], want[3::9] = low, 0.0
    for iters in (1, 2, 5):
        r = scores.balance(s, eps=0.2, iters=iters, g=g)
        f, w, _ = reference(want, 0.2, iters, None, None, g)
        f[3::9] -= low                                           # (a row's constant)
        # as in `check`: |S + f + g| below 10 of the ordinary rows and columns
        tol = U * 0.2 * 2 * iters * (4 * (10 / 0.2 + 16) + GAMMA + max(s.shape) / 32)
        close(r.g, w, tol + 8 * U * w.abs(), "g")
        close(r.f, f, tol + 8 * U * f.abs(), "f")


def test_balance_start_that_is_no_number():
    s = make(700, 16, torch.float32, scale=1.0)
    for bad in (math.nan, INF):
        g = torch.zeros(16, device="cuda")
        g[3] = bad
        r = scores.balance(s, eps=0.2, iters=2, g=g)
        assert torch.isnan(r.f).all() and torch.isnan(r.g).all()


# log_probs -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cols", [40, 3001, 70000])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("offset,temperature", [(-3e9, 1.0), (-1e10, 1.0), (7e11, 1.0), (0.0, 1e-10), (-1e20, 1.7),
                                                (1e28, 0.3)])
def test_log_probs_far_scores(cols, dtype, offset, temperature):
    """Scores whose multiple by log2(e) / T rounds by more than the exponential's range, on rows of equal scores, too."""
    if dtype == "f16" and offset:
        offset, temperature = math.copysign(30000.0, offset), temperature * 3e4 / abs(offset)
    s = make(5, cols, torch.float32, seed=cols).double()
    s[1:] += offset
    s[2] = offset * 1.0001
    s[3, ::2] = -INF
    s[4] = torch.where(torch.arange(cols, device="cuda") % 3 == 0, offset + abs(offset) * 2.0 ** -7, offset)
    t = torch.randint(cols, (5, 2), generator=gen(1), device="cuda")
    check_log_probs(s.to(TYPES[dtype]), t, 5, temperature)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1e-10, 1e-25])
def test_log_probs_gradient_of_masked_rows_at_small_temperatures(dtype, temperature):
    s = make(6, 1003, torch.float32, seed=4, scale=2.0 * temperature)
    s[1:, ::3] = -INF
    s[2] = -INF
    s[3, 5:] = torch.finfo(torch.float32).min
    check_gradient(s.to(TYPES[dtype]), torch.randint(1003, (6, 2), generator=gen(7), device="cuda"), 3, temperature)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_log_probs_gradient_of_masked_rows_with_large_upstream_values(dtype):
    """A scaled loss: 2^24 on the entropy at T = 0.02. The gradient is p (log p + H) g / T in 64 bits, p off by
    (8 |log p| + the chain + 2 GAMMA) u and log p + H by 8 u of its terms."""
    s = make(4, 2003, TYPES[dtype], seed=4, scale=0.05)
    s[1:, ::3] = -INF
    s[2, 4:] = -INF
    leaf = s.detach().requires_grad_()
    r = scores.log_probs(leaf, temperature=0.02)
    up = torch.full_like(r.entropy, 2.0 ** (3 if dtype == "f16" else 24))
    grad, = torch.autograd.grad(r.entropy, leaf, up)
    w = lp_reference(s, torch.zeros(4, 1, dtype=torch.int64, device="cuda"), 1, 0.02)
    log_p = torch.where(w["p"] > 0, w["log_p"], 0.0)
    each = w["p"] * up.double()[:, None] / 0.02
    want = -each * (log_p + w["h"][:, None])
    u = 2.0 ** -53 if dtype == "f64" else U
    size = log_p.abs() + w["h"][:, None] + 1
    tol = each * size * u * (8 * log_p.abs() + 2003 / 256 + 8 + 2 * GAMMA + 8 * size)
    tol = (tol + torch.finfo(s.dtype).eps / 2 * want.abs()) * (1 + torch.finfo(s.dtype).eps)
    close(grad, want, tol + torch.finfo(s.dtype).smallest_normal, "grad")
    assert (grad[s == -INF] == 0).all()


def test_log_probs_gradient_of_a_row_that_is_no_number():
    s = make(3, 300, torch.float32)
    s[1, 7] = math.nan
    s[2, 9] = INF
    leaf = s.requires_grad_()
    r = scores.log_probs(leaf, torch.zeros(3, dtype=torch.int64, device="cuda"))
    grad, = torch.autograd.grad((r.log_prob.sum() + r.entropy.sum()), leaf)
    assert torch.isfinite(grad[0]).all() and torch.isnan(grad[1:]).all()


def test_gradient_rows_between_the_scores_rows():
    """Scores and gradient as the halves of one buffer's rows, through the C calls."""
    from trnopt import _capi
    rows, cols = 37, 200
    buf = torch.zeros(rows, 2 * cols + 8, device="cuda")
    s, grad = buf[:, :cols], buf[:, cols + 4:2 * cols + 4]
    s.copy_(make(rows, cols, torch.float32, seed=3))
    buf[:, 2 * cols + 4:] = 7.0
    leaf = s.clone().requires_grad_()
    t = torch.randint(cols, (rows,), generator=gen(1), device="cuda")
    up = torch.randn(rows, generator=gen(2), device="cuda")
    want, = torch.autograd.grad(scores.log_probs(leaf, t).log_prob, leaf, up)
    numbers = [torch.empty(rows, device="cuda") for _ in range(5)]
    at, pitch, stream = [n.data_ptr() for n in numbers], buf.stride(0), torch.cuda.current_stream().cuda_stream
    _capi.check(_capi.lib.trnopt_log_probs(0, s.data_ptr(), pitch, rows, cols, 1.0, t.data_ptr(), 1, 0, at[0], at[1], at[2],
                                           None, None, at[3], at[4], stream), "log_probs")
    _capi.check(_capi.lib.trnopt_log_probs_grad(0, s.data_ptr(), pitch, rows, cols, 1.0, t.data_ptr(), 1, None, 0, at[3], at[4],
                                                at[1], up.data_ptr(), None, None, None, grad.data_ptr(), pitch, stream),
                "log_probs_grad")
    assert torch.equal(grad, want) and torch.equal(s, leaf) and (buf[:, cols:cols + 4] == 0).all()
    r = scores.route(leaf, 3)
    d = torch.randn(rows, 3, generator=gen(4), device="cuda")
    want, = torch.autograd.grad(r.weight, leaf, d)
    _capi.check(_capi.lib.trnopt_route_grad(0, s.data_ptr(), pitch, rows, cols, 3, 0, 1, 1.0, r.index.data_ptr(), d.data_ptr(),
                                            grad.data_ptr(), pitch, stream), "route_grad")
    assert torch.equal(grad, want) and torch.equal(s, leaf) and (buf[:, 2 * cols + 4:] == 7).all()
