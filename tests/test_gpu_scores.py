"""The score-matrix operators (trnopt.scores) against plain 64-bit formulas: values, gradients, masks, ties, sizes from
one column up, strides, streams, captured graphs, and what they refuse.

Tolerances. u = 2^-24 is half a step of float32 relative to a value. A float32 sum of n terms kept in c chains of equal
length and joined pairwise is off by at most (n / c + log2 c) u of the sum of absolute terms; the kernels hold at least 256
chains per row of log_probs and 32 per row of the others. Every term's own exponential adds a few u (GAMMA below covers the
exponential's and the products' roundings: expf and ex2 are documented to 2 units in the last place = 4 u, the scaled
difference rounds up to 3 times, which the exponential turns into 3 u |d| relative). A stored gradient is off by half a
step of its type, finfo.eps / 2."""

import math

import pytest
import torch

from trnopt import scores

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GAMMA = 16
INF = math.inf
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}


def unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else U


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(rows, cols, dtype, seed=0, scale=2.0):
    return (scale * torch.randn(rows, cols, generator=gen(seed), device="cuda")).to(dtype)


# log_probs -----------------------------------------------------------------------------------------------------------

def lp_reference(s, targets, top, temperature):
    """From the definition, float64: per row over its columns above -inf."""
    s = s.double()
    m = s.amax(-1, keepdim=True)
    empty = m == -INF
    d = torch.where(s == -INF, -INF, (s - torch.where(empty, 0.0, m)) / temperature)
    p = torch.exp(d)
    total = p.sum(-1, keepdim=True)
    log_p = torch.where(empty, -INF, d - total.log())
    p = torch.where(empty, 0.0, p / total)
    h = -torch.where(p > 0, p * log_p, 0.0).sum(-1)
    lse = torch.where(empty, -INF, m / temperature + total.log())[:, 0]
    lp = torch.where(targets >= 0, log_p.gather(1, targets.clamp(min=0)), 0.0)
    order = s.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    order = torch.nn.functional.pad(order, (0, top - order.shape[1]), value=0)
    value = log_p.gather(1, order)
    absent = (torch.arange(top, device=s.device) >= s.shape[1]) | (s.gather(1, order) == -INF)
    return dict(lp=lp, h=h, lse=lse, top_lp=torch.where(absent, -INF, value), top_i=torch.where(absent, -1, order),
                p=p, log_p=log_p, m=m)


def close(got, want, tol, name):
    """|got - want| <= tol elementwise, infinities and NaN in the same places."""
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and not torch.isinf(got[~inf]).any(), name
    off = ((got - want).abs() - tol)[torch.isfinite(want)]
    assert off.numel() == 0 or off.max() <= 0, f"{name}: {off.max().item():.3g} over the tolerance"


def check_log_probs(s, targets, top, temperature):
    r = scores.log_probs(s, targets, top=top, temperature=temperature)
    w = lp_reference(s, targets, top, temperature)
    u, cols = unit(s.dtype), s.shape[1]
    chain = cols / 256 + 8
    spread = torch.where(w["p"] > 0, w["log_p"], 0.0).abs()
    # log s: chain of terms with GAMMA + 3 |d| roundings each, weighted by p; the differences round three times
    base = u * (chain + GAMMA + 4 * (w["p"] * spread).sum(-1) + 4 * w["h"].abs())
    fin = lambda t: torch.where(torch.isfinite(t), t, 0.0).abs()
    close(r.log_prob, w["lp"], base[:, None] + 4 * u * fin(w["lp"]), "log_prob")
    close(r.lse, w["lse"], base + 4 * u * fin(w["lse"]) + 4 * u * fin(w["m"][:, 0] / temperature), "lse")
    # H = log s - sum e d / s: the second sum's terms are |d| times larger, with its own chain
    close(r.entropy, w["h"], base + u * (chain + GAMMA) * (w["p"] * spread).sum(-1)
          + 4 * u * (w["p"] * spread * spread).sum(-1), "entropy")
    if top:
        assert torch.equal(r.top_index, w["top_i"])
        close(r.top_log_prob, w["top_lp"], base[:, None] + 4 * u * fin(w["top_lp"]), "top_log_prob")
    return r, w


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (2, 31), (5, 257), (4, 1000), (3, 4099), (2, 8191), (2, 8192),
                                       (2, 16385), (1, 50001), (1, 131072), (1, 262144), (300, 700)])
def test_log_probs_values(rows, cols, dtype):
    s = make(rows, cols, TYPES[dtype], seed=rows * 7 + cols)
    t = torch.randint(cols, (rows, 3), generator=gen(1), device="cuda")
    check_log_probs(s, t, min(20, cols + 2), 1.0)


@pytest.mark.parametrize("top", [0, 1, 2, 8, 9, 33, 64])
@pytest.mark.parametrize("rows,cols", [(2, 40), (3, 5000), (2, 70000)])
def test_log_probs_number_of_best_columns(top, rows, cols):
    s = make(rows, cols, torch.bfloat16, seed=top)
    check_log_probs(s, torch.zeros(rows, 1, dtype=torch.int64, device="cuda"), top, 0.7)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("temperature", [0.05, 3.0, 1e-3])
def test_log_probs_temperature(dtype, temperature):
    s = make(4, 3001, TYPES[dtype], seed=5)
    check_log_probs(s, torch.randint(3001, (4, 2), generator=gen(2), device="cuda"), 5, temperature)


def patterns(cols, dtype):
    """Rows where a best-columns search or a masked sum can go wrong."""
    low = torch.finfo(dtype).min
    i = torch.arange(cols, device="cuda", dtype=torch.float64)
    base = make(1, cols, torch.float32, seed=9)[0].double()
    rows = [torch.full_like(i, 1.25),                                # all equal
            i / 64,                                                  # ascending: every column beats the ones before
            -i / 64,                                                 # descending
            torch.where(i % 7 == 3, 2.0, 0.0),                       # ties across the row
            torch.full_like(i, -INF),                                # nothing open
            torch.where(i == cols - 1, 0.5, -INF),                   # only the last column open
            torch.where(i < 5, base, -INF),                          # fewer open than wanted
            torch.full_like(i, low),                                 # all the type's lowest value
            torch.where(i % 11 == 0, base, low),                     # masked by the lowest value
            torch.where(i % 2 == 0, 1.0, -1.0) * 0.0,                # +0 and -0 are equal
            torch.where(i == cols // 2, 60.0, base),                 # one column has nearly everything
            base]
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", [9, 300, 9000, 33333])
def test_log_probs_patterns(cols, dtype):
    s = patterns(cols, TYPES[dtype])
    t = torch.stack([torch.zeros(len(s)), torch.full((len(s),), cols - 1), torch.full((len(s),), -3)], 1)
    check_log_probs(s, t.long().cuda(), min(20, cols), 1.0)


@pytest.mark.parametrize("repeats", [1, 40, 100, 250])      # few rows on many warps each, to many rows on one warp each
@pytest.mark.parametrize("dtype,cols,top", [("bf16", 5003, 64), ("f32", 5000, 30), ("f16", 2600, 7), ("f64", 1500, 64)])
def test_log_probs_patterns_in_many_rows(dtype, cols, top, repeats):
    s = patterns(cols, TYPES[dtype]).repeat(repeats, 1)
    s = s[torch.randperm(len(s), generator=gen(1), device="cuda")]
    check_log_probs(s, torch.randint(cols, (len(s), 1), generator=gen(2), device="cuda"), top, 1.0)


def test_log_probs_entropy_is_not_negative():
    s = make(3000, 500, torch.float32, scale=30.0)
    s[:, 7] += 200.0
    for temperature in (1.0, 0.013):
        assert (scores.log_probs(s, temperature=temperature).entropy >= 0).all()


def test_log_probs_extreme_scores_and_temperatures():
    """Scaled scores beyond float32's range: the differences to the row's maximum decide."""
    t = torch.randint(2000, (6, 1), generator=gen(2), device="cuda")
    for scale, temperature in ((1e31, 1e30), (1e37, 1.0), (1e37, 1e5)):
        s = make(6, 2000, torch.float32, scale=scale)
        s[1] = make(1, 2000, torch.float32, seed=3)[0] - 3e38
        r = scores.log_probs(s, t, top=4, temperature=temperature)
        w = lp_reference(s, t, 4, temperature)
        assert torch.equal(r.top_index, w["top_i"])
        close(r.log_prob, w["lp"], 1e-5 * (1 + w["lp"].abs()), "log_prob")
        close(r.entropy, w["h"], 2e-5 * (1 + w["h"]), "entropy")
    r = scores.log_probs(s[1:2], t[1:2], top=4)
    assert torch.isfinite(r.log_prob).all() and torch.isfinite(r.entropy).all()
    tiny = scores.log_probs(make(1, 2000, torch.float32), top=2, temperature=1e-30)      # one column has everything
    assert tiny.entropy.item() == 0 and tiny.top_log_prob[0, 0].item() == 0


@pytest.mark.parametrize("cols", [33, 20000])
def test_log_probs_infinite_and_nan_rows(cols):
    for dtype in TYPES.values():
        s = make(4, cols, dtype)
        s[1, cols // 2], s[2, cols - 1] = INF, math.nan
        t = torch.tensor([[0, -1], [1, -1], [2, -1], [cols + 5, -1]], device="cuda")
        r = scores.log_probs(s, t, top=3)
        assert torch.isnan(r.log_prob[1:, 0]).all() and not torch.isnan(r.log_prob[0, 0])
        assert (r.log_prob[:, 1] == 0).all()
        for v in (r.entropy, r.lse):
            assert torch.equal(torch.isnan(v), torch.tensor([False, True, True, False], device="cuda"))
        assert (r.top_index[1:3] == -1).all() and torch.isnan(r.top_log_prob[1:3]).all()
        check_log_probs(s[[0, 3]], torch.zeros(2, 1, dtype=torch.int64, device="cuda"), 3, 1.0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("offset,pitch,cols", [(0, 513, 513), (1, 520, 513), (3, 1029, 1000), (5, 4111, 4099)])
def test_log_probs_strides(dtype, offset, pitch, cols):
    buf = make(1, 6 * pitch + 16, TYPES[dtype], seed=3)[0]
    s = buf.as_strided((6, cols), (pitch, 1), offset)
    t = torch.randint(cols, (6, 2), generator=gen(4), device="cuda")
    check_log_probs(s, t, 7, 1.0)
    # a row repeated, and columns that are not neighbours (copied first)
    check_log_probs(s[:1].expand(3, cols), t[:3], 7, 1.0)
    w = make(cols, 5, TYPES[dtype], seed=6).t()
    check_log_probs(w, t[:5] % cols, 4, 1.0)


def test_log_probs_leading_shapes():
    s = make(6, 77, torch.float32).view(2, 3, 77)
    t = torch.randint(77, (2, 3), generator=gen(0), device="cuda", dtype=torch.int32)
    r = scores.log_probs(s, t, top=4)
    flat = scores.log_probs(s.view(6, 77), t.view(6), top=4)
    assert r.log_prob.shape == (2, 3) and r.entropy.shape == (2, 3) and r.top_index.shape == (2, 3, 4)
    assert torch.equal(r.log_prob.view(6), flat.log_prob) and torch.equal(r.top_index.view(6, 4), flat.top_index)
    one = scores.log_probs(s[0, 0], t[0, 0])
    assert one.log_prob.shape == () and one.log_prob == r.log_prob[0, 0] and one.top_index is None
    none = scores.log_probs(s[:0], top=2)
    assert none.log_prob is None and none.lse.shape == (0, 3) and none.top_index.shape == (0, 3, 2)


def test_log_probs_offsets_past_32_bits():
    """Rows that start more than 2^31 elements into the buffer, read and written through a row pitch."""
    pitch, cols = (1 << 30) + 24, 1500
    buf = torch.empty(2 * pitch + cols, dtype=torch.bfloat16, device="cuda")
    s = buf.as_strided((3, cols), (pitch, 1))
    s.copy_(make(3, cols, torch.bfloat16, seed=8))
    t = torch.randint(cols, (3, 1), generator=gen(4), device="cuda")
    check_log_probs(s, t, 5, 1.0)
    check_gradient(s, t, 2, 1.0)


def test_log_probs_longest_row():
    """2^31 - 1 columns, off a 16-byte boundary, with the gradient. A lane adds its scores in 32,768 chunks of 32 and the
    lanes' sums are joined, so sums are off by GAMMA = 33,000 roundings at most (relative to sums of magnitudes)."""
    cols, step = 2 ** 31 - 1, 1 << 26
    buf = torch.randn(cols + 1, generator=gen(3), device="cuda", dtype=torch.bfloat16)
    s = buf[1:].view(1, cols)
    named = [cols - 1, 2 ** 30 + 3, 7]
    s[0, named] = torch.tensor([20.0, 19.0, 18.0], dtype=torch.bfloat16, device="cuda")
    s.requires_grad_()
    targets = torch.tensor([[7, cols - 1, 2 ** 30 + 5, -1]], device="cuda")
    r = scores.log_probs(s, targets, top=3)
    total = weighted = 0.0
    for j in range(0, cols, step):
        d = s.detach()[0, j:j + step].double() - 20
        e = d.exp()
        total += float(e.sum())
        weighted += float((e * d).sum())
    lse, far = 20 + math.log(total), -weighted / total
    sums = 33_000 * U
    assert r.top_index.tolist() == [named]
    assert abs(r.lse.item() - lse) <= sums + 64 * U
    assert abs(r.entropy.item() - (math.log(total) + far)) <= 2 * sums * (1 + far)
    log_p = s.detach()[0, [7, cols - 1, 2 ** 30 + 5]].double() - lse
    assert (r.log_prob[0, :3].double() - log_p).abs().max() <= sums + 64 * U and r.log_prob[0, 3] == 0

    up = torch.tensor([[0.25, 0.5, 0.125, 9.0]], device="cuda")         # the last one's target is padding
    grad, = torch.autograd.grad((r.log_prob * up).sum() + r.lse.sum(), s)
    for j in range(0, cols, step):
        want = (s.detach()[0, j:j + step].double() - lse).exp() * (1 - 0.875)
        for t, g in zip(targets[0, :3].tolist(), up[0].tolist()):
            if j <= t < j + step:
                want[t - j] += g
        assert ((grad[0, j:j + step].double() - want).abs() <= want * (2.0 ** -8 + 2 * sums)).all()


def test_log_probs_most_rows():
    """More rows than one launch takes (2^30): the rows on both sides of the border, with the gradient of lse (p)."""
    rows, border = 2 ** 30 + 37, 2 ** 30
    s = torch.randn(rows, 2, generator=gen(6), device="cuda", dtype=torch.bfloat16).requires_grad_()
    r = scores.log_probs(s)
    grad, = torch.autograd.grad(r.lse, s, torch.ones_like(r.lse))
    for part in (slice(0, 1000), slice(border - 1000, rows)):
        x = s.detach()[part].double()
        lse, p = x.logsumexp(-1), x.softmax(-1)
        # lse = m + log(sum): sum in [1, 2], off by 8 roundings and ex2's 2 u; the sum of m and the log rounded once more
        assert ((r.lse[part].detach().double() - lse).abs() <= (GAMMA + lse.abs()) * U).all()
        assert ((r.entropy[part].detach().double() + (p * p.log()).sum(-1)).abs() <= 8 * GAMMA * U).all()
        assert ((grad[part].double() - p).abs() <= p * (2.0 ** -8 + 32 * U)).all()


# gradient -------------------------------------------------------------------------------------------------------------

def upstream(rows, n, dtype, seed):
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    return torch.randn(rows, n, generator=gen(seed), device="cuda").to(wide)


def check_gradient(s, targets, top, temperature, use=("log_prob", "entropy", "lse", "top")):
    leaf = s.detach().requires_grad_()
    r = scores.log_probs(leaf, targets, top=top, temperature=temperature)
    rows, n = targets.shape
    up = dict(log_prob=upstream(rows, n, s.dtype, 1), entropy=upstream(rows, 1, s.dtype, 2)[:, 0],
              lse=upstream(rows, 1, s.dtype, 3)[:, 0], top=upstream(rows, top, s.dtype, 4))
    outs = dict(log_prob=r.log_prob, entropy=r.entropy, lse=r.lse, top=r.top_log_prob)
    used = [k for k in use if not (k == "top" and top == 0)]
    grad, = torch.autograd.grad([outs[k] for k in used], [leaf], [up[k] for k in used])
    assert grad.dtype == s.dtype and grad.shape == s.shape
    # the formula in 64 bits
    w = lp_reference(s, targets, top, temperature)
    p, zero = w["p"], torch.zeros((), dtype=torch.float64, device="cuda")
    g = torch.where(targets >= 0, up["log_prob"].double(), zero) if "log_prob" in used else torch.zeros_like(targets).double()
    on = torch.zeros_like(p).scatter_add_(1, targets.clamp(min=0), g)
    total, size = g.sum(-1, keepdim=True), g.abs().sum(-1, keepdim=True)
    if "top" in used:
        gt = torch.where(w["top_i"] >= 0, up["top"].double(), zero)
        on.scatter_add_(1, w["top_i"].clamp(min=0), gt)
        total, size = total + gt.sum(-1, keepdim=True), size + gt.abs().sum(-1, keepdim=True)
    if "lse" in used:
        total, size = total - up["lse"].double()[:, None], size + up["lse"].double().abs()[:, None]
    log_p = torch.where(p > 0, w["log_p"], 0.0)
    gh = up["entropy"].double()[:, None] if "entropy" in used else zero
    empty = w["m"] == -INF
    want = torch.where(empty, 0.0, (on - p * (total + gh * (log_p + w["h"][:, None]))) / temperature)
    # p is off by (GAMMA + 8 |log p| + the row sum's chain) u relative, log p + H by that absolutely
    u = unit(s.dtype)
    chain = s.shape[1] / 256 + 8
    rel = u * (chain + 2 * GAMMA + 8 * log_p.abs() + 8 * w["h"][:, None])
    parts = p * (size + gh.abs() * (log_p.abs() + w["h"][:, None] + 1))
    entries = n + top + 4
    tol = (rel * parts + u * entries * (on.abs() + size * p) * 2) / temperature
    tol = tol + torch.finfo(s.dtype).eps / 2 * want.abs() + torch.finfo(s.dtype).smallest_normal * torch.finfo(s.dtype).eps
    # given columns that meet: their upstream gradients are added one after the other
    tol = tol + u * entries * torch.zeros_like(p).scatter_add_(1, targets.clamp(min=0), g.abs()) / temperature
    tol = tol * (1 + 2 * torch.finfo(s.dtype).eps)          # the last rounding acts on the value before it
    close(grad, want, tol, "grad")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols,n,top", [(1, 1, 1, 1), (3, 5, 2, 3), (4, 1000, 1, 0), (3, 4099, 8, 0), (2, 20001, 16, 5),
                                             (2, 65536, 1, 64), (37, 300, 3, 2)])
def test_log_probs_gradient(rows, cols, n, top, dtype):
    s = make(rows, cols, TYPES[dtype], seed=cols)
    t = torch.randint(cols, (rows, n), generator=gen(7), device="cuda")
    t[:, -1:] = t[:, :1]                              # a column given twice
    if n > 2:
        t[0, 1] = -1
    check_gradient(s, t, top, 0.8)


@pytest.mark.parametrize("use", [("log_prob",), ("entropy",), ("lse",), ("top",), ("log_prob", "top")])
def test_log_probs_gradient_of_each_output(use):
    s = make(5, 900, torch.float32, seed=2)
    check_gradient(s, torch.randint(900, (5, 2), generator=gen(7), device="cuda"), 4, 1.0, use)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_log_probs_gradient_patterns(dtype):
    s = patterns(3000, TYPES[dtype])
    t = torch.stack([torch.zeros(len(s)), torch.full((len(s),), 2999), torch.full((len(s),), -1)], 1).long().cuda()
    check_gradient(s, t, 5, 1.0)


def test_log_probs_gradient_strides_and_out_of_range():
    buf = make(1, 5 * 1111, torch.float16, seed=3)[0]
    s = buf.as_strided((4, 1003), (1111, 1), 3)
    check_gradient(s, torch.randint(1003, (4, 2), generator=gen(4), device="cuda"), 3, 1.0)
    # an index past the last column adds nothing
    a, b = s.detach().clone().requires_grad_(), s.detach().clone().requires_grad_()
    t = torch.tensor([[5, 2000]] * 4, device="cuda")
    ga, = torch.autograd.grad(scores.log_probs(a, t).log_prob[:, 0].sum(), a)
    gb, = torch.autograd.grad(scores.log_probs(b, t[:, :1]).log_prob.sum(), b)
    assert torch.equal(ga, gb)


def test_log_probs_gradient_by_differences():
    s = make(2, 40, torch.float64, seed=1).requires_grad_()
    t = torch.tensor([[3, 3, -1], [7, 39, 0]], device="cuda")
    fn = lambda x: tuple(scores.log_probs(x, t, top=2, temperature=0.9)[:4])
    assert torch.autograd.gradcheck(fn, (s,), eps=1e-6, atol=1e-7)


def test_log_probs_repeats_to_the_bit():
    s = make(50, 30000, torch.bfloat16).requires_grad_()
    t = torch.randint(30000, (50, 4), generator=gen(0), device="cuda")
    runs = []
    for _ in range(2):
        r = scores.log_probs(s, t, top=10)
        g, = torch.autograd.grad((r.log_prob.sum() + r.entropy.sum()), s)
        runs.append([*r, g])
    for x, y in zip(*runs):
        assert torch.equal(x, y)


# balance -------------------------------------------------------------------------------------------------------------

def balance_reference(s, eps, iters, a, b, g):
    """The half-steps in 64 bits; a row or column without terms has potential 0."""
    s = s.double()
    n, e = s.shape
    la = torch.full((n,), -math.log(n), dtype=torch.float64, device="cuda") if a is None else a.double().log()
    lb = torch.full((e,), -math.log(e), dtype=torch.float64, device="cuda") if b is None else b.double().log()
    g = torch.zeros(e, dtype=torch.float64, device="cuda") if g is None else g.double()
    for _ in range(iters):
        f = -eps * torch.logsumexp(lb + (g + s) / eps, 1)
        f = torch.where(torch.isinf(f), 0.0, f)
        g = -eps * torch.logsumexp(la[:, None] + (f[:, None] + s) / eps, 0)
        g = torch.where(torch.isinf(g), 0.0, g)
    return f, g


def check_balance(s, eps, iters, a=None, b=None, g=None):
    r = scores.balance(s, eps=eps, iters=iters, a=a, b=b, g=g)
    f, w = balance_reference(s, eps, iters, a, b, g)
    # a half-step does not enlarge differences of its input, so each of the 2 iters half-steps adds its own rounding:
    # terms of size z = |S + f + g| / eps + |log b| round 4 times, the sum is a chain of rows / 32 or columns / 32 terms
    fin = lambda t: torch.where(torch.isfinite(t), t, 0.0).abs().max().item()
    size = (fin(s.double()) + fin(f) + fin(w) + (0 if g is None else fin(g))) / eps + 16
    tol = U * eps * 2 * iters * (4 * size + GAMMA + max(s.shape) / 32) + 4 * U * max(fin(f), fin(w))
    close(r.f, f, tol, "f")
    close(r.g, w, tol, "g")
    return r


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (9, 1), (33, 31), (100, 64), (1000, 24), (777, 256), (130, 1000),
                                       (5000, 100), (300, 1024), (20011, 60)])
def test_balance_values(rows, cols, dtype):
    check_balance(make(rows, cols, TYPES[dtype], seed=rows + cols, scale=1.0), 0.3, 5)


@pytest.mark.parametrize("iters", [1, 2, 3, 30])
@pytest.mark.parametrize("eps", [0.02, 0.25, 4.0])
def test_balance_eps_and_iterations(eps, iters):
    check_balance(make(515, 40, torch.float32, scale=1.0), eps, iters)


def test_balance_far_columns():
    """Columns hundreds of eps apart: the first sums underflow unless every column keeps its own maximum."""
    s = make(400, 16, torch.float32, scale=0.5) + torch.linspace(-40, 0, 16, device="cuda")
    check_balance(s, 0.05, 6)
    check_balance(s, 0.05, 2, g=torch.linspace(3, -60, 16, device="cuda"))


def test_balance_masses_and_masks():
    s = make(300, 20, torch.bfloat16, scale=1.0)
    a = torch.rand(300, generator=gen(1), device="cuda")
    a[250:] = 0
    a /= a.sum()
    b = torch.rand(20, generator=gen(2), device="cuda") + 0.1
    b[7] = 0
    b /= b.sum()
    r = check_balance(s, 0.2, 12, a, b, 0.1 * make(1, 20, torch.float32)[0])
    # padding rows do not move the columns
    assert torch.equal(r.g, scores.balance(torch.cat([s[:250], s[:50]]), eps=0.2, iters=12, a=a, b=b,
                                           g=0.1 * make(1, 20, torch.float32)[0]).g)
    s[40] = -INF                       # a row, a column and half the rest are closed
    s[:, 3] = -INF
    s[::2, 5] = -INF
    check_balance(s, 0.2, 4)
    check_balance(torch.full((5, 4), -INF, device="cuda"), 0.2, 2)


def test_balance_rows_without_open_columns():
    """Rows whose only scores are on columns of mass 0: potential 0, and their terms still reach those columns."""
    s = make(70, 9, torch.float32, scale=1.0)
    b = torch.full((9,), 1 / 7, device="cuda")
    b[[2, 6]] = 0
    s[10, [0, 1, 3, 4, 5, 7, 8]] = -INF
    s[11] = -INF
    g = 0.5 * make(1, 9, torch.float32, seed=2)[0]
    for iters in (1, 2, 7):
        check_balance(s, 0.4, iters, None, b, g)


def test_balance_more_rows_than_shared_memory_holds():
    check_balance(make(70001, 40, torch.float32, scale=1.0), 0.3, 3)
    check_balance(make(40000, 301, torch.bfloat16, scale=1.0), 0.3, 3)


@pytest.mark.parametrize("rows,cols", [(5000, 16), (3001, 100), (40000, 256), (700, 1000)])
def test_balance_far_columns_over_several_ctas(rows, cols):
    """Sums far from 1 in the first iterations, which the CTAs do not exchange in fixed point, and near 1 later."""
    far = torch.linspace(-40, 0, cols, device="cuda")[torch.randperm(cols, generator=gen(0), device="cuda")]
    s = make(rows, cols, torch.float32, scale=0.5) + far
    s[: rows // 3] += 2 * far.flip(0)                      # (two kinds of rows: iterations that do not converge at once)
    for iters in (2, 3, 4, 9):
        check_balance(s, 0.5, iters)
    check_balance(s, 0.5, 3, g=torch.linspace(3, -60, cols, device="cuda"))


@pytest.mark.parametrize("rows,cols", [(5000, 16), (30000, 90), (2000, 1000)])
def test_balance_masses_and_masks_over_several_ctas(rows, cols):
    s = make(rows, cols, torch.bfloat16, scale=1.0)
    a = torch.rand(rows, generator=gen(1), device="cuda")
    a[-rows // 5:] = 0
    b = torch.rand(cols, generator=gen(2), device="cuda") ** 4 + 1e-6
    b[7] = 0
    g = 0.1 * make(1, cols, torch.float32)[0]
    check_balance(s, 0.2, 6, a / a.sum(), b / b.sum(), g)
    check_balance(s, 0.2, 6, 1000 * a / a.sum(), b / b.sum(), g)        # sums that do not agree: k = 1000 throughout
    s[40] = -INF
    s[:, 3] = -INF
    s[::2, 5] = -INF
    check_balance(s, 0.2, 6)
    check_balance(s, 0.2, 6, a / a.sum(), b / b.sum(), g)
    check_balance(torch.full((rows, cols), -INF, device="cuda"), 0.2, 3)
    s[rows // 2, 2] = float("nan")
    r = scores.balance(s, eps=0.2, iters=4)
    assert r.g[2].isnan() and r.f[rows // 2].isnan()


def test_balance_most_rows():
    """2^31 - 1 rows of one column: f = -S and g = 0. Column sums are of 28,341 terms a lane, then of 512 lanes in 148
    CTAs: N = 28,341 + 200 roundings at most, which move g by eps N u; f besides by three roundings of |S| log2(e) / eps."""
    rows, eps = 2 ** 31 - 1, 0.5
    s = torch.randn(rows, generator=gen(5), device="cuda", dtype=torch.bfloat16).view(rows, 1)
    r = scores.balance(s, eps=eps, iters=3)
    off = eps * 28_541 * U
    assert r.g.abs().item() <= off
    for i in range(0, rows, 1 << 28):
        x = s[i:i + (1 << 28), 0].float()
        assert ((r.f[i:i + (1 << 28)] + x).abs() <= off + 4 * U * x.abs()).all()


def test_balance_marginals_agree_with_sinkhorn():
    """Converged potentials on S = -C are sinkhorn()'s up to its constant shift, and the plan's columns sum to b."""
    from trnopt import Backend, SinkhornOptions, sinkhorn
    x, y = make(256, 4, torch.float32, 1, 0.3), make(40, 4, torch.float32, 2, 0.3)
    c = torch.cdist(x.double(), y.double()) ** 2
    r = scores.balance(-c.float(), eps=0.2, iters=200)
    plan = torch.exp((r.f.double()[:, None] + r.g.double() - c) / 0.2) / (256 * 40)
    assert (plan.sum(0) * 40 - 1).abs().max() < 1e-5 and (plan.sum(1) * 256 - 1).abs().max() < 1e-4
    ref = sinkhorn(x.cpu().numpy(), y.cpu().numpy(),
                   opts=SinkhornOptions(eps=0.2, max_iters=400, fixed_iters=True, normalize=False,
                                        backend=Backend.preset("cuda-fused")))
    shift = r.g.cpu().double() - torch.as_tensor(ref.g)
    assert (shift - shift.mean()).abs().max() < 1e-4 * 0.2


def test_balance_strides_shapes_and_repeats():
    buf = make(1, 40 * 700 + 9, torch.bfloat16, scale=1.0)[0]
    check_balance(buf.as_strided((600, 33), (37, 1), 3), 0.3, 4)
    check_balance(buf.as_strided((600, 32), (40, 1), 8), 0.3, 4)
    s = make(60, 12, torch.float32)
    r = scores.balance(s.view(3, 20, 12), eps=0.5, iters=3)
    assert r.f.shape == (3, 20) and torch.equal(r.f.view(60), scores.balance(s, eps=0.5, iters=3).f)
    s = make(30000, 250, torch.bfloat16, scale=1.0)
    x, y = scores.balance(s, eps=0.1, iters=10), scores.balance(s, eps=0.1, iters=10)
    assert torch.equal(x.f, y.f) and torch.equal(x.g, y.g)


def test_balance_nan_reaches_the_result():
    s = make(64, 8, torch.float32)
    s[5, 2] = math.nan
    r = scores.balance(s, iters=2)
    assert torch.isnan(r.f[5]) and torch.isnan(r.g).all()


# route ---------------------------------------------------------------------------------------------------------------

def route_reference(s, top, kind, bias, bias_on, groups, top_groups, group_top, renormalize, scale):
    """64 bits, from the definition; differentiable in s. Closed slots: index -1, weight 0."""
    rows, cols = s.shape
    log_share = torch.log_softmax(s, -1) if kind == "softmax" else torch.nn.functional.logsigmoid(s)
    log_share = torch.where((s.detach() == -INF).all(-1, keepdim=True), -INF, log_share)
    share = log_share.detach().exp()
    key, rank = s.detach(), share
    if bias is not None:
        key = rank = (share if bias_on == "scores" else s.detach()) + bias.double()
    closed = (s.detach() == -INF) | (key == -INF)
    key, rank = key.masked_fill(closed, -INF), rank.masked_fill(closed, -INF)
    if groups > 1:
        best = rank.view(rows, groups, -1).sort(-1, descending=True).values[..., :group_top]
        score = torch.where(best[..., :1].squeeze(-1) == -INF, -INF, torch.where(best == -INF, 0.0, best).sum(-1))
        order = score.sort(dim=-1, descending=True, stable=True).indices
        place = order.argsort(-1)
        shut = (place >= top_groups) | (score == -INF)
        key = key.masked_fill(shut.repeat_interleave(cols // groups, 1), -INF)
    v = key.sort(dim=-1, descending=True, stable=True)
    index = torch.where(v.values[:, :top] == -INF, -1, v.indices[:, :top])
    chosen = torch.where(index >= 0, log_share.gather(1, index.clamp(min=0)), -INF)
    if renormalize:
        none = (index[:, :1] < 0)
        weight = torch.softmax(torch.where(none, torch.zeros((), dtype=s.dtype, device=s.device), chosen), -1)
        weight = torch.where(index >= 0, weight, 0.0)
    else:
        weight = torch.where(index >= 0, torch.where(index >= 0, chosen, 0.0).exp(), 0.0)
    return index, scale * weight


def check_route(s, top, kind="softmax", bias=None, bias_on="scores", groups=1, top_groups=None, group_top=2,
                renormalize=True, scale=1.0):
    leaf = s.detach().requires_grad_()
    r = scores.route(leaf, top, kind=kind, bias=bias, bias_on=bias_on, groups=groups, top_groups=top_groups,
                     group_top=group_top, renormalize=renormalize, scale=scale, load=True)
    wide = s.detach().double().requires_grad_()
    index, weight = route_reference(wide, top, kind, bias, bias_on, groups, top_groups or groups, group_top,
                                    renormalize, scale)
    assert torch.equal(r.index, index)
    # a share is off by its exponential and a row sum's chain; log shares of size L round a few times
    x = torch.where(index >= 0, s.double().gather(1, index.clamp(min=0)), 0.0).abs()
    rel = U * (GAMMA + s.shape[1] / 32 + 8 + 6 * (x + s.double().masked_fill(s == -INF, 0).abs().amax(-1, keepdim=True)))
    close(r.weight, weight.detach(), rel * weight.detach().abs() * 2 + 1e-44, "weight")
    counts = torch.bincount(index[index >= 0], minlength=s.shape[1])
    assert r.load.dtype == torch.int32 and torch.equal(r.load.long(), counts)
    d = torch.randn(index.shape, generator=gen(5), device="cuda")
    grad, = torch.autograd.grad(r.weight, leaf, d)
    want, = torch.autograd.grad(weight, wide, d.double())
    want = torch.where((index < 0).all(-1, keepdim=True), 0.0, torch.nan_to_num(want))
    # a chosen column's value is a share times (d - mean): both terms count; another's is a share times the mean
    size = scale * d.double().abs().amax(-1, keepdim=True) * weight.detach().new_ones(()) * torch.ones_like(want)
    part = torch.softmax(s.double(), -1) if kind == "softmax" else torch.ones_like(want)
    part = torch.nan_to_num(part)
    if renormalize or kind == "sigmoid":
        part = torch.zeros_like(want).scatter(1, index.clamp(min=0), weight.detach() / scale)
    tol = 4 * rel.amax(-1, keepdim=True) * part * size * (2 + top) + torch.finfo(s.dtype).eps / 2 * want.abs() * 1.01
    tol = tol + torch.finfo(s.dtype).smallest_normal * torch.finfo(s.dtype).eps + 1e-44
    # columns whose gradient is zero by cancellation: the 64-bit reference adds 2 + top terms of at most `size` (shares
    # are at most 1), each with a rounding of 2^-53 through the log-softmax and the softmax: below 4 (2 + top) 2^-53 size
    tol = tol + 4 * (2 + top) * 2.0 ** -53 * size
    assert grad.dtype == s.dtype
    close(grad, want, tol, "grad")
    return r


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,top", [(1, 1, 1), (3, 2, 2), (5, 8, 2), (65, 33, 4), (1000, 64, 6), (7, 256, 8),
                                           (33, 1000, 32), (4, 1024, 5), (501, 60, 1)])
@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
def test_route_values(rows, cols, top, kind, dtype):
    s = make(rows, cols, TYPES[dtype], seed=rows + cols, scale=1.5)
    for renormalize in (True, False):
        check_route(s, top, kind, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("bias_on", ["scores", "logits"])
@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups,group_top", [(1, 1, 2), (8, 4, 2), (8, 3, 1), (4, 4, 2), (32, 5, 2)])
def test_route_bias_and_groups(bias_on, kind, groups, top_groups, group_top):
    s = make(400, 96, torch.float32, seed=groups, scale=1.5)
    bias = 0.1 * make(1, 96, torch.float32, seed=1)[0]
    for renormalize in (True, False):
        check_route(s, 6, kind, bias, bias_on, groups, top_groups, group_top, renormalize)
    check_route(s, 6, kind, None, bias_on, groups, top_groups, group_top)


def test_route_ties():
    """Few distinct scores: equal keys and equal groups go to the lower index."""
    for dtype in (torch.float32, torch.bfloat16):
        s = torch.randint(-2, 3, (3000, 64), generator=gen(0), device="cuda").to(dtype)
        for bias in (None, torch.zeros(64, device="cuda"), torch.full((64,), 0.3, device="cuda")):
            for groups, top_groups in ((1, 1), (8, 3)):
                check_route(s, 7, "sigmoid", bias, "scores", groups, top_groups)
                check_route(s, 7, "softmax", bias, "logits", groups, top_groups)


def test_route_many_equal_keys():
    """More equal keys than a row's candidates have places."""
    for dtype in (torch.float32, torch.bfloat16):
        s = torch.zeros(20, 256, dtype=dtype, device="cuda")
        s[1, 100:] = 1.0
        s[2, ::2] = -3.0
        s[3, :250] = -INF
        for bias in (None, torch.zeros(256, device="cuda")):
            for groups, top_groups in ((1, 1), (8, 3)):
                check_route(s, 9, "softmax", bias, "scores", groups, top_groups)
                check_route(s, 9, "sigmoid", bias, "logits", groups, top_groups)


@pytest.mark.parametrize("cols,groups,top_groups,top", [(1020, 5, 2, 9), (1023, 3, 2, 4), (96, 3, 2, 5), (60, 6, 4, 7),
                                                       (84, 12, 5, 6), (25, 5, 3, 12), (32, 32, 9, 9), (14, 7, 7, 14),
                                                       (512, 1, 1, 32), (1024, 32, 8, 32)])
def test_route_group_layouts(cols, groups, top_groups, top):
    """Groups that are no power of two, of odd sizes, and of more columns than a lane's 32; the most choices."""
    for dtype in (torch.float32, torch.bfloat16):
        s = make(150, cols, dtype, seed=cols, scale=1.5)
        bias = 0.1 * make(1, cols, torch.float32, seed=1)[0]
        check_route(s, top, "sigmoid", bias, "scores", groups, top_groups)
        check_route(s, top, "softmax", bias, "logits", groups, top_groups, 1, False)
        check_route(s, top, "softmax", None, "scores", groups, top_groups)


def test_route_infinite_bias():
    """+inf puts a column first (several: by index), -inf closes it."""
    s = make(30, 40, torch.float32)
    bias = 0.1 * make(1, 40, torch.float32, seed=1)[0]
    bias[[9, 30]], bias[[3, 17]] = INF, -INF
    for bias_on in ("scores", "logits"):
        r = check_route(s, 5, "sigmoid", bias, bias_on)
        assert (r.index[:, 0] == 9).all() and (r.index[:, 1] == 30).all()


def test_route_keys_closer_than_float32():
    """Biased shares that differ by less than a float32 step are ordered by their 64-bit values."""
    s = torch.linspace(0.5, 0.5 + 2e-5, 64, device="cuda").repeat(200, 1)
    s = s[:, torch.randperm(64, generator=gen(3), device="cuda")]
    share = torch.sigmoid(s[0].double())
    bias = (1.0 - share).float()                     # the sum is 1 up to the bias's own rounding
    for groups, top_groups in ((1, 1), (4, 2)):
        check_route(s, 8, "sigmoid", bias, "scores", groups, top_groups)
    check_route(s, 8, "softmax", (1.0 - torch.softmax(s[0].double(), -1)).float(), "scores", 4, 2)


def test_route_masks():
    s = make(40, 32, torch.float32)
    s[0] = -INF                                       # nothing open
    s[1, 3:] = -INF                                   # fewer open than wanted
    s[2, :8] = -INF                                   # a whole group closed
    s[3, 1::2] = -INF
    s[4] = torch.finfo(torch.float32).min             # the lowest value is a score like another
    s[5, 4:] = torch.finfo(torch.float32).min
    s[6] = -200.0 - torch.arange(32, device="cuda")   # sigmoids that underflow keep their ratio
    s[7] = 300.0
    bias = 0.1 * make(1, 32, torch.float32, seed=1)[0]
    shut = bias.clone()
    shut[5:12] = -INF
    for kind in ("softmax", "sigmoid"):
        for groups, top_groups in ((1, 1), (4, 2)):
            for renormalize in (True, False):
                check_route(s[:4], 5, kind, None, "scores", groups, top_groups, 2, renormalize)
                check_route(s[:4], 5, kind, bias, "scores", groups, top_groups, 2, renormalize)
                check_route(s[8:], 5, kind, shut, "logits", groups, top_groups, 2, renormalize)
        check_route(s[4:8], 5, kind)


def test_route_nan_rows():
    s = make(4, 16, torch.bfloat16).requires_grad_()
    with torch.no_grad():
        s[1, 3], s[2, 0] = math.nan, INF
    for kind in ("softmax", "sigmoid"):
        r = scores.route(s, 3, kind=kind, renormalize=False, load=True)
        assert (r.index[1:3] == -1).all() and torch.isnan(r.weight[1:3]).all() and int(r.load.sum()) == 6
        g, = torch.autograd.grad(r.weight[0].sum(), s, retain_graph=True)
        assert (g[1:3] == 0).all()
    bias = torch.zeros(16, device="cuda")
    bias[2] = math.nan
    r = scores.route(s, 3, bias=bias)
    assert (r.index == -1).all() and torch.isnan(r.weight).all()


def test_route_strides_and_shapes():
    buf = make(1, 70 * 50 + 5, torch.bfloat16)[0]
    check_route(buf.as_strided((50, 48), (69, 1), 3), 4, "sigmoid")
    check_route(buf.as_strided((50, 48), (64, 1), 8), 4)
    check_route(make(1, 24, torch.float32).expand(9, 24), 4)
    s = make(12, 16, torch.float32)
    r = scores.route(s.view(3, 4, 16), 2)
    assert r.index.shape == (3, 4, 2) and r.load is None
    assert torch.equal(r.weight.view(12, 2), scores.route(s, 2).weight)
    r = scores.route(s[:0], 2, load=True)
    assert r.index.shape == (0, 2) and int(r.load.sum()) == 0


def test_route_gradient_by_differences_of_its_weights():
    """Central differences of the float32 weights: the choice is fixed for steps this small."""
    s = make(3, 10, torch.float32, seed=4)
    d = torch.randn(3, 4, generator=gen(1), device="cuda")
    for kind in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            call = lambda x: scores.route(x, 4, kind=kind, renormalize=renormalize)
            leaf = s.clone().requires_grad_()
            r = call(leaf)
            grad, = torch.autograd.grad(r.weight, leaf, d)
            h = 2.0 ** -8
            for j in range(10):
                e = torch.zeros_like(s)
                e[:, j] = h
                up, down = call(s + e), call(s - e)
                if not (torch.equal(up.index, r.index) and torch.equal(down.index, r.index)):
                    continue
                slope = ((up.weight.double() - down.weight.double()) * d).sum(-1) / (2 * h)
                # third derivatives of a share are below 1: h^2 / 6; weights are off by at most 2^-20 each
                assert (slope - grad[:, j]).abs().max() < d.abs().sum(-1).max() * (h * h / 6 + 2.0 ** -20 / h)


# together, streams, graphs -------------------------------------------------------------------------------------------

def test_inputs_are_left_as_they_were_and_outputs_stay_inside():
    """Guard values around every output buffer of the C calls: odd sizes, a gradient with a pitch."""
    from trnopt import _capi
    rows, cols, top = 7, 301, 5
    s = make(rows, cols, torch.bfloat16, seed=1)
    before = s.clone()
    t = torch.randint(cols, (rows, 2), generator=gen(1), device="cuda")

    def guarded(*shape, dtype=torch.float32, fill=77):
        n = math.prod(shape)
        whole = torch.full((n + 64,), fill, dtype=dtype, device="cuda")
        return whole, whole[32:32 + n]

    def intact(whole, fill=77):
        return bool((whole[:32] == fill).all() and (whole[-32:] == fill).all())

    st = torch.cuda.current_stream().cuda_stream
    bufs = {k: guarded(*shape, dtype=d) for k, shape, d in (
        ("lp", (rows, 2), torch.float32), ("h", (rows,), torch.float32), ("lse", (rows,), torch.float32),
        ("tl", (rows, top), torch.float32), ("ti", (rows, top), torch.int64), ("m", (rows,), torch.float32),
        ("ls", (rows,), torch.float32), ("f", (rows,), torch.float32), ("g", (cols,), torch.float32),
        ("ri", (rows, 3), torch.int64), ("rw", (rows, 3), torch.float32), ("ld", (cols,), torch.int32))}
    at = {k: v[1].data_ptr() for k, v in bufs.items()}
    _capi.check(_capi.lib.trnopt_log_probs(2, s.data_ptr(), cols, rows, cols, 1.0, t.data_ptr(), 2, top, at["lp"], at["h"],
                                           at["lse"], at["tl"], at["ti"], at["m"], at["ls"], st), "log_probs")
    pitch = 309
    grad, inner = guarded(rows, pitch, dtype=torch.bfloat16)
    _capi.check(_capi.lib.trnopt_log_probs_grad(2, s.data_ptr(), cols, rows, cols, 1.0, t.data_ptr(), 2, at["ti"], top,
                                                at["m"], at["ls"], at["h"], at["lp"], at["h"], None, None,
                                                inner.data_ptr(), pitch, st), "log_probs_grad")
    assert intact(grad) and (inner.view(rows, pitch)[:, cols:] == 77).all()
    ws = torch.full((_capi.lib.trnopt_balance_workspace_size(rows, cols) + 256,), 7, dtype=torch.uint8, device="cuda")
    _capi.check(_capi.lib.trnopt_balance(2, s.data_ptr(), cols, rows, cols, 0.5, 3, None, None, None, at["f"], at["g"],
                                         ws.data_ptr(), ws.numel() - 256, st), "balance")
    assert (ws[-256:] == 7).all()
    _capi.check(_capi.lib.trnopt_route(2, s.data_ptr(), cols, rows, cols, 3, 1, None, 0, 1, 1, 2, 1, 1.0, at["ri"], at["rw"],
                                       at["ld"], st), "route")
    grad, inner = guarded(rows, pitch, dtype=torch.bfloat16)
    _capi.check(_capi.lib.trnopt_route_grad(2, s.data_ptr(), cols, rows, cols, 3, 1, 1, 1.0, at["ri"], at["rw"],
                                            inner.data_ptr(), pitch, st), "route_grad")
    assert intact(grad) and (inner.view(rows, pitch)[:, cols:] == 77).all()
    assert all(intact(whole) for whole, _ in bufs.values()) and torch.equal(s, before)
    assert not any((v == 77).any() for k, (_, v) in bufs.items() if k not in ("ti", "ri", "ld"))


def test_workspace_too_small_is_refused():
    from trnopt import _capi
    s, f, g = make(4000, 64, torch.float32), torch.empty(4000, device="cuda"), torch.empty(64, device="cuda")
    need = _capi.lib.trnopt_balance_workspace_size(4000, 64)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    call = lambda at, n: _capi.lib.trnopt_balance(0, s.data_ptr(), 64, 4000, 64, 0.5, 3, None, None, None, f.data_ptr(),
                                                  g.data_ptr(), at, n, torch.cuda.current_stream().cuda_stream)
    assert call(ws.data_ptr(), need - 1) == -3 and call(None, need) == -3 and call(ws.data_ptr() + 16, need) == -2
    assert call(ws.data_ptr(), need) == 0


def test_balanced_router_step():
    """The three operators as a router's step uses them: potentials, a balanced choice, its weights' gradient, entropy."""
    s = (make(2048, 16, torch.float32, scale=1.0) + torch.linspace(2, -2, 16, device="cuda")).requires_grad_()
    plain = scores.route(s, 2, load=True)
    g = scores.balance(s, eps=0.25, iters=50).g
    r = scores.route(s, 2, bias=g, bias_on="logits", load=True)
    assert r.load.max() < 0.5 * plain.load.max() and int(r.load.sum()) == 4096
    h = scores.log_probs(s).entropy
    (r.weight[:, 0].sum() + h.mean()).backward()
    w = s.detach().double().requires_grad_()
    chosen = w.gather(1, r.index)
    (torch.softmax(chosen, -1)[:, 0].sum() + torch.distributions.Categorical(logits=w).entropy().mean()).backward()
    assert (s.grad - w.grad).abs().max() < 64 * U * w.grad.abs().max()


def steps(s, t):
    leaf = s.detach().requires_grad_()
    r = scores.log_probs(leaf, t, top=5)
    grad, = torch.autograd.grad(r.log_prob.sum() + r.entropy.sum(), leaf)
    b = scores.balance(s[:, :64], eps=0.3, iters=6)
    q = scores.route(s[:, :64], 4, bias=b.g, bias_on="logits", load=True)
    return [*r, grad, b.f, b.g, *q]


def test_side_stream():
    s, t = make(500, 3000, torch.bfloat16), torch.randint(3000, (500, 2), generator=gen(0), device="cuda")
    want = steps(s, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = steps(s, t)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(want, got):
        assert torch.equal(x, y)


def test_captured_graphs_replayed_together():
    """Two graphs of the same calls, replayed in turn and on two streams at once, on changing inputs."""
    state = [(make(300, 2500, torch.bfloat16, seed=k), torch.randint(2500, (300, 2), generator=gen(k), device="cuda"))
             for k in range(2)]
    graphs, outs = [], []
    for s, t in state:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            steps(s, t)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = steps(s, t)
        graphs.append(graph)
        outs.append(out)
    for k, (s, t) in enumerate(state):
        s.copy_(make(300, 2500, torch.bfloat16, seed=10 + k))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (s, t), out in zip(state, outs):
        for x, y in zip(steps(s, t), out):
            assert torch.equal(x, y)


def test_calls_on_two_streams_at_once():
    s, t = make(2000, 2000, torch.float32), torch.randint(2000, (2000, 1), generator=gen(0), device="cuda")
    want = steps(s, t)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for stream in streams:
        with torch.cuda.stream(stream):
            got.append(steps(s, t))
    torch.cuda.synchronize()
    for out in got:
        for x, y in zip(want, out):
            assert torch.equal(x, y)


def test_large_balances_on_several_streams():
    """Grids that fill the GPU each and wait within themselves, queued on three streams beside other work."""
    from trnopt import _capi
    s = [make(65536, 256, torch.bfloat16, seed=k, scale=1.0) for k in range(3)]
    want = [scores.balance(x, eps=0.1, iters=4) for x in s]
    m, other = make(4096, 4096, torch.bfloat16), torch.cuda.Stream()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        with torch.cuda.stream(other):
            m @ m
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((k, scores.balance(s[k], eps=0.1, iters=4)))
    torch.cuda.synchronize()
    assert all(torch.equal(r.f, want[k].f) and torch.equal(r.g, want[k].g) for k, r in got)
    assert _capi.device_error_flags() == 0


def test_refusals():
    s = make(4, 10, torch.float32)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    bad = [lambda: scores.log_probs(s.int()), lambda: scores.log_probs(s[:, :0]), lambda: scores.log_probs(s, top=65),
           lambda: scores.log_probs(s, top=-1), lambda: scores.log_probs(s, temperature=0.0),
           lambda: scores.log_probs(s, temperature=math.nan), lambda: scores.log_probs(s, t.cpu()),
           lambda: scores.log_probs(s, t.float()), lambda: scores.log_probs(s, t[:3]),
           lambda: scores.log_probs(s, t.repeat(1025, 1).t()),
           lambda: scores.balance(s.double()), lambda: scores.balance(s, eps=0.0), lambda: scores.balance(s, iters=0),
           lambda: scores.balance(s[:0]), lambda: scores.balance(make(2, 1025, torch.float32)),
           lambda: scores.balance(s, a=torch.ones(3, device="cuda")), lambda: scores.balance(s, b=torch.ones(10)),
           lambda: scores.balance(s, g=torch.ones(10, device="cuda").double()),
           lambda: scores.route(s, 0), lambda: scores.route(s, 11), lambda: scores.route(s, 2, kind="relu"),
           lambda: scores.route(s, 2, bias_on="weights"), lambda: scores.route(s, 2, groups=3),
           lambda: scores.route(s, 2, groups=5, top_groups=6), lambda: scores.route(s, 3, groups=5, top_groups=1),
           lambda: scores.route(s, 2, groups=5, group_top=3), lambda: scores.route(s, 2, scale=math.inf),
           lambda: scores.route(s, 2, bias=torch.zeros(9, device="cuda")), lambda: scores.route(s.double(), 2),
           lambda: scores.route(make(2, 64, torch.float32), 33)]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", k)


# the plan's rows -----------------------------------------------------------------------------------------------------

def test_refusals_of_too_many_rows():
    s = torch.zeros(1, 8, device="cuda").expand(2 ** 31, 8)
    with pytest.raises(ValueError, match="rows"):
        scores.route(s, 1, load=True)
    with pytest.raises(ValueError, match="rows"):
        scores.balance(s)


def test_descendants(monkeypatch):
    import numpy as np
    from oracle import trnopt_oracle as O
    from trnopt import plan
    rng = np.random.default_rng(0)
    n, m, d = 130, 77, 5
    x, y = rng.normal(size=(n, d)), rng.normal(size=(m, d)) * 0.7 + 0.2
    a, b = rng.random(n) + 0.1, rng.random(m) + 0.1
    r = O.Result(f=rng.normal(size=n), g=rng.normal(size=m), iterations=0, error=0.0, converged=True,
                 cost=float("nan"), seconds=0.0, eps=0.7, rho=None, center=rng.normal(size=d) * 0.1, cost_scale=1.3)
    P = O.transport_plan(x, y, r, a, b)
    cond = P / P.sum(1, keepdims=True)
    monkeypatch.setattr(plan, "_BLOCK", 50 * m)          # several blocks, the last one short
    t = rng.integers(m, size=(n, 3))
    got = plan.descendants(x, y, r, targets=t, top=6, a=a, b=b)
    order = np.argsort(-cond, axis=1, kind="stable")[:, :6]
    np.testing.assert_array_equal(got.top_index, order)
    np.testing.assert_allclose(got.top_log_prob, np.log(np.take_along_axis(cond, order, 1)), rtol=0, atol=1e-11)
    np.testing.assert_allclose(got.log_prob, np.log(np.take_along_axis(cond, t, 1)), rtol=0, atol=1e-11)
    np.testing.assert_allclose(got.entropy, -(cond * np.log(cond)).sum(1), rtol=0, atol=1e-11)
    np.testing.assert_allclose(got.log_mass, np.log(P.sum(1)), rtol=0, atol=1e-11)
    some = plan.descendants(x, y, r, rows=[5, -1], targets=[1, -1], top=0, a=a, b=b)
    assert some.log_prob[0] == pytest.approx(np.log(cond[5, 1]), abs=1e-11) and some.log_prob[1] == 0
    assert some.top_index.shape == (2, 0)
    none = plan.descendants(x, y, r, rows=[], top=3, a=a, b=b)
    assert none.entropy.shape == (0,) and none.top_index.shape == (0, 3) and none.log_prob is None
    for bad in (dict(rows=[n]), dict(rows=[0], targets=[m])):
        with pytest.raises(IndexError):
            plan.descendants(x, y, r, a=a, b=b, **bad)
    for bad in (dict(top=65), dict(rows=[0], targets=[0.5]), dict(rows=[0], targets=[0, 1])):
        with pytest.raises(ValueError):
            plan.descendants(x, y, r, a=a, b=b, **bad)


def test_gradients_are_differentiable_once():
    """A second derivative is refused when it is asked for; a graph of the first alone is fine."""
    s = make(3, 20, torch.float32).requires_grad_()
    for out in (scores.log_probs(s).entropy.sum(), scores.route(s, 2).weight[:, 0].sum()):
        g, = torch.autograd.grad(out, s, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), s)
