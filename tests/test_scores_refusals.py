"""What the score-matrix operators refuse, before any GPU work: the C ABI's argument checks (called with addresses that
are never read) and the Python layer's refusal of CPU tensors. CPU only."""

import ctypes

import pytest
import torch

from trnopt import _capi, scores

A = 1 << 20          # an aligned address; every call here is refused before it could be used
OK, INVALID, ALIGN, WS, UNSUPPORTED = 0, -1, -2, -3, -4
F32, F16, BF16, F64 = 0, 1, 2, 3


def log_probs(type=F32, scores=A, ld=10, rows=4, cols=10, temperature=1.0, targets=A, n_targets=1, top=2, log_prob=A,
              entropy=A, lse=A, top_log_prob=A, top_index=A, row_max=None, log_sum=None):
    return _capi.lib.trnopt_log_probs(type, scores, ld, rows, cols, temperature, targets, n_targets, top, log_prob,
                                      entropy, lse, top_log_prob, top_index, row_max, log_sum, None)


def log_probs_grad(type=F32, scores=A, ld=10, rows=4, cols=10, temperature=1.0, targets=A, n_targets=1, top_index=A,
                   top=2, row_max=A, log_sum=A, entropy=A, d=(None,) * 4, grad=A, ld_grad=10):
    return _capi.lib.trnopt_log_probs_grad(type, scores, ld, rows, cols, temperature, targets, n_targets, top_index,
                                           top, row_max, log_sum, entropy, *d, grad, ld_grad, None)


def balance(type=F32, scores=A, ld=8, rows=4, cols=8, eps=0.1, iters=2, a=None, b=None, g0=None, f=A, g=A, ws=A,
            ws_bytes=1 << 30):
    return _capi.lib.trnopt_balance(type, scores, ld, rows, cols, eps, iters, a, b, g0, f, g, ws, ws_bytes, None)


def route(type=F32, scores=A, ld=8, rows=4, cols=8, top=2, kind=0, bias=None, bias_on=0, groups=1, top_groups=1,
          group_top=2, renormalize=1, scale=1.0, index=A, weight=A, load=None):
    return _capi.lib.trnopt_route(type, scores, ld, rows, cols, top, kind, bias, bias_on, groups, top_groups,
                                  group_top, renormalize, scale, index, weight, load, None)


def route_grad(type=F32, scores=A, ld=8, rows=4, cols=8, top=2, kind=0, renormalize=1, scale=1.0, index=A, d_weight=A,
               grad=A, ld_grad=8):
    return _capi.lib.trnopt_route_grad(type, scores, ld, rows, cols, top, kind, renormalize, scale, index, d_weight,
                                       grad, ld_grad, None)


@pytest.mark.parametrize("call,status", [
    (dict(type=4), UNSUPPORTED), (dict(type=-1), UNSUPPORTED), (dict(scores=None), INVALID), (dict(rows=-1), INVALID),
    (dict(cols=0), INVALID), (dict(ld=-1), INVALID), (dict(scores=A + 2), ALIGN), (dict(type=F64, scores=A + 4), ALIGN),
    (dict(type=BF16, scores=A + 1), ALIGN), (dict(temperature=0.0), INVALID), (dict(temperature=-1.0), INVALID),
    (dict(temperature=float("nan")), INVALID), (dict(temperature=float("inf")), INVALID), (dict(n_targets=-1), INVALID),
    (dict(n_targets=1025), INVALID), (dict(targets=None), INVALID), (dict(log_prob=None), INVALID),
    (dict(top=-1), INVALID), (dict(top=65), INVALID), (dict(top_index=None), INVALID), (dict(entropy=None), INVALID),
    (dict(lse=None), INVALID), (dict(row_max=A), INVALID), (dict(targets=A + 4), ALIGN), (dict(lse=A + 2), ALIGN),
    (dict(type=F64, lse=A + 4), ALIGN)])
def test_log_probs_arguments(call, status):
    assert log_probs(**call) == status


@pytest.mark.parametrize("call,status", [
    (dict(ld_grad=9), INVALID), (dict(grad=None), INVALID), (dict(grad=A + 2), ALIGN), (dict(row_max=None), INVALID),
    (dict(entropy=None), INVALID), (dict(top_index=None), INVALID), (dict(top=65), INVALID),
    (dict(temperature=0.0), INVALID), (dict(d=(A + 2, None, None, None)), ALIGN), (dict(type=7), UNSUPPORTED)])
def test_log_probs_grad_arguments(call, status):
    assert log_probs_grad(**call) == status


@pytest.mark.parametrize("call,status", [
    (dict(type=F64), UNSUPPORTED), (dict(cols=1025, ld=1025), UNSUPPORTED), (dict(rows=0), INVALID),
    (dict(iters=0), INVALID), (dict(eps=0.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(f=None), INVALID),
    (dict(g=None), INVALID), (dict(g=A + 2), ALIGN), (dict(a=A + 1), ALIGN)])
def test_balance_arguments(call, status):
    assert balance(**call) == status


def test_balance_workspace_size_refuses_bad_shapes():
    for rows, cols in ((0, 8), (-1, 8), (8, 0), (8, 1025)):
        assert _capi.lib.trnopt_balance_workspace_size(rows, cols) == 0


@pytest.mark.parametrize("call,status", [
    (dict(type=F64), UNSUPPORTED), (dict(cols=1025, ld=1025), UNSUPPORTED), (dict(top=33, cols=64), UNSUPPORTED),
    (dict(groups=64, cols=64), UNSUPPORTED), (dict(top=0), INVALID), (dict(top=9), INVALID), (dict(groups=3), INVALID),
    (dict(groups=4, top_groups=5), INVALID), (dict(groups=4, top_groups=0), INVALID),
    (dict(groups=4, top_groups=1, top=3), INVALID), (dict(group_top=3), INVALID), (dict(kind=2), INVALID),
    (dict(bias_on=2), INVALID), (dict(scale=float("inf")), INVALID), (dict(index=None), INVALID),
    (dict(weight=None), INVALID), (dict(index=A + 4), ALIGN), (dict(bias=A + 2), ALIGN)])
def test_route_arguments(call, status):
    assert route(**call) == status


@pytest.mark.parametrize("call,status", [
    (dict(type=F64), UNSUPPORTED), (dict(ld_grad=7), INVALID), (dict(top=33), UNSUPPORTED), (dict(top=0), INVALID),
    (dict(index=None), INVALID), (dict(d_weight=None), INVALID), (dict(kind=5), INVALID), (dict(grad=A + 2), ALIGN)])
def test_route_grad_arguments(call, status):
    assert route_grad(**call) == status


def test_no_rows_launch_nothing():
    assert log_probs(rows=0) == OK
    assert log_probs_grad(rows=0) == OK
    assert route(rows=0) == OK
    assert route_grad(rows=0) == OK


def test_cpu_tensors_are_refused():
    s = torch.zeros(3, 4)
    for call in (lambda: scores.log_probs(s), lambda: scores.balance(s), lambda: scores.route(s, 1)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError):
        scores.log_probs([1.0, 2.0])


def test_route_load_counts_in_32_bits():
    assert route(rows=1 << 31, load=A) == INVALID


def test_forward_mode_derivatives_are_refused():
    """log_probs and route have no forward-mode derivative: a dual tensor would come back without its tangent."""
    s = torch.zeros(3, 4)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(s, torch.ones_like(s))
        for call in (lambda: scores.log_probs(dual), lambda: scores.route(dual, 1)):
            with pytest.raises(ValueError, match="forward"):
                call()
        with pytest.raises(ValueError, match="CUDA tensor"):          # a tensor without a tangent is as elsewhere
            scores.log_probs(s)


def test_tracing_is_refused():
    """torch.jit.trace records the outputs' allocation and not the call that fills them."""
    for fn in (lambda s: scores.log_probs(s).lse, lambda s: scores.balance(s).g, lambda s: scores.route(s, 1).weight):
        with pytest.raises(ValueError, match="trace"):
            torch.jit.trace(fn, torch.zeros(3, 4), check_trace=False)


@pytest.mark.parametrize("grad_call", [log_probs_grad, route_grad])
def test_gradient_in_the_scores_place_is_refused(grad_call):
    """Scores are read after parts of the gradient are written, so the two must not share elements."""
    row = dict(rows=1, ld=0)
    for offset in (0, 4, 28):                          # the same rows, and rows that begin inside the scores' rows
        assert grad_call(cols=8, ld=8, ld_grad=8, grad=A + offset) == INVALID
    assert grad_call(cols=8, ld=16, ld_grad=16, grad=A + 28) == INVALID
    assert grad_call(cols=8, ld=16, ld_grad=16, grad=A + 36) == INVALID
    assert grad_call(cols=8, ld=16, ld_grad=24, grad=A + 40) == INVALID       # other pitches: the whole ranges
    assert grad_call(cols=8, ld_grad=8, grad=A + 28, **row) == INVALID
    assert grad_call(cols=8, ld=8, ld_grad=8, grad=A - 4 * 8 * 4 + 4) == INVALID
