"""Assignment of rows to columns from a score matrix that a program already holds, on the GPU.

sinkhorn() and trnopt.plan take two point clouds and never store their scores. Here the scores S (rows x columns) are
given, as by a model's output layer or a router, and three operators work on them:

    log_probs(S, targets, top=k)   each row's softmax: log-probabilities of given columns, entropy, log-sum-exp, the k
                                   best columns; differentiable
    balance(S, eps=, iters=)       Sinkhorn on S: the potentials f, g of the entropic transport plan between rows and
                                   columns, P_ij = a_i b_j exp((f_i + g_j + S_ij) / eps)
    route(S, k, ...)               each row's k best columns by softmax or sigmoid scores, with a bias for balance
                                   (balance's g, or one of the program's own), groups and weights; differentiable

A balanced router is the three in a row: g = balance(S).g; r = route(S, k, bias=g, bias_on="logits"); the entropy of
log_probs(S) tells how decided the rows are. trnopt.plan.descendants applies log_probs to the rows of a plan.

Scores are CUDA tensors of any leading shape and row pitch (a last dimension that is not contiguous is copied first).
The calls queue on the scores' device, on that device's current stream, return without waiting, and can be captured into
a CUDA graph (backward() as torch asks for it: on a side stream, with no eager graph of the same leaves alive), but not
traced (torch.jit.trace is refused, as are forward-mode tangents: derivatives are backward's). There is no CPU path. What a
call rejects it rejects before anything is queued, with ValueError; values on the device (an index out of range, NaN)
never raise and show in the results as described.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _capi

MAX_TOP = 64             # log_probs: best columns per row
MAX_TARGETS = 1024       # log_probs: given columns per row
MAX_COLUMNS = 1024       # balance, route: columns
MAX_CHOICES = 32         # route: choices per row, groups

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float64: 3}
_KIND = {"softmax": 0, "sigmoid": 1}
_BIAS_ON = {"scores": 0, "logits": 1}


class LogProbs(NamedTuple):
    log_prob: torch.Tensor | None       # targets' shape
    entropy: torch.Tensor               # scores.shape[:-1], nats
    lse: torch.Tensor                   # scores.shape[:-1]: log sum_j exp(S_j / temperature)
    top_log_prob: torch.Tensor | None   # scores.shape[:-1] + (top,), best first
    top_index: torch.Tensor | None      # the same shape, int64


class Balance(NamedTuple):
    f: torch.Tensor                     # scores.shape[:-1], float32
    g: torch.Tensor                     # (columns,), float32


class Routing(NamedTuple):
    index: torch.Tensor                 # scores.shape[:-1] + (top,), int64, best first
    weight: torch.Tensor                # the same shape, float32
    load: torch.Tensor | None           # (columns,) int32: rows that chose each column


def _matrix(scores: torch.Tensor, double: bool, differentiable: bool = True) -> torch.Tensor:
    """The scores as a 2-d view with unit column stride (a copy only where there is no such view)."""
    if torch.jit.is_tracing():
        raise ValueError("the score kernels cannot be traced (torch.jit.trace would record empty outputs)")
    if differentiable and forward_ad._current_level >= 0 and isinstance(scores, torch.Tensor) and \
            forward_ad.unpack_dual(scores).tangent is not None:
        raise ValueError("the score kernels have no forward-mode derivatives")
    if not isinstance(scores, torch.Tensor) or not scores.is_cuda:
        raise ValueError("scores must be a CUDA tensor (the score kernels have no CPU path)")
    if scores.dtype not in _TYPE or (scores.dtype == torch.float64 and not double):
        raise ValueError(f"scores of type {scores.dtype} are not supported")
    if scores.dim() < 1 or scores.shape[-1] < 1:
        raise ValueError("scores need at least one column")
    if scores.shape[-1] >= 2 ** 31:
        raise ValueError("scores have too many columns")
    s = scores if scores.dim() == 2 else scores.reshape(-1, scores.shape[-1])
    return s if s.stride(1) == 1 or s.shape[1] == 1 else s.contiguous()


def _small(t: torch.Tensor | None, n: int, name: str, like: torch.Tensor) -> torch.Tensor | None:
    """A float32 vector of n values on the scores' device."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.device != like.device or t.dtype != torch.float32 or t.numel() != n:
        raise ValueError(f"{name} must hold {n} float32 values on {like.device}")
    return t.detach().contiguous()


# The current stream's handle on a device, without making a Stream object for it where torch offers that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, index: int, *args) -> None:
    """A C call on device `index`, on that device's current stream."""
    fn = getattr(_capi.lib, name)
    if index == torch.cuda.current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status != 0:
        _capi.check(status, name)


def _at(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _once(backward):
    """A backward pass that cannot be differentiated itself: torch's guard, entered only where a graph of it is wanted."""
    guarded = torch.autograd.function.once_differentiable(backward)
    return staticmethod(lambda ctx, *up: (guarded if torch.is_grad_enabled() else backward)(ctx, *up))


# log_probs -----------------------------------------------------------------------------------------------------------

def _log_probs_forward(s, lead, targets, n_targets, top, temperature, keep):
    """The call's outputs, in the shapes the user sees, and the rows' (maximum, log sum) if they are to be kept."""
    rows, cols = s.shape
    wide = torch.float64 if s.dtype == torch.float64 else torch.float32
    new = s.new_empty
    log_prob = None if targets is None else new(targets.shape, dtype=wide)
    entropy, lse = new(lead, dtype=wide), new(lead, dtype=wide)
    top_log_prob, top_index = (new((*lead, top), dtype=wide), new((*lead, top), dtype=torch.int64)) if top else (None,) * 2
    kept = new((2, rows), dtype=wide) if keep else None
    row_max = _at(kept)
    log_sum = row_max + rows * wide.itemsize if keep else None
    _call("trnopt_log_probs", s.get_device(), _TYPE[s.dtype], s.data_ptr(), s.stride(0), rows, cols, temperature,
          _at(targets), n_targets, top, _at(log_prob), entropy.data_ptr(), lse.data_ptr(), _at(top_log_prob),
          _at(top_index), row_max, log_sum)
    return log_prob, entropy, lse, top_log_prob, top_index, kept


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, targets, call):
        lead, n_targets, top, temperature = call
        log_prob, entropy, lse, top_log_prob, top_index, kept = _log_probs_forward(s, lead, targets, n_targets, top,
                                                                                   temperature, True)
        ctx.save_for_backward(s, targets, top_index, kept, entropy)
        ctx.call = call
        if top:
            ctx.mark_non_differentiable(top_index)
        ctx.set_materialize_grads(False)
        return log_prob, entropy, lse, top_log_prob, top_index

    @_once
    def backward(ctx, d_log_prob, d_entropy, d_lse, d_top, _):
        s, targets, top_index, kept, entropy = ctx.saved_tensors
        _, n_targets, top, temperature = ctx.call
        rows, cols = s.shape
        grad = s.new_empty((rows, cols))
        up = [None if d is None else d.contiguous() for d in (d_log_prob, d_entropy, d_lse, d_top)]
        row_max = kept.data_ptr()
        _call("trnopt_log_probs_grad", s.get_device(), _TYPE[s.dtype], s.data_ptr(), s.stride(0), rows, cols, temperature,
              _at(targets), n_targets, _at(top_index), top, row_max, row_max + rows * kept.element_size(),
              entropy.data_ptr(), *map(_at, up), grad.data_ptr(), cols)
        return grad, None, None


def log_probs(scores: torch.Tensor, targets: torch.Tensor | None = None, *, top: int = 0,
              temperature: float = 1.0) -> LogProbs:
    """The softmax of scores / temperature over the last dimension, never stored: the log-probabilities of given
    columns, the entropy (nats), the log-sum-exp, and the `top` best columns (score descending, equal scores by lower
    index).

    scores   float32, float16, bfloat16 or float64, any leading shape L and row pitch
    targets  int64 (int32 is converted), of shape L or L + (T,): column indices per row. Negative ones are padding
             (log_prob 0, no gradient), ones past the last column give NaN (and no gradient)
    Results are float32 (float64 for float64 scores). Columns of score -inf are closed: probability 0. In a row of
    nothing else log_prob and lse are -inf, entropy 0, and gradients 0; best columns beyond the open ones are -inf with
    index -1. A row holding NaN or +inf has NaN values and top_index -1. All floating outputs are differentiable with
    respect to the scores (once); the gradient has the scores' type."""
    s = _matrix(scores, True)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must lie in 0 .. {MAX_TOP}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be positive and finite (1e-30 .. 1e30)")
    lead, n_targets = scores.shape[:-1], 0
    if targets is not None:
        if not isinstance(targets, torch.Tensor) or targets.device != scores.device or \
                targets.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"targets must be an int64 or int32 tensor on {scores.device}")
        if targets.shape == lead:
            n_targets = 1
        elif targets.shape[:-1] == lead:
            n_targets = targets.shape[-1]
        else:
            raise ValueError(f"targets must have shape {tuple(lead)} or {tuple(lead)} + (T,)")
        if n_targets > MAX_TARGETS:
            raise ValueError(f"at most {MAX_TARGETS} targets a row")
        if targets.dtype != torch.int64 or not targets.is_contiguous():
            targets = targets.to(torch.int64).contiguous()
    if s.requires_grad and torch.is_grad_enabled():
        return LogProbs(*_LogProbs.apply(s, targets, (lead, n_targets, int(top), float(temperature))))
    return LogProbs(*_log_probs_forward(s, lead, targets, n_targets, int(top), float(temperature), False)[:5])


# balance -------------------------------------------------------------------------------------------------------------

def balance(scores: torch.Tensor, *, eps: float = 0.05, iters: int = 20, a: torch.Tensor | None = None,
            b: torch.Tensor | None = None, g: torch.Tensor | None = None) -> Balance:
    """`iters` Sinkhorn iterations on a score matrix, from the column potential g (None: 0):

        f_i = -eps LSE_j(log b_j + (g_j + S_ij) / eps),   g_j = -eps LSE_i(log a_i + (f_i + S_ij) / eps)

    the half-steps of sinkhorn() for the cost -S. After the last one the columns of P_ij = a_i b_j exp((f_i + g_j +
    S_ij) / eps) sum to b exactly and its rows to a as far as the iteration has converged; route(..., bias=g,
    bias_on="logits") chooses each row's largest entries of P / b.

    scores   float32, float16 or bfloat16, at most 1024 columns
    a, b     row and column masses, float32, >= 0 (None: 1 / rows, 1 / columns). Padding rows have mass 0: they move no
             column, and still get their f. Masses are used as given (their sums should agree)
    g        a starting potential, for instance the last step's; -inf leaves a column out of the first f
    A row or column whose terms are all zero (scores -inf, masses 0) has potential 0; a score more than 2.3e38 eps below
    its row's largest (among columns with mass) is as good as -inf. Rows and columns masked by large finite scores do not cost the others accuracy
    (but time: beyond about 700 eps from the others, terms are formed from pairs of float32). The potentials are constants
    to autograd."""
    s = _matrix(scores, False, False)
    rows, cols = s.shape
    if cols > MAX_COLUMNS:
        raise ValueError(f"at most {MAX_COLUMNS} columns")
    if rows < 1 or rows >= 2 ** 31:
        raise ValueError("scores need between 1 and 2**31 - 1 rows")
    if not 1e-30 <= eps <= 1e30:
        raise ValueError("eps must be positive and finite (1e-30 .. 1e30)")
    if not 1 <= iters <= 1 << 24:
        raise ValueError("iters must lie in 1 .. 2**24")
    a, b, g = _small(a, rows, "a", s), _small(b, cols, "b", s), _small(g, cols, "g", s)
    index = s.get_device()
    f = s.new_empty(scores.shape[:-1], dtype=torch.float32)
    g_out = s.new_empty((cols,), dtype=torch.float32)
    ws = s.new_empty((_balance_workspace(index, rows, cols),), dtype=torch.uint8)
    _call("trnopt_balance", index, _TYPE[s.dtype], s.data_ptr(), s.stride(0), rows, cols, float(eps), int(iters), _at(a),
          _at(b), _at(g), f.data_ptr(), g_out.data_ptr(), ws.data_ptr(), ws.numel())
    return Balance(f, g_out)


@lru_cache(maxsize=256)
def _balance_workspace(index: int, rows: int, cols: int) -> int:
    with torch.cuda.device(index):
        return max(256, int(_capi.lib.trnopt_balance_workspace_size(rows, cols)))


# route ---------------------------------------------------------------------------------------------------------------

def _route_forward(s, lead, top, kind, bias, bias_on, groups, top_groups, group_top, renormalize, scale, load):
    rows, cols = s.shape
    shape = (*lead, top)
    index, weight = s.new_empty(shape, dtype=torch.int64), s.new_empty(shape, dtype=torch.float32)
    counts = s.new_empty((cols,), dtype=torch.int32) if load else None
    _call("trnopt_route", s.get_device(), _TYPE[s.dtype], s.data_ptr(), s.stride(0), rows, cols, top, kind, _at(bias),
          bias_on, groups, top_groups, group_top, renormalize, scale, index.data_ptr(), weight.data_ptr(), _at(counts))
    return index, weight, counts


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, *call):
        index, weight, counts = _route_forward(s, *call)
        _, top, kind, *_, renormalize, scale, _ = call
        ctx.save_for_backward(s, index)
        ctx.call = (top, kind, renormalize, scale)
        ctx.mark_non_differentiable(*((index,) if counts is None else (index, counts)))
        ctx.set_materialize_grads(False)
        return index, weight, counts

    @_once
    def backward(ctx, _, d_weight, *__):
        if d_weight is None:
            return (None,) * 12
        s, index = ctx.saved_tensors
        rows, cols = s.shape
        grad = s.new_empty((rows, cols))
        d_weight = d_weight.contiguous()
        _call("trnopt_route_grad", s.get_device(), _TYPE[s.dtype], s.data_ptr(), s.stride(0), rows, cols, *ctx.call,
              index.data_ptr(), d_weight.data_ptr(), grad.data_ptr(), cols)
        return (grad,) + (None,) * 11


def route(scores: torch.Tensor, top: int, *, kind: str = "softmax", bias: torch.Tensor | None = None,
          bias_on: str = "scores", groups: int = 1, top_groups: int | None = None, group_top: int = 2,
          renormalize: bool = True, scale: float = 1.0, load: bool = False) -> Routing:
    """Each row's `top` best columns and their weights.

    kind         a column's share of a row: "softmax" over the row, or "sigmoid" of its score
    bias         (columns,) float32, in the choice only: added to the shares (bias_on="scores") or to the scores
                 themselves (bias_on="logits": balance's g). -inf closes a column. Without a bias columns go by their
                 scores
    groups       columns form `groups` equal runs; the `top_groups` (None: all) runs with the largest sum of their
                 `group_top` (1 or 2) largest biased shares (bias on the logits: biased scores) stay open
    weight       scale * share, or with renormalize scale * share / (sum of the row's chosen shares)
    load         count the rows that chose each column (of fewer than 2**31 rows)

    scores are float32, float16 or bfloat16, of at most 1024 columns; top and groups are at most 32. The order is that
    of the keys in 64 bits, equal keys by lower index. Columns of score -inf are closed; slots that no open column fills
    hold index -1 and weight 0. A row holding NaN or +inf (or a NaN bias) chooses nothing: index -1, weight NaN. The
    weights are differentiable with respect to the scores (once; the choice and the bias are constants); a row that
    chose nothing has gradient 0."""
    s = _matrix(scores, False)
    rows, cols = s.shape
    if cols > MAX_COLUMNS:
        raise ValueError(f"at most {MAX_COLUMNS} columns")
    if kind not in _KIND:
        raise ValueError(f"kind={kind!r}: choose 'softmax' or 'sigmoid'")
    if bias_on not in _BIAS_ON:
        raise ValueError(f"bias_on={bias_on!r}: choose 'scores' or 'logits'")
    if not 1 <= groups <= MAX_CHOICES or cols % groups:
        raise ValueError(f"groups must divide the columns and lie in 1 .. {MAX_CHOICES}")
    top_groups = groups if top_groups is None else top_groups
    if not 1 <= top_groups <= groups:
        raise ValueError("top_groups must lie in 1 .. groups")
    if group_top not in (1, 2):
        raise ValueError("group_top must be 1 or 2")
    if not 1 <= top <= min(MAX_CHOICES, top_groups * (cols // groups)):
        raise ValueError(f"top must lie in 1 .. {MAX_CHOICES} and not exceed the columns of the open groups")
    if not abs(scale) < 1e30:
        raise ValueError("scale must be finite")
    if load and rows >= 2 ** 31:
        raise ValueError("load counts fewer than 2**31 rows")
    bias = _small(bias, cols, "bias", s)
    forward = _Route.apply if s.requires_grad and torch.is_grad_enabled() else _route_forward
    return Routing(*forward(s, scores.shape[:-1], int(top), _KIND[kind], bias, _BIAS_ON[bias_on], int(groups),
                            int(top_groups), int(group_top), int(bool(renormalize)), float(scale), bool(load)))
