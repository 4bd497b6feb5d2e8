"""The operators over an explicit score matrix (trnopt.scores): what is measured, and their plain forms.

A score matrix has one row per thing to be assigned (a position of a sequence, a token, a cell) and one column per thing
it can be assigned to (a vocabulary entry, an expert, a cell of the next day).

    log_probs   log-probabilities of given columns, entropy and the best columns of each row's softmax; with gradient
    balance     the potentials of an entropic transport plan between rows and columns (Sinkhorn on the score matrix)
    route       each row's best columns by softmax or sigmoid scores, with a bias, groups and weights; with gradient
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}


def _log_probs_case(name, rows, cols, dtype, targets=1, top=0, train=False, temperature=1.0, masked=False, pad=0):
    return {"name": name, "op": "log_probs", "rows": rows, "cols": cols, "dtype": dtype, "targets": targets, "top": top,
            "train": train, "temperature": temperature, "masked": masked, "pad": pad}


def _balance_case(name, rows, cols, dtype, iters, eps, padded=False, warm=False):
    return {"name": name, "op": "balance", "rows": rows, "cols": cols, "dtype": dtype, "iters": iters, "eps": eps,
            "padded": padded, "warm": warm}


def _route_case(name, rows, cols, dtype, top, kind, bias="none", groups=1, top_groups=1, renormalize=True, train=False):
    return {"name": name, "op": "route", "rows": rows, "cols": cols, "dtype": dtype, "top": top, "kind": kind,
            "bias": bias, "groups": groups, "top_groups": top_groups, "renormalize": renormalize, "train": train}


def listed():
    return [
        # one sequence being decoded: the token's log-probability and twenty alternatives, latency counts
        _log_probs_case("log_probs_1x131072_bf16", 1, 131072, "bf16", top=20),
        # a served batch with a constrained vocabulary (masked columns), sampling temperature, scores inside a padded buffer
        _log_probs_case("log_probs_61x50001_f32_masked", 61, 50001, "f32", top=8, temperature=0.7, masked=True, pad=47),
        # scoring a long prompt: every position's token and five alternatives (the largest case)
        _log_probs_case("log_probs_4096x131072_bf16", 4096, 131072, "bf16", top=5),
        # the plan's rows between two days of cells, in the plan's own float64: ten most probable descendants
        _log_probs_case("log_probs_735x896_f64", 735, 896, "f64", targets=4, top=10),
        # a policy-gradient step: log-probabilities and entropy with their gradient
        _log_probs_case("log_probs_train_8192x32768_bf16", 8192, 32768, "bf16", train=True),
        # training against eight given alternatives a row, odd vocabulary
        _log_probs_case("log_probs_train_1023x50001_f16", 1023, 50001, "f16", targets=8, train=True, temperature=2.0),
        # balancing a small batch over a few experts from the last step's potentials
        _balance_case("balance_509x24_f32", 509, 24, "f32", iters=4, eps=0.5, warm=True),
        # balancing a padded training batch
        _balance_case("balance_8192x64_bf16_padded", 8192, 64, "bf16", iters=10, eps=0.25, padded=True),
        # a large batch over many experts, to near convergence
        _balance_case("balance_65536x256_bf16", 65536, 256, "bf16", iters=20, eps=0.1),
        # one decoded token through a router with groups and a bias for balance
        _route_case("route_1x256_f32_grouped", 1, 256, "f32", 8, "sigmoid", bias="scores", groups=8, top_groups=4),
        # a prefill batch through the same router, with its gradient
        _route_case("route_train_32768x256_f32_grouped", 32768, 256, "f32", 8, "sigmoid", bias="scores", groups=8,
                    top_groups=4, train=True),
        # a softmax router that follows balance's potentials, odd sizes, plain softmax weights
        _route_case("route_train_10007x60_bf16", 10007, 60, "bf16", 6, "softmax", bias="logits", renormalize=False,
                    train=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs", "balance", "route"])
    if op == "log_probs":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32", "f64"])
        train = rng.random() < 0.4
        cols = _spread(rng, 500, 20000 if dtype == "f64" else 262144)
        rows = _spread(rng, 1, max(1, min(8192, 2 ** (26 if train or dtype == "f64" else 28) // cols)))
        case = _log_probs_case("", rows, cols, dtype, targets=rng.choice([1, 1, 2, 5, 16]),
                               top=0 if train else rng.choice([0, 1, 5, 20, 33, 64]), train=train,
                               temperature=rng.choice([1.0, 1.0, 0.6, 1.7]), masked=rng.random() < 0.3,
                               pad=rng.choice([0, 0, 1, 24]))
    elif op == "balance":
        cols = _spread(rng, 4, 384)
        rows = _spread(rng, 1, min(65536, 2 ** 24 // cols))
        case = _balance_case("", rows, cols, rng.choice(["bf16", "f16", "f32"]), rng.randint(1, 16),
                             rng.choice([0.05, 0.1, 0.3, 1.0]), padded=rng.random() < 0.3, warm=rng.random() < 0.5)
    else:
        groups = rng.choice([1, 1, 4, 8])
        cols = groups * _spread(rng, 4, 256 // groups + 10)
        top_groups = rng.randint((groups + 1) // 2, groups)
        top = rng.randint(1, min(12, top_groups * (cols // groups)))
        case = _route_case("", _spread(rng, 1, 32768), cols, rng.choice(["bf16", "f16", "f32"]), top,
                           rng.choice(["softmax", "sigmoid"]), bias=rng.choice(["none", "scores", "logits"]), groups=groups,
                           top_groups=top_groups, renormalize=rng.random() < 0.6, train=rng.random() < 0.5)
    del case["name"]
    return case


def _api():
    package = os.path.join(os.getcwd(), "trainium-sinkhorn_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from trnopt import scores
    return scores


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    rows, cols, dtype = case["rows"], case["cols"], _TYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["op"] == "log_probs":
        # scores of a trained model: a common frequency term a column, noise, and a few strong columns a row
        buffer = torch.empty(rows, cols + case["pad"], dtype=dtype, device=dev)
        common = normal(cols + case["pad"])
        for r in range(0, rows, 1024):
            block = normal(min(1024, rows - r), cols + case["pad"]).mul_(2.0).add_(common)
            strong = torch.randint(cols, (block.shape[0], 4), generator=gen, device=dev)
            block.scatter_add_(1, strong, 6.0 + 2.0 * normal(*strong.shape))
            buffer[r:r + 1024] = block
        scores = buffer[:, :cols]
        if case["masked"]:
            closed = torch.rand(cols, generator=gen, device=dev) < 0.3
            scores.masked_fill_(closed, -math.inf)
            scores[rows // 2 + 1::17] = -math.inf                   # rows of slots that are not in use
        targets = torch.randint(cols, (rows, case["targets"]), generator=gen, device=dev)
        targets[torch.rand(rows, case["targets"], generator=gen, device=dev) < 0.05] = -1      # padding
        out = torch.float64 if dtype == torch.float64 else torch.float32
        state.update(scores=scores, targets=targets, d_log_prob=normal(rows, case["targets"]).to(out),
                     d_entropy=0.1 * normal(rows).to(out))
        return state
    # router scores: a popularity term a column and noise
    state["scores"] = (normal(rows, cols) + 0.7 * normal(cols)).to(dtype)
    if case["op"] == "balance":
        a = torch.full((rows,), 1.0, device=dev)
        if case["padded"]:
            a[rows - rows // 8:] = 0.0
        state["a"] = a / a.sum() if case["padded"] else None
        b = 0.5 + torch.rand(cols, generator=gen, device=dev)
        state["b"] = b / b.sum() if case["padded"] else None
        state["g"] = 0.3 * normal(cols) if case["warm"] else None
    else:
        scale = {"none": 0.0, "scores": 0.05, "logits": 0.7}[case["bias"]]
        state["bias"] = scale * normal(cols) if case["bias"] != "none" else None
        state["d_weight"] = normal(rows, case["top"])
    return state


# The plain forms ---------------------------------------------------------------------------------------------------

def _ordered(values):
    """Whole numbers in the order of the float32 values (equal values equal)."""
    bits = (values + 0.0).view(torch.int32).long()
    return torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))


def _best(values, k):
    """The k largest of each row by (value, lower index first): indices."""
    if values.dtype == torch.float64:
        return values.sort(dim=-1, descending=True, stable=True).indices[..., :k]
    cols = values.shape[-1]
    index = torch.arange(cols, device=values.device)
    key = _ordered(values) * cols + (cols - 1 - index)
    return key.topk(k, dim=-1).indices


def _plain_log_probs(state):
    case, scores, targets = state["case"], state["scores"], state["targets"]
    kept = scores.double() if scores.dtype == torch.float64 else scores.float()
    z = kept / case["temperature"]
    peak = z.amax(-1, keepdim=True)
    peak = torch.where(peak == -math.inf, torch.zeros_like(peak), peak)
    down = z - peak
    e = down.exp()
    total = e.sum(-1, keepdim=True)
    lse = peak + total.log()
    empty = total == 0
    entropy = total.log() - torch.where(e > 0, e * down, torch.zeros_like(e)).sum(-1, keepdim=True) / total
    entropy = torch.where(empty, torch.zeros_like(entropy), entropy)

    def log_p(index):
        return torch.where(empty, torch.full_like(lse, -math.inf), z.gather(1, index) - lse)

    given = targets >= 0
    log_prob = torch.where(given, log_p(targets.clamp(min=0)), torch.zeros_like(lse))
    out = {"log_prob": log_prob, "entropy": entropy[:, 0], "lse": lse[:, 0]}
    if case["top"]:
        index = _best(kept, case["top"])
        value = log_p(index)
        out["top_log_prob"] = value
        out["top_index"] = torch.where(kept.gather(1, index) == -math.inf, -1, index)
    if case["train"]:
        g = torch.where(given, state["d_log_prob"], torch.zeros_like(log_prob))
        p = torch.where(empty, torch.zeros_like(e), e / total)
        log_all = torch.where(p > 0, z - lse, torch.zeros_like(p))
        grad = -p * (g.sum(-1, keepdim=True) + state["d_entropy"][:, None] * (log_all + entropy))
        grad = grad.scatter_add(1, targets.clamp(min=0), torch.where(empty, torch.zeros_like(g), g))
        out["grad"] = (grad / case["temperature"]).to(scores.dtype)
    return out


def _lse(t, dim):
    peak = t.amax(dim, keepdim=True)
    return (peak + (t - peak).exp().sum(dim, keepdim=True).log()).squeeze(dim)


def _plain_balance(state):
    # potentials are differences of logarithms many times their size: 64 bits
    case, scores = state["case"], state["scores"].double()
    rows, cols, eps = case["rows"], case["cols"], case["eps"]
    uniform_a = torch.full((rows,), -math.log(rows), dtype=torch.float64, device=scores.device)
    uniform_b = torch.full((cols,), -math.log(cols), dtype=torch.float64, device=scores.device)
    log_a = state["a"].double().log() if state["a"] is not None else uniform_a
    log_b = state["b"].double().log() if state["b"] is not None else uniform_b
    g = state["g"].double() if state["g"] is not None else torch.zeros_like(uniform_b)
    for _ in range(case["iters"]):
        f = -eps * _lse(log_b + (g + scores) / eps, 1)
        g = -eps * _lse(log_a[:, None] + (f[:, None] + scores) / eps, 0)
    return {"f": f.float(), "g": g.float()}


def _plain_route(state):
    case, scores, bias = state["case"], state["scores"].float(), state["bias"]
    rows, cols = scores.shape
    # the order of columns is a comparison of close values: 64 bits
    wide = scores.double()
    if case["kind"] == "softmax":
        e = (wide - wide.amax(-1, keepdim=True)).exp()
        share = e / e.sum(-1, keepdim=True)
    else:
        share = 1.0 / (1.0 + (-wide).exp())
    if case["bias"] == "scores":
        key = share + bias.double()
    elif case["bias"] == "logits":
        key = wide + bias.double()
    else:
        key = wide
    if case["groups"] > 1:
        # without a bias on the scores a group still goes by its scores' sum
        rank = share if case["bias"] == "none" else key
        parts = rank.view(rows, case["groups"], -1)
        group = parts.sort(-1, descending=True).values[..., :2].sum(-1)
        kept = _best(group, case["top_groups"])
        open_ = torch.zeros_like(group, dtype=torch.bool).scatter(1, kept, True)
        key = torch.where(open_[..., None].expand_as(parts).reshape(rows, cols), key, torch.full_like(key, -math.inf))
    index = _best(key, case["top"])
    share = share.float()
    chosen = share.gather(1, index)
    weight = chosen / chosen.sum(-1, keepdim=True) if case["renormalize"] else chosen
    load = torch.zeros(cols, dtype=torch.int32, device=scores.device)
    load = load.index_add(0, index.reshape(-1), torch.ones(index.numel(), dtype=torch.int32, device=scores.device))
    out = {"index": index, "weight": weight, "load": load}
    if case["train"]:
        d = state["d_weight"]
        if case["renormalize"]:
            d = (d - (d * weight).sum(-1, keepdim=True)) / chosen.sum(-1, keepdim=True)
        d_share = torch.zeros_like(share).scatter(1, index, d)
        if case["kind"] == "softmax":
            grad = share * (d_share - (d_share * share).sum(-1, keepdim=True))
        else:
            grad = d_share * share * (1.0 - share)
        out["grad"] = grad.to(state["scores"].dtype)
    return out


# The framework's calls -----------------------------------------------------------------------------------------------

def _own_log_probs(state):
    case, scores = state["case"], state["scores"]
    if case["train"]:
        scores = scores.detach().requires_grad_()
    r = _api().log_probs(scores, state["targets"], top=case["top"], temperature=case["temperature"])
    out = {"log_prob": r.log_prob.detach(), "entropy": r.entropy.detach(), "lse": r.lse.detach()}
    if case["top"]:
        out["top_log_prob"], out["top_index"] = r.top_log_prob, r.top_index
    if case["train"]:
        out["grad"], = torch.autograd.grad((r.log_prob, r.entropy), (scores,), (state["d_log_prob"], state["d_entropy"]))
    return out


def _own_balance(state):
    case = state["case"]
    r = _api().balance(state["scores"], eps=case["eps"], iters=case["iters"], a=state["a"], b=state["b"], g=state["g"])
    return {"f": r.f, "g": r.g}


def _own_route(state):
    case, scores = state["case"], state["scores"]
    if case["train"]:
        scores = scores.detach().requires_grad_()
    r = _api().route(scores, case["top"], kind=case["kind"], bias=state["bias"],
                     bias_on="logits" if case["bias"] == "logits" else "scores", groups=case["groups"],
                     top_groups=case["top_groups"], renormalize=case["renormalize"], load=True)
    out = {"index": r.index, "weight": r.weight.detach(), "load": r.load}
    if case["train"]:
        out["grad"], = torch.autograd.grad((r.weight,), (scores,), (state["d_weight"],))
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"log_probs": _own_log_probs, "balance": _own_balance, "route": _own_route}[op](state)
    return {"log_probs": _plain_log_probs, "balance": _plain_balance, "route": _plain_route}[op](state)


def work(case):
    rows, cols = case["rows"], case["cols"]
    matrix = rows * cols * {"bf16": 2, "f16": 2, "f32": 4, "f64": 8}[case["dtype"]]
    if case["op"] == "log_probs":
        size = 8 if case["dtype"] == "f64" else 4
        small = rows * (case["targets"] * (8 + size) + 2 * size + case["top"] * (8 + size))
        if case["train"]:
            # scores in and their gradient out
            return {"bytes": 2 * matrix + small + rows * (case["targets"] + 1) * size, "flops": 10 * rows * cols}
        return {"bytes": matrix + small, "flops": 5 * rows * cols}
    if case["op"] == "balance":
        # one exponential an element and iteration serves both half-steps: product-sum, exp, sum, product-sum
        return {"bytes": matrix + 4 * (rows + cols), "flops": 6 * rows * cols * case["iters"]}
    small = rows * case["top"] * 12 + cols * 8
    if case["train"]:
        return {"bytes": 2 * matrix + small + rows * case["top"] * 4, "flops": 10 * rows * cols}
    return {"bytes": matrix + small, "flops": 6 * rows * cols}


# From the definitions, in 64 bits --------------------------------------------------------------------------------------

def _exact_log_probs(state):
    case = state["case"]
    done = []
    for r in range(0, case["rows"], 512):
        s = state["scores"][r:r + 512].double()
        t = state["targets"][r:r + 512]
        full = torch.log_softmax(s / case["temperature"], -1)
        none = (s == -math.inf).all(-1)
        full_or_0 = torch.where((s == -math.inf), torch.zeros_like(full), full)
        lp = torch.where(t >= 0, full.gather(1, t.clamp(min=0)), torch.zeros_like(full[:, :1]))
        lp = torch.where(none[:, None] & (t >= 0), torch.full_like(lp, -math.inf), lp)
        h = -(full_or_0.exp() * full_or_0).masked_fill(s == -math.inf, 0.0).sum(-1)
        part = {"log_prob": lp, "entropy": h, "lse": torch.logsumexp(s / case["temperature"], -1)}
        if case["top"]:
            v = s.sort(dim=-1, descending=True, stable=True)
            i = v.indices[:, :case["top"]]
            part["top_log_prob"] = torch.where(none[:, None], torch.full((1, 1), -math.inf, dtype=s.dtype, device=s.device),
                                               full.gather(1, i))
            part["top_index"] = torch.where(v.values[:, :case["top"]] == -math.inf, -1, i)
        if case["train"]:
            # by the chain rule on log p of each column: d/ds_j log p_t = (1[j = t] - p_j) / T
            p = torch.where(none[:, None], torch.zeros_like(full), full.exp())
            g = torch.where(t >= 0, state["d_log_prob"][r:r + 512].double(), torch.zeros((), dtype=s.dtype, device=s.device))
            g = torch.where(none[:, None], torch.zeros_like(g), g)
            on = torch.zeros_like(p).scatter_add_(1, t.clamp(min=0), g)
            through_p = state["d_entropy"][r:r + 512].double()[:, None] * -(full_or_0 + 1.0)     # dH / dp
            through_p = torch.where(p > 0, through_p, torch.zeros_like(p))
            through_p = through_p - (p * through_p).sum(-1, keepdim=True)
            part["grad"] = (on - p * g.sum(-1, keepdim=True) + p * through_p) / case["temperature"]
        done.append(part)
    return {k: torch.cat([d[k] for d in done]) for k in done[0]}


def _exact_balance(state):
    case, s = state["case"], state["scores"].double()
    eps = case["eps"]
    a = state["a"].double() if state["a"] is not None else torch.full_like(s[:, 0], 1.0 / case["rows"])
    b = state["b"].double() if state["b"] is not None else torch.full_like(s[0], 1.0 / case["cols"])
    g = state["g"].double() if state["g"] is not None else torch.zeros_like(s[0])
    for _ in range(case["iters"]):
        f = -eps * torch.logsumexp((g + s) / eps + torch.log(b), dim=1)
        g = -eps * torch.logsumexp(((f + eps * torch.log(a))[:, None] + s) / eps, dim=0)
    return {"f": f, "g": g}


def _exact_route(state):
    case = state["case"]
    s = state["scores"].double().requires_grad_(case["train"])
    rows, cols = s.shape
    share = torch.softmax(s, -1) if case["kind"] == "softmax" else torch.sigmoid(s)
    key, rank = s.detach(), share.detach()
    if case["bias"] != "none":
        key = rank = (rank if case["bias"] == "scores" else key) + state["bias"].double()
    if case["groups"] > 1:
        score = rank.reshape(rows, case["groups"], -1).topk(2, -1).values.sum(-1)
        order = score.argsort(dim=-1, descending=True, stable=True)
        place = order.argsort(dim=-1)                             # of each group in that order
        closed = (place >= case["top_groups"]).repeat_interleave(cols // case["groups"], dim=1)
        key = key.masked_fill(closed, -math.inf)
    index = key.argsort(dim=-1, descending=True, stable=True)[:, :case["top"]]
    weight = share.gather(1, index)
    if case["renormalize"]:
        weight = weight / weight.sum(-1, keepdim=True)
    out = {"index": index, "weight": weight.detach(), "load": torch.bincount(index.reshape(-1), minlength=cols).int()}
    if case["train"]:
        out["grad"], = torch.autograd.grad((weight,), (s,), (state["d_weight"].double(),))
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"log_probs": _exact_log_probs, "balance": _exact_balance, "route": _exact_route}[case["op"]](state)
