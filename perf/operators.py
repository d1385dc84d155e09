"""What is measured of the operators that work on a row's labels: the log probabilities of a row of
scores (label_scores), rows sorted by label and back (row_groups), and the codebook lookup with its
gradient (codebook).

`listed()` and `draw(rng)` give cases, `prepare(case, seed)` what a program holds before the call,
`run(state)` one pass: the operators' plain form in elementary torch operations, or, where `own` is
set, the framework's calls.  `exact(case, seed)` is the same from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "euclid-cuda_b200")
_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one new row's answer: its scores over a large set of labels, the log probability of the label
        # that was drawn, the entropy and the 20 best alternatives; latency counts
        dict(name="scores_one_row", op="scores", rows=1, cols=131072, dtype="bf16", scale=1.25, top=20, pad=0,
             mask=False, train=False),
        # soft assignment of a block of points to 1024 centers from their squared distances
        dict(name="scores_posterior", op="scores", rows=131072, cols=1024, dtype="fp32", scale=-0.5, top=8, pad=0,
             mask=False, train=False),
        # odd sizes, rows of a wider buffer, masked labels and rows with no label left
        dict(name="scores_masked_odd", op="scores", rows=777, cols=32771, dtype="fp16", scale=1.0, top=5, pad=13,
             mask=True, train=False),
        # a training step's loss over a large label set: log probability, entropy and the scores' gradient
        dict(name="scores_train", op="scores", rows=4096, cols=131072, dtype="bf16", scale=1.0, top=0, pad=0,
             mask=False, train=True),
        # a serving step of a few rows, each to 4 of 64 clusters and back; latency counts
        dict(name="groups_step", op="groups", rows=16, picks=4, clusters=64, dim=2048, dtype="bf16", drop=False,
             train=False),
        # a long input: every row to 8 of 128 clusters and back
        dict(name="groups_long", op="groups", rows=16384, picks=8, clusters=128, dim=2048, dtype="bf16", drop=False,
             train=False),
        # a training step: there, back, and both gradients
        dict(name="groups_train", op="groups", rows=8192, picks=4, clusters=256, dim=4096, dtype="bf16", drop=False,
             train=True),
        # odd sizes, and picks outside the clusters, which are dropped
        dict(name="groups_odd", op="groups", rows=5003, picks=3, clusters=37, dim=1001, dtype="fp32", drop=True,
             train=True),
        # a serving step of a few rows from a large table; latency counts
        dict(name="lookup_step", op="lookup", rows=8, clusters=32768, dim=4096, dtype="bf16", scale=64.0, drop=False,
             skew=True, train=False),
        # points replaced by their centers (vector quantisation), with the centers' gradient
        dict(name="lookup_points", op="lookup", rows=1048576, clusters=1024, dim=128, dtype="fp32", scale=1.0,
             drop=False, skew=False, train=True),
        # a training batch over a large table, few labels frequent and most rare
        dict(name="lookup_train", op="lookup", rows=65536, clusters=131072, dim=1024, dtype="bf16", scale=32.0,
             drop=False, skew=True, train=True),
        # odd sizes, and labels outside the table
        dict(name="lookup_odd", op="lookup", rows=30011, clusters=4099, dim=77, dtype="fp16", scale=0.5, drop=True,
             skew=True, train=True),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["scores", "groups", "lookup"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    train = rng.random() < 0.5
    if op == "scores":
        cols = _between(rng, 2, 131072)
        rows = _between(rng, 1, max(1, min(131072, (1 << 27) // cols)))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, scale=rng.choice([1.0, 0.7, -0.5, 2.5, -1.0]),
                    top=min(cols, rng.choice([0, 1, 2, 5, 8, 20, 32])), pad=rng.choice([0, 0, 1, 13, 64]),
                    mask=rng.random() < 0.3, train=train)
    if op == "groups":
        dim = _between(rng, 16, 4096)
        picks = rng.randint(1, 8)
        rows = _between(rng, 1, max(1, min(65536, (1 << 26) // (dim * picks))))
        return dict(op=op, rows=rows, picks=picks, clusters=_between(rng, 2, 4096), dim=dim, dtype=dtype,
                    drop=rng.random() < 0.4, train=train)
    dim = _between(rng, 4, 4096)
    return dict(op=op, rows=_between(rng, 1, min(1048576, (1 << 26) // dim)),
                clusters=_between(rng, 2, min(131072, (1 << 26) // dim)), dim=dim, dtype=dtype,
                scale=rng.choice([1.0, 0.5, 8.0, 27.7]), drop=rng.random() < 0.4, skew=rng.random() < 0.5, train=train)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda", dtype=torch.float64)

    def labels(shape, k, skew, drop):
        u = uniform(*shape)
        # skewed: the frequency of a label falls as one over its rank
        lab = ((k + 1.0) ** u - 1.0).long() if skew else (u * k).long()
        lab = lab.clamp_(0, k - 1)
        if drop:  # one in ten outside [0, k), on both sides
            r = uniform(*shape)
            lab = torch.where(r < 0.05, -1, torch.where(r > 0.95, k, lab))
        return lab.contiguous()

    state = dict(case=case)
    if case["op"] == "scores":
        n, m = case["rows"], case["cols"]
        buf = normal(n, m + case["pad"])
        # squared distances where the scale is negative, scores of a last layer otherwise
        buf = buf.mul_(4.0).add_(30.0).clamp_min_(0.0) if case["scale"] < 0 else buf.mul_(3.0)
        x = buf.to(dt)[:, :m]
        del buf
        if case["mask"]:
            out = -math.copysign(math.inf, case["scale"])
            x.masked_fill_(torch.rand(n, m, generator=gen, device="cuda") < 0.3, out)
            x[5::97] = out  # rows with no label left
        state.update(scores=x, labels=labels((n,), m, False, False))
        if case["train"]:
            state.update(grad_log_probs=normal(n), grad_entropy=normal(n) * 0.1)
    elif case["op"] == "groups":
        n, p, d = case["rows"], case["picks"], case["dim"]
        w = uniform(n, p).float() + 0.05
        state.update(X=normal(n, d).to(dt), Z=normal(n * p, d).to(dt), weights=w / w.sum(1, keepdim=True),
                     labels=labels((n, p), case["clusters"], False, case["drop"]))
        if case["train"]:
            state.update(grad_out=normal(n, d).to(dt), grad_Y=normal(n * p, d).to(dt))
    else:
        n, k, d = case["rows"], case["clusters"], case["dim"]
        state.update(C=normal(k, d).to(dt), labels=labels((n,), k, case["skew"], case["drop"]))
        if case["train"]:
            state.update(G=normal(n, d).to(dt))
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        return {"scores": _own_scores, "groups": _own_groups, "lookup": _own_lookup}[op](state)
    return {"scores": _plain_scores, "groups": _plain_groups, "lookup": _plain_lookup}[op](state)


def _own_scores(s):
    from label_scores import label_log_probs, label_log_probs_grad
    c = s["case"]
    r = label_log_probs(s["scores"], s["labels"], scale=c["scale"], top=c["top"])
    out = dict(log_probs=r.log_probs, entropy=r.entropy)
    if c["top"]:
        out.update(top_log_probs=r.top_log_probs, top_labels=r.top_labels)
    if c["train"]:
        out["grad"] = label_log_probs_grad(s["scores"], s["labels"], r.row_stats, s["grad_log_probs"],
                                           s["grad_entropy"], scale=c["scale"])
    return out


def _own_groups(s):
    from row_groups import group_rows, rows_from_groups, rows_from_groups_grad, rows_to_groups
    c = s["case"]
    g = group_rows(s["labels"], c["clusters"])
    out = dict(offsets=g.offsets, order=g.order, position=g.position, Y=rows_to_groups(s["X"], g),
               out=rows_from_groups(s["Z"], g, s["weights"]))
    if c["train"]:
        out["grad_Z"], out["grad_weights"] = rows_from_groups_grad(s["grad_out"], s["Z"], g, s["weights"])
        out["grad_X"] = rows_from_groups(s["grad_Y"], g)
    return out


def _own_lookup(s):
    from codebook import lookup, lookup_grad
    c = s["case"]
    out = dict(rows=lookup(s["C"], s["labels"], scale=c["scale"]))
    if c["train"]:
        out["grad_C"] = lookup_grad(s["G"], s["labels"], c["clusters"], scale=c["scale"])
    return out


def _plain_scores(s):
    c = s["case"]
    x, lab = s["scores"], s["labels"]
    n, m = x.shape
    y = x.float() if c["scale"] > 0 else -x.float()
    hi = y.amax(1)
    none_left = hi == -math.inf
    shift = torch.where(none_left, 0.0, hi)
    d = (y - shift[:, None]) * abs(c["scale"])
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, e * d, 0.0).sum(1)
    entropy = torch.where(none_left, 0.0, log_total - weighted / total)
    at = d.gather(1, lab[:, None])[:, 0]
    log_probs = torch.where(none_left, -math.inf, at - log_total)
    out = dict(log_probs=log_probs, entropy=entropy)
    if c["top"]:
        # one whole number per score, ordered as the scores are and, where those tie, by the lower index
        bits = (y + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (bits << 32) + (m - 1 - torch.arange(m, device=x.device))
        top = (m - 1) - (torch.topk(key, c["top"], dim=1).values & 0xFFFFFFFF)
        out["top_labels"] = top
        out["top_log_probs"] = torch.where(none_left[:, None], -math.inf, d.gather(1, top) - log_total[:, None])
    if c["train"]:
        p = torch.where(none_left[:, None], 0.0, e / total[:, None])
        log_p = torch.where(p > 0, d - log_total[:, None], 0.0)
        gl, ge = s["grad_log_probs"][:, None], s["grad_entropy"][:, None]
        grad = -p * (gl + ge * (log_p + entropy[:, None]))
        hit = torch.where(none_left, 0.0, s["grad_log_probs"])
        grad.scatter_add_(1, lab[:, None], hit[:, None])
        out["grad"] = (grad * c["scale"]).to(x.dtype)
    return out


def _plain_groups(s):
    c = s["case"]
    k, (n, p) = c["clusters"], s["labels"].shape
    flat = s["labels"].reshape(-1)
    kept = (flat >= 0) & (flat < k)
    key = torch.where(kept, flat, k)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=k + 1)[:k]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    rank = torch.arange(n * p, device=flat.device)
    filled = rank < offsets[k]
    position = torch.empty_like(order)
    position[order] = rank
    position = torch.where(kept, position, -1)
    src = order // p

    def there(rows):  # the rows' copies in sorted order, zeros after the last
        return torch.where(filled[:, None], rows[src], torch.zeros((), dtype=rows.dtype, device=rows.device))

    slot = position.clamp_min(0)
    w = torch.where(kept, s["weights"].reshape(-1), 0.0)

    def back(rows, weight):  # 32-bit sums of each row's picks
        return (rows[slot].float() * weight[:, None]).view(n, p, -1).sum(1).to(rows.dtype)

    out = dict(offsets=offsets.int(), order=torch.where(filled, order, -1).int(), position=position.view(n, p).int(),
               Y=there(s["X"]), out=back(s["Z"], w))
    if c["train"]:
        g = s["grad_out"].float()
        gz = g[src] * torch.where(filled, w[order], 0.0)[:, None]
        out["grad_Z"] = gz.to(s["Z"].dtype)
        dots = (g.repeat_interleave(p, 0) * s["Z"][slot].float()).sum(1)
        out["grad_weights"] = torch.where(kept, dots, 0.0).view(n, p)
        out["grad_X"] = back(s["grad_Y"], kept.float())
    return out


def _plain_lookup(s):
    c = s["case"]
    k, lab = c["clusters"], s["labels"]
    kept = (lab >= 0) & (lab < k)
    slot = torch.where(kept, lab, 0)
    out = dict(rows=torch.where(kept[:, None], s["C"][slot].float() * c["scale"], 0.0).to(s["C"].dtype))
    if c["train"]:
        g = torch.where(kept[:, None], s["G"].float(), 0.0)
        sums = torch.zeros(k, c["dim"], device=lab.device).index_add_(0, slot, g)
        out["grad_C"] = (sums * c["scale"]).to(s["G"].dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = _SIZE[case["dtype"]]
    n = case["rows"]
    if case["op"] == "scores":
        m, t = case["cols"], case["top"]
        each = n * m
        byts = each * b + n * (8 + 4 + 4) + n * t * (4 + 8)
        flops = 6 * each
        if case["train"]:  # scores read again, gradient written
            byts += 2 * each * b + n * (8 + 4 + 4)
            flops += 8 * each
        return {"bytes": byts, "flops": flops}
    d = case["dim"]
    if case["op"] == "groups":
        slots = n * case["picks"]
        byts = slots * (8 + 4 + 4 + 4) + (case["clusters"] + 1) * 4
        byts += (n + slots) * d * b + (slots + n) * d * b  # there, and back
        flops = 2 * slots * d
        if case["train"]:
            byts += (n + 2 * slots) * d * b + slots * (4 + 4) + (slots + n) * d * b
            flops += 4 * slots * d
        return {"bytes": byts, "flops": flops}
    # rows of the table that a batch can touch, at most
    byts = n * 8 + min(n, case["clusters"]) * d * b + n * d * b
    flops = n * d
    if case["train"]:
        byts += n * d * b + case["clusters"] * d * b
        flops += n * d
    return {"bytes": byts, "flops": flops}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"scores": _exact_scores, "groups": _exact_groups, "lookup": _exact_lookup}[case["op"]](case, s)


def _exact_scores(c, s):
    z = s["scores"].double() * c["scale"]
    n, m = z.shape
    lse = torch.logsumexp(z, 1)
    left = lse > -math.inf
    logp = z - torch.where(left, lse, 0.0)[:, None]
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(1)
    out = dict(log_probs=logp.gather(1, s["labels"][:, None])[:, 0], entropy=entropy)
    if c["top"]:
        best = torch.topk(logp, c["top"], dim=1).values
        out.update(top_log_probs=best, top_labels=None)
    if c["train"]:
        onehot = torch.zeros_like(z).scatter_(1, s["labels"][:, None], 1.0)
        grad = s["grad_log_probs"].double()[:, None] * (onehot - p)
        grad -= s["grad_entropy"].double()[:, None] * (plogp + p * entropy[:, None])
        out["grad"] = torch.where(left[:, None], grad, 0.0) * c["scale"]
    return out


def _exact_groups(c, s):
    k, p, n = c["clusters"], c["picks"], c["rows"]
    lab = s["labels"]
    ok = ((lab >= 0) & (lab < k))
    slots = torch.nonzero(ok.reshape(-1))[:, 0]
    which = lab.reshape(-1)[slots]
    sorted_slots = slots[torch.argsort(which * (n * p) + slots)]
    row = torch.div(sorted_slots, p, rounding_mode="floor")
    used = sorted_slots.numel()
    offsets = torch.searchsorted(which.sort().values, torch.arange(k + 1, device=lab.device))
    order = torch.full((n * p,), -1, dtype=torch.int32, device=lab.device)
    order[:used] = sorted_slots.int()
    position = torch.full((n * p,), -1, dtype=torch.int32, device=lab.device)
    position[sorted_slots] = torch.arange(used, dtype=torch.int32, device=lab.device)
    Y = torch.zeros(n * p, c["dim"], dtype=torch.float64, device=lab.device)
    Y[:used] = s["X"].double()[row]
    w = s["weights"].double().reshape(-1)[sorted_slots]
    zeros = torch.zeros(n, c["dim"], dtype=torch.float64, device=lab.device)
    res = zeros.index_add(0, row, s["Z"][:used].double() * w[:, None])
    out = dict(offsets=offsets.int(), order=order, position=position.view(n, p), Y=Y, out=res)
    if c["train"]:
        g = s["grad_out"].double()[row]
        gz = torch.zeros_like(Y)
        gz[:used] = g * w[:, None]
        gw = torch.zeros(n * p, dtype=torch.float64, device=lab.device)
        gw[sorted_slots] = (g * s["Z"][:used].double()).sum(1)
        out.update(grad_Z=gz, grad_weights=gw.view(n, p),
                   grad_X=zeros.index_add(0, row, s["grad_Y"][:used].double()))
    return out


def _exact_lookup(c, s):
    k, lab = c["clusters"], s["labels"]
    at = torch.nonzero((lab >= 0) & (lab < k))[:, 0]
    rows = torch.zeros(c["rows"], c["dim"], dtype=torch.float64, device=lab.device)
    rows[at] = s["C"].double()[lab[at]] * c["scale"]
    out = dict(rows=rows)
    if c["train"]:
        grad = torch.zeros(k, c["dim"], dtype=torch.float64, device=lab.device)
        out["grad_C"] = grad.index_add_(0, lab[at], s["G"][at].double()) * c["scale"]
    return out
