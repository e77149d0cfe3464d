"""What the operators at the two ends of a training step are timed on: the log probabilities of given classes with entropy and the likeliest
alternatives, and the norm of all gradients with clipping.

    own                 False: `run` computes the plain form; True: it calls the framework's operators
    listed()            the cases that are always timed
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program has in hand before the call
    run(state)          one pass, returning everything it computes
    work(case)          bytes and floating-point operations that a pass cannot do without
    exact(case, seed)   the same outputs from the definitions in 64 bits

Kinds of a case:

    score   log probabilities of the labels, entropy and the `top` likeliest classes with their log probabilities (`log_probabilities`)
    train   the same with the gradient of the logits
    norm    the norm of a list of gradients (`gradient_norm`)
    clip    the gradients scaled so that their norm is at most `max_norm`, with the norm before it (`clip_gradients`)

Logits come as rows [batch, classes], as maps [batch, classes, height, width] or as sequences [batch, positions, classes] without their last
position, which has no successor.  With m the largest logit of a position, d_c = x_c - m and S = sum exp(d_c):

    log p_c = d_c - log S,   entropy = log S - sum exp(d_c) d_c / S

A label outside [0, classes) has log probability 0 and no gradient.  Logits of -infinity are classes that cannot be; where all of them are, every log
probability is -infinity, the entropy 0 and the gradient 0.  Alternatives go by falling logit, equal ones by index; one that cannot be has index -1.
"""
import math

import torch

own = False

INF = float("inf")


# ------------------------------------------------------------------------------------------------------------- the cases
def _score(layout, batch, classes, height, width, top, entropy, labels, f64=False, masked=False):
    """layout: rows (height = width = 1), map, or sequence (height positions of which the last is left out, width = 1); masked: a share of the
    classes, and every class of some positions, cannot be."""
    return dict(kind="score", layout=layout, batch=batch, classes=classes, height=height, width=width, top=top, entropy=entropy, labels=labels,
                f64=f64, masked=masked)


def _train(*args, **kw):
    return dict(_score(*args, **kw), kind="train")


def _gradients(kind, tensors, values, order, f64, clipped):
    """tensors: how many; values: about how many numbers in all; order 0: the largest magnitude; clipped: whether the norm is above the limit."""
    return dict(kind=kind, tensors=tensors, values=values, order=order, f64=f64, clipped=clipped)


def listed():
    return [
        # the answer of the 1x28x28 example network for one image: the smallest call, all latency
        dict(_score("rows", 1, 10, 1, 1, 3, True, False), name="answer for one image"),
        # a loss made of log probabilities and entropies behind the 3x32x32 network, at its training batch
        dict(_train("rows", 2048, 10, 1, 1, 0, True, True), name="train ten classes"),
        # one position over a large set of classes: the next symbol of one sequence
        dict(_score("rows", 1, 131072, 1, 1, 8, True, True), name="one of many classes"),
        # scoring whole sequences, classes that divide nothing, the last position of each left out: the most memory traffic of a forward pass
        dict(_score("sequence", 8, 65537, 257, 1, 5, True, True), name="score sequences"),
        # training over many classes of which some cannot be, with padded positions: the most memory traffic of a training step
        dict(_train("rows", 2048, 32000, 1, 1, 0, True, True, masked=True), name="train many classes"),
        # a map of a few dozen classes, as a network without a head for whole images gives, with alternatives that a second network learns from
        dict(_train("map", 32, 150, 64, 64, 3, False, True), name="train a map"),
        # double precision and odd sizes, as gradient checks have them
        dict(_train("map", 7, 37, 45, 37, 4, True, True, f64=True), name="gradient check of a map"),
        # small maps of many classes, as the last stages of the 3x32x32 network have them
        dict(_score("map", 512, 512, 4, 4, 8, True, False), name="score small maps"),
        # the gradients of the 3x32x32 network, every step: latency
        dict(_gradients("clip", 6, 770000, 2, False, True), name="clip a small network"),
        # many tensors of very different sizes, the limit not reached, as most steps of a long training have it
        dict(_gradients("clip", 61, 5.0e7, 2, False, False), name="clip many tensors below the limit"),
        # the gradients of a large network: the most memory traffic
        dict(_gradients("clip", 24, 2.6e8, 2, False, True), name="clip a large network"),
        # double precision, the largest magnitude, more tensors than one launch takes
        dict(_gradients("norm", 1500, 1.2e7, 0, True, False), name="largest gradient of many tensors"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# A drawn case has at most this many logits or gradients, which the largest listed one of its kind nearly reaches.
_MOST = {"score": 1.2e8, "train": 6.0e7, "clip": 2.4e8, "norm": 2.4e8}


def draw(rng):
    kind = rng.choice(["score", "score", "train", "train", "clip", "norm"])
    f64 = rng.random() < 0.2
    if kind in ("clip", "norm"):
        values = _log(rng, 100, int(_MOST[kind]) // (2 if f64 else 1))
        return _gradients(kind, _log(rng, 1, min(60 if kind == "clip" else 2000, values)), values, rng.choice([2, 2, 0]), f64, kind == "clip" and rng.random() < 0.6)
    most = _MOST[kind] / (2 if f64 else 1)
    layout = rng.choice(["rows", "map", "sequence"])
    if layout == "map":
        h, w = _log(rng, 1, 96), _log(rng, 1, 96)
        k = _log(rng, 2, 1024)
    else:
        h, w = (_log(rng, 2, 512) if layout == "sequence" else 1), 1
        k = _log(rng, 2, 131072)
    while h * w * k > most / 2:
        h, w = max(2 if layout == "sequence" else 1, h // 2), max(1, w // 2)
    batch = _log(rng, 1, max(1, min(4096, int(most / (h * w * k)))))
    top, entropy = rng.randint(0, min(8, k)), rng.random() < 0.7
    labels = rng.random() < 0.8 or not (top or entropy)
    return (_score if kind == "score" else _train)(layout, batch, k, h, w, top, entropy, labels, f64, rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _axis(case):
    return 2 if case["layout"] == "sequence" else 1


def _logits_shape(case):
    b, k, h, w = (case[n] for n in ("batch", "classes", "height", "width"))
    return (b, k) if case["layout"] == "rows" else (b, h, k) if case["layout"] == "sequence" else (b, k, h, w)


def _positions_shape(case):
    b, h, w = (case[n] for n in ("batch", "height", "width"))
    return (b,) if case["layout"] == "rows" else (b, h - 1) if case["layout"] == "sequence" else (b, h, w)


def _top_shape(case):
    shape = list(_positions_shape(case))
    shape.insert(_axis(case), case["top"])
    return tuple(shape)


def _sizes(case):
    """Sizes of the tensors: spread over two orders of magnitude, the same for every seed, odd ones among them."""
    n, total = case["tensors"], int(case["values"])
    share = [math.exp(4.0 * ((7 * i) % n) / n) for i in range(n)]
    return [max(1, int(total * s / sum(share))) for s in share]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], dict(case=case)
    real = torch.float64 if case["f64"] else torch.float32

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=real)

    if kind in ("clip", "norm"):
        sizes = _sizes(case)
        # (views of one bucket, as a data-parallel program keeps them)
        flat = 0.02 * normal(sum(sizes))
        state["grads"] = list(flat.split(sizes))
        if kind == "clip":
            state["flat_out"] = torch.empty_like(flat)
            state["out"] = list(state["flat_out"].split(sizes))
            typical = 0.02 * (math.sqrt(sum(sizes)) if case["order"] else math.sqrt(2.0 * math.log(sum(sizes) + 1.0)))
            state["max_norm"] = (0.1 if case["clipped"] else 10.0) * typical
        return state
    x = 3.0 * normal(*_logits_shape(case))
    axis, k = _axis(case), case["classes"]
    if case["masked"]:
        cannot = torch.rand(k, generator=gen, device="cuda") < 0.05
        cannot[0] = False
        x = torch.where(cannot.view((1,) * axis + (k,) + (1,) * (x.dim() - axis - 1)), -INF, x)
        padded = torch.rand([s if i != axis else 1 for i, s in enumerate(x.shape)], generator=gen, device="cuda") < 0.02
        x = torch.where(padded, -INF, x)
    state["logits"] = x[:, :-1] if case["layout"] == "sequence" else x
    if case["labels"]:
        at = torch.randint(0, k, _positions_shape(case), generator=gen, device="cuda")
        state["labels"] = torch.where(torch.rand(at.shape, generator=gen, device="cuda") < 0.05, -1, at)
        if case["masked"]:          # a program does not ask for what cannot be
            lost = torch.gather(state["logits"], axis, state["labels"].clamp(min=0).unsqueeze(axis)).squeeze(axis) == -INF
            state["labels"] = torch.where(lost, -1, state["labels"])
    if kind == "train":
        state["grad_label"] = normal(*_positions_shape(case)) if case["labels"] else None
        state["grad_entropy"] = 0.1 * normal(*_positions_shape(case)) if case["entropy"] else None
        state["grad_top"] = normal(*_top_shape(case)) if case["top"] else None
    return state


# ----------------------------------------------------------------------------------------------------------- plain forms
def _plain_score(s, case):
    x, axis, top = s["logits"], _axis(case), case["top"]
    m = x.amax(axis, keepdim=True)
    nothing = m == -INF
    d = x - torch.where(nothing, 0.0, m)
    e = d.exp()
    total = e.sum(axis, keepdim=True)
    log_total = torch.where(nothing, 0.0, total.log())
    out = dict(label=None, entropy=None, top_index=None, top=None)
    d_here = torch.where(d == -INF, 0.0, d)
    entropy = torch.where(nothing, 0.0, log_total - (e * d_here).sum(axis, keepdim=True) / total)
    if s.get("labels") is not None:
        known = (s["labels"] >= 0) & (s["labels"] < case["classes"])
        at = torch.where(known, s["labels"], 0).unsqueeze(axis)
        out["label"] = torch.where(known, (d.gather(axis, at) - log_total).squeeze(axis), 0.0)
    if case["entropy"]:
        out["entropy"] = entropy.squeeze(axis)
    if top:
        value, index = x.sort(dim=axis, descending=True, stable=True)
        value, index = value.narrow(axis, 0, top), index.narrow(axis, 0, top)
        out["top"] = torch.where(value == -INF, -INF, d.gather(axis, index) - log_total)
        out["top_index"] = torch.where(value == -INF, -1, index).int()
    if case["kind"] == "score":
        return out
    p = torch.where(nothing, 0.0, e / total)
    dx = torch.zeros_like(p)
    taken = torch.zeros_like(m)
    if s["grad_label"] is not None:
        g = torch.where(known, s["grad_label"], 0.0).unsqueeze(axis)
        dx.scatter_add_(axis, at, g)
        taken = taken + g
    if s["grad_top"] is not None:
        g = torch.where(out["top_index"] < 0, 0.0, s["grad_top"])
        dx.scatter_add_(axis, index, g)
        taken = taken + g.sum(axis, keepdim=True)
    dx -= p * taken
    if s["grad_entropy"] is not None:
        dx -= p * s["grad_entropy"].unsqueeze(axis) * (d_here - log_total + entropy)
    out["dlogits"] = torch.where(nothing, 0.0, dx)
    return out


def _plain_norm(s, case):
    if case["order"] == 0:
        return torch.stack([g.abs().max() for g in s["grads"]]).max()
    return torch.stack([g.square().sum() for g in s["grads"]]).sum().sqrt()


def _plain_clip(s, case):
    norm = _plain_norm(s, case)
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0)
    for g, o in zip(s["grads"], s["out"]):
        torch.mul(g, scale, out=o)
    return dict(norm=norm, clipped=s["flat_out"])


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own_run(s, case):
    from simnets_tf_b200.ops.gradients import clip_gradients, gradient_norm
    from simnets_tf_b200.ops.likelihood import log_probabilities
    if case["kind"] == "norm":
        return gradient_norm(s["grads"], order=case["order"] or INF)
    if case["kind"] == "clip":
        return dict(norm=clip_gradients(s["grads"], s["max_norm"], order=case["order"] or INF, out=s["out"]), clipped=s["flat_out"])
    kw = dict(labels=s.get("labels"), top_k=case["top"], entropy=case["entropy"], axis=_axis(case))
    if case["kind"] == "score":
        return log_probabilities(s["logits"], **kw)._asdict()
    logits = s["logits"].detach().requires_grad_()
    got = log_probabilities(logits, **kw)
    wanted = [(v, s[g]) for v, g in ((got.label, "grad_label"), (got.entropy, "grad_entropy"), (got.top, "grad_top")) if v is not None]
    dlogits, = torch.autograd.grad([v for v, _ in wanted], [logits], [g for _, g in wanted])
    out = {name: None if v is None else v.detach() for name, v in got._asdict().items()}
    return dict(out, dlogits=dlogits)


def run(state):
    case = state["case"]
    if own:
        return _own_run(state, case)
    return _plain_norm(state, case) if case["kind"] == "norm" else _plain_clip(state, case) if case["kind"] == "clip" else _plain_score(state, case)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    """Every input read once and every output written once."""
    size = 8 if case["f64"] else 4
    if case["kind"] in ("clip", "norm"):
        n = sum(_sizes(case))
        return dict(bytes=size * n * (2 if case["kind"] == "clip" else 1), flops=n * (3 if case["kind"] == "clip" else 2))
    positions = math.prod(_positions_shape(case))
    logits = positions * case["classes"]
    answers = positions * ((8 + size if case["labels"] else 0) + (size if case["entropy"] else 0) + case["top"] * (4 + size))
    if case["kind"] == "score":
        return dict(bytes=size * logits + answers, flops=6 * logits)
    asked = positions * size * ((1 if case["labels"] else 0) + (1 if case["entropy"] else 0) + case["top"])
    return dict(bytes=2 * size * logits + answers + asked, flops=11 * logits)


# ------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_rows(x, labels, case, s, top_index):
    """Answers for logits [positions, classes] in 64 bits."""
    log_p = torch.log_softmax(x, 1)
    empty = (x == -INF).all(1)
    log_p[empty] = -INF
    p = log_p.exp()
    terms = torch.special.entr(p)
    entropy = terms.sum(1)
    rows = torch.arange(x.shape[0], device=x.device)
    known = None if labels is None else (labels >= 0) & (labels < case["classes"])
    label = None if labels is None else torch.where(known, log_p[rows, labels.clamp(0, case["classes"] - 1)], 0.0)
    top = None if top_index is None else torch.where(top_index < 0, -INF, log_p.gather(1, top_index.clamp(min=0).long()))
    if s is None:
        return label, entropy, top, None
    g_label, g_entropy, g_top = s
    # every output that is asked for is linear in the log probabilities or the terms of the entropy: the gradient with respect to the log
    # probabilities, then through the softmax
    up = torch.zeros_like(x)
    if g_label is not None:
        up[rows, labels.clamp(0, case["classes"] - 1)] += torch.where(known, g_label, 0.0)
    if g_top is not None:
        up.scatter_add_(1, top_index.clamp(min=0).long(), torch.where(top_index < 0, 0.0, g_top))
    if g_entropy is not None:
        up -= g_entropy[:, None] * p * (torch.where(p > 0, log_p, 0.0) + 1.0)
    dx = up - p * up.sum(1, keepdim=True)
    dx[empty] = 0.0
    return label, entropy, top, dx


def _first_largest(x, top):
    """Index of the `top` largest of every row, equal ones by index, -1 for -infinity."""
    x, place, out = x.clone(), torch.arange(x.shape[1], device=x.device)[None], []
    for _ in range(top):
        best = x.max(1, keepdim=True).values
        at = torch.where(x == best, place, x.shape[1]).min(1, keepdim=True).values
        out.append(torch.where(best == -INF, -1, at))
        x.scatter_(1, at, -INF)
    return torch.cat(out, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("clip", "norm"):
        flat = torch.cat([g.double() for g in s["grads"]])
        norm = flat.abs().max() if case["order"] == 0 else torch.linalg.vector_norm(flat)
        if case["kind"] == "norm":
            return norm
        return dict(norm=norm, clipped=flat * min(1.0, s["max_norm"] / float(norm)))
    axis, shape, train = _axis(case), _positions_shape(case), case["kind"] == "train"

    def by_row(v, last):
        """[positions] or, where there is an axis more, [positions, last] of a tensor of the case."""
        return None if v is None else v.reshape(-1) if last is None else v.movedim(axis, -1).reshape(-1, last)

    x = by_row(s["logits"], case["classes"])
    labels = by_row(s.get("labels"), None)
    grads = [by_row(s.get(n), last) for n, last in (("grad_label", None), ("grad_entropy", None), ("grad_top", case["top"]))] if train else None
    # (in parts, for the memory of 64-bit copies)
    step = max(1, int(2.0e7) // case["classes"])
    parts = []
    for i in range(0, x.shape[0], step):
        at = slice(i, i + step)
        top_index = _first_largest(x[at], case["top"]) if case["top"] else None
        given = [None if g is None else g[at].double() for g in grads] if train else None
        parts.append(_exact_rows(x[at].double(), None if labels is None else labels[at], case, given, top_index) + (top_index,))
    label, entropy, top, dx, top_index = (None if v[0] is None else torch.cat(v) for v in zip(*parts))

    def back(v):
        return v.reshape(shape + (-1,)).movedim(-1, axis)

    out = dict(label=None if label is None else label.view(shape), entropy=entropy.view(shape) if case["entropy"] else None,
               top_index=None if top_index is None else back(top_index), top=None if top is None else back(top))
    if train:
        out["dlogits"] = back(dx)
    return out
