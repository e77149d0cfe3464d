"""Plain restatements, in numpy and 64 bits, of the operators on whole activation tensors: 8-bit checkpoints and routing."""
import numpy as np

NAN, INF = float("nan"), float("inf")


def pack(x, group):
    """(codes, ranges) of an array, by the definition in include/simnets_b200.h: what is held in the type of the values is rounded to it."""
    kind, flat = x.dtype, x.reshape(-1)
    groups = -(-flat.size // group)
    codes, ranges = np.zeros(flat.size, np.uint8), np.zeros((groups, 2), kind)
    two, half = kind.type(2), kind.type(0.5)
    for g in range(groups):
        v = flat[g * group:(g + 1) * group]
        fine = v[np.isfinite(v)]
        lo, hi = (fine.min(), fine.max()) if fine.size else (kind.type(0), kind.type(0))
        step = (hi * half - lo * half) / kind.type(126)
        if step < np.finfo(kind).tiny:
            step = kind.type(0)
        with np.errstate(invalid="ignore", over="ignore"):
            d = v * half - lo * half
            per = two / step if step > 0 else kind.type(0)
            # (float32: the product of two numbers is exact in 64 bits; float64: longdouble rounds it to 64 bits of mantissa)
            wide = np.float64 if kind == np.float32 else np.longdouble
            c = np.rint(d.astype(wide) * wide(per)).astype(np.float64)
        c = np.where(np.isnan(v), 255, np.where(v == -INF, 253, np.where(v == INF, 254, c)))
        codes[g * group:(g + 1) * group], ranges[g] = c.astype(np.uint8), (lo, step)
    return codes, ranges


def unpack(codes, ranges, shape, group):
    """The values in 64 bits, rounded once to the type of the ranges."""
    g = np.arange(codes.size) // group
    wide = np.float64 if ranges.dtype == np.float32 else np.longdouble
    v = ranges[g, 0].astype(wide) + codes.astype(wide) * ranges[g, 1].astype(wide)
    with np.errstate(over="ignore"):
        v = np.minimum(v.astype(ranges.dtype), np.finfo(ranges.dtype).max)
    return np.where(codes == 253, -INF, np.where(codes == 254, INF, np.where(codes == 255, NAN, v))).astype(ranges.dtype).reshape(shape)


def route(scores, top_k, prior=None, bias=None, groups=1, top_groups=None, sigmoid=False, scale=1.0):
    """(index, weights, load, dense, mass, eligible logits): the choice from sums in the type of the scores, the rest in 64 bits."""
    b, k = scores.shape[:2]
    flat = scores.reshape(b, k, -1)
    n = flat.shape[2]
    top_groups = groups if top_groups is None else top_groups
    index, weights = np.full((b, top_k, n), -1, np.int32), np.zeros((b, top_k, n))
    dense, load = np.zeros((b, k, n)), np.zeros(k, np.int64)
    with np.errstate(invalid="ignore", over="ignore"):
        logit = flat if prior is None else flat + prior[None, :, None]
        value = logit if bias is None else logit + bias[None, :, None]
    value = np.where(np.isnan(value), -INF, value)
    for i in range(b):
        for j in range(n):
            v = value[i, :, j].copy()
            if top_groups < groups:
                best = v.reshape(groups, -1).max(1)
                keep = [g for g in np.argsort(-best, kind="stable")[:top_groups] if best[g] > -INF]
                mask = np.isin(np.arange(k) // (k // groups), keep)
                v = np.where(mask, v, -INF)
            order = [c for c in np.argsort(-v, kind="stable")[:top_k] if v[c] > -INF]
            if not order:
                continue
            l = logit[i, order, j].astype(np.float64)
            with np.errstate(over="ignore"):
                ls = np.where(l >= 0, -np.log1p(np.exp(-np.abs(l))), l - np.log1p(np.exp(-np.abs(l)))) if sigmoid else l
            e = np.where(ls == ls.max(), 1.0, np.exp(np.where(ls == ls.max(), 0.0, ls - ls.max())))
            w = scale * e / e.sum()
            index[i, :len(order), j], weights[i, :len(order), j] = order, w
            dense[i, order, j] = w
            load[order] += 1
    tail = scores.shape[2:]
    return index.reshape((b, top_k) + tail), weights.reshape((b, top_k) + tail), load, dense.reshape(scores.shape), dense.sum((0, 2)), logit.reshape(scores.shape)


def route_gradient(index, weights, grad, logit, sigmoid=False, scale=1.0):
    """dscores of the gradient of the weights, in 64 bits."""
    b, top = index.shape[:2]
    idx, w, g = (a.reshape(b, top, -1) for a in (index, weights.astype(np.float64), grad.astype(np.float64)))
    l, out = logit.reshape(b, logit.shape[1], -1).astype(np.float64), np.zeros((b, logit.shape[1], idx.shape[2]))
    for i in range(b):
        for j in range(idx.shape[2]):
            on = idx[i, :, j] >= 0
            c, wj, gj = idx[i, on, j], w[i, on, j], g[i, on, j]
            d = wj * (gj - (wj * gj).sum() / scale)
            if sigmoid:
                with np.errstate(over="ignore"):
                    d = d / (1.0 + np.exp(l[i, c, j]))
            out[i, c, j] = d
    return out.reshape(logit.shape)


def route_sorted(scores, top_k, prior=None, bias=None, groups=1, top_groups=None, sigmoid=False, scale=1.0):
    """`route` for torch tensors with many positions, by a stable sort: (index, weights, load, chosen logits), weights and logits in 64 bits."""
    import torch
    along = lambda v: v.view((1, -1) + (1,) * (scores.dim() - 2))
    logit = scores if prior is None else scores + along(prior)
    value = logit if bias is None else logit + along(bias)
    value = torch.where(value.isnan(), -INF, value)
    if top_groups is not None and top_groups < groups:
        best, order = value.unflatten(1, (groups, -1)).amax(2).sort(dim=1, descending=True, stable=True)
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order[:, :top_groups], best[:, :top_groups] > -INF)
        value = torch.where(keep.repeat_interleave(value.shape[1] // groups, 1), value, -INF)
    best, order = value.sort(dim=1, descending=True, stable=True)
    some = best[:, :top_k] > -INF
    index = torch.where(some, order[:, :top_k], -1)
    chosen = logit.gather(1, index.clamp(min=0)).double()
    l = torch.where(some, torch.nn.functional.logsigmoid(chosen) if sigmoid else chosen, -INF)
    hi = l.amax(1, keepdim=True)
    e = torch.where(some, torch.where(l == hi, 1.0, (l - hi).exp()), 0.0)
    weights = scale * e / e.sum(1, keepdim=True).clamp(min=1.0)
    return index, weights, torch.bincount(index[some], minlength=scores.shape[1]), chosen
