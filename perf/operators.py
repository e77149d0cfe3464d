"""What the operators on whole activation tensors are timed on: 8-bit checkpoints of activations with the MEX and Similarity gradients
taken at them, and the routing of positions to the components of a mixture.

    own                 False: `run` computes the plain form; True: it calls the framework's operators
    listed()            the cases that are always timed
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program has in hand before the call
    run(state)          one pass, returning everything it computes
    work(case)          bytes and floating-point operations that a pass cannot do without
    exact(case, seed)   the same outputs from the definitions in 64 bits

Kinds of a case:

    pack        an activation to 8 bits and back (`checkpoint_pack`, `checkpoint_unpack`)
    unpack      a checkpoint back to an activation
    mex         both gradients of a MEX layer at a checkpoint of its input (`mex_checkpoint_backward`)
    similarity  all three gradients of a Similarity layer at a checkpoint of its input (`similarity_checkpoint_backward`)
    route       the components that every position goes to, with weights and loads (`route`), and for training the gradient of the weights
    dense       the same as a tensor of responsibilities with the components' masses (`responsibilities`)

A checkpoint holds, for every `group` consecutive values, the lowest finite value `base` and `step` = range / 252 in the type of the values
(0 where the range is below 252 of the type's smallest normal number), and for every value a byte: round((x - base) / step), computed as
round((x / 2 - base / 2) * (2 / step)) with x / 2 - base / 2 and 2 / step rounded to the type and the product exact, or 253, 254, 255 for
-infinity, infinity, NaN.  It stands for base + code * step, rounded once.
"""
import math

import torch

own = False

NAN, INF = float("nan"), float("inf")


# ------------------------------------------------------------------------------------------------------------- the cases
def _pack(shape, group, f64, missing):
    return dict(kind="pack", batch=shape[0], channels=shape[1], height=shape[2], width=shape[3], group=group, f64=f64, missing=missing)


def _unpack(shape, group, f64, missing):
    return dict(_pack(shape, group, f64, missing), kind="unpack")


def _mex(batch, channels, height, width, instances, block_c, block, region, pooled, epsilon, group):
    """Disjoint blocks of block_c x block x block; region: 0 = one offsets table, n = unshared n x n regions; pooled: the gradient of a 2x2
    sum pooling of the output comes in."""
    return dict(kind="mex", batch=batch, channels=channels, height=height, width=width, instances=instances, block_c=block_c, block=block,
                region=region, pooled=pooled, epsilon=epsilon, group=group)


def _similarity(batch, channels, height, width, templates, block, stride, pad, missing, group):
    """missing: L2 with the normalisation term over data with missing entries, else plain L2."""
    return dict(kind="similarity", batch=batch, channels=channels, height=height, width=width, templates=templates, block=block, stride=stride,
                pad=pad, missing=missing, group=group)


def _route(batch, components, height, width, top, groups, top_groups, sigmoid, biased, gradient):
    return dict(kind="route", batch=batch, components=components, height=height, width=width, top=top, groups=groups, top_groups=top_groups,
                sigmoid=sigmoid, biased=biased, gradient=gradient)


def _dense(batch, components, height, width, top, biased):
    return dict(_route(batch, components, height, width, top, 1, 1, False, biased, False), kind="dense")


def listed():
    return [
        # what the second layer of the 1x28x28 example network keeps of one image: the smallest call, all latency
        dict(_pack((1, 32, 16, 16), 128, False, False), name="pack one image"),
        # the input of the first MEX layer of the 3x32x32 network at its training batch: the most memory traffic
        dict(_pack((2048, 64, 32, 32), 128, False, False), name="pack first stage"),
        # double precision, sizes that divide nothing, missing and infinite entries, as gradient checks have them
        dict(_unpack((37, 19, 45, 37), 32, True, True), name="unpack odd map"),
        # the input of the second MEX layer at the training batch, as the backward pass wants it back
        dict(_unpack((2048, 128, 16, 16), 128, False, False), name="unpack second stage"),
        # a small MEX layer with unshared regions
        dict(_mex(64, 32, 16, 16, 64, 32, 1, 2, False, 1.0, 128), name="mex small unshared"),
        # the first MEX stage of the 3x32x32 network, pooled, at a quarter of its training batch
        dict(_mex(512, 64, 32, 32, 128, 64, 1, 2, True, 1.0, 128), name="mex first stage"),
        # blocks that tile channels and rows and share one table: few taps under many instances
        dict(_mex(32, 256, 32, 32, 256, 4, 2, 0, False, 0.5, 64), name="mex wide shared"),
        # a wide inner Similarity layer on data with missing entries: the most arithmetic
        dict(_similarity(64, 64, 32, 32, 128, 3, 1, 1, True, 128), name="similarity missing data"),
        # odd sizes, strides and padding
        dict(_similarity(37, 19, 45, 37, 100, 3, 2, 1, False, 256), name="similarity ragged"),
        # a gated choice in groups with its gradient, as a training step has it
        dict(_route(64, 192, 15, 15, 6, 8, 3, True, True, True), name="route in groups"),
        # every patch of a small batch to its nearest centre
        dict(_dense(8, 64, 30, 30, 1, False), name="assign small batch"),
        # the responsibilities of one EM update of the 3x32x32 network's first layer, cut to four, with a bias for balance
        dict(_dense(512, 64, 30, 30, 4, True), name="responsibilities cut to four"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# A drawn case stays below these, which the largest listed case of its kind reaches or nearly reaches.
_MOST = {"pack": 1.3e8, "unpack": 6.0e7, "mex": 2.5e10, "similarity": 2.0e10, "route": 3.0e7, "dense": 3.0e7}


def draw(rng):
    kind = rng.choice(["pack", "unpack", "mex", "mex", "similarity", "route", "dense"])
    group = rng.choice([32, 64, 128, 256])
    if kind in ("pack", "unpack"):
        c, h, w = _log(rng, 1, 256), _log(rng, 1, 64), _log(rng, 1, 64)
        shape = (_log(rng, 1, max(1, min(2048, int(_MOST[kind] / (c * h * w))))), c, h, w)
        return (_pack if kind == "pack" else _unpack)(shape, group, rng.random() < 0.3, rng.random() < 0.4)
    if kind == "mex":
        if rng.random() < 0.6:          # over the channels of each pixel, regions unshared n x n
            c, region = _log(rng, 8, 160), rng.choice([0, 2, 2])
            h, w = 2 * _log(rng, 1, 16), 2 * _log(rng, 1, 16)
            m, bc, block, eps, pooled = _log(rng, 8, 256), c, 1, 1.0, rng.random() < 0.5
        else:                           # disjoint blocks of a few channels, rows and columns
            bc, block, region, pooled = _log(rng, 1, 8), rng.choice([1, 2, 3]), 0, False
            c, h, w = bc * _log(rng, 1, 48), block * rng.randint(2, 12), block * rng.randint(2, 12)
            m, eps = _log(rng, 8, 256), rng.choice([0.5, 1.0])
        flops = work(_mex(1, c, h, w, m, bc, block, region, pooled, eps, group))["flops"]
        return _mex(_log(rng, 1, max(1, min(512, int(_MOST[kind] / flops)))), c, h, w, m, bc, block, region, pooled, eps, group)
    if kind == "similarity":
        block, missing = rng.randint(1, 4), rng.random() < 0.4
        args = (_log(rng, 1, 64), _log(rng, 6, 45), _log(rng, 6, 45), _log(rng, 8, 128), block, rng.randint(1, 2), rng.randint(0, block // 2), missing, group)
        flops = work(_similarity(1, *args))["flops"]
        return _similarity(_log(rng, 1, max(1, min(128, int(_MOST[kind] / flops)))), *args)
    h, w = _log(rng, 1, 40), _log(rng, 1, 40)
    if kind == "dense":
        k = _log(rng, 2, 256)
        return _dense(_log(rng, 1, max(1, min(512, int(_MOST[kind] / (k * h * w))))), k, h, w, rng.randint(1, min(8, k)), rng.random() < 0.5)
    groups = rng.choice([1, 1, 2, 4, 8])
    k = groups * _log(rng, 2, 48)
    top_groups = rng.randint(1, groups)
    top = rng.randint(1, min(8, top_groups * (k // groups)))
    b = _log(rng, 1, max(1, min(512, int(_MOST[kind] / (k * h * w)))))
    return _route(b, k, h, w, top, groups, top_groups, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _shape(case):
    return (case["batch"], case["channels"], case["height"], case["width"])


def _mex_out(case):
    return (case["channels"] // case["block_c"], case["height"] // case["block"], case["width"] // case["block"])


def _sim_out(case):
    return tuple((s + 2 * case["pad"] - case["block"]) // case["stride"] + 1 for s in (case["height"], case["width"]))


def _made_missing(x, gen, infinite):
    """A share of the entries missing, whole groups of them too, and where the path may meet them infinite ones."""
    u = torch.rand(x.shape, generator=gen, device="cuda")
    x = torch.where(u < 0.05, NAN, x)
    if infinite:
        x = torch.where((u > 0.95) & (u < 0.97), -INF, x)
        x = torch.where(u > 0.995, INF, x)
    x[:1, :1] = NAN
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    kind, state = case["kind"], dict(case=case)
    if kind in ("route", "dense"):
        b, k, h, w = case["batch"], case["components"], case["height"], case["width"]
        state["scores"] = 2.0 * normal(b, k, h, w)
        state["prior"] = 0.5 * normal(k) if kind == "dense" else None
        state["bias"] = 0.3 * normal(k) if case["biased"] else None
        if case["gradient"]:
            state["grad"] = normal(b, case["top"], h, w)
        return state
    x = normal(*_shape(case))
    if kind in ("pack", "unpack"):
        x = (3.0 * x - 40.0).to(torch.float64 if case["f64"] else torch.float32)       # log-likelihoods
        if case["missing"]:
            x = _made_missing(x, gen, True)
        if kind == "pack":
            return dict(state, x=x)
    elif kind == "mex":
        co, ho, wo = _mex_out(case)
        taps, regions = case["block_c"] * case["block"] ** 2, case["region"] ** 2 if case["region"] else 1
        x = 2.0 * x - 20.0
        offsets = 2.0 * normal(regions, case["instances"], taps)                       # log-weights spread over a few nats
        state["offsets"] = (offsets - torch.logsumexp(offsets, 2, keepdim=True)).view(regions, case["instances"], case["block_c"], case["block"], case["block"])
        half = 2 if case["pooled"] else 1
        state["dy"] = normal(case["batch"], case["instances"] * co, ho // half, wo // half)
    else:
        if case["missing"]:
            x = _made_missing(x, gen, False)
        params = (case["templates"], case["channels"], case["block"], case["block"])
        state["templates"] = normal(*params)
        state["weights"] = 0.1 + torch.rand(params, generator=gen, device="cuda")
        state["dy"] = normal(case["batch"], case["templates"], *_sim_out(case))
    state["codes"], state["ranges"] = _plain_pack(x, case["group"])
    return state


# ----------------------------------------------------------------------------------------------------------- plain forms
def _grouped(x, group, fill):
    flat = x.reshape(-1)
    return torch.cat([flat, flat.new_full((-flat.numel() % group,), fill)]).view(-1, group)


def _plain_pack(x, group):
    """(codes, ranges): codes one byte a value, ranges [groups, 2] = base and step."""
    v = _grouped(x, group, NAN)
    fine = v.isfinite()
    lo, hi = torch.where(fine, v, INF).amin(1), torch.where(fine, v, -INF).amax(1)
    some = fine.any(1)
    lo, hi = torch.where(some, lo, 0.0), torch.where(some, hi, 0.0)
    step = (hi * 0.5 - lo * 0.5) / torch.full_like(hi, 126.0)      # (a division: by a number it would be a product with 1 / 126)
    step = torch.where(step < torch.finfo(x.dtype).tiny, 0.0, step)
    per = torch.where(step > 0, 2.0 / step, 0.0)
    # (64 bits: a product next to the border of two codes)
    code = ((v * 0.5 - lo[:, None] * 0.5).double() * per.double()[:, None]).round()
    code = torch.where(v == -INF, 253.0, torch.where(v == INF, 254.0, torch.where(v.isnan(), 255.0, code)))
    return code.to(torch.uint8).view(-1)[:x.numel()].contiguous(), torch.stack([lo, step], 1)


def _plain_unpack(codes, ranges, shape, group):
    c = _grouped(codes, group, 0).double()
    v = (ranges[:, :1].double() + c * ranges[:, 1:].double()).to(ranges.dtype).clamp(max=torch.finfo(ranges.dtype).max)
    v = torch.where(c == 253, -INF, torch.where(c == 254, INF, torch.where(c == 255, NAN, v)))
    return v.view(-1)[:codes.numel()].view(shape)


def _mex_taps(case):
    """Index inside a sample of every tap [regions, taps, positions of a region], and of the positions [regions, positions]."""
    co, ho, wo = _mex_out(case)
    bc, b, n = case["block_c"], case["block"], case["region"] or 1
    pos = torch.arange(co * ho * wo, device="cuda").view(co, ho // n, n, wo // n, n).permute(2, 4, 0, 1, 3).reshape(n * n, -1)
    c, h, w = pos // (ho * wo), pos // wo % ho, pos % wo
    k = torch.arange(bc * b * b, device="cuda")[None, :, None]
    taps = ((c[:, None] * bc + k // (b * b)) * case["height"] + h[:, None] * b + k // b % b) * case["width"] + w[:, None] * b + k % b
    return taps, pos


def _mex_dy(case, dy):
    if case["pooled"]:
        dy = dy.repeat_interleave(2, 2).repeat_interleave(2, 3)
    return dy.reshape(case["batch"], case["instances"], -1)


def _plain_mex(s, case):
    x = _plain_unpack(s["codes"], s["ranges"], _shape(case), case["group"]).reshape(case["batch"], -1)
    taps, pos = _mex_taps(case)
    eps, off = case["epsilon"], s["offsets"].flatten(2)
    xt = x[:, taps]                                                                     # [batch, regions, taps, positions]
    ex = (eps * (xt - xt.amax(2, keepdim=True))).exp()
    eo = (eps * (off - off.amax(2, keepdim=True))).exp()                                # [regions, instances, taps]
    q = _mex_dy(case, s["dy"])[:, :, pos].transpose(1, 2) / (eo @ ex)                   # [batch, regions, instances, positions]
    dx = torch.zeros_like(x)
    dx[:, taps] = ex * (eo.transpose(1, 2) @ q)
    doff = eo * (q @ ex.transpose(2, 3)).sum(0, dtype=torch.float64).float()
    return dx.view(_shape(case)), doff.view(s["offsets"].shape)


def _sim_patches(case, x, fill):
    """[batch, channels, block, block, out_h, out_w]"""
    p, b, st = case["pad"], case["block"], case["stride"]
    padded = x.new_full((x.shape[0], x.shape[1], x.shape[2] + 2 * p, x.shape[3] + 2 * p), fill)
    padded[:, :, p:p + x.shape[2], p:p + x.shape[3]] = x
    oh, ow = _sim_out(case)
    i = torch.arange(b, device="cuda")[:, None] + st * torch.arange(oh, device="cuda")
    j = torch.arange(b, device="cuda")[:, None] + st * torch.arange(ow, device="cuda")
    return padded[:, :, i[:, None, :, None], j[None, :, None, :]], padded, i, j


def _plain_similarity(s, case):
    # (sums over every position of a batch, of squares that cancel: 64 bits)
    x = _plain_unpack(s["codes"], s["ranges"], _shape(case), case["group"])
    half = 0.5 if case["missing"] else 1.0
    there = (~x.isnan()).float()
    here = _sim_patches(case, there, 1.0)[0]
    patch, padded, i, j = _sim_patches(case, torch.where(x.isnan(), 0.0, x), 0.0)
    b, m, taps = case["batch"], case["templates"], case["channels"] * case["block"] ** 2
    xk = patch.reshape(b, taps, -1)
    t, w, dy = s["templates"].reshape(m, taps), s["weights"].reshape(m, taps), s["dy"].reshape(b, m, -1)
    k = here.reshape(b, taps, -1)
    dxk = 2.0 * half * k * ((w * t).t() @ dy - xk * (w.t() @ dy))
    c = torch.arange(case["channels"], device="cuda").view(-1, 1, 1, 1, 1)
    place = (c * padded.shape[2] + i[:, None, :, None]) * padded.shape[3] + j[None, :, None, :]
    dp = torch.zeros_like(padded)
    dp.view(b, -1).index_add_(1, place.reshape(-1), dxk.reshape(b, -1))
    p = case["pad"]
    dx = dp[:, :, p:p + x.shape[2], p:p + x.shape[3]].contiguous()
    xk, k, t, w, dy = (v.double() for v in (xk, k, t, w, dy))
    s0, s1, s2 = ((dy @ v.transpose(1, 2)).sum(0) for v in (k, xk, xk * xk))
    dt = 2.0 * half * w * (s1 - t * s0)
    dw = -(s2 - 2.0 * t * s1 + t * t * s0) * half
    if case["missing"]:
        dw = dw + half * s0 / (w + FUDGE)
    return dx, dt.float().view(s["templates"].shape), dw.float().view(s["templates"].shape)


FUDGE = 0.001


def _plain_route(s, case):
    """(indices, weights, load, the chosen scores): components by falling score + prior + bias, ties to the lowest."""
    logit = s["scores"] if s["prior"] is None else s["scores"] + s["prior"].view(1, -1, 1, 1)
    v = logit if s["bias"] is None else logit + s["bias"].view(1, -1, 1, 1)
    g = case["groups"]
    if case["top_groups"] < g:
        by_group = v.unflatten(1, (g, -1)).amax(2)
        rank = by_group.sort(dim=1, descending=True, stable=True)[1].argsort(1)
        v = torch.where((rank < case["top_groups"]).repeat_interleave(v.shape[1] // g, 1), v, -INF)
    index = v.sort(dim=1, descending=True, stable=True)[1][:, :case["top"]]
    chosen = logit.gather(1, index)
    value = 1.0 / (1.0 + (-chosen).exp()) if case["sigmoid"] else (chosen - chosen.amax(1, keepdim=True)).exp()
    weights = value / value.sum(1, keepdim=True)
    load = torch.zeros(v.shape[1], dtype=torch.int64, device="cuda").index_add_(0, index.reshape(-1), torch.ones_like(index).reshape(-1))
    return index, weights, load, chosen


def _plain_run(s, case):
    kind = case["kind"]
    if kind == "pack":
        codes, ranges = _plain_pack(s["x"], case["group"])
        return _plain_unpack(codes, ranges, _shape(case), case["group"])
    if kind == "unpack":
        return _plain_unpack(s["codes"], s["ranges"], _shape(case), case["group"])
    if kind == "mex":
        return _plain_mex(s, case)
    if kind == "similarity":
        return _plain_similarity(s, case)
    index, weights, load, chosen = _plain_route(s, case)
    if kind == "dense":
        resp = torch.zeros_like(s["scores"]).scatter_(1, index, weights)
        return resp, resp.sum((0, 2, 3), dtype=torch.float64).float(), load
    if not case["gradient"]:
        return index.int(), weights, load
    g = s["grad"]
    dchosen = weights * (g - (weights * g).sum(1, keepdim=True))
    if case["sigmoid"]:
        dchosen = dchosen / (1.0 + chosen.exp())
    return index.int(), weights, load, torch.zeros_like(s["scores"]).scatter_(1, index, dchosen)


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own_run(s, case):
    from simnets_tf_b200.ops import checkpoint, routing
    kind = case["kind"]
    if kind == "pack":
        return checkpoint.checkpoint_unpack(checkpoint.checkpoint_pack(s["x"], group=case["group"]))
    if kind in ("route", "dense"):
        kw = dict(top_k=case["top"], prior=s["prior"], bias=s["bias"])
        if kind == "dense":
            return routing.responsibilities(s["scores"], **kw)
        kw.update(groups=case["groups"], top_groups=case["top_groups"], sigmoid=case["sigmoid"])
        if not case["gradient"]:
            return routing.route(s["scores"], **kw)
        scores = s["scores"].detach().requires_grad_()
        index, weights, load = routing.route(scores, **kw)
        return index, weights.detach(), load, torch.autograd.grad(weights, scores, s["grad"])[0]
    kept = checkpoint.Checkpoint(s["codes"], s["ranges"], _shape(case), case["group"])
    if kind == "unpack":
        return checkpoint.checkpoint_unpack(kept)
    if kind == "mex":
        blocks = [case["block_c"], case["block"], case["block"]]
        regions = dict(use_unshared_regions=True, unshared_offset_region=[case["region"]]) if case["region"] else dict(use_unshared_regions=False, shared_offset_region=[-1])
        return checkpoint.mex_checkpoint_backward(kept, s["offsets"], s["dy"], case["instances"], pooled=case["pooled"], blocks=blocks, strides=blocks,
                                                  epsilon=case["epsilon"], softmax_mode=True, **regions)
    return checkpoint.similarity_checkpoint_backward(kept, s["templates"], s["weights"], s["dy"], blocks=[case["block"]] * 2, strides=[case["stride"]] * 2,
                                                     padding=[case["pad"]] * 2, normalization_term=case["missing"], ignore_nan_input=case["missing"],
                                                     normalization_term_fudge=FUDGE)


def run(state):
    return _own_run(state, state["case"]) if own else _plain_run(state, state["case"])


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    """Every input read once and every output written once; multiply-adds of the products as two operations."""
    kind = case["kind"]
    if kind in ("route", "dense"):
        positions = case["batch"] * case["height"] * case["width"]
        scores, top = positions * case["components"], positions * case["top"]
        if kind == "dense":
            return dict(bytes=8 * scores + 16 * case["components"], flops=3 * scores + 8 * top)
        return dict(bytes=4 * scores + 8 * top + 12 * case["components"] + (4 * top + 4 * scores if case["gradient"] else 0), flops=2 * scores + 8 * top)
    n = math.prod(_shape(case))
    size = 8 if case.get("f64") else 4
    kept = n + -(-n // case["group"]) * 2 * size
    if kind == "pack":
        return dict(bytes=2 * size * n + 2 * kept, flops=6 * n)
    if kind == "unpack":
        return dict(bytes=size * n + kept, flops=2 * n)
    if kind == "mex":
        co, ho, wo = _mex_out(case)
        taps, outputs = case["block_c"] * case["block"] ** 2, case["batch"] * case["instances"] * co * ho * wo
        table = case["instances"] * taps * (case["region"] ** 2 if case["region"] else 1)
        # (the sums of the outputs, the input's gradient and the offsets' gradient: three products)
        return dict(bytes=kept + 4 * n + outputs * (1 if case["pooled"] else 4) + 8 * table, flops=6 * outputs * taps)
    oh, ow = _sim_out(case)
    taps, outputs = case["channels"] * case["block"] ** 2, case["batch"] * case["templates"] * oh * ow
    # (for every template, tap and position a difference, and three products of it)
    return dict(bytes=kept + 4 * n + 4 * outputs + 16 * case["templates"] * taps, flops=7 * outputs * taps)


# ------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_pack(x, group):
    kind = x.dtype
    flat = x.reshape(-1).double()
    full = torch.nn.functional.pad(flat, (0, -flat.numel() % group), value=NAN).view(-1, group)
    fine = full.isfinite()
    lo = full.masked_fill(~fine, INF).min(1, keepdim=True).values
    hi = full.masked_fill(~fine, -INF).max(1, keepdim=True).values
    none = ~fine.any(1, keepdim=True)
    lo, hi = lo.masked_fill(none, 0.0), hi.masked_fill(none, 0.0)

    def held(v):                        # the two numbers of a group, the differences and the reciprocal are held in the type of the values
        return v.to(kind).double()

    step = held(held(hi / 2 - lo / 2) / torch.full_like(hi, 126.0))
    flat_group = step < torch.finfo(kind).tiny
    step = step.masked_fill(flat_group, 0.0)
    per = held(2 / step.masked_fill(flat_group, 1.0)).masked_fill(flat_group, 0.0)
    codes = torch.round(held(full / 2 - lo / 2) * per)
    values = torch.where(fine, lo + codes * step, full)
    return values.view(-1)[:flat.numel()].view(x.shape)


def _exact_unpack(codes, ranges, shape, group):
    n = codes.numel()
    g = torch.arange(n, device="cuda") // group
    c, r = codes.double(), ranges.double()
    v = r[g, 0] + c * r[g, 1]
    v[codes == 253], v[codes == 254], v[codes == 255] = -INF, INF, NAN
    return v.view(shape)


def _exact_mex(s, case):
    x = _exact_unpack(s["codes"], s["ranges"], _shape(case), case["group"]).reshape(case["batch"], -1)
    taps, pos = _mex_taps(case)
    dy, off, eps = _mex_dy(case, s["dy"]).double(), s["offsets"].flatten(2).double(), case["epsilon"]
    dx, doff = torch.zeros_like(x), torch.zeros_like(off)
    for r in range(taps.shape[0]):
        xt = x[:, taps[r]]
        part = torch.zeros_like(xt)
        for m in range(case["instances"]):
            p = torch.softmax(eps * (xt + off[r, m][None, :, None]), 1) * dy[:, m, pos[r]][:, None]
            part += p
            doff[r, m] = p.sum((0, 2))
        dx[:, taps[r]] = part
    return dx.view(_shape(case)), doff.view(s["offsets"].shape)


def _exact_similarity(s, case):
    x = _exact_unpack(s["codes"], s["ranges"], _shape(case), case["group"])
    half, b, p = (0.5 if case["missing"] else 1.0), case["block"], case["pad"]
    st, (oh, ow) = case["stride"], _sim_out(case)
    full = torch.nn.functional.pad(x, (p, p, p, p))
    dfull = torch.zeros_like(full)
    t, w, dy = s["templates"].double(), s["weights"].double(), s["dy"].double()
    dt, dw = torch.zeros_like(t), torch.zeros_like(w)
    for i in range(b):
        for j in range(b):
            at = (slice(None), slice(None), slice(i, i + st * (oh - 1) + 1, st), slice(j, j + st * (ow - 1) + 1, st))
            xs = full[at]
            for m in range(case["templates"]):
                d = torch.nan_to_num(xs - t[m, :, i, j][None, :, None, None], nan=0.0)
                e = dy[:, m][:, None]
                ed = e * d
                dfull[at] -= 2 * half * w[m, :, i, j][None, :, None, None] * ed
                dt[m, :, i, j] = 2 * half * w[m, :, i, j] * ed.sum((0, 2, 3))
                dw[m, :, i, j] = -half * (ed * d).sum((0, 2, 3))
                if case["missing"]:
                    dw[m, :, i, j] += half * (e * ~xs.isnan()).sum((0, 2, 3)) / (w[m, :, i, j] + FUDGE)
    return dfull[:, :, p:p + x.shape[2], p:p + x.shape[3]].contiguous(), dt, dw


def _exact_route(s, case):
    scores = s["scores"]
    logit = scores if s["prior"] is None else scores + s["prior"][:, None, None]         # (sums in 32 bits are the definition of the choice)
    v = (logit if s["bias"] is None else logit + s["bias"][:, None, None]).clone()
    size, taken = v.shape[1] // case["groups"], []
    if case["top_groups"] < case["groups"]:
        best = torch.stack([v[:, g * size:(g + 1) * size].max(1).values for g in range(case["groups"])], 1)
        keep = torch.zeros_like(best, dtype=torch.bool)
        for _ in range(case["top_groups"]):
            first = _first_largest(best)
            keep.scatter_(1, first, True)
            best.scatter_(1, first, -INF)
        v[~keep[:, :, None].expand(-1, -1, size, -1, -1).reshape(v.shape)] = -INF
    for _ in range(case["top"]):
        taken.append(_first_largest(v))
        v.scatter_(1, taken[-1], -INF)
    index = torch.cat(taken, 1)
    l = logit.gather(1, index).double()
    log_value = torch.nn.functional.logsigmoid(l) if case["sigmoid"] else l
    return index, torch.softmax(log_value, 1), l


def _first_largest(v):
    """Index of the first of the largest values along axis 1."""
    place = torch.arange(v.shape[1], device="cuda").view(1, -1, 1, 1)
    return torch.where(v == v.max(1, keepdim=True).values, place, v.shape[1]).min(1, keepdim=True).values


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "pack":
        return _exact_pack(s["x"], case["group"])
    if kind == "unpack":
        return _exact_unpack(s["codes"], s["ranges"], _shape(case), case["group"])
    if kind == "mex":
        return _exact_mex(s, case)
    if kind == "similarity":
        return _exact_similarity(s, case)
    index, weights, l = _exact_route(s, case)
    load = torch.bincount(index.reshape(-1), minlength=case["components"])
    if kind == "dense":
        resp = torch.zeros(s["scores"].shape, dtype=torch.float64, device="cuda").scatter_(1, index, weights)
        return resp, resp.sum((0, 2, 3)), load
    if not case["gradient"]:
        return index.int(), weights, load
    g = s["grad"].double()
    d = weights * g - weights * (weights * g).sum(1, keepdim=True)
    if case["sigmoid"]:
        d = d * torch.sigmoid(-l)
    return index.int(), weights, load, torch.zeros(s["scores"].shape, dtype=torch.float64, device="cuda").scatter_(1, index, d)
