"""MEX gradients at a checkpoint where a CTA has several tiles, where quotients leave the range of float32, and on the route through the other
entry points with a pooled gradient: against the oracle and against plain sums in 64 bits."""
import numpy as np
import pytest
import torch

import cases
from simnets_tf_b200 import abi
from simnets_tf_b200.ops import checkpoint as ck
from simnets_tf_b200.ops.routing import route
from test_checkpoint_gpu import DISJOINT, _dev, _mex_inputs, _mex_oracle, _mex_tolerance

pytestmark = pytest.mark.gpu
NAMES = ["k17", "k64", "k100", "tiles_4x2x2"]


def _named(name):
    return next(c for c in DISJOINT if c["name"] == name)


@pytest.mark.parametrize("name", NAMES)
def test_infinite_gradients_come_back_as_infinities(port, name):
    """Where the formula gives infinity (a weight above 0 times an infinite dy) the answer is infinity of that sign, not NaN, whatever the
    spread of the offsets; everything else is what it was."""
    c = _named(name)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    kept = ck.checkpoint_pack(_dev(x), 32)
    at = ck.checkpoint_unpack(kept).cpu().numpy()
    call = lambda g: ck.mex_checkpoint_backward(kept, _dev(off), _dev(g), c["M"], **cases.mex_attrs(c))
    clean = [t.cpu().numpy() for t in call(dy)]
    bad = dy.copy()
    bad[0, 1, 0, 0], bad[-1, -1, -1, -1] = np.inf, -np.inf
    got = [t.cpu().numpy() for t in call(bad)]
    refs, _ = _mex_oracle(port, c, at, off, bad)
    for g, ref, want in zip(got, refs, clean):
        assert np.isposinf(ref).any() and np.isneginf(ref).any() and not np.isnan(ref).any()
        assert np.array_equal(np.where(np.isinf(g), g, 0), np.where(np.isinf(ref), ref, 0))
        fine = np.isfinite(ref)
        assert np.array_equal(g[fine], want[fine])


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("exponent", [36, 60, 100])
def test_gradients_whose_quotients_are_no_floats(port, name, exponent):
    """Sums of exponentials near the least that the factors hold (e^-58) under a dy of 2^exponent: quotients of up to 2^(exponent + 84), gradients
    of 2^exponent."""
    c = _named(name)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    x, off = x.copy(), off.copy() * np.float32(0.1)
    b, (ch, h, w) = x.shape[0], c["blocks"]
    x.reshape(b, x.shape[1] // ch, ch, x.shape[2] // h, h, x.shape[3] // w, w)[:, :, 0, :, 0, :, 0] -= 57.0      # the first tap of every patch is low
    off.reshape(off.shape[0], off.shape[1], -1)[:, :, 0] += 57.0                                                 # ... where its offset is high
    dy = (dy * np.float32(2.0) ** exponent).astype(np.float32)
    kept = ck.checkpoint_pack(_dev(x), 32)
    at = ck.checkpoint_unpack(kept).cpu().numpy()
    dx, doff = ck.mex_checkpoint_backward(kept, _dev(off), _dev(dy), c["M"], **cases.mex_attrs(c))
    (rdx, rdoff), (adx, adoff) = _mex_oracle(port, c, at, off, dy)
    tol = _mex_tolerance(torch.float32, c, at, off, dy.size // c["M"])
    for got, ref, size in ((dx.cpu().numpy(), rdx, adx), (doff.cpu().numpy(), rdoff, adoff)):
        assert (np.abs(got - ref) <= tol * size + 1e-30 * 2.0 ** exponent).all()


def test_second_derivatives_are_refused():
    """A term with a second derivative must not be dropped: the gradients of a graph that is kept lead to a refusal."""
    torch.manual_seed(6)
    x, off = torch.randn(2, 8, 4, 4, device="cuda"), torch.randn(1, 5, 8, 1, 1, device="cuda")
    t, w = torch.randn(5, 8, 2, 2, device="cuda"), torch.rand(5, 8, 2, 2, device="cuda")
    mex = dict(blocks=[8, 1, 1], strides=[8, 1, 1], softmax_mode=True, use_unshared_regions=False, shared_offset_region=[-1])
    calls = {"Route": (lambda v: route(v, top_k=3)[1], x), "MexCheckpoint": (lambda v: ck.mex_checkpointed(v, off, 5, **mex), x),
             "MexCheckpoint of offsets": (lambda v: ck.mex_checkpointed(x, v, 5, **mex), off),
             "SimilarityCheckpoint": (lambda v: ck.similarity_checkpointed(v, t, w, blocks=[2, 2], strides=[1, 1]), x),
             "SimilarityCheckpoint of weights": (lambda v: ck.similarity_checkpointed(x, t, v, blocks=[2, 2], strides=[1, 1]), w)}
    for name, (call, at) in calls.items():
        v = at.clone().requires_grad_()
        y = call(v)
        weigh = torch.randn_like(y).requires_grad_()
        first = torch.autograd.grad((y * weigh).sum(), v, retain_graph=True)[0]
        kept = torch.autograd.grad((y * weigh).sum(), v, create_graph=True)[0]
        assert torch.equal(first, kept) and not first.requires_grad
        for inputs in (v, weigh):
            with pytest.raises(RuntimeError, match=name.split()[0] + "Backward is differentiable once"):
                torch.autograd.grad(kept.square().sum() + v.sum() + weigh.sum(), inputs, retain_graph=True)


# ---- CTAs with several tiles of positions -------------------------------------------------------------------------------------------
def _tap_index(c):
    """Index inside a sample of every tap of every position [positions, taps], the region of every position."""
    (_, ch, h, w), (bc, bh, bw) = c["shape"], c["blocks"]
    co, ho, wo = ch // bc, h // bh, w // bw
    i, j, k = torch.meshgrid(torch.arange(co), torch.arange(ho), torch.arange(wo), indexing="ij")
    i, j, k = (v.reshape(-1, 1) for v in (i, j, k))
    t = torch.arange(bc * bh * bw)
    taps = ((i * bc + t // (bh * bw)) * h + j * bh + t // bw % bh) * w + k * bw + t % bw
    n = c["unshared_region"][0] if c["unshared"] else 1
    return taps.cuda(), ((j % n) * n + k % n).reshape(-1).cuda()


def _plain_gradients(c, x, off, dy):
    """(dx, doff) in 64 bits and the sums of the terms' magnitudes, from the definition."""
    taps, region = _tap_index(c)
    x, off, dy = x.double().reshape(x.shape[0], -1), off.double().flatten(2), dy.double().reshape(x.shape[0], c["M"], -1)
    out = [torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(off), torch.zeros_like(off)]
    for r in range(off.shape[0]):
        at = (region == r).nonzero().view(-1)
        xt = x[:, taps[at]]
        sums = [torch.zeros_like(xt), torch.zeros_like(xt)]
        for m in range(c["M"]):
            p = torch.softmax(c["eps"] * (xt + off[r, m]), 2)
            for i, d in enumerate((dy, dy.abs())):
                v = d[:, m, at].unsqueeze(2) * p
                sums[i] += v
                out[2 + i][r, m] = v.sum((0, 1))
        for i in range(2):
            out[i][:, taps[at].reshape(-1)] = sums[i].reshape(x.shape[0], -1)
    return out


def _blocks(name, batch, shape, m, region, blocks=None, pooled=False, **kw):
    blocks = blocks or (shape[0], 1, 1)
    c = cases.mex_case(name, (batch,) + shape, m, blocks, blocks, softmax=True, unshared=region > 0, unshared_region=(region,) if region else (-1,), **kw)
    return dict(c, pooled=pooled)


# A CTA takes 128 positions of one region, and there are as many CTAs as multiprocessors (148): more than 18944 positions give it a second tile.  For each
# number of taps (16, 32, 64, 128): instances that fill one step and several, offsets that stay in shared memory and that do not, regions, pooling.
TILES = [
    _blocks("k13_m20", 44, (13, 32, 31), 20, 0), _blocks("k16_m300", 43, (16, 32, 32), 300, 2, pooled=True), _blocks("k16_m1200", 22, (16, 32, 31), 1200, 0),
    _blocks("k4x2x2_m150", 30, (16, 32, 32), 150, 0, blocks=(4, 2, 2), eps=0.5), _blocks("k20_m40_16_regions", 42, (20, 32, 32), 40, 4),
    _blocks("k32_m130", 43, (32, 32, 32), 130, 2), _blocks("k30_m600", 23, (30, 31, 33), 600, 0, eps=-0.7),
    _blocks("k64_m128", 43, (64, 32, 32), 128, 2, pooled=True), _blocks("k64_m100_uneven", 44, (64, 31, 33), 100, 2), _blocks("k50_m200", 30, (50, 32, 31), 200, 0),
    _blocks("k128_m64", 43, (128, 32, 32), 64, 2), _blocks("k100_m100", 30, (100, 31, 33), 100, 0), _blocks("k128_m150", 24, (128, 32, 32), 150, 2, pooled=True),
]


@pytest.mark.parametrize("c", TILES, ids=lambda c: c["name"])
def test_several_tiles_a_cta(c):
    gen = torch.Generator("cuda").manual_seed(11)
    normal = lambda *s: torch.randn(s, device="cuda", generator=gen)
    regions, ho, wo = c["unshared_region"][0] ** 2 if c["unshared"] else 1, c["shape"][2] // c["blocks"][1], c["shape"][3] // c["blocks"][2]
    kept = ck.checkpoint_pack(2 * normal(*c["shape"]) - 20, 64)
    x = ck.checkpoint_unpack(kept)
    off = 2 * normal(regions, c["M"], *c["blocks"])
    off -= torch.logsumexp(off.flatten(2), 2).view(regions, c["M"], 1, 1, 1)
    half = 2 if c["pooled"] else 1
    dy = normal(c["shape"][0], c["M"] * (c["shape"][1] // c["blocks"][0]), ho // half, wo // half)
    call = lambda: ck.mex_checkpoint_backward(kept, off, dy, c["M"], pooled=c["pooled"], **cases.mex_attrs(c))
    dx, doff = call()
    for a, b in zip(call(), (dx, doff)):
        assert torch.equal(a, b)                                                    # the same on every run
    full = dy.repeat_interleave(half, 2).repeat_interleave(half, 3)
    rdx, adx, rdoff, adoff = _plain_gradients(c, x, off, full)
    # sums of instances in pieces of 16; of positions: a tile's in pieces of 16, three tiles and 148 CTAs one after the other (a unit each)
    host = x.cpu().numpy(), off.cpu().numpy()
    for got, ref, size, n in ((dx, rdx, adx, c["M"]), (doff, rdoff, adoff, 128 + 16 * (3 + 148))):
        tol = float(_mex_tolerance(torch.float32, c, *host, n))
        assert bool(((got.double().view_as(ref) - ref).abs() <= tol * size + 1e-30).all())
    # each gradient alone
    for i, t in enumerate((x, off)):
        t = t.clone().requires_grad_()
        y = ck.mex_checkpointed(*((t, off) if i == 0 else (x, t)), c["M"], group=64, sum_pool2=c["pooled"], **cases.mex_attrs(c))
        got, = torch.autograd.grad(y, t, dy)
        # (packed again: the values of a checkpoint are at most a unit or so from those of their own checkpoint)
        again = ck.mex_checkpoint_backward(ck.checkpoint_pack(x, 64), off, dy, c["M"], pooled=c["pooled"], **cases.mex_attrs(c))[i]
        assert torch.equal(got, again)


def test_inputs_of_more_than_31_bits():
    """The last samples of an input of 2^31 values have the gradients that they have alone, and the offsets' are the sum over all."""
    batch, shape, m, group = (1 << 15) + 5, (64, 32, 32), 3, 128
    n = 64 * 32 * 32
    gen = torch.Generator("cuda").manual_seed(12)
    codes = torch.empty(batch * n, dtype=torch.uint8, device="cuda").random_(0, 253, generator=gen)
    ranges = torch.stack([torch.randn(batch * n // group, device="cuda", generator=gen) - 20, torch.full((batch * n // group,), 0.02, device="cuda")], 1)
    off, dy = torch.randn(4, m, 64, 1, 1, device="cuda", generator=gen), torch.randn(batch, m, 32, 32, device="cuda", generator=gen)
    attrs = dict(blocks=[64, 1, 1], strides=[64, 1, 1], softmax_mode=True, use_unshared_regions=True, unshared_offset_region=[2])

    def part(lo, hi):
        kept = ck.Checkpoint(codes[lo * n:hi * n], ranges[lo * n // group:hi * n // group], (hi - lo,) + shape, group)
        return ck.mex_checkpoint_backward(kept, off, dy[lo:hi], m, **attrs)
    dx, doff = part(0, batch)
    total = torch.zeros_like(doff, dtype=torch.float64)
    for lo in range(0, batch, 4096):
        a, b = part(lo, min(batch, lo + 4096))
        assert torch.equal(dx[lo:lo + 4096], a)                                     # (a position's gradients are its own)
        total += b.double()
    # sums of 2^15 x 256 terms of either sign: per CTA (148) some 445 tiles one after the other, half a unit each of what has been added so far
    weight = dy.abs().double().sum() / 4 / m
    assert bool(((doff.double() - total).abs() <= (445 + 148 + 64) * 2.0 ** -24 * weight).all())


# ---- a pooled gradient on the route through the other entry points ------------------------------------------------------------------------
def _pooled_case(name, batch, k, h, w, m, region, **kw):
    return _blocks(name, batch, (k, h, w), m, region, normalize=True, **kw)


POOLED = [_pooled_case("k129", 2, 129, 6, 6, 60, 2, seed=41), _pooled_case("k200", 3, 200, 8, 8, 96, 2, seed=42), _pooled_case("k160_few", 2, 160, 6, 8, 20, 0, seed=43),
          _pooled_case("k16_few", 2, 16, 10, 6, 16, 0, seed=44), _pooled_case("k8_few", 2, 8, 6, 6, 8, 2, seed=45), _pooled_case("k32", 2, 32, 16, 16, 64, 2, seed=46),
          _pooled_case("k64", 2, 64, 8, 8, 128, 2, seed=47), _pooled_case("k100_few", 3, 100, 6, 8, 30, 0, seed=48)]


@pytest.mark.parametrize("raw", [False, True])
@pytest.mark.parametrize("kind,flags", [(torch.float64, 0), (torch.float32, 0), (torch.float32, abi.FLAG_MEX_CHECKPOINT_TENSORCORE),
                                        (torch.float32, abi.FLAG_MEX_CHECKPOINT_TENSORCORE | abi.FLAG_MEX_NO_SMALL_TILES), (torch.float32, abi.FLAG_MEX_NO_TENSORCORE)])
@pytest.mark.parametrize("c", POOLED, ids=lambda c: c["name"])
def test_a_pooled_gradient_by_way_of_the_values(port, c, kind, flags, raw):
    """More than 128 taps, float64, or tensor cores forbidden: the bytes become x again and y is made from it, in a workspace that serves a pass at
    full resolution and gradients at half of it."""
    x, off, dy = _mex_inputs(port, c, kind)
    pooled = np.random.default_rng(5).normal(size=dy.shape[:2] + (dy.shape[2] // 2, dy.shape[3] // 2)).astype(dy.dtype)
    up = np.repeat(np.repeat(pooled, 2, axis=2), 2, axis=3)
    given = off
    if raw:
        given = off + np.random.default_rng(1).normal(size=off.shape[:2] + (1, 1, 1)).astype(off.dtype) * 5
        flags |= abi.FLAG_MEX_NORMALIZED_OFFSETS
    kept = ck.checkpoint_pack(_dev(x), 64)
    at = ck.checkpoint_unpack(kept).cpu().numpy()
    dx, doff = ck.mex_checkpoint_backward(kept, _dev(given), _dev(pooled), c["M"], flags=flags, pooled=True, **cases.mex_attrs(c))
    r = given.astype(np.float64).reshape(off.shape[0], off.shape[1], -1)
    if raw:
        r = r - (np.log(np.exp(r - r.max(2, keepdims=True)).sum(2, keepdims=True)) + r.max(2, keepdims=True))
    (rdx, rdoff), (adx, adoff) = _mex_oracle(port, c, at, r.reshape(off.shape), up)
    if raw:
        flat = lambda a: a.reshape(r.shape)
        rdoff = (flat(rdoff) - np.exp(r) * flat(rdoff).sum(2, keepdims=True)).reshape(off.shape)
        adoff = (flat(adoff) + np.exp(r) * flat(adoff).sum(2, keepdims=True)).reshape(off.shape)
    positions = dy.size // c["M"]
    tol = _mex_tolerance(kind, c, at, given, positions)
    if flags & abi.FLAG_MEX_CHECKPOINT_TENSORCORE:              # y and the sums of the products are 3 x 2^-23 off for every eight terms
        tol += 3 * 2.0 ** -23 * (np.prod(c["blocks"]) + max(c["M"], positions)) / 8
    for got, ref, size in ((dx.cpu().numpy(), rdx, adx), (doff.cpu().numpy(), rdoff, adoff)):
        assert (np.abs(got - ref) <= tol * size + 1e-30).all(), float((np.abs(got - ref) / (tol * size + 1e-30)).max())
