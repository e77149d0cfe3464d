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
