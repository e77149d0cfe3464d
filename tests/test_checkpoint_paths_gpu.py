"""MEX gradients at a checkpoint where a CTA has several tiles, where quotients leave the range of float32, and on the route through the other
entry points with a pooled gradient: against the oracle and against plain sums in 64 bits."""
import numpy as np
import pytest
import torch

import cases
from simnets_tf_b200 import abi
from simnets_tf_b200.ops import checkpoint as ck
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
