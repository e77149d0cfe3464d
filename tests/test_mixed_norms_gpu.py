"""Norms of float32 and float64 tensors together, where one type's squares decide and the other's are an infinity, a NaN, or nothing beside them."""
import math

import numpy as np
import pytest
import torch

import plain_training as plain
from simnets_tf_b200.ops.gradients import clip_gradients, gradient_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", [2, math.inf])
@pytest.mark.parametrize("f32", [0.0, 1e-45, 1e-38, 1.0, 3e38, math.inf, math.nan])
@pytest.mark.parametrize("f64", [0.0, 5e-324, 1e-300, 1e-140, 1e-20, 1.0, 1e150, 1e300, math.inf, math.nan])
def test_both_types(f32, f64, order):
    arrays = [np.full(5, f32, np.float32), np.full(7, f64)]
    tensors = [torch.from_numpy(a).cuda() for a in arrays]
    with np.errstate(over="ignore"):
        want = np.float64(plain.norm(arrays, order))
    for given in (tensors, tensors[::-1]):
        n = gradient_norm(given, order=order)
        assert n.dtype == torch.float64
        got = float(n)
        # Roundings of half an eps: a thread adds up to four squares, five times two lanes' sums are added, and then those of the two types (what else is added is 0):
        # ten of a sum of one sign, five of its root, and the root's own.  (The last is a step where the norm is no normal number.)
        assert (math.isnan(got) and math.isnan(want)) or got == want or abs(got - want) <= 3 * np.finfo(np.float64).eps * want + 5e-324, (got, want)
    if order == 2 and 0 < want < math.inf:
        _, clipped = plain.clipped(arrays, 0.5 * want)
        clip_gradients(tensors, 0.5 * want)
        # (those six, of the quotient and, on the other side, of the norm; the product's on both)
        for t, w in zip(tensors, clipped):
            assert (abs(t.cpu().numpy().astype(np.longdouble) - w) <= (4 * np.finfo(np.float64).eps + np.finfo(w.dtype).eps) * abs(w.astype(np.longdouble)) + np.finfo(w.dtype).smallest_subnormal).all()
