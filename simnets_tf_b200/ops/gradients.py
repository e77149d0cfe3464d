"""The norm of all gradients of a network and their clipping, between the backward pass and the step.  `dp.GradBucket` offers both for its bucket.
The reference leaves its gradients to the optimisers of its framework (HUJI-Deep/simnets-tf README.md:108-111)."""
import math

from .. import _lib
from .. import _torch_glue


def _order(order):
    """2, or 0 for the largest magnitude as the library has it."""
    if _torch_glue.is_tracing():
        raise RuntimeError("norms of gradients cannot be recorded by torch.jit.trace")
    if order not in (2, math.inf):
        raise ValueError("order must be 2 or infinity, got %r" % (order,))
    return 2 if order == 2 else 0


def gradient_norm(tensors, order=2):
    """The norm of all values of all `tensors` together (None is left out), as a 0-d tensor on their device: order 2, or math.inf for the largest
    magnitude.  float32 and float64 tensors may be mixed; the norm is float64 if one of them is.  Summed in 64 bits and in a fixed order."""
    return _lib.ops().gradient_norm(tensors, _order(order))


def clip_gradients(tensors, max_norm, order=2, out=None):
    """Scales `tensors` in place by max_norm / norm where their norm (see `gradient_norm`) is above `max_norm`, and returns the norm before.
    out: a list of tensors alike that the result goes to instead (a bucket that is added to further keeps its sums).  A norm that is NaN or
    infinite changes nothing: the norm that is returned tells.  The host waits for nothing, so a call can be part of a CUDA graph.
    No tensor that is written may share memory with another one that is given, as a slice of it, say; a tensor may be its own destination."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative, got %r" % max_norm)
    return _lib.ops().clip_gradients(tensors, max_norm, _order(order), out)
