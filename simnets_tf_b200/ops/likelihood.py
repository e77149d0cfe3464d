"""Log probabilities of given classes with the entropy and the likeliest alternatives: what a classifier answers, and what losses per position (maps,
sequences, padded batches, entropy terms, a second network's alternatives) are made of.  `ops.loss.softmax_cross_entropy` is their sum as one
number over rows.  The reference has its framework's softmax and cross-entropy (HUJI-Deep/simnets-tf README.md:108-111)."""
from collections import namedtuple

from .. import _lib
from .. import _torch_glue

LogProbabilities = namedtuple("LogProbabilities", ["label", "entropy", "top_index", "top"])


def log_probabilities(logits, labels=None, top_k=0, entropy=False, axis=1):
    """(label, entropy, top_index, top) of logits with the classes on `axis`, 1 or the last one; None in the place of what is not asked for.

    label: log probabilities of the classes in `labels` (int64, the logits' shape without `axis`), 0 where a label is outside [0, classes);
    entropy: of the classes of every position; top_index, top: the `top_k` (at most 16) classes with the largest logits by falling logit, ties to
    the lowest index, as int32 and their log probabilities, with top_k in the place of the classes.  A logit of -infinity is a class
    that cannot be: where fewer than top_k can, the index is -1 and the log probability -infinity; where none can, the entropy is 0 and every log
    probability -infinity.  A NaN or infinity makes the log probabilities and the entropy of its position NaN.

    label, entropy and top are differentiable with respect to the logits, once; the logits and three numbers per position stay for it.  A
    position where no class can be has the gradient 0.  float32 and float64, any strides (what has neither classes nor positions
    side by side is copied)."""
    if _torch_glue.is_tracing():
        raise RuntimeError("log_probabilities cannot be recorded by torch.jit.trace: its alternatives depend on the values")
    if type(top_k) is not int or type(axis) is not int:
        raise ValueError("top_k and axis must be whole numbers, got %r and %r" % (top_k, axis))
    return LogProbabilities(*_lib.ops().log_probabilities(logits, labels, top_k, bool(entropy), axis + logits.dim() if axis < 0 else axis))
