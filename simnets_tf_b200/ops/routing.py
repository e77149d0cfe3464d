"""Routing of positions to the components of a mixture: of every position's scores the largest few, with weights that sum to one.  The
unsupervised initialisation assigns patches to templates with it (k-means takes one, a mixture that is cut short a few), with a bias
against components that nothing goes to.  The reference's estimators know full responsibilities only
(HUJI-Deep/simnets-tf python/simnets/unsupervised/gmm.py:37-71)."""
from .. import _lib
from .. import _torch_glue


def _checked(scores, top_k, prior, bias, groups, top_groups):
    """top_groups of a call whose arguments fit together (a ValueError, or the TypeError or RuntimeError of an operator, if they do not)."""
    if _torch_glue.is_tracing():
        raise RuntimeError("routing cannot be recorded by torch.jit.trace: its choice depends on the values")
    top_groups = groups if top_groups is None else top_groups
    k = scores.shape[1] if scores.dim() > 1 else 0
    whole = type(top_k) is type(groups) is type(top_groups) is int
    if not (whole and 1 <= k <= 4096 and 1 <= top_k <= 16 and 1 <= top_groups <= groups and k % groups == 0 and top_k <= top_groups * (k // groups) and
            (top_groups == groups or groups <= 64 and top_groups <= 16)):
        _explain(scores, k, top_k, groups, top_groups)
    for name, v in (("prior", prior), ("bias", bias)):
        if v is None:
            continue
        if v.dim() != 1 or v.shape[0] != k:
            raise ValueError("%s must hold one value per component, got %s" % (name, tuple(v.shape)))
        if v.requires_grad:
            raise ValueError("%s is a constant of the choice: it has no gradient" % name)
    return top_groups


def _explain(scores, k, top_k, groups, top_groups):
    if k < 1:
        raise ValueError("scores must have the components on axis 1, got %s" % (tuple(scores.shape),))
    for name, v in (("top_k", top_k), ("groups", groups), ("top_groups", top_groups)):
        if type(v) is not int or v < 1:
            raise ValueError("%s must be a positive whole number, got %r" % (name, v))
    if k % groups or top_groups > groups:
        raise ValueError("%d components do not fall into %d groups of which %d are taken" % (k, groups, top_groups))
    if top_k > top_groups * (k // groups):
        raise ValueError("top_k = %d of %d components" % (top_k, top_groups * (k // groups)))
    raise ValueError("at most 4096 components, top_k = 16, and where groups are chosen 16 of 64, got %d, %d, %d of %d" % (k, top_k, top_groups, groups))


def route(scores, top_k=1, prior=None, bias=None, groups=1, top_groups=None, sigmoid=False, scale=1.0):
    """(index, weights, load) for scores [batch, components, ...]: per position the `top_k` components with the largest
    v = (score + prior) + bias, ties to the lowest index.  index: int32 [batch, top_k, ...] by falling v; weights: alike, `scale` times
    exp(score + prior), or sigmoid(score + prior), over its sum over the chosen, so that `bias` changes who is chosen and not what they
    weigh; load: int64 [components], positions that chose each.

    With groups > 1 the components are that many runs of equal length, and only the `top_groups` of them with the largest v
    are in the choice.  A component whose v is NaN or -infinity is not chosen; where fewer than `top_k` are left the index
    is -1 and the weight 0.  Chosen components with an infinite score share alike.

    The weights are differentiable with respect to the scores, once; what stays for the gradient are index and weights, and the scores with
    sigmoid=True."""
    top_groups = _checked(scores, top_k, prior, bias, groups, top_groups)
    return _lib.ops().route_apply(scores, prior, bias, top_k, groups, top_groups, bool(sigmoid), float(scale))


def responsibilities(scores, top_k=1, prior=None, bias=None, groups=1, top_groups=None, sigmoid=False):
    """(responsibilities, mass, load): the weights of `route` as a tensor of the scores' shape, 0 where a component is not chosen, and
    their sum per component over all positions.  What the moments of a mixture take; constants of the scores (not differentiable)."""
    top_groups = _checked(scores, top_k, prior, bias, groups, top_groups)
    return _lib.ops().responsibilities(scores, prior, bias, top_k, groups, top_groups, bool(sigmoid))
