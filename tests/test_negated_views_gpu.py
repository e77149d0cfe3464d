"""Tensors that stand for the negated values of their memory (`is_neg()`), as inputs and as incoming gradients of every operator: the answers are those for the
values.  Autograd hands such gradients to a node itself, where its output was made complex and conjugated."""
import pytest
import torch

import cases
from simnets_tf_b200 import keras
from simnets_tf_b200.ops import checkpoint as ck
from simnets_tf_b200.ops.gradients import clip_gradients, gradient_norm
from simnets_tf_b200.ops.likelihood import log_probabilities
from simnets_tf_b200.ops.loss import softmax_cross_entropy
from simnets_tf_b200.ops.mex import mex, mex_sum_pool2, sum_pool2x2
from simnets_tf_b200.ops.routing import responsibilities, route
from simnets_tf_b200.ops.similarity import similarity

pytestmark = pytest.mark.gpu
KINDS = [torch.float32, torch.float64]


def negated(v):
    """The values of v as a contiguous view of their negatives."""
    t = torch._neg_view((-v).contiguous())
    assert t.is_neg() and t.is_contiguous() and t.contiguous().is_neg()
    return t


def rand(*shape, kind=torch.float32, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=kind)


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("shape,axis", [((1, 9), 1), ((5, 700), 1), ((3, 40, 6), 1), ((2, 4, 300), 2)], ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_gradients_into_log_probabilities(shape, axis, kind):
    x = rand(*shape, kind=kind).requires_grad_()
    labels = torch.randint(0, shape[axis], [s for i, s in enumerate(shape) if i != axis], device="cuda")
    got = log_probabilities(x, labels, 2, True, axis)
    outs = [got.label, got.entropy, got.top]
    gs = [rand(*o.shape, kind=kind, seed=i) for i, o in enumerate(outs)]
    for some in ([0], [1], [2], [0, 1, 2]):
        want, = torch.autograd.grad([outs[i] for i in some], [x], [gs[i] for i in some], retain_graph=True)
        have, = torch.autograd.grad([outs[i] for i in some], [x], [negated(gs[i]) for i in some], retain_graph=True)
        assert bool((have == want).all())
    # and the labels
    again = log_probabilities(x, negated(labels), 2, True, axis)
    assert all(bool((u == v).all()) for u, v in zip(got, again))


def test_an_answer_that_is_made_complex_and_conjugated():
    """One position and several: a gradient of one value counts as contiguous, one of several lies apart in the complex one's memory."""
    for n in (1, 4):
        x = rand(n, 9).requires_grad_()
        labels = torch.arange(n, device="cuda")
        z = rand(n) + 1j * rand(n, seed=1)
        label = log_probabilities(x, labels).label
        have, = torch.autograd.grad(torch.complex(torch.zeros_like(label), label).conj(), x, z)
        want, = torch.autograd.grad(log_probabilities(x, labels).label, x, -z.imag.contiguous())
        assert bool((have == want).all())


OPS = {
    "mex": (lambda x, o: mex(x, o, 4, blocks=[3, 2, 2], strides=[3, 2, 2], epsilon=0.7, use_unshared_regions=False), [(2, 3, 8, 8), (1, 4, 3, 2, 2)]),
    "mex pooled": (lambda x, o: mex_sum_pool2(x, o, num_instances=4, blocks=[3, 1, 1], strides=[3, 1, 1], epsilon=0.7, use_unshared_regions=False), [(2, 3, 8, 8), (1, 4, 3, 1, 1)]),
    "mex with a checkpoint": (lambda x, o: ck.mex_checkpointed(x, o, 4, blocks=[3, 2, 2], strides=[3, 2, 2], epsilon=0.7, use_unshared_regions=False), [(2, 3, 8, 8), (1, 4, 3, 2, 2)]),
    "similarity": (lambda x, t, w: similarity(x, t, w, similarity_function="L2", blocks=[2, 2], strides=[2, 2]), [(2, 3, 8, 8), (5, 3, 2, 2), (5, 3, 2, 2)]),
    "similarity with a checkpoint": (lambda x, t, w: ck.similarity_checkpointed(x, t, w, similarity_function="L2", blocks=[2, 2], strides=[2, 2]), [(2, 3, 8, 8), (5, 3, 2, 2), (5, 3, 2, 2)]),
    "routing": (lambda s: route(s, top_k=2)[1], [(2, 7, 5)]),
    "routing with sigmoids": (lambda s: route(s, top_k=2, sigmoid=True)[1], [(2, 7, 5)]),
    "normalized offsets": (lambda o: keras._NormalizeOffsets.apply(o), [(2, 4, 3, 2, 2)]),
    "log probabilities": (lambda x: log_probabilities(x, entropy=True).entropy, [(6, 50)]),
}


@pytest.mark.parametrize("name", sorted(OPS))
def test_inputs_and_incoming_gradients(name):
    op, shapes = OPS[name]
    inputs = [rand(*s, seed=i).abs() if i == 2 else rand(*s, seed=i) for i, s in enumerate(shapes)]           # (weights are not negative)
    leaves = [v.clone().requires_grad_() for v in inputs]
    y = op(*leaves)
    dy = rand(*y.shape, seed=9)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    # (the same kernels on the same values; sums of parameter gradients may be taken in another order from run to run)
    for have, w in zip(torch.autograd.grad(y, leaves, negated(dy)), want):
        cases.assert_parity(have.cpu().numpy(), w.cpu().numpy(), tol=1e-5, what=name)
    twice = [negated(v).requires_grad_() for v in inputs]
    again = op(*twice)
    cases.assert_parity(again.detach().cpu().numpy(), y.detach().cpu().numpy(), tol=1e-5, what=name)
    for have, w in zip(torch.autograd.grad(again, twice, negated(dy)), want):
        cases.assert_parity(have.cpu().numpy(), w.cpu().numpy(), tol=1e-5, what=name)


def test_operators_without_gradients():
    s, y = rand(2, 7, 5), rand(2, 3, 4, 4)
    prior, bias = rand(7, seed=1), rand(7, seed=2)
    for a, b in zip(responsibilities(s, 2, prior, bias), responsibilities(negated(s), 2, negated(prior), negated(bias))):
        cases.assert_parity(a.cpu().numpy(), b.cpu().numpy(), tol=1e-6, what="responsibilities")
    assert bool((sum_pool2x2(negated(y)) == sum_pool2x2(y)).all())
    x = rand(300, 5)
    kept, again = ck.checkpoint_pack(x), ck.checkpoint_pack(negated(x))
    assert bool((kept.codes == again.codes).all()) and bool((kept.ranges == again.ranges).all())
    handmade = ck.Checkpoint(kept.codes, negated(kept.ranges), kept.shape, kept.group)
    assert bool((ck.checkpoint_unpack(handmade) == ck.checkpoint_unpack(kept)).all())
    logits = rand(6, 10)
    labels = torch.arange(6, device="cuda")
    assert bool(softmax_cross_entropy(negated(logits), negated(labels)) == softmax_cross_entropy(logits, labels))
    g = rand(5000)
    assert bool(gradient_norm([negated(g)]) == gradient_norm([g]))
    out = torch.zeros(5000, device="cuda")
    want = g.clone()
    clip_gradients([want], 1.0)
    clip_gradients([negated(g)], 1.0, out=[out])
    assert bool((out == want).all())
