"""Tensors whose storage has been given back (sharded training does that between two uses) are refused; zeros that need no memory count as zeros.  Neither reaches
a kernel, which would read at an address of null."""
import pytest
import torch

from simnets_tf_b200 import _torch_glue, keras
from simnets_tf_b200.ops import checkpoint as ck
from simnets_tf_b200.ops.gradients import clip_gradients, gradient_norm
from simnets_tf_b200.ops.likelihood import log_probabilities
from simnets_tf_b200.ops.loss import softmax_cross_entropy
from simnets_tf_b200.ops.mex import mex, sum_pool2x2
from simnets_tf_b200.ops.routing import route
from simnets_tf_b200.ops.similarity import similarity


def freed(*shape, dtype=torch.float32, device="cuda", view=lambda t: t):
    t = torch.zeros(shape, dtype=dtype, device=device)
    v = view(t)                             # (of a tensor that is empty already torch makes none)
    t.untyped_storage().resize_(0)
    return v


def test_the_check_itself():
    with pytest.raises(RuntimeError, match="no memory"):
        _torch_glue.plain(freed(3, device="cpu"))
    assert _torch_glue.plain(torch._efficientzerotensor(3)).tolist() == [0.0] * 3
    assert _torch_glue.plain(torch.zeros(0)).numel() == 0


@pytest.mark.gpu
def test_storage_that_has_been_given_back():
    ok, labels = torch.zeros(4, 6, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    image, block = torch.zeros(1, 2, 4, 4, device="cuda"), torch.zeros(3, 2, 2, 2, device="cuda")
    offsets, kw = torch.zeros(1, 3, 2, 1, 1, device="cuda"), dict(blocks=[2, 1, 1], strides=[2, 1, 1], use_unshared_regions=False)
    for call in (lambda: log_probabilities(freed(4, 6), entropy=True), lambda: log_probabilities(ok, freed(4, dtype=torch.int64)),
                 lambda: log_probabilities(freed(4, 12, view=lambda t: t[:, ::2].t()), entropy=True, axis=1), lambda: softmax_cross_entropy(freed(4, 6), labels),
                 lambda: softmax_cross_entropy(ok, freed(4, dtype=torch.int64)), lambda: gradient_norm([ok, freed(5)]), lambda: clip_gradients([freed(5)], 1.0),
                 lambda: clip_gradients([freed(4, 6, view=lambda t: t[:, :3])], 1.0), lambda: clip_gradients([ok], 1.0, out=[freed(4, 6)]), lambda: route(freed(2, 5, 3)),
                 lambda: mex(freed(1, 2, 4, 4), offsets, 3, **kw), lambda: mex(image, freed(1, 3, 2, 1, 1), 3, **kw),
                 lambda: similarity(freed(1, 2, 4, 4), block, block, blocks=[2, 2]), lambda: similarity(image, block, freed(3, 2, 2, 2), blocks=[2, 2]),
                 lambda: ck.checkpoint_pack(freed(40)), lambda: sum_pool2x2(freed(1, 1, 2, 2)), lambda: keras._NormalizeOffsets.apply(freed(1, 3, 2, 1, 1))):
        with pytest.raises(RuntimeError, match="no memory"):
            call()
    assert bool((ok == 0).all())
    # between the two passes
    x = ok.clone().requires_grad_()
    got = log_probabilities(x, entropy=True)
    x.data.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="no memory"):
        got.entropy.sum().backward()


@pytest.mark.gpu
def test_zeros_that_need_no_memory():
    def zeros(*shape, dtype=torch.float32):
        t = torch._efficientzerotensor(shape, dtype=dtype, device="cuda")
        assert t._is_zerotensor()
        return t
    x = torch.randn(4, 6, device="cuda").requires_grad_()
    got = log_probabilities(x, torch.zeros(4, dtype=torch.int64, device="cuda"), 2, True)
    for out in (got.label, got.entropy, got.top):
        dx, = torch.autograd.grad(out, x, zeros(*out.shape), retain_graph=True)
        assert bool((dx == 0).all())
    even = log_probabilities(zeros(4, 6), zeros(4, dtype=torch.int64), 2, True)
    want = log_probabilities(torch.zeros(4, 6, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), 2, True)
    assert all(bool((u == v).all()) for u, v in zip(even, want))
    s = torch.randn(2, 5, 3, device="cuda").requires_grad_()
    ds, = torch.autograd.grad(route(s, top_k=2)[1], s, zeros(2, 2, 3))
    assert bool((ds == 0).all())
    assert float(gradient_norm([zeros(5), torch.full((4,), 2.0, device="cuda")])) == 4.0
    out = torch.ones(5, device="cuda")
    assert float(clip_gradients([zeros(5)], 1.0, out=[out])) == 0.0 and bool((out == 0).all())
    for call in (lambda: clip_gradients([zeros(5)], 1.0), lambda: clip_gradients([torch.ones(5, device="cuda")], 1.0, out=[zeros(5)])):
        with pytest.raises(ValueError, match="no memory"):
            call()
