"""What a position answers does not depend on the others: the same bits alone and inside a batch where both take the same kernel (the number of positions chooses
it, and with it the order of the sums), and the same bits whatever the others are."""
import pytest
import torch

from simnets_tf_b200.ops.likelihood import log_probabilities

pytestmark = pytest.mark.gpu
KINDS = [torch.float32, torch.float64]
NAN, INF = float("nan"), float("inf")


def everything(x, labels, axis=1):
    leaf = x.detach().requires_grad_()
    got = log_probabilities(leaf, labels, min(4, x.shape[axis]), True, axis)
    dx, = torch.autograd.grad([got.label, got.entropy, got.top], [leaf], [torch.ones_like(got.label), torch.full_like(got.entropy, 0.3), torch.full_like(got.top, -0.7)])
    return [got.label.detach(), got.entropy.detach(), got.top_index, got.top.detach(), dx]


def make(shape, axis, kind):
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = 3 * torch.randn(shape, generator=gen, device="cuda", dtype=kind)
    return x, torch.randint(0, shape[axis], [s for i, s in enumerate(shape) if i != axis], generator=gen, device="cuda")


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("shape", [(40, 300), (33, 10), (50, 33), (9, 511), (6, 20, 33), (5, 70, 40), (3, 300, 64)], ids=lambda v: "x".join(map(str, v)))
def test_alone_and_in_a_batch(shape, kind):
    """(Up to 512 classes rows go to warps of their own however many they are, and up to ten tiles of positions are shared by as many warps as one is; a slice starts where
    the sample in the batch does.)"""
    x, labels = make(shape, 1, kind)
    whole = everything(x, labels)
    for i in (0, 1, shape[0] // 2, shape[0] - 1):
        for part, w in zip(everything(x[i:i + 1], labels[i:i + 1]), whole):
            assert bool((part == w[i:i + 1]).all())


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("shape,axis", [((40, 300), 1), ((20, 9001), 1), ((300, 5000), 1), ((17000, 40), 1), ((3000, 1500), 1), ((6, 20, 33), 1), ((70, 66, 16), 1), ((4, 9, 700), 2), ((1, 40, 20000), 1)],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_whatever_the_others_are(shape, axis, kind):
    x, labels = make(shape, axis, kind)
    whole = everything(x, labels, axis)
    rows = x.movedim(axis, -1)
    keep = torch.rand(rows.shape[:-1], generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.5
    for fill in (NAN, INF, -INF, torch.finfo(kind).max, torch.finfo(kind).min):
        other = torch.where(keep.unsqueeze(-1), rows, torch.full((), fill, dtype=kind, device="cuda")).movedim(-1, axis).contiguous()
        for part, w in zip(everything(other, labels, axis), whole):
            if part.dim() > keep.dim():
                part, w = part.movedim(axis, -1), w.movedim(axis, -1)
            assert bool((part[keep] == w[keep]).all())
