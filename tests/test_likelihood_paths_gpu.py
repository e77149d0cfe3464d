"""Log probabilities on every path that sizes and layouts choose, and beyond 31 bits; the checks are those of test_likelihood_gpu.py."""
import numpy as np
import pytest
import torch

import plain_training as plain
from simnets_tf_b200.ops.likelihood import log_probabilities
from test_likelihood_gpu import KINDS, chain_of, make, near, rows_of, verify

pytestmark = pytest.mark.gpu

# rows of many and few classes in many and few rows; maps whose positions one, two, four or sixteen warps share, with classes that divide nothing
SHAPES = [(20000, 40), (17000, 100), (40000, 10), (16384, 33), (16384, 256), (300, 256), (300, 257), (2000, 513), (150, 2052), (3000, 4097), (700, 5003), (2, 4096), (2, 4095), (299, 4093),
          (5, 64, 33), (3, 65, 1000), (1, 40, 40000), (2, 17, 30000), (1, 9, 100000), (4, 1000, 7), (1, 4099, 5), (70, 66, 16), (600, 70, 4)]


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("style,top_k", [("plain", 3), ("ties", 16), ("masked", 8), ("broken", 1), ("rising", 5)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda v: "x".join(map(str, v)))
def test_every_path(shape, style, top_k, kind):
    if kind == torch.float64 and np.prod(shape) > 1200000:
        shape = (max(1, shape[0] // 2),) + shape[1:]
    x, labels = make(shape, 1, style, kind, seed=len(shape))
    top_k = min(top_k, shape[1])
    verify(x, labels, 1, top_k, True, torch.from_numpy(x).cuda())


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("top_k", [0, 1, 4, 16])
def test_rows_at_every_address(top_k, kind):
    """Rows whose starts lie to 16 bytes in every way, in gradients that lie otherwise."""
    for rows, classes in ((6, 700), (5, 9001), (3, 2), (17000, 35)):
        for shift in range(4):
            x, labels = make((rows, classes), 1, "plain", kind, seed=shift)
            wide = torch.full((rows, classes + 5), 7.0, dtype=kind, device="cuda")
            wide[:, shift:shift + classes] = torch.from_numpy(x).cuda()
            verify(x, labels, 1, min(top_k, classes), True, wide[:, shift:shift + classes])


@pytest.mark.parametrize("top_k", [2, 16])
def test_equal_classes_everywhere(top_k):
    """Heads of zeros: the alternatives are the first classes, whatever shares them."""
    for shape in ((3, 50), (2, 300), (2, 600), (1, 4096), (2, 70000), (1, 300000), (2, 80, 9), (1, 5000, 3), (2, 30, 700), (17000, 40)):
        x = torch.zeros(shape, device="cuda")
        got = log_probabilities(x, top_k=top_k, entropy=True)
        want = torch.arange(top_k, device="cuda", dtype=torch.int32).view((1, top_k) + (1,) * (x.dim() - 2))
        assert bool((got.top_index == want).all()), shape
        # S is the number of classes, exactly; its logarithm is off by a few units, and log S - 0 is the entropy
        k = shape[1]
        assert bool(((got.entropy.double() - np.log(k)).abs() <= 4 * np.finfo(np.float32).eps * np.log(k)).all())
        # later equals do not get in front: a class in the middle and one at the end
        x[:, k // 2] = 1.0
        x[:, -1] = 1.0
        got = log_probabilities(x, top_k=top_k)
        assert bool((got.top_index[:, 0] == k // 2).all()) and bool((got.top_index[:, 1] == k - 1).all())


def _rows(logits, labels, at, top_k, chain):
    return plain.Rows(np.ascontiguousarray(logits[at].cpu().numpy()), labels[at].cpu().numpy(), top_k, chain)


def test_rows_beyond_31_bits():
    rows, classes = 33000, 65537
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, classes, generator=gen, device="cuda", requires_grad=True)
    labels = torch.randint(0, classes, (rows,), generator=gen, device="cuda")
    got = log_probabilities(x, labels, 4, True)
    g = torch.randn(rows, generator=gen, device="cuda")
    dx, = torch.autograd.grad(got.label, x, g)
    at = torch.tensor([0, 1, 16384, 32766, 32767, 32768, 32769, 32998, 32999], device="cuda")
    r = _rows(x.detach(), labels, at, 4, classes // 2048 + 64)
    assert np.array_equal(got.top_index[at].cpu().numpy(), r.top_index)
    near(got.label.detach()[at].cpu().numpy(), *r.label(), "label")
    near(got.entropy.detach()[at].cpu().numpy(), r.entropy, r.off_entropy, "entropy")
    near(dx[at].cpu().numpy(), *r.gradient(g_label=g[at].cpu().numpy()), "gradient")


def test_maps_beyond_31_bits():
    classes, positions = 40, 1 << 26
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(1, classes, positions, generator=gen, device="cuda", requires_grad=True)
    labels = torch.randint(0, classes, (1, positions), generator=gen, device="cuda")
    got = log_probabilities(x, labels, 2, True)
    g = torch.randn(1, positions, generator=gen, device="cuda")
    dx, = torch.autograd.grad(got.entropy, x, g)
    at = torch.cat([torch.arange(4, device="cuda"), torch.arange(positions - 4, positions, device="cuda"), torch.randint(0, positions, (64,), generator=gen, device="cuda")])
    r = plain.Rows(np.ascontiguousarray(x.detach()[0, :, at].t().cpu().numpy()), labels[0, at].cpu().numpy(), 2, chain_of(classes))
    assert np.array_equal(got.top_index[0, :, at].t().cpu().numpy(), r.top_index)
    near(got.label.detach()[0, at].cpu().numpy(), *r.label(), "label")
    near(dx[0, :, at].t().cpu().numpy(), *r.gradient(g_entropy=g[0, at].cpu().numpy()), "gradient")
