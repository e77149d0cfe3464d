"""Whether two tensors share memory, which clipping asks before it writes: against the sets of their bytes, on the host; and the calls that it refuses."""
import itertools
import time

import numpy as np
import pytest
import torch

from simnets_tf_b200 import _lib
from simnets_tf_b200.ops.gradients import clip_gradients, gradient_norm


def bytes_of(t):
    at = np.array([t.data_ptr()])
    for size, stride in zip(t.shape, t.stride()):
        at = (at[:, None] + stride * t.element_size() * np.arange(size)).reshape(-1)
    return set((at[:, None] + np.arange(t.element_size())).reshape(-1).tolist())


def agree(a, b):
    want = bool(bytes_of(a) & bytes_of(b))
    share = _lib.ops().share_memory
    assert share(a, b) == want == share(b, a), (a.shape, a.stride(), a.storage_offset(), a.dtype, b.shape, b.stride(), b.storage_offset(), b.dtype)


@pytest.mark.parametrize("seed", range(8))
def test_any_two_strided_views(seed):
    rng = np.random.default_rng(seed)
    flat = torch.zeros(4000)
    hits = 0
    for _ in range(400):
        def view():
            base = flat.view(torch.float64) if rng.random() < 0.3 else flat
            dims = int(rng.integers(0, 5))
            size, stride = [int(s) for s in rng.integers(1, 6, dims)], [int(s) for s in rng.choice([0, 1, 1, 2, 3, 4, 6, 10, 12, 20, 60, 61, 100], dims)]
            return base.as_strided(size, stride, int(rng.integers(0, 300)))
        a, b = view(), view()
        agree(a, b)
        hits += bool(bytes_of(a) & bytes_of(b))
    assert 20 < hits < 380


def test_views_of_one_matrix():
    a = torch.zeros(12, 10)
    views = [a, a[:, :3], a[:, 2:5], a[:, 3:], a[3], a[4:8], a[::2], a[1::2], a[::3, ::2], a[1::3, 1::2], a.t(), a.t()[:3], a[:, 3:].t(), a[2:4, 3:5], a.view(torch.float64)[:, 2:],
             a[0, 0], a[5, 5], a.view(-1)[::7], a.view(-1)[3::7], a.view(-1)[::11], a.view(-1).unfold(0, 5, 3), a[:, 4].expand(3, 12), a[:0]]
    for x, y in itertools.product(views, views):
        if x.numel() and y.numel():
            agree(x, y)
        else:
            assert not _lib.ops().share_memory(x, y)


def test_many_values_take_no_longer():
    """What the strides tell, without looking at every value."""
    a = torch.empty(2048, 2048)
    share, begin = _lib.ops().share_memory, time.perf_counter()
    assert not share(a[:, :1000], a[:, 1000:]) and share(a[:, :1000], a[:, 999:])
    assert not share(a.view(-1)[::2], a.view(-1)[1::4]) and share(a.view(-1)[1::2], a.view(-1)[3::4])
    assert not share(a.t()[::2, ::2], a[1::2, 1::2]) and not share(a[:, 5], a[:, 6]) and share(a[:, 5], a[5])
    assert time.perf_counter() - begin < 1.0


@pytest.mark.gpu
def test_clipping_refuses_tensors_that_share_some_of_their_memory():
    a, to = torch.ones(10, 6, device="cuda"), torch.zeros(10, 6, device="cuda")
    ok = torch.ones(10, 3, device="cuda")
    for bad, out in (([a[:, :3], a[:, 2:5]], None), ([a[1], a[:, :3]], None), ([a[:, :3], a[4]], None), ([a[::2, :3], a[2:7, 1:5]], None), ([a[:, ::2], a[:, 2:4]], None),
                     ([a[:, :3], a[:, 3:]], [to[:, :3], to[:, 2:5]]), ([ok, a[0]], [to[:, 1:4], to[3]]), ([a[0], ok], [to[3], to[:, 1:4]]), ([a[:, :3]], [a[:, 1:4]]),
                     ([a[:, :3], ok], [to[:, :3], a[:, 2:5]]), ([a[:6, :6]], [a[:6, :6].t()]), ([a[:3, :3]], [a[:3, :3].t()])):
        with pytest.raises(ValueError, match="share memory"):
            clip_gradients(bad, 1.0, out=out)
    assert bool((a == 1).all()) and bool((to == 0).all()) and bool((ok == 1).all())
    # side by side, and as their own destinations
    n = clip_gradients([a[:, :3], a[:, 3:5], a[:, 5]], 1.0, out=[a[:, :3], to[:, 3:5], to[:, 0]])
    assert abs(float(n) - 60 ** 0.5) < 1e-5
    assert torch.allclose(a[:, :3], 1 / n, rtol=1e-6, atol=0) and bool((a[:, 3:] == 1).all()) and torch.allclose(to[:, 3:5], 1 / n, rtol=1e-6, atol=0)
    assert torch.allclose(to[:, 0], 1 / n, rtol=1e-6, atol=0) and bool((to[:, 1:3] == 0).all()) and bool((to[:, 5] == 0).all())
    b = torch.full((8, 8), 3.0, device="cuda")
    n = clip_gradients([b[::2, ::2], b[1::2, 1::2], b[::2, 1::2], b[1::2, ::2]], 1.0)
    assert float(n) == 24.0 and torch.allclose(b, torch.full_like(b, 3.0 / 24.0), rtol=1e-6, atol=0)
    # where nothing is written a tensor may be counted twice
    assert abs(float(gradient_norm([ok[:, :2], ok[:, 1:]])) - 40 ** 0.5) < 1e-5
