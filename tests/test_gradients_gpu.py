"""Norms and clipping of gradients on the GPU against the restatement in plain_training.py."""
import math

import numpy as np
import pytest
import torch

import plain_training as plain
from simnets_tf_b200 import _lib, dp
from simnets_tf_b200.ops.gradients import clip_gradients, gradient_norm

pytestmark = pytest.mark.gpu
INF = math.inf
SIZES = [(1,), (3,), (7, 5), (4096,), (4097,), (64, 64, 3), (100003,), (0,), (2, 0, 3), (), (300001,)]


def make(sizes, kinds, seed=0, scale=1.0):
    rng = np.random.default_rng(seed)
    return [np.asarray(scale * rng.normal(size=s)).astype(kinds[i % len(kinds)]) for i, s in enumerate(sizes)]


def dev(arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).reshape(a.shape).cuda() for a in arrays]


def agree(norm, got, want_norm, want, arrays, limit):
    """The norm is a sum in 64 bits, rounded once to its type: a step of it.  The scale is off by as much, and the product rounded once."""
    eps = np.finfo(want_norm.dtype).eps
    n = norm.cpu().numpy()
    assert n.dtype == want_norm.dtype and n.shape == ()
    assert (np.isnan(n) and np.isnan(want_norm)) or n == want_norm or abs(np.longdouble(n) - want_norm) <= eps * abs(np.longdouble(want_norm)) + np.finfo(n.dtype).smallest_subnormal, (n, want_norm)
    for g, w, a in zip(got, want, arrays):
        g = g.cpu().numpy()
        assert g.dtype == a.dtype and g.shape == a.shape
        if not np.isfinite(want_norm) or want_norm <= limit:
            assert np.array_equal(g, a, equal_nan=True)
        else:
            off = (eps + np.finfo(a.dtype).eps) * abs(w.astype(np.longdouble)) + np.finfo(a.dtype).smallest_subnormal
            assert (abs(g.astype(np.longdouble) - w) <= off).all()


@pytest.mark.parametrize("order", [2, INF])
@pytest.mark.parametrize("kinds", [[np.float32], [np.float64], [np.float32, np.float64]], ids=["f32", "f64", "both"])
@pytest.mark.parametrize("count", [1, 4, 11, 30, 1000, 2500])
def test_norm_and_clipping(count, kinds, order):
    sizes = [SIZES[i % len(SIZES)] if count <= 30 else (1 + i % 37,) for i in range(count)]
    arrays = make(sizes, kinds)
    n0 = plain.clipped(arrays, INF, order)[0]
    for limit in (0.3 * float(n0), 3.0 * float(n0), 0.0, INF):
        want_norm, want = plain.clipped(arrays, limit, order)
        tensors = dev(arrays)
        agree(gradient_norm(tensors, order=order), [], want_norm, [], [], limit)
        out = [torch.full_like(t, 7.0) for t in tensors]
        agree(clip_gradients(tensors, limit, order=order, out=out), out, want_norm, want, arrays, limit)
        assert all(np.array_equal(t.cpu().numpy(), a) for t, a in zip(tensors, arrays))
        agree(clip_gradients(tensors, limit, order=order), tensors, want_norm, want, arrays, limit)


@pytest.mark.parametrize("order", [2, INF])
def test_values_whose_squares_do_not_fit(order):
    for kind, scales in ((np.float32, (1e-44, 1e-38, 1e-30, 1e18, 1e37)), (np.float64, (1e-320, 1e-300, 1e-170, 1e-140, 1e140, 1e160, 1e300))):
        for scale in scales:
            arrays = make([(1000,), (77,)], [kind], scale=scale)
            limit = 0.5 * float(plain.norm(arrays, order))
            want_norm, want = plain.clipped(arrays, limit, order)
            tensors = dev(arrays)
            agree(clip_gradients(tensors, limit, order=order), tensors, want_norm, want, arrays, limit)
    # tiny ones beside one that is not
    arrays = [np.full(100, 1e-200), np.array([2.0]), np.full(9, 1e-30, np.float32)]
    assert float(gradient_norm(dev(arrays))) == 2.0
    arrays = [np.full(100, 1e-30, np.float32), np.full(1, 1e200)]
    assert abs(float(gradient_norm(dev(arrays))) / 1e200 - 1) < 1e-15


@pytest.mark.parametrize("order", [2, INF])
@pytest.mark.parametrize("bad", [math.nan, INF, -INF])
def test_a_norm_that_is_no_number_changes_nothing(bad, order):
    for kind in (np.float32, np.float64):
        for place in (0, 1):
            arrays = make([(5000,), (33,)], [kind])
            arrays[place][17] = bad
            tensors = dev(arrays)
            n = clip_gradients(tensors, 1.0, order=order)
            assert bool(n.isnan()) if math.isnan(bad) else bool(n.isinf())
            assert all(np.array_equal(t.cpu().numpy(), a, equal_nan=True) for t, a in zip(tensors, arrays))
    # a norm beyond float32: as it is returned, infinite
    t = torch.full((4,), 3e38, device="cuda")
    assert bool(clip_gradients([t], 1.0).isinf()) and bool((t == 3e38).all())


@pytest.mark.parametrize("kind", [torch.float32, torch.float64])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_tensors_at_any_address_and_what_lies_beside_them(kind, shift):
    """Views of one buffer, one behind the other with a value between: what is between stays."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    sizes = [1, 2, 3, 5, 4093, 4096, 8191, 12289]
    flat = torch.randn(sum(sizes) + 16, generator=gen, device="cuda", dtype=kind)
    kept = flat.clone()
    views, at, used = [], shift, torch.zeros_like(flat, dtype=torch.bool)
    for n in sizes:
        views.append(flat[at:at + n])
        used[at:at + n] = True
        at += n + 1
    want = kept[used].double().square().sum().sqrt()
    n = clip_gradients(views, 1.0)
    assert abs(float(n) / float(want) - 1) < 1e-6
    assert bool((flat[~used] == kept[~used]).all())
    assert torch.allclose(flat[used], kept[used] / n.to(kind), rtol=1e-6 if kind == torch.float32 else 1e-14, atol=0)
    # into places that lie differently to 16 bytes
    for other in range(4):
        src, to = kept[shift:shift + 9001], torch.full((9100,), 7.0, device="cuda", dtype=kind)
        clip_gradients([src], 1.0, out=[to[other:other + 9001]])
        alone = src.clone()
        clip_gradients([alone], 1.0)
        # The sums are grouped by the 16-byte pieces in which the values lie, and src and alone lie differently.  Two orders of a sum of n terms
        # of one sign part by at most n eps of it, its root by half of that; then the root, the scale and the product are each rounded
        # (float32: the norm and the product to that type), on both sides.
        tol = (9001 / 2 + 6) * np.finfo(np.float64).eps + (0 if kind == torch.float64 else 2 * np.finfo(np.float32).eps)
        assert bool(((to[other:other + 9001] - alone).abs() <= tol * alone.abs()).all()) and bool((to[:other] == 7).all()) and bool((to[other + 9001:] == 7).all())


def test_tensors_that_are_not_dense():
    a = torch.randn(40, 30, device="cuda")
    ref = a.clone()
    n = clip_gradients([a[:, :10], a[:, 10:].t()], 1.0)                      # (columns of one matrix, one part transposed)
    assert abs(float(n) / float(ref.norm()) - 1) < 1e-6 and torch.allclose(a, ref / n, rtol=1e-6, atol=0)
    b, out = torch.randn(6, 8, device="cuda").t(), torch.zeros(8, 6, device="cuda")
    n = clip_gradients([b], 1.0, out=[out])
    assert torch.allclose(out, b / n, rtol=1e-6, atol=0)
    out = torch.zeros(8, 12, device="cuda")
    n = clip_gradients([b], 1.0, out=[out[:, ::2]])
    assert torch.allclose(out[:, ::2], b / n, rtol=1e-6, atol=0) and bool((out[:, 1::2] == 0).all())
    e = torch.full((1, 5), 2.0, device="cuda").expand(8, 5)
    assert abs(float(gradient_norm([e])) - math.sqrt(160)) < 1e-5           # (every element counts)


def test_a_tensor_that_is_not_dense_is_given_once_too():
    a = torch.ones(10, 6, device="cuda")
    for bad in ([a[:, :3], a[:, :3]], [a[:, ::2], a], [a[:, :3], a[:4, :2]], [a[3, 2:], a[3:, 2:4]]):
        with pytest.raises(ValueError, match="share memory"):
            clip_gradients(bad, 1.0)
    to = torch.zeros(10, 6, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([a[:, :3], a[:, 3:]], 1.0, out=[to[:, :3], to[:, :3]])
    assert bool((a == 1).all()) and bool((to == 0).all())
    assert abs(float(gradient_norm([a[:, :3], a[:, :3]])) - math.sqrt(60)) < 1e-5
    # into itself, and into the other's place
    n = clip_gradients([a[:, :3], a[:, 3:]], 1.0, out=[a[:, :3], to[:, 3:]])
    assert torch.allclose(a[:, :3], 1 / n, rtol=1e-6, atol=0) and bool((a[:, 3:] == 1).all()) and torch.allclose(to[:, 3:], 1 / n, rtol=1e-6, atol=0)


def test_what_is_refused():
    a = torch.ones(10, device="cuda")
    for bad in ([a, a], [a, a[2:5]], [a[:6], a[5:]]):
        with pytest.raises(ValueError, match="share memory"):
            clip_gradients(bad, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([a[:4], a[4:8]], 1.0, out=[a[4:8], torch.ones(4, device="cuda")])
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([a[:4]], 1.0, out=[a[1:5]])
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([torch.ones(1, device="cuda").expand(5)], 1.0)
    for out in (torch.ones(9, device="cuda"), torch.ones(10, device="cuda", dtype=torch.float64), torch.ones(10)):
        with pytest.raises(ValueError, match="out must have"):
            clip_gradients([a], 1.0, out=[out])
    p = torch.ones(4, device="cuda", requires_grad=True)
    for call in (lambda: gradient_norm([p]), lambda: clip_gradients([p], 1.0), lambda: clip_gradients([torch.ones(4, device="cuda")], 1.0, out=[p])):
        with pytest.raises(ValueError, match="detach"):
            call()
    with torch.no_grad():
        assert float(gradient_norm([p])) == 2.0
    with pytest.raises(RuntimeError, match="no CPU kernels"):
        clip_gradients([a, torch.ones(3)], 1.0)
    assert bool((a == 1).all())
    # the same tensor may be counted twice where nothing is written, and be its own destination
    assert abs(float(gradient_norm([a, a])) - math.sqrt(20)) < 1e-5
    clip_gradients([a, None], 1.0, out=[a, None])
    assert abs(float(gradient_norm([a])) - 1) < 1e-6


def test_autograd_sees_that_a_tensor_was_written():
    w = torch.randn(5, device="cuda", requires_grad=True)
    g = torch.randn(5, device="cuda")
    y = (w * g).sum()
    clip_gradients([g], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_the_same_sum_on_every_run_and_stream_and_in_a_graph():
    arrays = make([(100003,), (5,), (70001,)], [np.float32])
    tensors, out = dev(arrays), dev(arrays)
    want = clip_gradients(tensors, 1.0, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            assert bool(gradient_norm(tensors) == want)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph, to = torch.cuda.CUDAGraph(), [torch.zeros_like(t) for t in tensors]
        with torch.cuda.graph(graph):
            n = clip_gradients(tensors, 1.0, out=to)
        graphs.append((graph, n, to))
    for t in tensors:
        t.mul_(2.0)
    for _ in range(2):
        for graph, _, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for _, n, to in graphs:
        assert bool(n == 2 * want) and all(bool((a == b).all()) for a, b in zip(to, out))


def test_two_launches():
    g = dev(make([(1000,), (20,)], [np.float32]))
    n = _lib.launch_count()
    clip_gradients(g, 1.0)
    assert _lib.launch_count() == n + 2
    gradient_norm(g)
    assert _lib.launch_count() == n + 4


def test_beyond_31_bits():
    """More than 2^31 values in one tensor, one of which decides."""
    n = (1 << 31) + 12345
    t = torch.zeros(n, device="cuda")
    t[n - 2] = 3.0
    t[1] = 4.0
    assert float(gradient_norm([t])) == 5.0 and float(gradient_norm([t], order=INF)) == 4.0
    assert float(clip_gradients([t], 2.5)) == 5.0
    assert float(t[n - 2]) == 1.5 and float(t[1]) == 2.0 and float(t[n - 1]) == 0.0


def test_a_bucket():
    a, b = torch.nn.Parameter(torch.zeros(7, 3, device="cuda")), torch.nn.Parameter(torch.zeros(5, device="cuda"))
    bucket = dp.GradBucket([a, b])
    a.grad.fill_(2.0)
    b.grad.fill_(4.0)
    want = math.sqrt(21 * 4 + 5 * 16)
    assert abs(float(bucket.norm()) / want - 1) < 1e-6 and float(bucket.norm(order=INF)) == 4.0
    assert abs(float(bucket.clip(1.0)) / want - 1) < 1e-6
    assert abs(float(a.grad[0, 0]) * want / 2 - 1) < 1e-6 and abs(float(b.grad[0]) * want / 4 - 1) < 1e-6


def test_views_that_stand_for_negated_values():
    z = torch.randn(5000, dtype=torch.complex64, device="cuda")
    x, want = z.conj().imag, (-z.imag).contiguous()
    assert x.is_neg()
    out = torch.zeros(5000, device="cuda")
    n = clip_gradients([x], 1.0, out=[out])
    clip_gradients([want], 1.0)
    assert bool((out == want).all()) and bool(n == gradient_norm([(-z.imag).contiguous()]))
    clip_gradients([x], 1.0)
    assert bool((x == want).all()) and bool((z.imag == -want).all())


def test_nothing_to_take_the_norm_of():
    """Through Python tensors without values, through the C entry point none at all."""
    assert float(gradient_norm([torch.zeros(0, device="cuda"), torch.zeros(3, 0, device="cuda")])) == 0.0
    assert float(clip_gradients([torch.zeros(0, device="cuda", dtype=torch.float64)], 1.0)) == 0.0
    lib = _lib.lib()
    size = lib.simnets_gradient_norm_workspace_bytes(0)
    ws, norm = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.full((3,), 7.0, device="cuda")
    _lib.check(lib.simnets_gradient_norm(2, 0, None, None, None, norm.data_ptr() + 4, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream))
    assert norm.tolist() == [7.0, 0.0, 7.0]
