"""Routing on the GPU against the restatement in plain_operators.py: choices and loads exactly, weights, masses and gradients in 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

import plain_operators as plain
from oracle import unsupervised_oracle as uo
from simnets_tf_b200 import abi, keras
from simnets_tf_b200 import unsupervised as un
from simnets_tf_b200.ops.routing import responsibilities, route

pytestmark = pytest.mark.gpu
KINDS = [torch.float32, torch.float64]


def _dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _inputs(shape, kind, style, seed=0):
    rng = np.random.default_rng(seed)
    dt = np.float32 if kind == torch.float32 else np.float64
    s = 2 * rng.normal(size=shape)
    if style == "ties":
        s = np.round(s)
    elif style == "masked":
        u = rng.random(shape)
        s = np.where(u < 0.4, -np.inf, np.where(u < 0.5, np.nan, np.where(u > 0.97, np.inf, s)))
        s[:, :, ::3] = -np.inf                                   # positions with nothing to go to
    elif style == "far":
        s = s * 200 - 1000                                        # exponentials of these do not fit
    prior, bias = rng.normal(size=shape[1]), 0.5 * rng.normal(size=shape[1])
    if style == "ties":
        prior, bias = np.round(prior), np.round(bias)
    if style == "masked":
        prior[0], bias[-1] = -np.inf, -np.inf
    return [a.astype(dt) for a in (s, prior, bias)]


SHAPES = [((1, 1, 1), 1, 1, 1), ((2, 5, 7, 3), 2, 1, 1), ((3, 64, 11, 13), 4, 1, 1), ((2, 192, 5, 5), 6, 8, 3), ((1, 130, 300), 16, 1, 1), ((4, 12, 33), 3, 4, 2), ((2, 33, 40), 1, 1, 1),
          ((1, 300, 9), 8, 1, 1), ((2, 128, 17), 5, 64, 16), ((1, 4096, 5), 3, 1, 1), ((5, 16, 1), 16, 1, 1), ((2, 256, 129), 7, 2, 1)]


def _units(kind, n):
    """Half-units of a weight: exponentials of differences of up to A nats (two units and A for the argument each), a sum of n, a quotient."""
    return n * np.finfo(np.float32 if kind == torch.float32 else np.float64).eps


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("style", ["plain", "ties", "masked", "far"])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("shape,top,groups,top_groups", SHAPES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_choice_weights_loads_and_gradient(shape, top, groups, top_groups, sigmoid, style, kind):
    s, prior, bias = _inputs(shape, kind, style)
    for p, b, scale in ((None, None, 1.0), (prior, bias, 2.5)):
        kw = dict(top_k=top, groups=groups, top_groups=top_groups, sigmoid=sigmoid)
        index, weights, load, dense, mass, logit = plain.route(s, prior=p, bias=b, scale=scale, **kw)
        x = _dev(s).requires_grad_()
        i, w, n = route(x, prior=_dev(p), bias=_dev(b), scale=scale, **kw)
        assert i.dtype == torch.int32 and n.dtype == torch.int64 and w.dtype == kind and tuple(i.shape) == tuple(w.shape) == index.shape
        assert np.array_equal(i.cpu().numpy(), index) and np.array_equal(n.cpu().numpy(), load)
        # differences of the chosen scores of up to A nats
        fine = np.isfinite(logit)
        a = 2 * np.abs(logit[fine]).max() if fine.any() else 0.0
        tol = _units(kind, 8 + top + 2 * min(a, 100.0))
        got = w.detach().cpu().numpy().astype(np.float64)
        assert (np.abs(got - weights) <= tol * np.abs(weights) + np.finfo(got.dtype).tiny + np.exp(-85.0 if kind == torch.float32 else -700.0)).all()
        g = np.random.default_rng(1).normal(size=weights.shape).astype(s.dtype)
        ds = torch.autograd.grad(w, x, _dev(g))[0].cpu().numpy()
        ref = plain.route_gradient(index, weights, g, logit, sigmoid, scale)
        # a difference of the gradient and its mean: relative to the larger of the two
        assert (np.abs(ds - ref) <= 4 * tol * np.abs(weights).max() * np.abs(g).max()).all() and np.array_equal(ds == 0, np.abs(ds) == 0)
        r, m, n = responsibilities(_dev(s), prior=_dev(p), bias=_dev(b), **kw)
        assert np.array_equal(n.cpu().numpy(), load)
        if scale == 1.0:                    # (64 bits: adding up in 32 bits with atomics flushes what is below the normal numbers)
            flat = torch.zeros_like(r, dtype=torch.float64).scatter_add_(1, i.long().clamp(min=0), torch.where(i >= 0, w.detach().double(), 0.0))
            assert bool((r.double() == flat).all())
        want = r.double().sum(dim=[0] + list(range(2, r.dim()))).cpu().numpy()
        # a mass is a sum of positive weights, 256 and the samples of a split one after the other at most
        assert (np.abs(m.cpu().numpy() - want) <= _units(kind, 300) * want + 1e-300).all()
        assert (np.abs(want - mass / scale) <= _units(kind, 8 + top + 2 * min(a, 100.0)) * mass / scale + 1e-30).all()


@pytest.mark.parametrize("shape,top", [((2, 64, 37), 4), ((1, 13, 300), 2), ((1, 256, 129), 7), ((1, 257, 40), 5), ((3, 40, 41), 16), ((700, 24, 110), 3)])
@pytest.mark.parametrize("style", ["neighbours", "below_zero", "zeros", "subnormal", "infinite", "few"])
def test_choices_between_values_that_are_nearly_equal(shape, top, style):
    """Values a few units in the last place apart, zeros of both signs, numbers below the normal ones, positions of which little is left."""
    rng = np.random.default_rng(9)
    near = np.array(1.75, np.float32).view(np.int32) + rng.integers(0, 90, shape)
    s = near.astype(np.int32).view(np.float32)
    if style == "below_zero":
        s = -s
    elif style == "zeros":
        s = np.where(rng.random(shape) < 0.5, np.float32(0.0), np.float32(-0.0)) * rng.choice(np.array([1.0, 0.0], np.float32), shape)
        s[rng.random(shape) < 0.02] = 1e-30
    elif style == "subnormal":
        s = (rng.integers(0, 300, shape) * rng.choice([-1, 1], shape)).astype(np.float32) * np.float32(1e-45)
    elif style == "infinite":
        s = np.where(rng.random(shape) < 0.1, np.float32(np.inf), s)
        s[:, :, ::2] = np.finfo(np.float32).max * rng.choice(np.array([-1.0, 1.0], np.float32), s[:, :, ::2].shape)
    elif style == "few":
        s = np.where(rng.random(shape) < 2.0 / shape[1], s, -np.float32(np.inf))
        s[:, 0, 1::5] = -np.finfo(np.float32).max
    s = s.astype(np.float32)
    for bias in (None, np.where(rng.random(shape[1]) < 0.5, np.float32(0), np.float32(2.0 ** -22))):
        if shape[0] > 100 and bias is not None:
            continue
        n = 3 if shape[0] > 100 else shape[0]               # (many samples: a lane has a whole position; the first ones tell)
        index, weights, load, dense, _, _ = plain.route(s[:n], top, bias=bias)
        i, w, _ = route(_dev(s), top_k=top, bias=_dev(bias))
        assert np.array_equal(i[:n].cpu().numpy(), index)
        r, _, count = responsibilities(_dev(s), top_k=top, bias=_dev(bias))
        assert np.array_equal((r[:n] > 0).cpu().numpy(), dense > 0)
        assert np.abs(w[:n].cpu().numpy() - weights).max() <= _units(torch.float32, 8 + top)      # (exponentials of differences near 0, or of infinities)
        if n == shape[0]:
            assert np.array_equal(count.cpu().numpy(), load)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_the_gradient_is_that_of_differences(sigmoid):
    torch.manual_seed(0)
    s = torch.randn(2, 9, 4, device="cuda", dtype=torch.float64, requires_grad=True)
    prior = torch.randn(9, device="cuda", dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda v: route(v, top_k=4, prior=prior, bias=-prior, sigmoid=sigmoid, scale=1.7)[1], (s,), eps=1e-6, atol=1e-7)


def test_strides_streams_graphs_and_empty_batches():
    torch.manual_seed(1)
    base = torch.randn(3, 8, 10, 48, device="cuda")
    view = base.permute(0, 3, 1, 2)
    a, b = route(view, top_k=5), route(view.contiguous(), top_k=5)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    for shape in ((0, 7, 4, 4), (3, 7, 0, 4)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        i, w, n = route(x, top_k=2)
        assert w.shape[1] == 2 and w.numel() == 0 and n.tolist() == [0] * 7
        assert torch.autograd.grad(w.sum(), x)[0].shape == shape
        r, m, n = responsibilities(x.detach(), top_k=2)
        assert r.shape == shape and m.tolist() == [0.0] * 7
    s = view.contiguous()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        responsibilities(s, top_k=5)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g):
        outs = responsibilities(s, top_k=5) + route(s, top_k=3, sigmoid=True)
    for scale in (1.0, -0.5):
        s.copy_(view * scale)
        want = [t.clone() for t in responsibilities(s, top_k=5) + route(s, top_k=3, sigmoid=True)]
        g.replay()
        assert all(torch.equal(u, v) for u, v in zip(outs, want))


def test_the_choice_is_no_input_of_the_gradient():
    x = torch.randn(2, 6, 5, device="cuda", requires_grad=True)
    i, w, n = route(x, top_k=2)
    assert w.requires_grad and not i.requires_grad and not n.requires_grad
    assert not any(t.requires_grad for t in responsibilities(x, top_k=2))
    with torch.no_grad():
        assert not route(x, top_k=2)[1].requires_grad
    with pytest.raises(RuntimeError, match="same device|CUDA"):
        route(x, top_k=2, bias=torch.zeros(6))
    with pytest.raises(TypeError):
        route(x, top_k=2, bias=torch.zeros(6, device="cuda", dtype=torch.float64))


def test_what_stays_for_the_gradient():
    """Index and weights; the scores only where the values are sigmoids of them."""
    s = torch.randn(4, 12, 50, device="cuda", dtype=torch.float64)
    g = torch.randn(4, 3, 50, device="cuda", dtype=torch.float64)
    for sigmoid in (False, True):
        x = s.clone().requires_grad_()
        y = x * 1.0
        i, w, _ = route(y, top_k=3, prior=torch.arange(12.0, device="cuda", dtype=torch.float64) / 8, sigmoid=sigmoid)
        want = torch.autograd.grad(w, x, g, retain_graph=True)[0]
        with torch.no_grad():
            y.zero_()
        if sigmoid:
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad(w, x, g)
        else:
            assert torch.equal(torch.autograd.grad(w, x, g)[0], want)


@pytest.mark.parametrize("kind", KINDS)
def test_masses_are_sums_of_scaled_weights(cuda_lib, kind):
    """simnets_route with the dense form and a scale, which `responsibilities` does not take."""
    s = torch.randn(3, 20, 70, device="cuda", dtype=kind)
    for top, groups, top_groups in ((1, 1, 1), (1, 5, 2), (4, 1, 1), (4, 5, 2)):
        d = abi.RouteDesc(dtype=abi.F32 if kind == torch.float32 else abi.F64, batch=3, components=20, top_k=top, groups=groups, top_groups=top_groups, positions=70, scale=2.5)
        dense, mass, load = torch.empty_like(s), torch.empty(20, device="cuda", dtype=kind), torch.empty(20, device="cuda", dtype=torch.int64)
        ws = torch.empty(cuda_lib.simnets_route_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
        assert cuda_lib.simnets_route(C.byref(d), s.data_ptr(), None, None, None, None, dense.data_ptr(), load.data_ptr(), mass.data_ptr(), ws.data_ptr(), ws.numel(),
                                      torch.cuda.current_stream().cuda_stream) == 0
        _, _, want_load, _, want, _ = plain.route(s.cpu().numpy(), top, groups=groups, top_groups=top_groups, scale=2.5)
        assert np.array_equal(load.cpu().numpy(), want_load)
        # (weights as in the test above, scores of up to 12 nats apart; a sum of 210 at most)
        assert (np.abs(mass.cpu().numpy() - want) <= _units(kind, 8 + top + 24 + 210) * want + 1e-30).all()
        assert torch.allclose(dense.sum(dim=(0, 2)), mass, rtol=_units(kind, 420), atol=0)


class Ops(uo.OraclePatchOps):
    def responsibilities(self, scores, top_k, prior=None, bias=None):
        a = [None if v is None else v.numpy() for v in (prior, bias)]
        _, _, load, dense, mass, _ = plain.route(scores.numpy(), top_k, *a)
        return torch.from_numpy(dense).to(scores.dtype), torch.from_numpy(mass).to(scores.dtype), torch.from_numpy(load)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what", ["kmeans", "gmm"])
def test_balanced_estimators_follow_the_restatement(what, kind):
    rng = np.random.default_rng(7)
    batches = [rng.normal(size=(4, 2, 9, 8)) for _ in range(4)]
    make = lambda ops: un.KMeans([3, 3], [1, 1], 7, ops=ops, balance=0.5) if what == "kmeans" else un.DiagonalGMM([3, 3], [1, 1], 7, ops=ops, top_k=3, balance=0.25)
    ours, ref = make(None), make(Ops((3, 3), (1, 1)))
    u, picks = rng.random(7), rng.integers(0, 100, 7)
    for est, dt, where in ((ours, kind, "cuda"), (ref, torch.float64, "cpu")):
        first = torch.from_numpy(batches[0]).to(where, dt)
        est.init(first, **(dict(uniforms=u) if what == "kmeans" else dict(picks=picks)))
        for b in batches:
            est.update(torch.from_numpy(b).to(where, dt))
    a, b = [(e.centres, e.counts) if what == "kmeans" else (e.means, e.covs) for e in (ours, ref)]
    # no choice in these batches is near enough to a tie for float32 to turn it
    for p, q in zip(a, b):
        assert torch.allclose(p.cpu().double(), q, rtol=1e-4 if kind == torch.float32 else 1e-9, atol=1e-5 if kind == torch.float32 else 1e-10)
    assert torch.equal(ours.bias.cpu().double(), ref.bias.double())


def test_initialisation_training_and_checkpoints_together():
    """What the operators are for, in one run: balanced initialisation of the first layer, then a step that keeps bytes."""
    from simnets_tf_b200.simnet import SPECS, SimNet
    rng = np.random.default_rng(8)
    data = rng.random((24, 1, 28, 28)).astype(np.float32) - 0.5
    net = SimNet(SPECS["cfg3"], seed=2, checkpoint=64)
    before = net.stages[0].templates.detach().clone()
    un.perform_unsupervised_init(net, kind="gmm", layers=[net.stages[0]], data=data, batch_size=12, top_k=4, balance=0.1)
    assert not torch.equal(before, net.stages[0].templates)
    x, labels = torch.from_numpy(data[:8]).cuda(), torch.arange(8, device="cuda") % 10
    net.loss(x, labels).backward()
    assert all(torch.isfinite(p.grad).all() and float(p.grad.abs().max()) > 0 for p in net.parameters())
    assert isinstance(net.stages[1], keras.Mex) and net.stages[1].checkpoint == 64
