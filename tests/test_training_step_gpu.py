"""A training step as a whole on the GPU: network, log probabilities and entropies, gradients in a bucket, their norm and clipping; eager, captured, and in the
data-parallel step."""
import numpy as np
import pytest
import torch

import cases
import plain_training as plain
from simnets_tf_b200 import dp
from simnets_tf_b200.netspec import SPECS
from simnets_tf_b200.ops.likelihood import log_probabilities
from simnets_tf_b200.simnet import SimNet

pytestmark = pytest.mark.gpu


def data(spec, n, dtype=torch.float32, seed=3):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.uniform(-0.5, 0.5, size=(n,) + tuple(spec["input_shape"]))).to("cuda", dtype)
    return x, torch.from_numpy(rng.integers(0, spec["classes"], size=n)).cuda()


def loss_of(got):
    return -(got.label.mean() + 0.05 * got.entropy.mean())


@pytest.mark.parametrize("name", ["cfg3", "cfg5"])
def test_gradients_of_a_network(name):
    """float64, as in test_simnet_gpu.py: the offsets' gradients cancel, which makes 1e-16 up to 1e-7 of them."""
    spec = SPECS[name]
    x, labels = data(spec, 5, torch.float64)
    net = SimNet(spec, seed=5, device="cuda", dtype=torch.float64)
    bucket = dp.GradBucket(net.parameters())
    bucket.zero()
    loss = loss_of(net.log_probabilities(x, labels, entropy=True))
    loss.backward()
    got, got_loss = [p.grad.clone() for p in net.parameters()], float(loss.detach())
    bucket.zero()
    l = torch.log_softmax(net(x), 1)
    want = -(l.gather(1, labels[:, None]).mean() - 0.05 * (l.exp() * l).sum(1).mean())
    want.backward()
    # (a mean of five, each of a handful of roundings)
    assert abs(got_loss - float(want.detach())) <= 64 * np.finfo(np.float64).eps * abs(got_loss)
    for i, (a, p) in enumerate(zip(got, net.parameters())):
        cases.assert_parity(a.cpu().numpy(), p.grad.cpu().numpy(), tol=1e-7, what="%s gradient %d" % (name, i))


def check_clipped(flat, norm, before, limit):
    """norm and flat as the restatement has them for the gradients before: the norm a step of its type off, products rounded once and by the norm's step."""
    eps = np.finfo(before.dtype).eps
    want_norm, (want,) = plain.clipped([before], limit)
    assert abs(float(norm) - float(want_norm)) <= eps * float(want_norm)
    assert (abs(flat.astype(np.longdouble) - want) <= 2 * eps * abs(want.astype(np.longdouble)) + np.finfo(before.dtype).smallest_subnormal).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_a_step_with_clipping(dtype):
    spec = SPECS["cfg3"]
    x, labels = data(spec, 8, dtype)
    net = SimNet(spec, seed=5, device="cuda", dtype=dtype)
    bucket = dp.GradBucket(net.parameters())
    bucket.zero()
    loss_of(net.log_probabilities(x, labels, entropy=True)).backward()
    before = bucket.flat.cpu().numpy()
    limit = 0.25 * float(plain.norm([before]))
    norm = bucket.clip(limit)
    check_clipped(bucket.flat.cpu().numpy(), norm, before, limit)
    old = [p.detach().clone() for p in net.parameters()]
    with torch.no_grad():
        for p in net.parameters():
            p -= 0.5 * p.grad
    assert all(bool((p == o - 0.5 * p.grad).all()) for p, o in zip(net.parameters(), old))


@pytest.mark.parametrize("limit", [1e-3, 1e-5])
def test_a_captured_step(limit):
    """Forward pass, answers, backward pass and clipping as one CUDA graph: what it leaves is within the limit, and is what the same step left without a
    graph.  (The norm is about 3e-5: the one limit is not reached.)"""
    spec = SPECS["cfg3"]
    x, labels = data(spec, 8)
    net = SimNet(spec, seed=5, device="cuda")
    bucket = dp.GradBucket(net.parameters())

    def step():
        bucket.zero()
        got = net.log_probabilities(x, labels, top_k=2, entropy=True)
        loss_of(got).backward()
        return got.top_index, bucket.clip(limit)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            index, norm = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    eager, eager_norm, eager_index = bucket.flat.clone(), float(norm), index.clone()
    del index, norm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        index, norm = step()
    for _ in range(2):
        bucket.flat.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert bool((index == eager_index).all())
        # (the two differ, if at all, by the order in which sums over the batch are taken: as in test_dp_nccl_gpu.py)
        assert float((bucket.flat - eager).abs().max()) <= 1e-6 * float(eager.abs().max()) and abs(float(norm) - eager_norm) <= 1e-5 * eager_norm
        # the norm of products that were each rounded, by a norm that was
        left = min(limit, float(norm))
        assert abs(float(plain.norm([bucket.flat.cpu().numpy()])) - left) <= 2 * np.finfo(np.float32).eps * left


@pytest.mark.parametrize("graphs", [False, True])
def test_the_data_parallel_step_clips(graphs):
    spec = SPECS["cfg5"]
    x, labels = data(spec, 8)
    net = SimNet(spec, seed=4, device="cuda")
    bucket = dp.GradBucket(net.parameters())
    plain_step = dp.OverlappedStep(net, bucket, x, labels, 8, graphs=False)
    plain_step.run()
    torch.cuda.synchronize()
    whole = float(bucket.norm())
    assert plain_step.norm is None
    del plain_step                          # (with its autograd graph)
    step = dp.OverlappedStep(net, bucket, x, labels, 8, graphs=graphs, max_norm=0.5 * whole)
    for _ in range(2):
        step.run()
        torch.cuda.synchronize()
        # (two backward passes: as far from one another as the data-parallel tests have them)
        assert abs(float(step.norm) - whole) <= 1e-5 * whole
        assert abs(float(plain.norm([bucket.flat.cpu().numpy()])) - 0.5 * whole) <= 2 * np.finfo(np.float32).eps * 0.5 * whole
    step.max_norm = 2.0 * whole
    step.run()
    assert abs(float(bucket.norm()) - whole) <= 1e-5 * whole


def test_a_network_that_answers_at_every_position():
    """Without its last layers a network gives a map: the instances of a MEX layer as classes at every position."""
    spec = dict(SPECS["cfg5"], layers=SPECS["cfg5"]["layers"][:3])
    x, _ = data(spec, 3)
    net = SimNet(spec, seed=4, device="cuda")
    with torch.no_grad():
        logits = net(x)
    assert tuple(logits.shape) == (3, 128, 16, 16)
    labels = torch.from_numpy(np.random.default_rng(1).integers(-1, 128, size=(3, 16, 16))).cuda()
    got = net.log_probabilities(x, labels, top_k=3, entropy=True)
    rows = np.ascontiguousarray(np.moveaxis(logits.cpu().numpy(), 1, -1)).reshape(-1, 128)
    r = plain.Rows(rows, labels.cpu().numpy().reshape(-1), 3, chain=64)
    assert np.array_equal(np.moveaxis(got.top_index.cpu().numpy(), 1, -1).reshape(-1, 3), r.top_index)
    for v, (want, off) in ((got.label, r.label()), (got.entropy, (r.entropy, r.off_entropy))):
        assert (abs(v.detach().cpu().numpy().reshape(-1) - want) <= off).all()
    g = torch.autograd.grad(loss_of(got) - got.top.mean(), list(net.parameters()))
    assert all(bool(v.isfinite().all()) for v in g)
    # and answers of rows in another order of memory: a layer with its channels last
    last = log_probabilities(logits.permute(0, 2, 3, 1).contiguous(), labels, 3, True, axis=-1)
    assert np.array_equal(last.top_index.cpu().numpy().reshape(-1, 3), r.top_index)


def test_two_calls_at_once():
    """On two streams, each with what it needs in memory of its own."""
    x = [torch.randn(64, 20000, device="cuda") for _ in range(2)]
    grads = [torch.randn(3000000, device="cuda") for _ in range(2)]
    want = [(log_probabilities(v, top_k=3, entropy=True), None) for v in x]
    norms = [float(g.double().norm()) for g in grads]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [[], []]
    buckets = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.numel(), device="cuda"))
        b = dp.GradBucket([p])
        b.flat.copy_(g)
        buckets.append(b)
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i].append((log_probabilities(x[i], top_k=3, entropy=True), buckets[i].norm()))
    torch.cuda.synchronize()
    for i in range(2):
        for got, norm in out[i]:
            assert all(u is v is None or bool((u == v).all()) for u, v in zip(got, want[i][0]))
            assert abs(float(norm) - norms[i]) <= 2 * np.finfo(np.float32).eps * norms[i]
