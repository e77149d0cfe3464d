"""Routing without a GPU: what its entry points refuse, the estimators that balance their components on stand-in statistics."""
import ctypes as C
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import plain_operators as plain
from oracle import unsupervised_oracle as uo
from simnets_tf_b200 import abi
from simnets_tf_b200 import unsupervised as un
from simnets_tf_b200.ops.routing import responsibilities, route


@pytest.mark.parametrize("call", [route, responsibilities])
def test_arguments_are_checked(call):
    s = torch.zeros(2, 12, 3, 3)
    for kw in (dict(top_k=0), dict(top_k=13), dict(top_k=1.5), dict(top_k=True), dict(groups=5), dict(groups=0), dict(groups=4, top_groups=5), dict(groups=4, top_groups=1, top_k=4),
               dict(groups=4, top_groups=0)):
        with pytest.raises(ValueError):
            call(s, **kw)
    for kw in (dict(prior=torch.zeros(11)), dict(bias=torch.zeros(12, 1)), dict(bias=torch.zeros(12, requires_grad=True))):
        with pytest.raises(ValueError, match="prior|bias"):
            call(s, **kw)
    for bad in (torch.zeros(4), torch.zeros(2, 0, 3)):
        with pytest.raises(ValueError, match="axis 1"):
            call(bad)
    with pytest.raises(ValueError, match="at most 4096"):
        call(torch.zeros(1, 4097, 1))
    with pytest.raises(ValueError, match="top_k = 16"):
        call(torch.zeros(1, 40, 1), top_k=17)
    with pytest.raises(ValueError, match="16 of 64"):
        call(torch.zeros(1, 130, 1), groups=65, top_groups=3)
    with pytest.raises(TypeError, match="float32 and float64"):
        call(s.half())
    with pytest.raises(RuntimeError, match="no CPU kernels"):
        call(s, top_k=2)


def test_the_c_entry_points_check_before_they_launch(cuda_lib):
    one = C.c_void_p(256)                   # (never dereferenced: every call below is refused)

    def call(ws=one, n=None, load=one, scores=one, mass=None, dense=None, **kw):
        d = abi.RouteDesc(**dict(dict(dtype=abi.F32, batch=2, components=12, top_k=2, groups=1, top_groups=1, positions=9, scale=1.0), **kw))
        need = cuda_lib.simnets_route_workspace_bytes(C.byref(d))
        rc = cuda_lib.simnets_route(C.byref(d), scores, None, None, one, one, dense, load, mass, ws, need if n is None else n, None)
        assert cuda_lib.simnets_route_gradient(C.byref(d), one, None, None, one, one, one, None) == (rc if need == 0 else abi.E_NULL)
        return rc
    assert C.sizeof(abi.RouteDesc) == 48
    assert call(dtype=3) == abi.E_DTYPE
    for kw in (dict(batch=-1), dict(positions=-1), dict(components=0), dict(top_k=0), dict(top_k=13), dict(groups=5), dict(top_groups=2), dict(reserved=1), dict(scale=0.0),
               dict(scale=float("inf")), dict(groups=4, top_groups=1, top_k=4)):
        assert call(**kw) == abi.E_DESC, kw
    for kw in (dict(components=4097), dict(components=40, top_k=17), dict(components=130, groups=65, top_groups=3), dict(components=170, groups=34, top_groups=17),
               dict(batch=1 << 20, positions=1 << 40)):
        assert call(**kw) == abi.E_UNSUPPORTED, kw
    assert call(load=None) == abi.E_NULL and call(scores=None) == abi.E_NULL and call(mass=one) == abi.E_NULL
    assert call(ws=None) == abi.E_WORKSPACE and call(n=8) == abi.E_WORKSPACE


def test_the_restatement_routes_by_value_and_index():
    s = np.zeros((1, 4, 2), np.float32)
    s[0, :, 1] = [np.nan, 1.0, -np.inf, 1.0]
    index, weights, load, dense, mass, _ = plain.route(s, 3)
    assert index[0, :, 0].tolist() == [0, 1, 2] and index[0, :, 1].tolist() == [1, 3, -1]
    assert np.allclose(weights[0, :, 0], 1 / 3) and weights[0, :, 1].tolist() == [0.5, 0.5, 0.0]
    assert load.tolist() == [1, 2, 1, 1] and np.allclose(mass, dense.sum((0, 2)))


class Ops(uo.OraclePatchOps):
    def responsibilities(self, scores, top_k, prior=None, bias=None):
        a = [None if v is None else v.numpy() for v in (prior, bias)]
        _, _, load, dense, mass, _ = plain.route(scores.numpy(), top_k, *a)
        return torch.from_numpy(dense).to(scores.dtype), torch.from_numpy(mass).to(scores.dtype), torch.from_numpy(load)


def test_a_mixture_cut_to_all_its_components_is_the_mixture():
    rng = np.random.default_rng(3)
    batches = [torch.from_numpy(rng.normal(size=(3, 2, 6, 7))) for _ in range(3)]
    picks = rng.integers(0, 60, 5)
    full, cut, two = (un.DiagonalGMM([3, 3], [1, 1], 5, ops=Ops((3, 3), (1, 1)), top_k=k) for k in (None, 5, 2))
    for est in (full, cut, two):
        est.init(batches[0], picks=picks)
        for b in batches:
            est.update(b)
    assert torch.allclose(full.means, cut.means, rtol=1e-10, atol=1e-12) and torch.allclose(full.covs, cut.covs, rtol=1e-9, atol=1e-12)
    assert not torch.allclose(full.means, two.means, rtol=1e-3)


@pytest.mark.parametrize("kind", ["kmeans", "gmm"])
def test_balance_brings_idle_components_into_use(kind):
    """Two components far from all data: without balance they stay where they are.  A patch is at about 4 x 12^2 = 576 from them (half of
    that in the mixture, whose variances are near one), and the biases of an idle and of a busy component part by at most
    2 x balance a step: 720 after 60."""
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.normal(size=(6, 1, 8, 8)))
    load = {}
    for balance in (0.0, 6.0):
        ops = Ops((2, 2), (2, 2))
        est = un.KMeans([2, 2], [2, 2], 6, ops=ops, balance=balance) if kind == "kmeans" else un.DiagonalGMM([2, 2], [2, 2], 6, ops=ops, top_k=1, balance=balance)
        est.init(x)
        centres = est.centres if kind == "kmeans" else est.means
        centres[4:] = 12.0
        for _ in range(60):
            est.update(x)
        centres = est.centres if kind == "kmeans" else est.means
        load[balance] = bool((centres[4:] < 11).any())
    assert load == {0.0: False, 6.0: True}


def _worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        rng = np.random.default_rng(4)
        first, batches = rng.normal(size=(4, 2, 5, 5)), [rng.normal(size=(4, 2, 5, 5)) for _ in range(3)]
        u, picks, res = rng.random(3), rng.integers(0, 36, 3), []
        for group, lo, hi in ((dist.group.WORLD, 2 * rank, 2 * rank + 2), (None, 0, 4)):
            km = un.KMeans((3, 3), (1, 1), 3, ops=Ops((3, 3), (1, 1)), group=group, balance=0.75)
            gm = un.DiagonalGMM((3, 3), (1, 1), 3, ops=Ops((3, 3), (1, 1)), group=group, top_k=2, balance=0.25)
            km.init(torch.from_numpy(first), uniforms=u)
            gm.init(torch.from_numpy(first), picks=picks)
            for b in batches:
                km.update(torch.from_numpy(b[lo:hi]))
                gm.update(torch.from_numpy(b[lo:hi]))
            res.append(torch.cat([km.centres.flatten(), km.counts, km.bias, gm.means.flatten(), gm.covs.flatten(), gm.bias]))
        if rank == 0:
            np.save(out, np.array([float((res[0] - res[1]).abs().max()), float(res[1].abs().max())]))
    finally:
        dist.destroy_process_group()


def test_balance_over_two_ranks_equals_the_unsharded_step(tmp_path):
    """Biases follow the loads of all ranks."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = str(tmp_path / "r.npy")
    mp.spawn(_worker, args=(2, port, out), nprocs=2, join=True)
    err, scale = np.load(out)
    assert scale > 0 and err < 1e-12 * max(scale, 1.0)


def test_estimators_check_their_new_arguments():
    class L(object):
        blocks, strides, num_instances = [3, 3], [1, 1], 4
    for kw in (dict(top_k=0), dict(top_k=5), dict(top_k=1.5), dict(top_k=True), dict(balance=1.0), dict(top_k=2, balance=-1.0), dict(top_k=2, balance=float("nan"))):
        with pytest.raises(ValueError):
            un.similarity_unsupervised_init("gmm", L(), **kw)
    for kw in (dict(top_k=1), dict(balance=-0.5), dict(balance=float("inf"))):
        with pytest.raises(ValueError):
            un.similarity_unsupervised_init("kmeans", L(), **kw)
    est = un.similarity_unsupervised_init("gmm", L(), top_k=2, balance=0.5)
    assert est.top_k == 2 and est.balance == 0.5 and est.bias is None


@pytest.mark.parametrize("top_k", [2, 2.0, np.int64(2), np.float32(2)])
def test_whole_numbers_of_any_type_are_taken_for_top_k(top_k):
    """What the constructor takes every update takes: `responsibilities` wants an int."""
    class Strict(Ops):
        def responsibilities(self, scores, top_k, prior=None, bias=None):
            assert type(top_k) is int
            return super(Strict, self).responsibilities(scores, top_k, prior, bias)
    x = torch.from_numpy(np.random.default_rng(6).normal(size=(3, 2, 5, 5)))
    est = un.DiagonalGMM([3, 3], [1, 1], 4, ops=Strict((3, 3), (1, 1)), top_k=top_k)
    est.init(x)
    est.update(x)
    assert est.top_k == 2


@pytest.mark.parametrize("dtype,scale,ok", [(abi.F32, 1e-50, False), (abi.F32, 1e-40, False), (abi.F32, -1e39, False), (abi.F32, 1.2e-38, True), (abi.F32, -3e38, True),
                                            (abi.F64, 1e-50, True), (abi.F64, 1e-310, False), (abi.F64, 1e300, True)])
def test_scales_must_be_numbers_of_the_weights_type(cuda_lib, dtype, scale, ok):
    """A scale that rounds to 0 or infinity in float32, or whose reciprocal (which the gradient takes) does, would give weights of 0 and
    gradients of 0 x infinity."""
    one = C.c_void_p(256)                   # (never dereferenced: every call below is refused)
    d = abi.RouteDesc(dtype=dtype, batch=2, components=12, top_k=2, groups=1, top_groups=1, positions=9, scale=scale)
    assert (cuda_lib.simnets_route_workspace_bytes(C.byref(d)) > 0) == ok
    rc = abi.E_NULL if ok else abi.E_DESC
    assert cuda_lib.simnets_route(C.byref(d), None, None, None, one, one, None, one, None, one, 1 << 30, None) == rc
    assert cuda_lib.simnets_route_gradient(C.byref(d), one, None, None, one, one, one, None) == rc


def test_estimators_stored_before_there_was_a_balance_go_on():
    """An estimator pickled by an earlier version has neither `balance` nor `bias` nor `top_k`."""
    x = torch.from_numpy(np.random.default_rng(6).normal(size=(3, 2, 5, 5)))
    for make in (lambda: un.KMeans([3, 3], [1, 1], 4, ops=Ops((3, 3), (1, 1))), lambda: un.DiagonalGMM([3, 3], [1, 1], 4, ops=Ops((3, 3), (1, 1)))):
        new, old = make(), make()
        new.init(x)
        old.init(x)
        for name in ("balance", "bias", "top_k"):
            old.__dict__.pop(name, None)
        for a, b in zip(new.update(x), old.update(x)):
            assert torch.equal(a, b)


def test_responsibilities_refuse_to_be_recorded():
    """torch.jit.trace would keep their result as a constant."""
    class Cut(torch.nn.Module):
        def forward(self, s):
            return responsibilities(s, top_k=2)[0]
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        torch.jit.trace(Cut(), (torch.zeros(2, 4, 3),), check_trace=False)


@pytest.mark.parametrize("kw", [dict(), dict(groups=4, top_groups=2), dict(sigmoid=True, scale=2.5)])
def test_the_two_restatements_agree(kw):
    rng = np.random.default_rng(2)
    s = np.round(2 * rng.normal(size=(3, 12, 40)))
    u = rng.random(s.shape)
    s = np.where(u < 0.4, -np.inf, np.where(u < 0.5, np.nan, np.where(u > 0.97, np.inf, s)))
    s[:, :, ::7] = -np.inf
    prior, bias = np.round(rng.normal(size=12)), np.round(rng.normal(size=12))
    for p, b in ((None, None), (prior, bias)):
        index, weights, load, _, _, _ = plain.route(s, 3, p, b, **kw)
        i, w, n, _ = plain.route_sorted(torch.from_numpy(s), 3, None if p is None else torch.from_numpy(p), None if b is None else torch.from_numpy(b), **kw)
        assert np.array_equal(i.numpy(), index) and np.array_equal(n.numpy(), load) and np.allclose(w.numpy(), weights, rtol=1e-12, atol=0)
