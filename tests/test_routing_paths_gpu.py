"""Routing where every position has a lane of its own and a CTA several tiles of them (short lists and long ones, groups, many components, float64),
positions beyond 31 bits, and gradients that are exactly 0 where nothing was chosen."""
import numpy as np
import pytest
import torch

import plain_operators as plain
from simnets_tf_b200.ops.routing import responsibilities, route
from test_routing_gpu import KINDS, _dev, _inputs, _units

pytestmark = pytest.mark.gpu

# (shape, top, groups, top_groups).  A lane a position from 512 positions a multiprocessor or 128 a component on (64 with groups); 12 CTAs of 128 threads
# a multiprocessor at most, fewer by registers.
MANY = [((2000, 24, 130), 3, 4, 2), ((2000, 48, 130), 8, 1, 1), ((2000, 40, 130), 16, 1, 1), ((2000, 33, 130), 6, 11, 5), ((2000, 48, 130), 7, 4, 2), ((1000, 300, 130), 5, 1, 1),
        ((1000, 200, 130), 2, 1, 1), ((2000, 64, 130), 1, 1, 1), ((1000, 96, 130), 12, 32, 16), ((1000, 100, 130), 4, 1, 1), ((1000, 5, 1031), 5, 1, 1), ((2000, 20, 130), 1, 5, 3)]
# the same with the lanes of a warp shared, in several tiles a CTA
SHARED = [((250, 300, 130), 1, 1, 1), ((200, 300, 130), 9, 1, 1), ((150, 1024, 130), 4, 1, 1), ((250, 512, 130), 5, 8, 3), ((140, 256, 130), 4, 1, 1)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("style", ["plain", "ties", "masked"])
@pytest.mark.parametrize("shape,top,groups,top_groups", MANY + SHARED, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_many_positions(shape, top, groups, top_groups, style, kind):
    s, prior, bias = [_dev(a) for a in _inputs(shape, kind, style)]
    for p, b, sigmoid, scale in ((None, None, False, 1.0), (prior, bias, True, 2.5)):
        kw = dict(top_k=top, groups=groups, top_groups=top_groups, sigmoid=sigmoid, prior=p, bias=b)
        index, weights, load, chosen = plain.route_sorted(s, scale=scale, **kw)
        x = s.clone().requires_grad_()
        i, w, n = route(x, scale=scale, **kw)
        assert torch.equal(i.long(), index) and torch.equal(n, load)
        on = index >= 0
        # differences of the chosen scores of up to A nats, as in test_routing_gpu.py
        fine = chosen[on & chosen.isfinite()]
        a = 2 * float(fine.abs().max()) if fine.numel() else 0.0
        tol = float(_units(kind, 8 + top + 2 * min(a, 100.0)))
        assert bool(((w.detach().double() - weights).abs() <= tol * weights + 1e-35).all())
        # the gradient: exactly 0 for what was not chosen; else a difference of two numbers of the position's gradients
        g = torch.randn(w.shape, device="cuda", dtype=kind, generator=torch.Generator("cuda").manual_seed(3))
        ds = torch.autograd.grad(w, x, g)[0]
        ref = weights * (g.double() - (weights * torch.where(on, g.double(), 0.0)).sum(1, keepdim=True) / scale)
        if sigmoid:
            ref = ref / (1.0 + chosen.exp())
        got = torch.where(on, ds.gather(1, index.clamp(min=0)), 0.0).double()
        assert bool(((got - torch.where(on, ref, 0.0)).abs() <= 4 * tol * weights * g.double().abs().amax(1, keepdim=True) + 1e-35).all())
        put = torch.zeros_like(s, dtype=torch.bool).scatter_(1, torch.where(on, index, index[:, :1].clamp(min=0)), on[:, :1] | on)
        assert bool((ds[~put] == 0).all())
        del ds, got, ref
        r, m, n = responsibilities(s, **kw)
        again = responsibilities(s, **kw)
        assert torch.equal(r, again[0]) and torch.equal(m, again[1])                # (masses are added up in a fixed order)
        assert torch.equal(n, load) and bool((r[~put] == 0).all())
        if scale == 1.0:
            assert torch.equal(torch.where(on, r.gather(1, index.clamp(min=0)), 0.0), w.detach())
        # positive numbers, at most 300 one after the other and then in pairs
        want = r.double().sum(dim=(0, 2))
        assert bool(((m.double() - want).abs() <= float(_units(kind, 320)) * want).all())


def test_gradients_of_what_was_not_chosen_are_zero():
    """Few positions, whose lanes are shared between components, and stale memory under the result."""
    for shape, kw in (((3, 64, 11, 13), dict(top_k=4)), ((2, 192, 5, 5), dict(top_k=6, groups=8, top_groups=3)), ((1, 4096, 5), dict(top_k=3)), ((2, 33, 40), dict(top_k=1))):
        torch.full(shape, float("nan"), device="cuda")                              # (freed at once: the allocator hands it to the gradient)
        x = torch.randn(shape, device="cuda", requires_grad=True)
        i, w, _ = route(x, sigmoid=True, **kw)
        ds = torch.autograd.grad(w, x, torch.randn_like(w))[0]
        mask = torch.zeros(shape, dtype=torch.bool, device="cuda").scatter_(1, i.long(), True)
        assert bool((ds[~mask] == 0).all())
        assert bool((ds[mask] != 0).any()) or kw["top_k"] == 1


def test_positions_beyond_31_bits():
    batch, n = (1 << 31) // 3 + 26, 3
    assert batch * n > 1 << 31
    step = 1 << 24
    gen = torch.Generator("cuda").manual_seed(4)
    x = torch.empty(batch, 2, n, device="cuda")
    for b in range(0, batch, step):
        x[b:b + step].normal_(generator=gen)
    x.requires_grad_()
    i, w, load = route(x, top_k=2)
    g = torch.empty_like(w)
    g[:, 0], g[:, 1] = 1.0, -0.5
    ds = torch.autograd.grad(w, x, g)[0]
    del g
    r, m, count = responsibilities(x.detach(), top_k=1)
    total, first = torch.zeros(2, dtype=torch.long, device="cuda"), torch.zeros(2, dtype=torch.long, device="cuda")
    for b in range(0, batch, step):
        index, weights, n_chosen, _ = plain.route_sorted(x[b:b + step].detach(), 2)
        total += n_chosen
        first += torch.bincount(index[:, 0].reshape(-1), minlength=2)
        assert torch.equal(i[b:b + step].long(), index)
        # scores of up to 12 nats apart: see _units
        tol = float(_units(torch.float32, 8 + 2 + 24))
        assert bool(((w[b:b + step].detach().double() - weights).abs() <= tol * weights).all())
        ref = weights[:, :1] * weights[:, 1:] * 1.5
        got = ds[b:b + step].gather(1, index).double()
        assert bool((torch.cat([got[:, :1] - ref, got[:, 1:] + ref], 1).abs() <= 4 * tol * weights).all())
        assert torch.equal(r[b:b + step], torch.zeros_like(r[b:b + step]).scatter_(1, index[:, :1], 1.0))
    assert torch.equal(load, total) and torch.equal(count, first)
    assert bool((m.double() - first.double()).abs().max() <= 2.0 ** -24 * float(first.max()))            # (one rounding)
