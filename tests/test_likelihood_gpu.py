"""Log probabilities, entropies and alternatives on the GPU against the restatement in plain_training.py: choices exactly, the rest within bounds
counted from the formulas."""
import ctypes as C

import numpy as np
import pytest
import torch

import plain_training as plain
from simnets_tf_b200 import _lib, abi
from simnets_tf_b200.ops.likelihood import log_probabilities

pytestmark = pytest.mark.gpu
KINDS = [torch.float32, torch.float64]
NAN, INF = float("nan"), float("inf")


def make(shape, axis, style, kind, seed=0):
    """(logits, labels) as numpy arrays"""
    axis %= len(shape)
    rng = np.random.default_rng(seed)
    dt = np.float32 if kind == torch.float32 else np.float64
    x = 3 * rng.normal(size=shape)
    if style == "ties":
        x = np.round(x / 3)
    elif style == "masked":
        x = np.where(rng.random(shape) < 0.5, -INF, x)
        x = np.where(np.expand_dims(rng.random([s for i, s in enumerate(shape) if i != axis]) < 0.2, axis), -INF, x)      # positions where nothing can be
    elif style == "lowest":
        x = np.where(rng.random(shape) < 0.5, np.finfo(dt).min, x)
        x = np.where(np.expand_dims(rng.random([s for i, s in enumerate(shape) if i != axis]) < 0.2, axis), np.finfo(dt).min, x)
    elif style == "broken":
        u = rng.random(shape)
        one = 0.3 / shape[axis]
        x = np.where(u < one, NAN, np.where(u < 2 * one, INF, np.where(u > 0.8, -INF, x)))
    elif style == "far":
        x = 300 * x - 5000
    elif style == "rising":                # every class is larger than those in front of it: the sums move to a new largest all the time
        k = shape[axis]
        x = 0.01 * x + np.arange(k).reshape([k if i == axis else 1 for i in range(len(shape))]) * (60.0 / k)
    at = rng.integers(-2, shape[axis] + 2, size=[s for i, s in enumerate(shape) if i != axis])
    return x.astype(dt), at.astype(np.int64)


def rows_of(a, axis):
    return np.ascontiguousarray(np.moveaxis(a, axis, -1)).reshape(-1, a.shape[axis])


def near(got, want, off, what):
    """Within the bounds where the reference is a number, equal elsewhere (a NaN for a NaN)."""
    got = got.astype(want.dtype)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what
    share = abs(got[fine] - want[fine]) / np.maximum(off[fine], 1e-300)
    assert bool((share <= 1).all()), "%s: %g of the bound" % (what, share.max())


def chain_of(k):
    """The longest chain of additions of a position's sums: eight at a time, and what a handful of partial sums take to be joined."""
    return k // 8 + 40


def verify(x, labels, axis, top_k, entropy, logits, call=log_probabilities, grads=True, chain=None):
    """Everything that a call returns for `logits`, a tensor of the values of x in any layout."""
    k = x.shape[axis]
    dt = x.dtype
    r = plain.Rows(rows_of(x, axis), None if labels is None else labels.reshape(-1), top_k, chain or chain_of(k))
    leaf = logits.detach().requires_grad_(grads)
    got = call(leaf, labels=None if labels is None else torch.from_numpy(labels).cuda(), top_k=top_k, entropy=entropy, axis=axis)
    others = [s for i, s in enumerate(x.shape) if i != axis % x.ndim]
    assert (got.label is None) == (labels is None) and (got.entropy is None) != entropy and (got.top is None) == (got.top_index is None) == (top_k == 0)
    outs, gs, args = [], [], {}
    rng = np.random.default_rng(9)
    if labels is not None:
        assert got.label.dtype == logits.dtype and list(got.label.shape) == others
        near(got.label.detach().cpu().numpy().reshape(-1), *r.label(), "label")
        args["g_label"] = rng.normal(size=others).astype(dt)
        outs.append(got.label)
    if entropy:
        assert got.entropy.dtype == logits.dtype and list(got.entropy.shape) == others
        near(got.entropy.detach().cpu().numpy().reshape(-1), r.entropy, r.off_entropy, "entropy")
        args["g_entropy"] = rng.normal(size=others).astype(dt)
        outs.append(got.entropy)
    if top_k:
        want = list(x.shape)
        want[axis] = top_k
        assert got.top_index.dtype == torch.int32 and list(got.top.shape) == list(got.top_index.shape) == want and not got.top_index.requires_grad
        assert np.array_equal(rows_of(got.top_index.cpu().numpy(), axis), r.top_index)
        near(rows_of(got.top.detach().cpu().numpy(), axis), *r.top(), "top")
        args["g_top"] = rng.normal(size=want).astype(dt)
        outs.append(got.top)
    if grads and outs:
        dx, = torch.autograd.grad(outs, [leaf], [torch.from_numpy(g).cuda() for g in args.values()])
        assert dx.shape == logits.shape and dx.dtype == logits.dtype
        flat = {n: rows_of(g, axis) if n == "g_top" else g.reshape(-1) for n, g in args.items()}
        near(rows_of(dx.cpu().numpy(), axis), *r.gradient(**flat), "gradient")
    return got


SHAPES = [((1, 1), 1), ((1, 10), 1), ((3, 7), 1), ((65, 33), 1), ((5, 200), 1), ((3, 1000), 1), ((2, 4099), 1), ((2, 5, 3), 1), ((3, 10, 4, 4), 1), ((1, 21, 37, 5), 1), ((2, 130, 33), 1),
          ((9, 64, 1, 1), 1), ((2, 3, 12), 2), ((1, 4, 2, 600), 3), ((3, 1, 50), -1), ((2, 1, 6), 1), ((4, 600, 2), 1)]


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("style", ["plain", "ties", "masked", "lowest", "broken", "far", "rising"])
@pytest.mark.parametrize("shape,axis", SHAPES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_everything_at_once(shape, axis, style, kind):
    x, labels = make(shape, axis, style, kind)
    verify(x, labels, axis, min(5, x.shape[axis]), True, torch.from_numpy(x).cuda())


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("top_k", [0, 1, 2, 4, 8, 9, 16])
@pytest.mark.parametrize("shape,axis", [((6, 16), 1), ((3, 600), 1), ((2, 9000), 1), ((2, 17, 40), 1), ((2, 300, 33), 1)], ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_each_number_of_alternatives_and_output(shape, axis, top_k, kind):
    for style in ("ties", "plain"):
        x, labels = make(shape, axis, style, kind, seed=top_k)
        dev = torch.from_numpy(x).cuda()
        for lab, ent in ((labels, False), (None, True), (None, False)):
            verify(x, lab, axis, top_k, ent, dev)


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("style", ["plain", "ties", "masked", "broken", "rising"])
@pytest.mark.parametrize("rows,classes", [(1, 131072), (1, 1 << 20), (3, 40001), (40, 8193), (300, 2049), (5, 1025), (9, 1024)])
def test_long_rows(rows, classes, style, kind):
    """Up to a million classes; 256 lanes at least share a row from 1025 on, which makes chains of classes / 2048."""
    x, labels = make((rows, classes), 1, style, kind)
    if style == "ties":
        x[0] = 1.0                          # (a head of zeros: every class is as likely)
        x[-1, classes // 2:] = 9.0
    verify(x, labels, 1, 8, True, torch.from_numpy(x).cuda(), chain=classes // 2048 + 64)


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
def test_any_layout(kind):
    """The same values wherever they lie: slices, transposed, channels last, every other value, broadcast, at an odd address."""
    def laid(x, how):
        t = torch.from_numpy(x).cuda()
        if how == "slice":
            big = torch.full([s + 3 for s in t.shape], 7.0, dtype=t.dtype, device="cuda")
            at = tuple(slice(2, 2 + s) for s in t.shape)
            big[at] = t
            return big[at]
        if how == "reversed":
            return t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))
        if how == "last":
            return t.movedim(1, -1).contiguous().movedim(-1, 1)
        if how == "other":
            big = torch.full([2 * s for s in t.shape], 7.0, dtype=t.dtype, device="cuda")
            at = tuple(slice(None, None, 2) for _ in t.shape)
            big[at] = t
            return big[at]
        flat = torch.full([t.numel() + 1], 7.0, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)
    for shape, axis in (((5, 37), 1), ((6, 3000), 1), ((3, 37, 5, 7), 1), ((3, 40, 9), 1), ((3, 11, 300), 2), ((2, 3, 5, 40), 3), ((1, 50, 33), 1)):
        x, labels = make(shape, axis, "plain", kind)
        for how in ("slice", "reversed", "last", "other", "odd"):
            verify(x, labels, axis, 3, True, laid(x, how))
    x, labels = make((1, 40, 6), 1, "plain", kind)
    wide = np.broadcast_to(x, (4, 40, 6))
    verify(np.ascontiguousarray(wide), np.broadcast_to(labels, (4, 6)).copy(), 1, 3, True, torch.from_numpy(x).cuda().expand(4, 40, 6))
    x, labels = make((3, 40, 1), 1, "plain", kind)
    verify(np.ascontiguousarray(np.broadcast_to(x, (3, 40, 5))), np.broadcast_to(labels, (3, 5)).copy(), 1, 3, True, torch.from_numpy(x).cuda().expand(3, 40, 5))


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
def test_runs_of_nan_and_alternatives_behind_them(kind):
    """Whole loads and whole chunks of NaN or of classes that cannot be, in front of the likeliest."""
    for shape in ((2, 300), (2, 5000), (1, 70000), (2, 300, 3)):
        for fill in (NAN, -INF, INF):
            x, labels = make(shape, 1, "plain", kind)
            x[:, :shape[1] * 3 // 4] = fill
            verify(x, labels, 1, 9, True, torch.from_numpy(x).cuda())
        x, labels = make(shape, 1, "plain", kind)
        x[:] = NAN
        x[:, -2] = 1.0
        verify(x, labels, 1, 9, True, torch.from_numpy(x).cuda())


def test_nothing_to_answer():
    for shape, axis in (((0, 5), 1), ((2, 5, 0), 1), ((0, 3, 5), 2), ((2, 0, 5), 2)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        others = [s for i, s in enumerate(shape) if i != axis]
        got = log_probabilities(x, torch.zeros(others, dtype=torch.int64, device="cuda"), 2, True, axis)
        assert list(got.label.shape) == list(got.entropy.shape) == others and got.top.numel() == 0
        (got.label.sum() + got.entropy.sum() + got.top.sum()).backward()
        assert x.grad.shape == x.shape
    got = log_probabilities(torch.zeros(2, 3, device="cuda", requires_grad=True))
    assert got == (None, None, None, None)


def test_gradients_of_one_output_and_by_differences():
    x, labels = make((4, 23, 6), 1, "plain", torch.float64)
    dev, lab = torch.from_numpy(x).cuda().requires_grad_(), torch.from_numpy(labels).cuda()

    def answers(t):
        got = log_probabilities(t, lab, 3, True)
        return got.label, got.entropy, got.top
    assert torch.autograd.gradcheck(answers, (dev,))
    # each output alone: what the others would have brought is missing, not garbage
    r = plain.Rows(rows_of(x, 1), labels.reshape(-1), 3, 64)
    for name in ("label", "entropy", "top"):
        got = log_probabilities(dev, lab, 3, True)
        out = getattr(got, name)
        dx, = torch.autograd.grad(out.sum(), dev)
        one = {"g_" + name: rows_of(np.ones(out.shape), 1) if name == "top" else np.ones(out.numel())}
        near(rows_of(dx.cpu().numpy(), 1), *r.gradient(**one), name)


def test_differentiable_once():
    x = torch.randn(3, 9, device="cuda", requires_grad=True)
    got = log_probabilities(x, torch.zeros(3, dtype=torch.int64, device="cuda"), 2, True)
    scale = torch.ones(3, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad([got.label, got.entropy], [x], [scale, torch.ones(3, device="cuda")], create_graph=True)
    for leaf in (x, scale):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(dx.sum(), leaf, retain_graph=True)
    y = log_probabilities(x, entropy=True).entropy.sum()
    y.backward()
    with pytest.raises(RuntimeError, match="second time|freed"):
        y.backward()


def test_tangents_and_records_are_refused():
    import torch.autograd.forward_ad as fwd
    x = torch.randn(3, 9, device="cuda")
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            log_probabilities(fwd.make_dual(x, torch.ones_like(x)), entropy=True)
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(lambda t: log_probabilities(t, entropy=True).entropy, (x,))


def test_what_a_position_answers_does_not_depend_on_the_others():
    """One position alone, and inside a batch: the same bits (every path takes the sums of a position in an order of its own)."""
    x, labels = make((40, 300), 1, "plain", torch.float32)
    dev, lab = torch.from_numpy(x).cuda(), torch.from_numpy(labels).cuda()
    a = log_probabilities(dev, lab, 4, True)
    b = log_probabilities(dev, lab, 4, True)
    for u, v in zip(a, b):
        assert bool((u == v).all())


def test_on_another_stream_and_in_a_graph():
    x, labels = make((33, 500), 1, "plain", torch.float32)
    dev, lab = torch.from_numpy(x).cuda(), torch.from_numpy(labels).cuda()
    want = log_probabilities(dev, lab, 3, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = log_probabilities(dev, lab, 3, True)
    side.synchronize()
    assert all(bool((u == v).all()) for u, v in zip(got, want))
    leaf = torch.zeros_like(dev).requires_grad_()
    with torch.cuda.stream(side):
        for _ in range(2):
            r = log_probabilities(leaf, lab, 3, True)
            torch.autograd.grad(r.label.sum() + r.entropy.sum(), leaf)
        del r
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = log_probabilities(leaf, lab, 3, True)
            dx, = torch.autograd.grad(r.label.sum() + r.entropy.sum(), leaf)
        graphs.append((graph, [t.detach() for t in r], dx))
        del r
    with torch.no_grad():
        leaf.copy_(dev)
    for _ in range(3):
        for graph, _, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    eager = log_probabilities(dev.requires_grad_(), lab, 3, True)
    ddev, = torch.autograd.grad(eager.label.sum() + eager.entropy.sum(), dev)
    for _, r, dx in graphs:
        assert all(bool((u == v).all()) for u, v in zip(r, want)) and bool((dx == ddev).all())


def test_the_library_launches_one_kernel_each_way():
    x = torch.randn(8, 100, device="cuda", requires_grad=True)
    n = _lib.launch_count()
    got = log_probabilities(x, torch.zeros(8, dtype=torch.int64, device="cuda"), 2, True)
    assert _lib.launch_count() == n + 1
    got.label.sum().backward()
    assert _lib.launch_count() == n + 2


def test_memory_in_front_of_and_behind_the_outputs_stays():
    """Through the C entry points, into the middle of buffers."""
    lib = _lib.lib()
    b, k, p, top = 3, 37, 11, 4
    x, labels = make((b, k, p), 1, "plain", torch.float32)
    dev, lab = torch.from_numpy(x).cuda(), torch.from_numpy(labels).cuda()
    pad, s = 64, torch.cuda.current_stream().cuda_stream
    sizes = dict(label=b * p, entropy=b * p, top_index=b * p * top, top=b * p * top, stats=3 * b * p, dlogits=b * k * p)
    bufs = {n: torch.full((v + 2 * pad,), 77, dtype=torch.int32 if n == "top_index" else torch.float32, device="cuda") for n, v in sizes.items()}
    at = {n: t.data_ptr() + 4 * pad for n, t in bufs.items()}
    d = abi.LikelihoodDesc(abi.F32, k, top, 0, b, p, k * p, p, 1)
    _lib.check(lib.simnets_log_probabilities(C.byref(d), dev.data_ptr(), lab.data_ptr(), at["label"], at["entropy"], at["top_index"], at["top"], at["stats"], None, 0, s))
    g = torch.ones(b * p * top, device="cuda")
    _lib.check(lib.simnets_log_probabilities_gradient(C.byref(d), dev.data_ptr(), lab.data_ptr(), at["stats"], at["top_index"], g.data_ptr(), g.data_ptr(), g.data_ptr(), at["dlogits"], s))
    torch.cuda.synchronize()
    for n, t in bufs.items():
        assert bool((t[:pad] == 77).all()) and bool((t[-pad:] == 77).all()), n
    got = log_probabilities(dev, lab, top, True)
    assert bool((bufs["label"][pad:-pad].view(b, p) == got.label).all()) and bool((bufs["top"][pad:-pad].view(b, top, p) == got.top).all())


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
def test_positions_that_are_nearly_sure(kind):
    """Log probabilities are at most 0 and entropies at least, whatever rounding does."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    for shape in ((4000, 10), (300, 700), (3, 20000), (5, 30, 500)):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=kind)
        x[:, 0] += torch.linspace(0, 40, x[:, 0].numel(), device="cuda", dtype=kind).view(x[:, 0].shape)
        got = log_probabilities(x, top_k=2, entropy=True)
        assert bool((got.entropy >= 0).all()) and bool((got.top <= 0).all())


def test_what_is_refused():
    x = torch.zeros(3, 7, 5, device="cuda")
    for bad in (torch.zeros(3, 7, dtype=torch.int64, device="cuda"), torch.zeros(3, 5, 1, dtype=torch.int64, device="cuda"), torch.zeros(15, dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError, match="labels must have shape"):
            log_probabilities(x, bad)
    with pytest.raises(TypeError, match="int64"):
        log_probabilities(x, torch.zeros(3, 5, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="labels must live"):
        log_probabilities(x, torch.zeros(3, 5, dtype=torch.int64))
    with pytest.raises(TypeError, match="float32 and float64"):
        log_probabilities(x.half())
    with pytest.raises(ValueError, match="at most the number of classes"):
        log_probabilities(x, top_k=8)


def test_autograd_sees_what_changes_between_the_passes():
    for change in ("logits", "labels", "index"):
        x, labels = torch.randn(3, 9, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
        leaf = x.clone().requires_grad_()
        mid = leaf * 1.0
        got = log_probabilities(mid, labels, 2)
        with torch.no_grad():
            dict(logits=mid, labels=labels, index=got.top_index)[change].fill_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            (got.label.sum() + got.top.sum()).backward()


def test_kept_graphs_shared_and_broadcast_logits():
    x = torch.randn(1, 40, 6, device="cuda", dtype=torch.float64, requires_grad=True)
    wide = x.expand(4, 40, 6)
    labels = torch.randint(0, 40, (4, 6), device="cuda")
    got = log_probabilities(wide, labels, entropy=True)
    total = got.label.sum() - 0.3 * got.entropy.sum()
    a, = torch.autograd.grad(total, x, retain_graph=True)
    b, = torch.autograd.grad(total, x)
    assert bool((a == b).all())
    r = plain.Rows(rows_of(x.detach().expand(4, 40, 6).cpu().numpy(), 1), labels.cpu().numpy().reshape(-1), 0, 64)
    want, off = r.gradient(np.ones(24), np.full(24, -0.3))
    want, off = want.reshape(4, 6, 40).sum(0), off.reshape(4, 6, 40).sum(0)
    # a sum of four, each within its bound, and three additions of numbers below 2.5 (the label's 1 - p and 0.3 p (log p + H), of which the latter is
    # at most 0.3 (1 / e + log 40) = 1.2), whose sums are below four times that
    assert (abs(rows_of(a.cpu().numpy(), 1) - want) <= off + 3 * 4 * 2.5 * np.finfo(np.float64).eps).all()
    # two calls on the same logits: their gradients add up
    y = torch.randn(5, 30, device="cuda", requires_grad=True)
    one, = torch.autograd.grad(log_probabilities(y, entropy=True).entropy.sum(), y)
    two, = torch.autograd.grad(log_probabilities(y, entropy=True).entropy.sum() + log_probabilities(y, entropy=True).entropy.sum(), y)
    assert bool((two == 2 * one).all())


def test_views_that_stand_for_negated_values():
    z = torch.randn(4, 300, dtype=torch.complex64, device="cuda")
    x = z.conj().imag
    assert x.is_neg()
    a, b = log_probabilities(x, top_k=3, entropy=True), log_probabilities((-z.imag).contiguous(), top_k=3, entropy=True)
    assert all(u is v is None or bool((u == v).all()) for u, v in zip(a, b))
