"""8-bit checkpoints on the GPU: bytes and values against the restatement in plain_operators.py, gradients at a checkpoint against the
oracle in 64 bits at the values that it stands for, the layers that use them."""
import importlib

import numpy as np
import pytest
import torch

import cases
import plain_operators as plain
from simnets_tf_b200 import abi, dp, keras
from simnets_tf_b200.ops import checkpoint as ck
from simnets_tf_b200.simnet import SPECS, SimNet

mex_ops = importlib.import_module("simnets_tf_b200.ops.mex")
sim_ops = importlib.import_module("simnets_tf_b200.ops.similarity")
pytestmark = pytest.mark.gpu

KINDS = [torch.float32, torch.float64]


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _values(rng, n, kind, style):
    x = rng.normal(size=n) * 3 - 40
    if style == "special":
        u = rng.random(n)
        x = np.where(u < 0.1, np.nan, np.where(u < 0.15, -np.inf, np.where(u < 0.2, np.inf, x)))
        x[:min(n, 300)] = np.nan                                # whole groups without a finite value
        x[-min(n, 40):] = -np.inf
    elif style == "wide":
        x = np.where(rng.random(n) < 0.5, 1.0, -1.0) * np.finfo(kind).max * rng.random(n)
    elif style == "tiny":
        x = rng.random(n) * np.finfo(kind).tiny * rng.choice([1.0, 100.0, 1e4], size=n)
    elif style == "flat":
        x = np.full(n, -7.25)
    return x.astype(kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group", ck.GROUPS)
@pytest.mark.parametrize("style", ["plain", "special", "wide", "tiny", "flat"])
def test_bytes_ranges_and_values_are_the_definitions(kind, group, style):
    rng = np.random.default_rng(group)
    for n in (1, 31, 32, 33, 127, 128, 129, 255, 257, 4099):
        x = _values(rng, n, torch.zeros((), dtype=kind).numpy().dtype, style)
        kept = ck.checkpoint_pack(_dev(x), group)
        codes, ranges = plain.pack(x, group)
        assert kept.shape == (n,) and kept.dtype == kind
        assert np.array_equal(kept.ranges.cpu().numpy(), ranges)
        assert np.array_equal(kept.codes.cpu().numpy(), codes), (n, np.flatnonzero(kept.codes.cpu().numpy() != codes)[:5])
        got, want = ck.checkpoint_unpack(kept).cpu().numpy(), plain.unpack(codes, ranges, x.shape, group)
        assert np.array_equal(np.isfinite(got), np.isfinite(x))
        # one rounding, of a sum that numpy rounds twice
        fine = np.isfinite(want)
        assert np.array_equal(np.where(fine, 0, got), np.where(fine, 0, want), equal_nan=True)
        assert (np.abs(got[fine] - want[fine]) <= np.spacing(np.abs(want[fine]))).all()


@pytest.mark.parametrize("kind", KINDS)
def test_views_offsets_and_empty_tensors(kind):
    base = torch.randn(4100, device="cuda", dtype=kind)
    for x in (base[1:4001], base[3:], base[:4096].view(4, 16, 8, 8).permute(0, 2, 3, 1), base[:4096].view(64, 64)[:, ::2], base[:0].view(0, 3, 4, 4)):
        kept = ck.checkpoint_pack(x, 64)
        codes, ranges = plain.pack(x.contiguous().cpu().numpy(), 64)
        assert np.array_equal(kept.codes.cpu().numpy(), codes) and np.array_equal(kept.ranges.cpu().numpy(), ranges)
        assert ck.checkpoint_unpack(kept).shape == x.shape
    # codes and ranges that lie anywhere in memory
    kept = ck.checkpoint_pack(base[:1000], 32)
    moved = torch.zeros(1003, dtype=torch.uint8, device="cuda")
    moved[3:] = kept.codes
    off = torch.zeros(2 * 32 + 1, dtype=kind, device="cuda")
    off[1:] = kept.ranges.reshape(-1)
    again = ck.Checkpoint(moved[3:], off[1:].view(32, 2), kept.shape, 32)
    assert torch.equal(ck.checkpoint_unpack(again), ck.checkpoint_unpack(kept))


def test_a_long_tensor_keeps_its_offsets_beyond_32_bits():
    n = (1 << 31) + (1 << 12) + 77
    x = torch.zeros(n, device="cuda")
    x[-1000:] = torch.linspace(-3, 5, 1000, device="cuda")
    kept = ck.checkpoint_pack(x, 256)
    tail = x[-1000 - (n - 1000) % 256:].clone()
    del x
    codes, ranges = plain.pack(tail.cpu().numpy(), 256)
    assert np.array_equal(kept.codes[-tail.numel():].cpu().numpy(), codes)
    assert np.array_equal(kept.ranges[-len(ranges):].cpu().numpy(), ranges)
    back = ck.checkpoint_unpack(kept)
    assert float(back[:1 << 20].abs().max()) == 0.0 and float(back[n // 2:n // 2 + 4096].abs().max()) == 0.0
    assert np.array_equal(back[-tail.numel():].cpu().numpy(), plain.unpack(codes, ranges, tail.shape, 256))


# ---- MEX ------------------------------------------------------------------------------------------------------------------------
def _mex_inputs(port, c, kind, spread=1.0):
    d = cases.mex_desc(c, dtype=abi.F32 if kind == torch.float32 else abi.F64)
    x, off, dy = cases.mex_inputs(c, port.mex_offsets_shape(d), port.mex_out_shape(d), np.float32 if kind == torch.float32 else np.float64)
    return x, (off * spread).astype(off.dtype), dy


def _mex_oracle(port, c, x, off, dy):
    """(dx, doff) in 64 bits and the same of |dy|: what the terms of the sums add up to."""
    d = cases.mex_desc(c, dtype=abi.F64)
    x, off, dy = (np.ascontiguousarray(a.astype(np.float64)) for a in (x, off, dy))
    y = port.mex_forward(d, x, off)
    return [(port.mex_input_grad(d, x, off, y, g), port.mex_offsets_grad(d, x, off, y, g)) for g in (dy, np.abs(dy))]


def _mex_tolerance(kind, c, x, off, positions):
    """Relative to the sum of the terms' magnitudes: arguments of exponentials of up to A nats are off by A half-units each for x and for the
    offsets, in numerator and sum; exponentials, quotient and products a few units more; sums of instances and positions in
    pieces of 16."""
    span = lambda a: float(np.ptp(a[np.isfinite(a)])) if np.isfinite(a).any() else 0.0
    a = min(abs(c["eps"]), 1e3) * (span(x) + span(off))
    return (4 * a + 32 + positions / 16) * np.finfo(np.float32 if kind == torch.float32 else np.float64).eps


FINITE = [c for c in cases.MEX_SMALL if np.isfinite(c["eps"]) and c["shape"][0] > 0]


def _check_mex(port, c, kind, x, off, dy, group, flags=0, pooled_dy=None, **kw):
    kept = ck.checkpoint_pack(_dev(x), group)
    at = ck.checkpoint_unpack(kept).cpu().numpy()
    given = dy if pooled_dy is None else pooled_dy
    dx, doff = ck.mex_checkpoint_backward(kept, _dev(off), _dev(given), c["M"], flags=c["flags"] | flags, pooled=pooled_dy is not None, **cases.mex_attrs(c), **kw)
    (rdx, rdoff), (adx, adoff) = _mex_oracle(port, c, at, off, dy)
    tol = _mex_tolerance(kind, c, at, off, dy.size // c["M"])
    assert dx.dtype == kind and doff.shape == off.shape
    for got, ref, size in ((dx.cpu().numpy(), rdx, adx), (doff.cpu().numpy(), rdoff, adoff)):
        assert (np.abs(got - ref) <= tol * size + 1e-30).all(), float((np.abs(got - ref) / (tol * size + 1e-30)).max())
    return dx, doff


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("c", FINITE, ids=lambda c: c["name"])
def test_mex_gradients_at_a_checkpoint(port, c, kind):
    x, off, dy = _mex_inputs(port, c, kind)
    _check_mex(port, c, kind, x, off, dy, 32)


def _pixel(name, batch, channels, height, width, m, region=2, **kw):
    return cases.mex_case(name, (batch, channels, height, width), m, (channels, 1, 1), (channels, 1, 1), softmax=True, unshared=region > 0,
                          unshared_region=(region,) if region else (-1,), normalize=True, **kw)


# over the channels of each pixel and over blocks that tile channels and rows: taps and instances around the sizes of tiles, few positions
# and many, one sample, odd maps, regions that divide the map unevenly
DISJOINT = [
    _pixel("one_tap", 3, 1, 5, 7, 4, seed=1), _pixel("few", 2, 8, 6, 6, 8, seed=2), _pixel("k15", 2, 15, 4, 6, 17, seed=3), _pixel("k16", 2, 16, 9, 5, 16, 0, seed=4),
    _pixel("k17", 3, 17, 8, 8, 33, seed=5), _pixel("k32", 2, 32, 16, 16, 64, seed=6), _pixel("k33", 5, 33, 6, 10, 65, 0, seed=7), _pixel("k64", 4, 64, 16, 16, 128, seed=8),
    _pixel("k64_m129", 3, 64, 8, 8, 129, seed=9), _pixel("k65", 2, 65, 10, 10, 70, seed=10), _pixel("k100", 3, 100, 6, 8, 200, seed=11), _pixel("k128", 2, 128, 16, 16, 256, seed=12),
    _pixel("k129", 2, 129, 6, 6, 60, seed=13), _pixel("uneven", 2, 40, 7, 9, 50, 4, seed=14), _pixel("one_position", 1, 24, 1, 1, 5, 0, seed=15),
    _pixel("many_instances", 2, 16, 6, 6, 1200, seed=22), _pixel("many_of_k64", 2, 50, 4, 4, 300, 0, seed=23), _pixel("many_of_k128", 1, 90, 4, 4, 400, seed=24),
    _pixel("eps_small", 2, 48, 8, 8, 48, seed=16, eps=0.25), _pixel("eps_negative", 2, 48, 8, 8, 48, 0, seed=17, eps=-1.5), _pixel("wide", 7, 20, 30, 30, 300, 0, seed=18),
    cases.mex_case("tiles_4x2x2", (3, 32, 8, 8), 60, (4, 2, 2), (4, 2, 2), eps=0.5, unshared=False, seed=19),
    cases.mex_case("tiles_2x3x3", (2, 8, 9, 12), 130, (2, 3, 3), (2, 3, 3), softmax=True, unshared_region=(2,), seed=20),
    cases.mex_case("channel_halves", (3, 64, 4, 6), 40, (32, 1, 1), (32, 1, 1), softmax=True, unshared=False, shared_region=(2, 2, 3), seed=21),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("c", DISJOINT, ids=lambda c: c["name"])
def test_mex_gradients_over_disjoint_blocks(port, c, kind):
    x, off, dy = _mex_inputs(port, c, kind, 3.0)
    dx, doff = _check_mex(port, c, kind, x * 2 - 30, off, dy, 64)
    again = _check_mex(port, c, kind, x * 2 - 30, off, dy, 64)
    assert torch.equal(dx, again[0]) and torch.equal(doff, again[1])            # the same on every run


@pytest.mark.parametrize("c", [c for c in DISJOINT if c["name"] in ("k16", "k32", "k64", "k100", "eps_negative")], ids=lambda c: c["name"])
def test_mex_gradients_of_a_pooled_output(port, c):
    b, _, h, w = c["shape"]
    c = dict(c, shape=(b, c["shape"][1], h + h % 2, w + w % 2))
    x, off, dy = _mex_inputs(port, c, torch.float32)
    pooled = np.random.default_rng(5).normal(size=dy.shape[:2] + (dy.shape[2] // 2, dy.shape[3] // 2)).astype(np.float32)
    up = np.repeat(np.repeat(pooled, 2, axis=2), 2, axis=3)
    _check_mex(port, c, torch.float32, x, off, up, 128, pooled_dy=pooled)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", ["k17", "k64", "k100", "tiles_4x2x2"])
def test_offsets_gradients_of_raw_offsets_and_sums_onto_others(port, name, kind):
    c = next(c for c in DISJOINT if c["name"] == name)
    x, off, dy = _mex_inputs(port, c, kind)
    raw = off + np.random.default_rng(1).normal(size=off.shape[:2] + (1, 1, 1)).astype(off.dtype) * 5
    kept = ck.checkpoint_pack(_dev(x), 64)
    dx, doff = ck.mex_checkpoint_backward(kept, _dev(raw), _dev(dy), c["M"], flags=abi.FLAG_MEX_NORMALIZED_OFFSETS, **cases.mex_attrs(c))
    r = raw.astype(np.float64).reshape(raw.shape[0], raw.shape[1], -1)
    lse = np.log(np.exp(r - r.max(2, keepdims=True)).sum(2, keepdims=True)) + r.max(2, keepdims=True)
    at = ck.checkpoint_unpack(kept).cpu().numpy()
    (rdx, rdoff), (adx, adoff) = _mex_oracle(port, c, at, (r - lse).reshape(raw.shape), dy)
    flat = lambda a: a.reshape(r.shape)
    want = flat(rdoff) - np.exp(r - lse) * flat(rdoff).sum(2, keepdims=True)
    size = flat(adoff) + np.exp(r - lse) * flat(adoff).sum(2, keepdims=True)
    tol = _mex_tolerance(kind, c, at, raw, dy.size // c["M"])
    assert (np.abs(dx.cpu().numpy() - rdx) <= tol * adx).all()
    assert (np.abs(flat(doff.cpu().numpy()) - want) <= tol * size).all()
    sums = torch.full_like(doff, 3.0)
    _, same = ck.mex_checkpoint_backward(kept, _dev(raw), _dev(dy), c["M"], flags=abi.FLAG_MEX_NORMALIZED_OFFSETS | abi.FLAG_ACCUMULATE, doff_out=sums, **cases.mex_attrs(c))
    assert same.data_ptr() == sums.data_ptr()
    eps = torch.finfo(kind).eps                                                 # (one rounding of the sum)
    assert bool(((sums - (doff + 3.0)).abs() <= eps * (doff.abs() + 3.0)).all())


@pytest.mark.parametrize("name", ["k17", "k64", "k100", "tiles_4x2x2", "tiles_2x3x3"])
def test_offsets_that_no_factorisation_takes(port, name):
    """Rows whose spread is beyond what exponentials of float32 hold."""
    c = next(c for c in DISJOINT if c["name"] == name)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    off = off.copy()
    off.reshape(off.shape[0], off.shape[1], -1)[:, ::2, 0] = 150.0
    _check_mex(port, c, torch.float32, x, off, dy, 64)
    off.reshape(off.shape[0], off.shape[1], -1)[:, 1::2, -1] = -np.inf
    _check_mex(port, c, torch.float32, x, off, dy, 64)


@pytest.mark.parametrize("name", ["k17", "k64", "k100", "tiles_4x2x2"])
def test_missing_and_infinite_activations(port, name):
    """-infinity is a tap of no weight; a patch with a NaN or infinity has NaN gradients, and so have the offsets that it adds to."""
    c = next(c for c in DISJOINT if c["name"] == name)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    x = x.copy()
    x[:, 1::3] = -np.inf
    _check_mex(port, c, torch.float32, x, off, dy, 32)
    x[0, 0, 0, 0], x[-1, 0, -1, -1] = np.nan, np.inf
    kept = ck.checkpoint_pack(_dev(x), 32)
    dx, doff = ck.mex_checkpoint_backward(kept, _dev(off), _dev(dy), c["M"], **cases.mex_attrs(c))
    (rdx, rdoff), (adx, _) = _mex_oracle(port, c, ck.checkpoint_unpack(kept).cpu().numpy(), off, dy)
    assert np.array_equal(np.isnan(dx.cpu().numpy()), np.isnan(rdx)) and np.array_equal(np.isnan(doff.cpu().numpy()), np.isnan(rdoff))


@pytest.mark.parametrize("name", ["k17", "k64", "k100", "tiles_4x2x2"])
def test_patches_that_hold_nothing(port, name):
    """Whole samples of -infinity have no weights: NaN there and in the offsets that they add to, as of the formula, and nowhere else."""
    c = next(c for c in DISJOINT if c["name"] == name)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    x, dy = x.copy(), dy.copy()
    x[0] = -np.inf
    kept = ck.checkpoint_pack(_dev(x), 32)
    dx, doff = (t.cpu().numpy() for t in ck.mex_checkpoint_backward(kept, _dev(off), _dev(dy), c["M"], **cases.mex_attrs(c)))
    (rdx, rdoff), _ = _mex_oracle(port, c, ck.checkpoint_unpack(kept).cpu().numpy(), off, dy)
    assert np.array_equal(np.isnan(dx), np.isnan(rdx)) and np.array_equal(np.isnan(doff), np.isnan(rdoff))
    assert np.isfinite(dx[1:]).all()


@pytest.mark.parametrize("name", ["k17", "k64", "k100", "tiles_4x2x2"])
def test_gradients_that_are_no_numbers_stay_where_they_are(port, name):
    """An infinity or NaN in dy: neither dx of its patch nor its instance's offsets are finite, and all others are what they were."""
    c = next(c for c in DISJOINT if c["name"] == name)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    kept = ck.checkpoint_pack(_dev(x), 32)
    at = ck.checkpoint_unpack(kept).cpu().numpy()
    dx, doff = ck.mex_checkpoint_backward(kept, _dev(off), _dev(dy), c["M"], **cases.mex_attrs(c))
    for bad in (np.inf, np.nan):
        b = dy.copy()
        b[0, 1, 0, 0] = bad
        dxb, doffb = ck.mex_checkpoint_backward(kept, _dev(off), _dev(b), c["M"], **cases.mex_attrs(c))
        for got, want in ((dxb, dx), (doffb, doff)):
            fine = torch.isfinite(got)
            assert bool((~fine).any()) and torch.equal(got[fine], want[fine])
        # (which those are depends on how the instances of several blocks lie in dy: the oracle's)
        (rdx, rdoff), _ = _mex_oracle(port, c, at, off, b)
        assert np.array_equal(torch.isfinite(dxb).cpu().numpy(), np.isfinite(rdx)) and np.array_equal(torch.isfinite(doffb).cpu().numpy(), np.isfinite(rdoff))
        assert (~np.isfinite(rdx)).sum() == (~np.isfinite(rdoff)).sum() == np.prod(c["blocks"])


@pytest.mark.parametrize("name", ["eps_pinf", "eps_ninf"])
def test_maxima_at_a_checkpoint(port, name):
    c = next(c for c in cases.MEX_SMALL if c["name"] == name)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    kept = ck.checkpoint_pack(_dev(x), 32)
    dx, doff = ck.mex_checkpoint_backward(kept, _dev(off), _dev(dy), c["M"], **cases.mex_attrs(c))
    d, at = cases.mex_desc(c), ck.checkpoint_unpack(kept).cpu().numpy()
    y = port.mex_forward(d, at, off)
    cases.assert_parity(dx.cpu().numpy(), port.mex_input_grad(d, at, off, y, dy), what="dx")
    cases.assert_parity(doff.cpu().numpy(), port.mex_offsets_grad(d, at, off, y, dy), what="doff")


def test_an_empty_batch():
    c = next(c for c in cases.MEX_SMALL if c["name"] == "empty_batch")
    kept = ck.checkpoint_pack(torch.zeros(c["shape"], device="cuda"), 32)
    layer = keras.Mex(3, blocks=[4, 1, 1], strides=[4, 1, 1], softmax_mode=True, checkpoint=32)
    x = torch.zeros(c["shape"], device="cuda", requires_grad=True)
    layer(x).sum().backward()
    assert x.grad.shape == c["shape"] and float(layer.offsets.grad.abs().max()) == 0.0
    dx, dt, dw = ck.similarity_checkpoint_backward(kept, torch.ones(2, 4, 3, 3, device="cuda"), torch.ones(2, 4, 3, 3, device="cuda"), torch.zeros(0, 2, 2, 2, device="cuda"))
    assert dx.shape == c["shape"] and float(dt.abs().max()) == 0.0 and float(dw.abs().max()) == 0.0


def test_a_wait_that_runs_out_is_reported_and_recomputed(port, cuda_lib):
    """abi.FLAG_MEX_TEST_EXPIRE_WAIT: the one-pass kernel's first product is withheld and its waits are short.  It must return (no hang, no
    fault), say so in word 1 of the workspace, and the gradients must be right because the kernel behind redoes them."""
    import ctypes as C
    for name in ("k17", "k64", "k100", "tiles_4x2x2"):
        c = next(c for c in DISJOINT if c["name"] == name)
        x, off, dy = _mex_inputs(port, c, torch.float32)
        kept = ck.checkpoint_pack(_dev(x), 64)
        (rdx, rdoff), (adx, adoff) = _mex_oracle(port, c, ck.checkpoint_unpack(kept).cpu().numpy(), off, dy)
        tol = _mex_tolerance(torch.float32, c, x, off, dy.size // c["M"])
        od, dyd = _dev(off), _dev(dy)
        unsafe = off.copy()
        unsafe.reshape(off.shape[0] * off.shape[1], -1)[0, 0] = 200.0
        for flags, given, want in ((0, od, (0, 0)), (abi.FLAG_MEX_TEST_EXPIRE_WAIT, od, (0, 1)), (0, _dev(unsafe), (1, 0)), (0, od, (0, 0))):
            d = cases.mex_desc(c, flags=flags)
            assert cuda_lib.simnets_mex_checkpoint_one_pass(C.byref(d)) == 1
            ws = torch.full((cuda_lib.simnets_mex_checkpoint_workspace_bytes(C.byref(d)),), 255, dtype=torch.uint8, device="cuda")
            dx, doff = torch.full(x.shape, float("nan"), device="cuda"), torch.full(off.shape, float("nan"), device="cuda")
            stream = torch.cuda.current_stream().cuda_stream
            assert cuda_lib.simnets_mex_checkpoint_gradients(C.byref(d), 64, kept.codes.data_ptr(), kept.ranges.data_ptr(), given.data_ptr(), dyd.data_ptr(), dx.data_ptr(),
                                                             doff.data_ptr(), ws.data_ptr(), ws.numel(), stream) == 0
            status = (C.c_int32 * 2)(7, 7)
            assert cuda_lib.simnets_mex_workspace_status(ws.data_ptr(), stream, status) == 0
            torch.cuda.synchronize()
            assert (status[0], status[1]) == want, (name, flags)
            if given is od:
                assert (np.abs(dx.cpu().numpy() - rdx) <= tol * adx + 1e-30).all() and (np.abs(doff.cpu().numpy() - rdoff) <= tol * adoff + 1e-30).all()


def test_long_patches_with_the_sums_of_the_ordinary_gradients(port):
    """abi.FLAG_MEX_CHECKPOINT_TENSORCORE: what the ordinary gradients give at the checkpoint's values, to the library's bound."""
    c = _pixel("k200", 3, 200, 16, 16, 96, seed=30, flags=abi.FLAG_MEX_NO_SMALL_TILES)
    x, off, dy = _mex_inputs(port, c, torch.float32)
    kept = ck.checkpoint_pack(_dev(x), 64)
    at = ck.checkpoint_unpack(kept)
    got = ck.mex_checkpoint_backward(kept, _dev(off), _dev(dy), 96, flags=c["flags"] | abi.FLAG_MEX_CHECKPOINT_TENSORCORE, **cases.mex_attrs(c))
    y = mex_ops.mex_forward(at, _dev(off), 96, flags=c["flags"], **cases.mex_attrs(c))
    for a, b in zip(got, mex_ops.mex_backward(at, _dev(off), y, _dev(dy), 96, flags=c["flags"], **cases.mex_attrs(c))):
        assert torch.equal(a, b)
    (rdx, rdoff), _ = _mex_oracle(port, c, at.cpu().numpy(), off, dy)
    # y and the sums over instances are each 3 x 2^-23 off for every eight terms (library bound on its tensor-core sums)
    for a, ref in zip(got, (rdx, rdoff)):
        assert np.abs(a.cpu().numpy() - ref).max() <= 3 * 2.0 ** -23 * ((200 + 96) / 8 + 768 / 8) * np.abs(ref).max()


def test_codes_and_ranges_anywhere_in_memory(cuda_lib):
    import ctypes as C
    c = next(c for c in DISJOINT if c["name"] == "k64")
    x, off, dy = (torch.randn(s, device="cuda") for s in (c["shape"], (4, 128, 64, 1, 1), (4, 128, 16, 16)))
    kept = ck.checkpoint_pack(x, 32)
    codes, ranges = torch.zeros(kept.codes.numel() + 3, dtype=torch.uint8, device="cuda"), torch.zeros(kept.ranges.numel() + 1, device="cuda")
    codes[3:], ranges[1:] = kept.codes, kept.ranges.reshape(-1)
    moved = ck.Checkpoint(codes[3:], ranges[1:].view(-1, 2), kept.shape, 32)
    assert moved.ranges.data_ptr() % 8 == 4 and moved.codes.data_ptr() % 4 == 3
    want = ck.mex_checkpoint_backward(kept, off, dy, 128, **cases.mex_attrs(c))
    for got, ref in zip(ck.mex_checkpoint_backward(moved, off, dy, 128, **cases.mex_attrs(c)), want):
        assert torch.equal(got, ref)
    odd_off, odd_dy = (torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (off, dy))
    assert odd_off.data_ptr() % 8 == 4 and odd_dy.data_ptr() % 8 == 4
    for got, ref in zip(ck.mex_checkpoint_backward(kept, odd_off, odd_dy, 128, **cases.mex_attrs(c)), want):
        assert torch.equal(got, ref)
    d = cases.mex_desc(c)
    ws = torch.empty(cuda_lib.simnets_mex_checkpoint_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
    assert cuda_lib.simnets_mex_checkpoint_gradients(C.byref(d), 32, moved.codes.data_ptr(), moved.ranges.data_ptr(), off.data_ptr(), dy.data_ptr(), x.data_ptr(), off.data_ptr(),
                                                     ws.data_ptr(), ws.numel(), None) == abi.E_UNSUPPORTED


def test_which_shapes_take_one_pass(cuda_lib):
    import ctypes as C
    ask = lambda c, dtype=abi.F32, flags=0: cuda_lib.simnets_mex_checkpoint_one_pass(C.byref(cases.mex_desc(c, dtype=dtype, flags=flags)))
    by_name = {c["name"]: c for c in DISJOINT + cases.MEX_SMALL}
    assert [ask(by_name[n]) for n in ("one_tap", "k64", "k128", "tiles_2x3x3", "k129", "tiled_padded", "eps_pinf", "head_overlap")] == [1, 1, 1, 1, 0, 0, 0, 0]
    assert ask(by_name["k64"], abi.F64) == 0 and ask(by_name["k64"], flags=abi.FLAG_MEX_EXACT) == 0
    assert ask(dict(by_name["k64"], eps=1e31)) == 0 and ask(dict(by_name["k64"], shape=(0, 64, 16, 16))) == 0


# ---- Similarity -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("c", cases.SIM_SMALL, ids=lambda c: c["name"])
def test_similarity_gradients_at_a_checkpoint(port, c, kind):
    d, d64 = (cases.sim_desc(c, dtype=k) for k in (abi.F32 if kind == torch.float32 else abi.F64, abi.F64))
    x, t, w, dy = cases.sim_inputs(c, port.sim_out_shape(d), np.float32 if kind == torch.float32 else np.float64)
    kept = ck.checkpoint_pack(_dev(x), 32)
    at = ck.checkpoint_unpack(kept).cpu().numpy()
    dx, dt, dw = ck.similarity_checkpoint_backward(kept, _dev(t), _dev(w), _dev(dy), flags=c["flags"], **cases.sim_attrs(c))
    full = [np.ascontiguousarray(a.astype(np.float64)) for a in (at, t, w, dy)]
    refs = [port.similarity_input_grad(d64, *full)] + list(port.similarity_params_grad(d64, *full))
    # the operator's own bound on its sums (acceptance rule of cases.py)
    for got, ref, what in zip((dx, dt, dw), refs, ("dx", "dt", "dw")):
        cases.assert_parity(got.cpu().numpy(), ref, what=c["name"] + " " + what)


# ---- through autograd, layers and networks ------------------------------------------------------------------------------------------
def _grads(call, *tensors):
    tensors = [t.detach().clone().requires_grad_() for t in tensors]
    y = call(*tensors)
    dy = torch.linspace(-1, 1, y.numel(), dtype=y.dtype, device="cuda").view(y.shape)
    return (y.detach(), dy) + torch.autograd.grad(y, tensors, dy)


ATTRS = dict(blocks=[8, 1, 1], strides=[8, 1, 1], softmax_mode=True, use_unshared_regions=False, shared_offset_region=[-1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pooled", [False, True])
def test_the_differentiable_mex_op_keeps_a_checkpoint(kind, pooled):
    torch.manual_seed(0)
    x, off = torch.randn(3, 16, 6, 8, device="cuda", dtype=kind), torch.randn(1, 20, 8, 1, 1, device="cuda", dtype=kind)
    y, dy, dx, doff = _grads(lambda x, o: ck.mex_checkpointed(x, o, 20, group=32, sum_pool2=pooled, **ATTRS), x, off)
    plain_y = mex_ops.mex_sum_pool2(x, off, 20, **ATTRS) if pooled else mex_ops.mex(x, off, 20, **ATTRS)
    assert torch.equal(y, plain_y)                                              # the forward pass is the op's
    if pooled and kind == torch.float64:
        dy, pooled = torch.nn.functional.interpolate(dy, scale_factor=2, mode="nearest"), False
    want = ck.mex_checkpoint_backward(ck.checkpoint_pack(x, 32), off, dy, 20, pooled=pooled, **ATTRS)
    for got, ref in zip((dx, doff), want):
        assert torch.allclose(got, ref, rtol=1e-12 if kind == torch.float64 else 1e-6, atol=1e-6 * float(ref.abs().max()) if kind == torch.float32 else 1e-12)


def test_the_differentiable_similarity_op_keeps_a_checkpoint():
    torch.manual_seed(0)
    x, t, w = torch.randn(3, 4, 9, 8, device="cuda"), torch.randn(6, 4, 3, 3, device="cuda"), torch.rand(6, 4, 3, 3, device="cuda")
    attrs = dict(blocks=[3, 3], strides=[1, 1], padding=[1, 1])
    y, dy, dx, dt, dw = _grads(lambda x, t, w: ck.similarity_checkpointed(x, t, w, group=64, **attrs), x, t, w)
    assert torch.equal(y, sim_ops.similarity(x, t, w, **attrs))
    for got, ref in zip((dx, dt, dw), ck.similarity_checkpoint_backward(ck.checkpoint_pack(x, 64), t, w, dy, **attrs)):
        assert torch.equal(got, ref)


def test_only_wanted_gradients_and_none_without_grad():
    x, off = torch.randn(3, 16, 6, 8, device="cuda"), torch.randn(1, 20, 8, 1, 1, device="cuda")
    both = _grads(lambda x, o: ck.mex_checkpointed(x, o, 20, **ATTRS), x, off)
    xg = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ck.mex_checkpointed(xg, off, 20, **ATTRS), xg, both[1])[0], both[2])
    og = off.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ck.mex_checkpointed(x, og, 20, **ATTRS), og, both[1])[0], both[3])
    with torch.no_grad():
        assert not ck.mex_checkpointed(xg, og, 20, **ATTRS).requires_grad


def test_what_stays_between_the_passes():
    """The bytes, the ranges and the parameters; the input may change."""
    x, off = torch.randn(4, 16, 8, 8, device="cuda"), torch.randn(1, 20, 8, 1, 1, device="cuda")
    want = _grads(lambda x, o: ck.mex_checkpointed(x, o, 20, group=64, **ATTRS), x, off)
    seen, og = [], off.clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append((t.dtype, t.numel())) or t.cpu(), lambda t: t.cuda()):
        y = ck.mex_checkpointed(x, og, 20, group=64, **ATTRS)
    assert seen == [(torch.uint8, x.numel()), (torch.float32, 2 * x.numel() // 64), (torch.float32, off.numel())]
    x.zero_()
    assert torch.equal(torch.autograd.grad(y, og, want[1])[0], want[3])


def test_layers_and_networks_with_checkpoints():
    spec = SPECS["cfg3"]
    x = torch.rand(6, 1, 28, 28, device="cuda") - 0.5
    labels = torch.arange(6, device="cuda") % 10
    net, kept = SimNet(spec, seed=3), SimNet(spec, seed=3, checkpoint=64)
    assert [m.checkpoint for m in kept.stages] == [None] + [64] * (len(kept.stages) - 1)
    assert torch.equal(net(x), kept(x))
    inputs = []
    handles = [m.register_forward_pre_hook(lambda m, a: inputs.append(a[0].detach())) for m in kept.stages]
    logits = kept(x)
    loss = kept.loss_of_logits(logits, labels)
    d = torch.autograd.grad(loss, logits, retain_graph=True)[0].reshape(6, 10, 1, 1)
    loss.backward()
    for h in handles:
        h.remove()
    # the same by the op's own calls, from the last layer to the first
    for layer, given in reversed(list(zip(kept.stages, inputs))[1:]):
        attrs, pooled = dict(layer._op_attrs()), layer is not kept.stages[-1] and tuple(d.shape[2:]) != tuple(layer.compute_output_shape(given.shape)[2:])
        if pooled and layer.compute_output_shape(given.shape)[2] % 2:
            break                                                               # (an odd map is pooled by torch)
        d, doff = ck.mex_checkpoint_backward(ck.checkpoint_pack(given, 64), layer.offsets.detach(), d, layer.num_instances, flags=abi.FLAG_MEX_NORMALIZED_OFFSETS,
                                             pooled=pooled, **attrs)
        assert torch.allclose(layer.offsets.grad, doff, rtol=1e-5, atol=1e-6 * float(doff.abs().max()))
    assert all(torch.isfinite(p.grad).all() for p in kept.parameters())
    # the layers keep bytes
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        kept.loss(x, labels)
    inputs = [t for t in held if t.dtype == torch.uint8]
    assert len(inputs) == len(kept.stages) - 1 and all(t.dim() != 4 or t.data_ptr() in (x.data_ptr(),) or t.shape[1] == 1 for t in held)


def test_layers_with_every_option_agree_with_the_op():
    torch.manual_seed(1)
    x = torch.randn(2, 9, 10, 16, device="cuda")                                 # channels last
    layer = keras.Mex(12, blocks=[16, 1, 1], strides=[16, 1, 1], normalize_offsets=True, channels_last=True, checkpoint=32)
    xg = x.clone().requires_grad_()
    y = layer(xg)
    dy = torch.randn_like(y)
    y.backward(dy)
    plain_layer = keras.Mex(12, blocks=[16, 1, 1], strides=[16, 1, 1], normalize_offsets=True, channels_last=True, offsets_initializer=lambda s, dtype=None: layer.offsets.detach().cpu().numpy())
    at = ck.checkpoint_unpack(ck.checkpoint_pack(x.permute(0, 3, 1, 2), 32)).permute(0, 2, 3, 1).contiguous().requires_grad_()
    plain_layer(at).backward(dy)
    # both sum in float32: see _mex_tolerance for what they may differ by
    for got, ref in ((xg.grad, at.grad), (layer.offsets.grad, plain_layer.offsets.grad)):
        assert torch.allclose(got, ref, rtol=1e-4, atol=1e-5 * float(ref.abs().max()))


def test_gradients_into_a_bucket():
    torch.manual_seed(2)
    x = torch.randn(6, 4, 8, 8, device="cuda")
    for layer in (keras.Mex(8, blocks=[4, 1, 1], strides=[4, 1, 1], softmax_mode=True, normalize_offsets=True, use_unshared_regions=False, checkpoint=True),
                  keras.Similarity(8, checkpoint=True)):
        layer(x).square().sum().backward()
        want = torch.cat([p.grad.reshape(-1) for p in layer.parameters()])
        for p in layer.parameters():
            p.grad = None
        bucket = dp.GradBucket(layer.parameters())
        bucket.zero()
        layer(x).square().sum().backward()
        assert torch.allclose(bucket.flat[:want.numel()], want, rtol=1e-6, atol=1e-6 * float(want.abs().max()))


def test_tangents_are_refused_and_recorded_calls_run_again():
    import torch.autograd.forward_ad as forward_ad
    x, off = torch.randn(3, 16, 6, 8, device="cuda"), torch.randn(1, 20, 8, 1, 1, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            ck.mex_checkpointed(forward_ad.make_dual(x, torch.ones_like(x)), off, 20, **ATTRS)
        with pytest.raises(NotImplementedError):
            ck.checkpoint_pack(forward_ad.make_dual(x, torch.ones_like(x)))
    net = SimNet(SPECS["cfg3"], seed=1, checkpoint=128)
    image = torch.rand(3, 1, 28, 28, device="cuda") - 0.5
    traced = torch.jit.trace(net, (image,), check_trace=False)
    for v in (image, image * 0.5, torch.rand(5, 1, 28, 28, device="cuda") - 0.5):
        assert torch.allclose(traced(v), net(v), rtol=1e-6, atol=1e-6)
        g = torch.autograd.grad(traced(v).square().sum(), list(net.parameters()))
        for got, ref in zip(g, torch.autograd.grad(net(v).square().sum(), list(net.parameters()))):
            assert torch.allclose(got, ref, rtol=1e-5, atol=1e-5 * float(ref.abs().max()))


def test_on_another_stream_and_in_a_graph():
    torch.manual_seed(3)
    c = next(c for c in DISJOINT if c["name"] == "k64")
    off = torch.randn(4, 128, 64, 1, 1, device="cuda")
    dy = torch.randn(4, 128, 16, 16, device="cuda")
    x = torch.randn(c["shape"], device="cuda")
    attrs = cases.mex_attrs(c)

    def both():
        kept = ck.checkpoint_pack(x, 64)
        return (ck.checkpoint_unpack(kept),) + ck.mex_checkpoint_backward(kept, off, dy, 128, **attrs)
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                                          # two graphs share a pool: neither may lean on what the other left
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            outs = both()
        graphs.append((g, outs))
    keep = x.clone()
    for scale in (1.0, 0.5):
        x.copy_(keep * scale)
        want = [t.clone() for t in both()]
        for g, outs in graphs:
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_the_captured_data_parallel_step_takes_checkpoints():
    spec = SPECS["cfg5"]
    torch.manual_seed(4)
    net = SimNet(spec, seed=5, checkpoint=128)
    x, labels = torch.rand(8, 3, 32, 32, device="cuda") - 0.5, torch.arange(8, device="cuda") % 10
    net.loss(x, labels).backward()
    want = [p.grad.clone() for p in net.parameters()]
    for p in net.parameters():
        p.grad = None
    bucket = dp.GradBucket(net.parameters())
    step = dp.OverlappedStep(net, bucket, x, labels, 8)
    step.run()
    torch.cuda.synchronize()
    for p, ref in zip(net.parameters(), want):
        assert torch.allclose(p.grad, ref, rtol=1e-5, atol=1e-6 * float(ref.abs().max()))


def test_refusals_with_tensors_on_the_gpu():
    kept = ck.checkpoint_pack(torch.randn(2, 8, 4, 4, device="cuda"), 32)
    off, dy = torch.randn(1, 5, 8, 1, 1, device="cuda"), torch.randn(2, 5, 4, 4, device="cuda")
    call = lambda off=off, dy=dy, **kw: ck.mex_checkpoint_backward(kept, off, dy, 5, **dict(ATTRS, **kw))
    call()
    with pytest.raises(ValueError, match="offsets must have shape"):
        call(off=off[:, :4])
    with pytest.raises(ValueError, match="output_grad must have shape"):
        call(dy=dy[:1])
    with pytest.raises(TypeError):
        call(off=off.double())
    with pytest.raises(RuntimeError):
        call(flags=abi.FLAG_MEX_WORKSPACE_PRIMED)
    t = torch.randn(5, 8, 2, 2, device="cuda")
    with pytest.raises(ValueError, match="output_grad must have shape"):
        ck.similarity_checkpoint_backward(kept, t, t, dy, blocks=[2, 2], strides=[1, 1])
    with pytest.raises(TypeError):
        ck.similarity_checkpoint_backward(kept, t.double(), t.double(), torch.randn(2, 5, 3, 3, device="cuda"), blocks=[2, 2], strides=[1, 1])
