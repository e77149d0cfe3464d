"""Norms and clipping of gradients without a GPU: what their entry points refuse, and the restatement that the GPU tests compare with."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import plain_training as plain
from simnets_tf_b200 import abi
from simnets_tf_b200.ops.gradients import clip_gradients, gradient_norm


def test_arguments_are_checked():
    g = [torch.zeros(3), torch.zeros(2, 2)]
    for call in (gradient_norm, lambda t, **kw: clip_gradients(t, 1.0, **kw)):
        with pytest.raises(ValueError, match="order"):
            call(g, order=1)
        with pytest.raises(ValueError, match="no tensors"):
            call([])
        with pytest.raises(ValueError, match="no tensors"):
            call([None])
        with pytest.raises(TypeError, match="float32 and float64"):
            call([torch.zeros(3).half()])
        with pytest.raises(TypeError, match="dense"):
            call([torch.zeros(3, 3).to_sparse()])
        with pytest.raises(RuntimeError, match="no CPU kernels"):
            call(g)
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(lambda t: call([t]), (torch.zeros(3),))
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_gradients(g, bad)
    with pytest.raises(ValueError, match="one tensor for each"):
        clip_gradients(g, 1.0, out=[torch.zeros(3)])


def test_the_c_entry_points_check_before_they_launch(cuda_lib):
    one = C.c_void_p(256)                   # (never dereferenced: every call below is refused)
    ws = cuda_lib.simnets_gradient_norm_workspace_bytes(2)
    assert ws > 0 and cuda_lib.simnets_gradient_norm_workspace_bytes(-1) == 0

    def both(order=2, n=2, dtypes=(0, 1), counts=(5, 6), tensors=(256, 512), out=(256, 512), norm=one, w=one, size=ws, limit=1.0):
        d = (C.c_int32 * len(dtypes))(*dtypes) if dtypes is not None else None
        c = (C.c_int64 * len(counts))(*counts) if counts is not None else None
        t = (C.c_void_p * len(tensors))(*tensors) if tensors is not None else None
        o = (C.c_void_p * len(out))(*out) if out is not None else None
        return (cuda_lib.simnets_gradient_norm(order, n, d, c, t, norm, w, size, None), cuda_lib.simnets_clip_gradients(order, limit, n, d, c, t, o, norm, w, size, None))
    assert both(order=1) == both(n=-1) == both(counts=(-1, 6)) == (abi.E_DESC,) * 2
    assert both(dtypes=(0, 2)) == (abi.E_DTYPE,) * 2
    assert both(counts=None) == both(tensors=None) == both(norm=None) == both(tensors=(256, None)) == (abi.E_NULL,) * 2
    assert both(w=None) == both(size=ws - 1) == (abi.E_WORKSPACE,) * 2
    assert both(counts=(1 << 40, 1)) == both(tensors=(257, 512)) == both(tensors=(256, 516)) == (abi.E_UNSUPPORTED,) * 2
    assert both(out=(256, 516))[1] == abi.E_UNSUPPORTED
    assert both(size=ws - 1, limit=-1.0)[1] == both(size=ws - 1, limit=math.nan)[1] == abi.E_DESC
    assert both(size=ws - 1, out=None)[1] == abi.E_NULL


def test_the_workspace_grows_with_the_list(cuda_lib):
    sizes = [cuda_lib.simnets_gradient_norm_workspace_bytes(n) for n in (0, 1, 24, 25, 5000, 100000)]
    assert sizes == sorted(sizes) and sizes[0] > 0


def test_the_restatement_clips():
    g = [np.array([3.0, 0.0], np.float32), np.array([[4.0]], np.float32)]
    assert plain.norm(g) == 5 and plain.norm(g, math.inf) == 4
    n, c = plain.clipped(g, 1.0)
    assert n == 5 and np.allclose(c[0], [0.6, 0]) and np.allclose(c[1], 0.8)
    assert all((a == b).all() for a, b in zip(plain.clipped(g, 5.0)[1], g))
    g[0][1] = np.nan
    n, c = plain.clipped(g, 1.0)
    assert np.isnan(n) and (c[1] == 4).all()
    big = [np.full(4, 1e300)]
    assert float(plain.clipped(big, 1.0)[0]) == 2e300
