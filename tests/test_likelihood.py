"""Log probabilities without a GPU: what their entry points refuse, and the restatement that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest
import torch

import plain_training as plain
from simnets_tf_b200 import abi
from simnets_tf_b200.ops.likelihood import log_probabilities


def test_arguments_are_checked():
    x = torch.zeros(2, 12, 3)
    for kw in (dict(top_k=-1), dict(top_k=13), dict(top_k=1.5), dict(top_k=True), dict(axis=0), dict(axis=1.0), dict(axis=-3), dict(axis=7), dict(axis=2, top_k=4)):
        with pytest.raises(ValueError):
            log_probabilities(x, **kw)
    with pytest.raises(ValueError, match="0 to 16"):
        log_probabilities(torch.zeros(1, 40), top_k=17)
    for bad in (torch.zeros(4), torch.zeros(2, 0), torch.zeros(())):
        with pytest.raises(ValueError):
            log_probabilities(bad)
    with pytest.raises(TypeError, match="float32 and float64"):
        log_probabilities(x.half())
    with pytest.raises(RuntimeError, match="no CPU kernels"):
        log_probabilities(x, entropy=True)
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(lambda t: log_probabilities(t, entropy=True).entropy, (x,))


def test_the_c_entry_points_check_before_they_launch(cuda_lib):
    one = C.c_void_p(256)                   # (never dereferenced: every call below is refused, or has nothing to do)

    def both(logits=one, labels=one, label=one, index=one, top=one, stats=one, **kw):
        d = abi.LikelihoodDesc(**dict(dict(dtype=abi.F32, classes=12, top_k=2, batch=2, positions=9, stride_batch=108, stride_class=9, stride_position=1), **kw))
        return (cuda_lib.simnets_log_probabilities(C.byref(d), logits, labels, label, None, index, top, stats, None, 0, None),
                cuda_lib.simnets_log_probabilities_gradient(C.byref(d), logits, labels, stats, index, label, None, top, one, None))
    assert C.sizeof(abi.LikelihoodDesc) == 56
    assert both(dtype=2) == (abi.E_DTYPE,) * 2
    for kw in (dict(classes=0), dict(batch=-1), dict(positions=-1), dict(top_k=-1), dict(top_k=13), dict(stride_batch=-1), dict(stride_class=-9), dict(stride_position=-1),
               dict(top_k=0), dict(top=None, index=None)):
        assert both(**kw) == (abi.E_DESC,) * 2, kw
    for kw in (dict(classes=40, top_k=17), dict(classes=(1 << 30) + 1), dict(batch=1 << 17, positions=1 << 17), dict(classes=1 << 20, batch=1 << 12, positions=1 << 12)):
        assert both(**kw) == (abi.E_UNSUPPORTED,) * 2, kw
    assert both(logits=C.c_void_p(258)) == (abi.E_UNSUPPORTED,) * 2 and both(logits=C.c_void_p(260), dtype=abi.F64) == (abi.E_UNSUPPORTED,) * 2
    for kw in (dict(logits=None), dict(labels=None), dict(index=None)):
        assert both(**kw) == (abi.E_NULL,) * 2, kw
    assert both(stats=None)[1] == abi.E_NULL
    assert both(batch=0, logits=None) == (0, 0) and both(positions=0, logits=None) == (0, 0)
    # one long row is shared by several CTAs, which leave what they find in a workspace
    long_row = dict(classes=100000, batch=1, positions=1, stride_class=1)
    assert both(**long_row)[0] == abi.E_WORKSPACE
    d = abi.LikelihoodDesc(dtype=abi.F32, top_k=2, **long_row)
    assert cuda_lib.simnets_log_probabilities_workspace_bytes(C.byref(d)) > 0 == cuda_lib.simnets_log_probabilities_workspace_bytes(None)
    assert cuda_lib.simnets_log_probabilities(None, *[one] * 8, 0, None) == abi.E_NULL
    assert cuda_lib.simnets_log_probabilities_gradient(None, *[one] * 8, None) == abi.E_NULL


def test_the_restatement_agrees_with_differences_and_with_softmax():
    rng = np.random.default_rng(0)
    x = rng.normal(size=(6, 9)) * 2
    x[1, 3:] = -np.inf
    x[2] = -np.inf
    labels = np.array([0, 2, 3, -1, 9, 8])
    r = plain.Rows(x, labels, 3)
    t = torch.from_numpy(x).requires_grad_()
    keep = [0, 1, 3, 4, 5]
    l = torch.log_softmax(t, 1)
    want = torch.where(torch.from_numpy((labels >= 0) & (labels < 9)), l.gather(1, torch.from_numpy(np.clip(labels, 0, 8))[:, None])[:, 0], torch.zeros(6, dtype=torch.float64))
    p = l.exp()
    ent = -torch.where(p > 0, p * torch.where(p > 0, l, 0.0), 0.0).sum(1)
    assert np.allclose(r.label()[0][keep].astype(float), want.detach().numpy()[keep], rtol=1e-14) and r.label()[0][2] == -np.inf
    assert np.allclose(r.entropy[keep].astype(float), ent.detach().numpy()[keep], rtol=1e-13) and r.entropy[2] == 0
    top, index = t.topk(3, 1)
    assert np.array_equal(r.top_index[keep], index.numpy()[keep]) and (r.top_index[2] == -1).all()
    g = rng.normal(size=(3, 6, 3))
    (want[keep] * torch.from_numpy(g[0, keep, 0])).sum().backward(retain_graph=True)
    assert np.allclose(r.gradient(g_label=g[0, :, 0])[0][keep].astype(float), t.grad.numpy()[keep], atol=1e-14)
    eps = 1e-6
    dx = r.gradient(g[0, :, 0], g[1, :, 0], g[2])[0]
    for c in range(9):
        for i in keep:
            if x[i, c] == -np.inf:
                continue
            def total(v):
                y = x.copy()
                y[i, c] += v
                q = plain.Rows(y, labels, 3)
                lab, tp = q.label()[0][i], q.top()[0][i]
                return float(lab * g[0, i, 0] + q.entropy[i] * g[1, i, 0] + (np.where(np.isfinite(tp), tp, 0) * g[2, i]).sum())
            assert abs((total(eps) - total(-eps)) / (2 * eps) - float(dx[i, c])) < 1e-7
    assert (dx[2] == 0).all()
