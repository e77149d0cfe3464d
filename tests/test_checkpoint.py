"""8-bit checkpoints without a GPU: what their entry points refuse, what the layers take, the restatement's own properties."""
import ctypes as C

import numpy as np
import pytest
import torch

import plain_operators as plain
from simnets_tf_b200 import _lib, abi, keras
from simnets_tf_b200.ops import checkpoint as ck


def _checkpoint(shape=(2, 3, 4, 4), group=32, dtype=torch.float32):
    n = int(np.prod(shape))
    return ck.Checkpoint(torch.zeros(n, dtype=torch.uint8), torch.zeros(-(-n // group), 2, dtype=dtype), shape, group)


@pytest.mark.parametrize("group", [0, 1, 16, 33, 512, True, None, "128"])
def test_other_groups_are_refused(group):
    with pytest.raises(ValueError, match="group"):
        ck.checkpoint_pack(torch.zeros(4), group=group)
    with pytest.raises(ValueError, match="group"):
        ck.Checkpoint(torch.zeros(4, dtype=torch.uint8), torch.zeros(1, 2), (4,), group)
    if group is not None and group is not True:
        with pytest.raises(ValueError, match="group"):
            keras.Mex(num_instances=3, checkpoint=group)


def test_codes_and_ranges_must_belong_to_the_shape():
    codes, ranges = torch.zeros(96, dtype=torch.uint8), torch.zeros(3, 2)
    assert ck.Checkpoint(codes, ranges, (2, 3, 4, 4), 32).nbytes() == 96 + 24
    for c, r, s, g in ((codes[:95], ranges, (2, 3, 4, 4), 32), (codes, ranges[:2], (2, 3, 4, 4), 32), (codes, ranges, (2, 3, 4, 5), 32), (codes, ranges, (2, 3, 4, 4), 64),
                       (codes, ranges.view(2, 3), (2, 3, 4, 4), 32), (codes, ranges, (-2, -48), 32)):
        with pytest.raises(ValueError, match="checkpoint"):
            ck.Checkpoint(c, r, s, g)
    with pytest.raises(TypeError, match="uint8"):
        ck.Checkpoint(codes.char(), ranges, (2, 3, 4, 4), 32)
    with pytest.raises(TypeError, match="float32 and float64"):
        ck.Checkpoint(codes, ranges.half(), (2, 3, 4, 4), 32)


def test_other_types_and_cpu_tensors_are_refused():
    with pytest.raises(TypeError, match="float32 and float64"):
        ck.checkpoint_pack(torch.zeros(4, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no CPU kernels"):
        ck.checkpoint_pack(torch.zeros(4))
    with pytest.raises(RuntimeError, match="no CPU kernels"):
        ck.checkpoint_unpack(_checkpoint())
    with pytest.raises(RuntimeError, match="no CPU kernels"):
        ck.mex_checkpoint_backward(_checkpoint(), torch.zeros(1, 5, 3, 1, 1), torch.zeros(2, 5, 4, 4), 5, blocks=[3, 1, 1], use_unshared_regions=False)
    with pytest.raises(RuntimeError, match="no CPU kernels"):
        ck.similarity_checkpoint_backward(_checkpoint(), torch.zeros(5, 3, 2, 2), torch.zeros(5, 3, 2, 2), torch.zeros(2, 5, 3, 3), blocks=[2, 2], strides=[1, 1])


def test_gradients_refuse_other_shapes():
    with pytest.raises(ValueError, match="4-D"):
        ck.mex_checkpoint_backward(_checkpoint((96,)), torch.zeros(1, 5, 3, 1, 1), torch.zeros(2, 5, 4, 4), 5)
    with pytest.raises(ValueError, match="4-D"):
        ck.similarity_checkpoint_backward(_checkpoint((6, 16)), torch.zeros(5, 3, 2, 2), torch.zeros(5, 3, 2, 2), torch.zeros(2, 5, 3, 3))
    with pytest.raises(ValueError, match="channels"):
        ck.similarity_checkpoint_backward(_checkpoint(), torch.zeros(5, 2, 2, 2), torch.zeros(5, 2, 2, 2), torch.zeros(2, 5, 3, 3), blocks=[2, 2])
    with pytest.raises(ValueError):
        ck.mex_checkpoint_backward(_checkpoint(), torch.zeros(1, 5, 9, 1, 1), torch.zeros(2, 5, 4, 4), 5, blocks=[9, 1, 1])


def test_the_c_entry_points_check_before_they_launch(cuda_lib):
    one = C.c_void_p(256)                   # (never dereferenced: every call below is refused)
    assert [cuda_lib.simnets_checkpoint_groups(n, 64) for n in (0, 1, 64, 65)] == [0, 1, 1, 2]
    for f in (cuda_lib.simnets_checkpoint_pack, cuda_lib.simnets_checkpoint_unpack):
        assert f(7, 10, 64, one, one, one, None) == abi.E_DTYPE
        assert f(abi.F32, -1, 64, one, one, one, None) == abi.E_DESC
        assert f(abi.F32, 10, 48, one, one, one, None) == abi.E_DESC
        assert f(abi.F32, 10, 64, None, one, one, None) == abi.E_NULL
        assert f(abi.F32, 0, 64, None, None, None, None) == abi.OK
    d = abi.make_mex_desc((2, 4, 6, 6), 5, blocks=(4, 1, 1), strides=(4, 1, 1), use_unshared_regions=False)
    need = cuda_lib.simnets_mex_checkpoint_workspace_bytes(C.byref(d))
    call = lambda group=64, codes=one, dx=one, doff=one, ws=one, n=need: cuda_lib.simnets_mex_checkpoint_gradients(
        C.byref(d), group, codes, one, one, one, dx, doff, ws, n, None)
    assert need > 0
    assert call(group=63) == abi.E_DESC and call(codes=None) == abi.E_NULL and call(dx=None, doff=None) == abi.E_NULL
    assert call(ws=None) == abi.E_WORKSPACE and call(n=need - 1) == abi.E_WORKSPACE
    for flag in (abi.FLAG_MEX_WORKSPACE_PRIMED, abi.FLAG_MEX_MAXIMA_GIVEN):
        d.flags = flag
        assert call() == abi.E_UNSUPPORTED
    s = abi.make_sim_desc((2, 4, 6, 6), 5)
    need = cuda_lib.simnets_similarity_checkpoint_workspace_bytes(C.byref(s))
    call = lambda group=64, dx=one, dt=one, dw=one, n=need: cuda_lib.simnets_similarity_checkpoint_gradients(
        C.byref(s), group, one, one, one, one, one, dx, dt, dw, one, n, None)
    assert call(group=0) == abi.E_DESC and call(dt=None) == abi.E_NULL and call(dx=None, dt=None, dw=None) == abi.E_NULL and call(n=need - 1) == abi.E_WORKSPACE


def test_layers_take_a_group_and_tell_it():
    assert keras.Mex(num_instances=3).checkpoint is None and "checkpoint" not in keras.Mex(num_instances=3).get_config()
    assert keras.Mex(num_instances=3, checkpoint=False).checkpoint is None
    for l in (keras.Mex(num_instances=3, checkpoint=True), keras.Similarity(num_instances=3, checkpoint=64)):
        assert l.get_config()["checkpoint"] == l.checkpoint == (128 if isinstance(l, keras.Mex) else 64)
        assert type(l)(**l.get_config()).checkpoint == l.checkpoint


@pytest.mark.parametrize("kind", [np.float32, np.float64])
def test_the_restatement_is_within_half_a_step(kind):
    rng = np.random.default_rng(0)
    x = (rng.normal(size=1000) * 3 - 40).astype(kind)
    x[5:37:3], x[40], x[41] = np.nan, np.inf, -np.inf
    codes, ranges = plain.pack(x, 64)
    v = plain.unpack(codes, ranges, x.shape, 64)
    fine = np.isfinite(x)
    assert np.array_equal(np.isnan(v), np.isnan(x)) and v[40] == np.inf and v[41] == -np.inf
    step = ranges[np.arange(1000) // 64, 1].astype(np.float64)
    # half a step; the roundings of x / 2 - base / 2, of 2 / step (each half a unit of at most 126 and 252 steps) and of the value
    eps = np.finfo(kind).eps
    assert (np.abs(v[fine] - x[fine]) <= (0.5 + 252 * eps) * step[fine] + eps * np.abs(x[fine])).all()
