"""Addresses that cannot hold what the C entry points read or write there are refused before anything is launched."""
import ctypes as C

import pytest

from simnets_tf_b200 import abi

AT = 4096                                   # (never dereferenced: every call below is refused)


@pytest.mark.parametrize("dtype", [abi.F32, abi.F64])
def test_log_probabilities(cuda_lib, dtype):
    size = 8 if dtype == abi.F64 else 4
    d = abi.LikelihoodDesc(dtype=dtype, classes=12, top_k=2, batch=2, positions=9, stride_batch=108, stride_class=9, stride_position=1)
    need = dict(logits=size, labels=8, label=size, entropy=size, top_index=4, top=size, stats=size, ws=8)
    order = list(need)
    for name in order:
        for off in {1, 2, need[name] // 2, need[name] - 1}:
            args = [C.c_void_p(AT + (off if n == name else 0)) for n in order]
            assert cuda_lib.simnets_log_probabilities(C.byref(d), *args, 0, None) == abi.E_UNSUPPORTED, (name, off)
    need = dict(logits=size, labels=8, stats=size, top_index=4, g_label=size, g_entropy=size, g_top=size, dlogits=size)
    order = list(need)
    for name in order:
        for off in {1, 2, need[name] // 2, need[name] - 1}:
            args = [C.c_void_p(AT + (off if n == name else 0)) for n in order]
            assert cuda_lib.simnets_log_probabilities_gradient(C.byref(d), *args, None) == abi.E_UNSUPPORTED, (name, off)


@pytest.mark.parametrize("dtypes,size", [((abi.F32, abi.F32), 4), ((abi.F32, abi.F64), 8), (None, 4)])
def test_norms(cuda_lib, dtypes, size):
    ws = cuda_lib.simnets_gradient_norm_workspace_bytes(2)
    types, counts = (C.c_int32 * 2)(*dtypes) if dtypes else None, (C.c_int64 * 2)(5, 6)
    tensors = (C.c_void_p * 2)(AT, 2 * AT)

    def both(norm=AT, w=AT):
        return (cuda_lib.simnets_gradient_norm(2, 2, types, counts, tensors, C.c_void_p(norm), C.c_void_p(w), ws, None),
                cuda_lib.simnets_clip_gradients(2, 1.0, 2, types, counts, tensors, tensors, C.c_void_p(norm), C.c_void_p(w), ws, None))
    for off in {1, 2, size // 2, size - 1}:
        assert both(norm=AT + off) == (abi.E_UNSUPPORTED,) * 2
    for off in (1, 4, 7):
        assert both(w=AT + off) == (abi.E_UNSUPPORTED,) * 2
