"""Log probabilities on both sides of every border at which sizes choose another number of warps a tile, or another kernel for rows; the checks are those of
test_likelihood_gpu.py."""
import numpy as np
import pytest
import torch

from test_likelihood_gpu import KINDS, make, verify

pytestmark = pytest.mark.gpu
MULTIPROCESSORS = 148


def _at(tiles):
    """Positions on both sides of a number of tiles of 32."""
    return (32 * tiles - 31, 32 * tiles + 1)


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("top_k", [0, 1, 4, 8, 16])
@pytest.mark.parametrize("classes", [96, 97, 128, 255, 256, 257, 512, 768])
def test_sixteen_warps_a_tile(classes, top_k, kind):
    for positions in (3, 32, 33, 100):
        x, labels = make((2, classes, positions), 1, "ties" if positions == 33 else "plain", kind, seed=classes)
        verify(x, labels, 1, top_k, True, torch.from_numpy(x).cuda())


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
def test_as_many_tiles_as_are_there_at_once(kind):
    """One and two rounds of sixteen warps a tile with as many classes as each wants, for answers and for gradients."""
    wave, wanted = (2, ((1, 97), (1, 256), (2, 256), (2, 768))) if kind == torch.float32 else (1, ((1, 97), (1, 256), (2, 512), (2, 1024)))
    for rounds, classes in wanted:
        for positions in _at(rounds * wave * MULTIPROCESSORS):
            x, labels = make((1, classes, positions), 1, "plain", kind, seed=rounds)
            verify(x, labels, 1, 3, True, torch.from_numpy(x).cuda())


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("classes", [15, 16, 31, 32, 64, 128])
def test_one_two_and_four_warps_a_tile(classes, kind):
    for ctas in (8, 16) if kind == torch.float32 else (3, 4, 6, 8, 16):
        if ctas * classes > 1024:               # (the restatement takes seconds for each)
            continue
        for positions in _at(ctas * MULTIPROCESSORS):
            x, labels = make((1, classes, positions), 1, "plain", kind, seed=classes)
            verify(x, labels, 1, 3, True, torch.from_numpy(x).cuda())


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("rows,classes", [(16384, 64), (17500, 130), (18900, 100), (18950, 64), (16384, 33)])
@pytest.mark.parametrize("top_k", [0, 5, 16])
def test_rows_of_some_classes_in_great_numbers(rows, classes, top_k, kind):
    x, labels = make((rows, classes), 1, "plain", kind, seed=rows)
    verify(x, labels, 1, top_k, True, torch.from_numpy(x).cuda())
