"""Log probabilities on both sides of every border at which sizes choose another number of warps a tile, or another kernel for rows; the checks are those of
test_likelihood_gpu.py."""
import numpy as np
import pytest
import torch

from simnets_tf_b200.ops.likelihood import log_probabilities
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


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f64"])
@pytest.mark.parametrize("top_k", [0, 5])
def test_rows_by_warps_and_by_streams(top_k, kind):
    """As many rows as are just enough for a warp each, and one fewer."""
    for classes in (513, 700, 2000, 4099):
        for of in (4,) if kind == torch.float32 else (2, 4):
            for rows in (-(-classes // of), -(-classes // of) - 1):
                x, labels = make((rows, classes), 1, "plain", kind, seed=rows)
                verify(x, labels, 1, top_k, True, torch.from_numpy(x).cuda())


def test_rows_of_two_to_the_24_logits():
    """float64 beyond the one border that counts logits: the answers of 2100 rows of 8000 by warps are those of half of them by streams."""
    x = torch.randn(2100, 8000, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(0))
    labels = torch.arange(2100, device="cuda")
    whole = log_probabilities(x, labels, 3, True)
    for at in (slice(0, 1050), slice(1050, 2100)):
        half = log_probabilities(x[at], labels[at], 3, True)
        assert bool((half.top_index == whole.top_index[at]).all())
        # log S of 8000 numbers, added up in two orders of chains of at most 8000 / 32 and what joins them: 300 units of S each, which are 300 of its logarithm,
        # and the same of the entropy's second sum, whose terms are below 8
        eps = torch.finfo(torch.float64).eps
        assert float((half.label - whole.label[at]).abs().max()) <= 600 * eps and float((half.top - whole.top[at]).abs().max()) <= 600 * eps
        assert float((half.entropy - whole.entropy[at]).abs().max()) <= 600 * 9 * eps
