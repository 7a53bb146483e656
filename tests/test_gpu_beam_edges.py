"""Beam search's selection and reordering at their edges, against the definitions of include/caten_hip.h in NumPy."""
import numpy as np
import pytest

from tests.test_gpu_beam import PAGE, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [1, 2, 5])
def test_infinite_scores_and_logits(K):
    """A score of infinity and a logit of infinity in one beam: the other tokens' scores, infinity less infinity, count as minus infinity."""
    from caten_amd import ops
    rng = np.random.default_rng(K)
    V = 700
    logits = rng.normal(0, 2, (3, K, V)).astype(np.float32)
    scores = np.full((3, K), -np.inf, np.float32)
    scores[0, 0] = scores[1] = scores[2, K - 1] = np.inf
    logits[0, 0, 7] = logits[1, 0, 9] = logits[1, 0, 600] = np.inf
    got = ops.beam_select(logits, scores)
    # one candidate of infinity, then beam 0's others from the highest logit down
    order = np.argsort(-logits[0, 0], kind="stable")[:K]
    assert np.array_equal(got["tokens"][0], order) and not got["parents"][0].any()
    assert got["scores"][0, 0] == np.inf and (got["scores"][0, 1:] == -np.inf).all()
    # all finite tokens of the other beams of request 1 are at infinity, behind beam 0's two in the order of beams
    best = [(0, 9), (0, 600)] + [(k, t) for k in range(1, K) for t in np.argsort(-logits[1, k], kind="stable")[:K]]
    if K > 1:
        assert [tuple(x) for x in zip(got["parents"][1], got["tokens"][1])] == best[:K] and (got["scores"][1] == np.inf).all()
    # an infinite score alone: the logits' order
    assert np.array_equal(got["tokens"][2], np.argsort(-logits[2, K - 1], kind="stable")[:K]) and (got["parents"][2] == K - 1).all()
