"""Beam search's selection from scores that are no numbers, against the plain implementation."""
import numpy as np
import pytest

import paged_ref as R
import test_gpu_beam as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,vocab", [(1, 5), (4, 3000), (8, 2049), (32, 64)])
def test_finished_hypotheses_with_scores_that_are_no_numbers(gpu, width, vocab):
    """A NaN score of a finished hypothesis counts as -inf like every other total: it is still a continuation, the last."""
    x, scores = B.inputs(gpu, 3, width, vocab, "f32", width)
    done = np.zeros((3, width), np.int32)
    done[0] = 1
    done[1, ::2] = 1
    scores[0] = np.nan  # nothing else is left of this group
    scores[1, ::2] = np.nan
    scores[2, 0] = np.nan  # (one that goes on: all its totals are NaN)
    total, parents, tokens, ended = B.run(gpu, x, scores, done, vocab - 1)
    logits = x.float().numpy().reshape(3, width, vocab)
    for g in range(3):
        best, parent, token = R.beam(logits[g], np.where(np.isnan(scores[g]), -np.inf, scores[g]).astype(np.float32), done[g], vocab - 1)
        assert parents[g].tolist() == parent and tokens[g].tolist() == token
        assert np.array_equal(np.isneginf(total[g]), np.isneginf(best)) and not np.isnan(total[g]).any()
        assert ended[g].tolist() == [int(done[g, p] != 0 or t == vocab - 1) for p, t in zip(parent, token)]
