"""rlq_beam_select of so many groups that they take several launches."""
import numpy as np
import pytest

from rlq_loader import load
from test_gpu_kv import cuda, raises, say

pytestmark = pytest.mark.gpu

rlq = load()
torch = rlq.torch


@pytest.mark.parametrize("groups,beams,vocabulary,best", [(65535, 64, 2, 64), (65535, 3, 5, 4), (1025, 64, 3, 5), (65535, 1, 7, 7)])
def test_select_of_very_many_groups(groups, beams, vocabulary, best):
    """Every group's choice, an error in a group of the last launch, and a workspace of one launch's rows."""
    say("select groups", groups, beams, vocabulary, best)
    own = rlq.Context(0)
    rng = np.random.default_rng(beams)
    z = (rng.standard_normal((groups, beams, vocabulary)) * 2).astype(np.float32)
    z[rng.random(z.shape) < 0.05] = -np.inf
    z[..., 0] = rng.standard_normal((groups, beams))
    scores = (-5 * rng.random((groups, beams))).astype(np.float32)
    bad = groups - 17
    z[bad, beams - 1, 1] = np.nan
    logits, score = cuda(z), cuda(scores)
    out = [torch.full((groups, best), 9.0, device="cuda")] + \
          [torch.full((groups, best), 9, dtype=torch.int32, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    room = torch.cuda.mem_get_info()[0]
    own.beam_select(logits, score, best, out=out)
    with raises("NonFinite", 4, bad):
        own.sync()
    taken = room - torch.cuda.mem_get_info()[0]
    print("scratch", taken, flush=True)
    # 65535 rows of a launch at most, each of best + 2 words for its list and 2 best for its ranks; allocations may round up
    assert taken <= 65535 * (3 * best + 2) * 8 + (16 << 20)
    got, parents, tokens = (t.cpu().numpy() for t in out)
    assert (got[bad] == -np.inf).all() and (parents[bad] == -1).all() and (tokens[bad] == -1).all()
    z[bad] = 0
    r = z.astype(np.float64)
    rank = (scores.astype(np.float64)[..., None] + r - np.log(np.exp(r).sum(-1, keepdims=True))).reshape(groups, -1)
    want = -np.sort(-rank, 1)[:, :best]
    others = np.arange(groups) != bad
    some = want > -np.inf
    assert np.array_equal(parents[others] >= 0, some[others]) and np.array_equal(tokens[others] >= 0, some[others])
    place = np.where(some, parents.astype(np.int64) * vocabulary + tokens, -1 - np.arange(best))  # (no candidate: all different)
    place[bad] = np.arange(best)
    assert (np.diff(np.sort(place, 1), axis=1) > 0).all()  # nothing is chosen twice
    chosen = np.take_along_axis(rank, np.maximum(place, 0), 1)
    # the sum's exponentials are each within 2^-22, so two candidates closer than twice that may change places; a score is rounded once
    near = 2.0 ** -21
    at = some & others[:, None]
    assert (np.abs(chosen[at] - want[at]) <= near).all()
    assert (np.abs(got[at] - chosen[at]) <= 2.0 ** -24 * np.abs(chosen[at]) + near).all()
    assert (got[~some & others[:, None]] == -np.inf).all()
    own.close()
