"""Losses from feedback where they can go wrong: plans used at once, masks of
finite values, log ratios at the end of float64's range, and the like, against
plain float64 forms (feedback_util)."""
import numpy as np
import pytest

import feedback_util as fu

gpu = pytest.mark.gpu


# ------------------------------------------------------------------- plans

@gpu
@pytest.mark.parametrize("n,P,turns", [(96, 48, 200), (3000, 4000, 60), (60_000, 200_000, 12)])
def test_plan_is_there_for_any_stream(mtlib, n, P, turns):
    """A plan made from recycled memory and used at once on a stream that
    does not wait for the legacy one, which has work of its own meanwhile.
    Per pair, in float64: x rounds to |x| steps, exp is within 2 + |x| steps,
    then 1 + e, its inverse and three products, or a log1p within 2 steps and a
    sum; both here and there, so 4 (14 + 4 |x|) half steps of a value below
    1 + |x| hold.  A gradient adds a pair's in any order and rounds to float32."""
    import torch
    rng = np.random.default_rng(n)
    side = torch.cuda.Stream()
    s = torch.from_numpy(rng.normal(size=n)).cuda()
    sd = s.cpu().numpy()
    x = 2 * np.abs(sd).max()
    term = 4 * (14 + 4 * x) * 2.0 ** -53
    busy = torch.zeros(1 << 26, device="cuda")
    torch.cuda.synchronize()
    for turn in range(turns):
        i = rng.integers(0, n, size=P)
        j = (i + 1 + rng.integers(0, n - 1, size=P)) % n
        busy.add_(1.0)  # the legacy stream is behind
        plan = mtlib.PreferencePlan(i, j, n)
        with torch.cuda.stream(side):
            loss, grad, hess = mtlib.preference_loss(plan, s)
        side.synchronize()
        L, g, h = fu.pairs_loss(sd, None, i, j, None, 1.0, 0.0, "logistic")
        assert np.abs(loss.cpu().numpy() - L).max() <= term * (1 + x), turn
        G = np.zeros(n)
        np.add.at(G, i, g)
        np.add.at(G, j, -g)
        degree = np.bincount(np.concatenate([i, j]), minlength=n)
        tol = np.abs(G) * fu.U32 * 1.01 + degree * (term + degree * 2.0 ** -52)
        assert (np.abs(grad.cpu().numpy() - G) <= tol).all(), turn
