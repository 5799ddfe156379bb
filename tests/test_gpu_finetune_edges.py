"""GPU tests at the edges of the fine-tuning operators, against definitions in float64 on the CPU: values past float32 inside a
loss, NaN that must show, gradients of unlikely classes, what a call keeps alive, and rows at any place.

Tolerances count roundings; U = 2^-24 is half a step of float32.
"""
import math

import pytest
import torch

from graphmaker_amd import autograd as ag
from test_gpu_finetune import DT, TYPES, U, check_norm, close, ratios, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return torch.device("cuda:0")


@pytest.mark.parametrize("offsets", [None, [0, 15, 40]])
def test_policy_loss_shows_nan_at_advantage_zero(dev, offsets):
    """A log-probability of NaN (a class outside the table) shows whatever its advantage, as r * 0 does; a masked one never."""
    M, at = 40, 7
    lp, old, _ = ratios(3, M)
    adv = torch.tensor([0.0, 1.0]) if offsets else torch.arange(M).float() - at
    kw = dict(offsets=torch.tensor(offsets, device=dev)) if offsets else {}

    def run(lp, old, **more):
        a = lp.to(dev).requires_grad_(True)
        loss, stats = ag.policy_loss(a, old.to(dev), adv.to(dev), **kw, **more)
        return loss.detach(), stats, torch.autograd.grad(loss, [a])[0]

    want = run(lp, old)
    assert all(t.isfinite().all() for t in want) and want[2][at] == 0
    for x, y in ((math.nan, -1.0), (-1.0, math.nan), (-1.0, -math.inf)):         # the last: a ratio of inf times 0
        bad, bad_old = lp.clone(), old.clone()
        bad[at], bad_old[at] = x, y
        loss, stats, dl = run(bad, bad_old)
        assert loss.isnan() and stats[0].isnan() and stats[2:].isfinite().all()
        assert dl[at].isnan() and dl[torch.arange(M, device=dev) != at].isfinite().all()
        mask = torch.arange(M, device=dev) != at
        assert all(t.isfinite().all() for t in run(bad, bad_old, mask=mask))
    for x, y in ((-math.inf, -1.0), (-1.0, -300.0), (-1.0, -3000.0)):            # a ratio of 0, and finite ones of any size
        fine, fine_old = lp.clone(), old.clone()
        fine[at], fine_old[at] = x, y
        for a, b in zip(run(fine, fine_old), want):
            assert torch.equal(a, b)
