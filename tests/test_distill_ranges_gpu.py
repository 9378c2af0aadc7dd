"""Distillation loss at the ends of its range: NaN in live rows, logits of any finite size."""
import numpy as np
import pytest

from tests import w4_plain as P
from tests.test_distill_gpu import TERM, Run, _problem

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


# sizes whose rows lie in one CTA, in several of a cluster, and in none
@pytest.mark.parametrize("n,kind", [(300, "f32"), (5001, "bf16"), (128000, "bf16"), (60000, "f16"), (256000, "f32"), (1 << 20, "f32")])
@pytest.mark.parametrize("tail", [False, True])
def test_nan_in_a_row_spoils_its_loss_and_gradient(hy, n, kind, tail):
    """All of a row, all of it outside the list, a quarter of it, one entry, all listed classes, one listed class, all but them minus
    infinity: the softmax of each is NaN; the rows beside them are untouched."""
    torch = _torch()
    rng = np.random.default_rng(n)
    k, rows = 8, 9
    z, ids, teacher, lse = _problem(rng, n, rows, k, kind, 1.0, tail)
    r = Run(hy, z, ids, teacher, 1.0, lse, None, kind)
    r.step()
    clean, clean_loss = r.dZ.clone(), r.loss.clone()
    out = [np.setdiff1d(np.arange(n), ids[t]) for t in range(rows)]
    z[1, :] = np.nan
    z[2, out[2]] = np.nan
    quarter = np.arange(n // 4, n // 2)
    z[3, np.intersect1d(quarter, out[3])] = np.nan
    z[4, out[4][n // 2]] = np.nan
    z[5, ids[5]] = np.nan
    z[6, ids[6, 3]] = np.nan
    z[7, out[7]] = -np.inf
    z[7, ids[7]] = np.nan
    r = Run(hy, z, ids, teacher, 1.0, lse, None, kind)
    r.step()
    loss = r.loss.cpu().numpy()
    assert np.isnan(loss[1:8]).all(), loss
    assert bool(torch.isnan(r.dZ[1:8, :n]).all())
    for t in (0, 8):
        assert torch.equal(r.dZ[t], clean[t]) and torch.equal(r.loss[t], clean_loss[t])
    once = r.loss.clone()
    r.step(grad=False)
    assert np.isnan(r.loss.cpu().numpy()[1:8]).all() and torch.equal(r.loss[[0, 8]], once[[0, 8]])
    r.dZ.fill_(9.0)
    d = r.grad()
    assert bool(torch.isnan(d[1:8, :n]).all()) and torch.equal(d[0], clean[0])
