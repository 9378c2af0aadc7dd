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


def _by_logarithms(z, ids, teacher, tau, lse):
    """Loss, gradient and a scale for its errors in 64 bits, by log-sum-exp throughout, for distinct ids.  Probabilities are formed
    relative to the largest logit: at 1e30 the logarithm of their number would be lost beside it."""
    u = z.astype(np.float64) / tau

    def lsumexp(a):
        top = a.max(1, keepdims=True)
        return top[:, 0] + np.log(np.exp(a - top).sum(1))

    def softmax(a):
        e = np.exp(a - a.max(1, keepdims=True))
        return e / e.sum(1, keepdims=True)
    rows = np.arange(len(z))[:, None]
    score = teacher.astype(np.float64) / tau
    logp = score - (lsumexp(score) if lse is None else lse.astype(np.float64))[:, None]
    p = np.exp(logp)
    rest = np.zeros(len(z)) if lse is None else np.maximum(0, 1 - p.sum(1))
    total = lsumexp(u)
    inside = np.zeros(z.shape, dtype=bool)
    inside[rows, ids] = True
    outside = lsumexp(np.where(inside, -np.inf, u))
    loss = (p * (logp - (u[rows, ids] - total[:, None]))).sum(1)
    loss += np.where(rest > 0, rest * (np.log(np.where(rest > 0, rest, 1)) - (outside - total)), 0)
    q = softmax(u)
    target = np.zeros(z.shape)
    target[rows, ids] = p
    share = rest[:, None] * softmax(np.where(inside, -np.inf, u))
    mass = (p.sum(1) + rest)[:, None]
    return loss, (q * mass - target - share) / tau, (q * mass + target + share) / tau


@pytest.mark.parametrize("n,kind", [(300, "f32"), (5001, "bf16"), (60000, "f16"), (128000, "bf16"), (1 << 20, "f32")])
@pytest.mark.parametrize("tau,tail", [(1.0, False), (1.0, True), (0.7, True), (3.0, False)])
def test_logits_of_any_finite_size(hy, n, kind, tau, tail):
    """Everything outside the list at one mask value, down to the type's lowest; one class far above all others; classes a few
    places apart far from zero."""
    torch = _torch()
    rng = np.random.default_rng(n)
    t, k = 8, 6
    top = float(torch.finfo(P.kinds()[kind][0]).max)
    size = (lambda v: min(v, top))
    z, ids, teacher, lse = _problem(rng, n, t, k, kind, tau, False)
    if tail:                                         # the rest weighs a third of the listed classes
        lse = (np.log(np.exp(teacher.astype(np.float64) / tau).sum(1)) + np.log(4 / 3)).astype(np.float32)
    inside = np.zeros(z.shape, dtype=bool)
    inside[np.arange(t)[:, None], ids] = True
    for row, value in ((1, 1e9), (2, 1e10), (3, 1e30), (4, top)):
        z[row] = np.where(inside[row], z[row], -size(value))
    z[5, np.flatnonzero(~inside[5])[n // 3]] = size(1e10)
    z[6, np.flatnonzero(~inside[6])[n // 2]] = size(1e30)
    z[7] = np.where(rng.random(n) < 0.5, 3e9, 3e9 + 256) if kind == "f32" else z[7]
    z = P.round_to(z, kind)
    r = Run(hy, z, ids, teacher, tau, lse, None, kind)
    d = r.step()
    want_loss, want, scale = _by_logarithms(z, ids, teacher, tau, lse)
    loss, g = r.loss.double().cpu().numpy(), d[:, :n].double().cpu().numpy()
    fits = np.abs(want_loss) < np.finfo(np.float32).max
    assert np.isfinite(loss[fits]).all() and np.isposinf(loss[~fits]).all()
    assert (np.abs(loss - want_loss)[fits] <= (P.HALF_STEP["f32"] * np.abs(want_loss) + 4 * TERM)[fits]).all()
    tol = P.HALF_STEP[kind] * np.abs(want) + 4 * TERM * scale + P.TINY[kind]
    assert np.isfinite(g).all() and (np.abs(g - want) <= tol).all(), (np.abs(g - want) / tol).max(axis=1)
    once = r.dZ.clone()
    r.dZ.fill_(9.0)
    assert torch.equal(r.grad(), once)


@pytest.mark.parametrize("n,repeat", [(1, False), (5, False), (64, False), (1000, False), (40, True)])
def test_a_list_of_every_class_leaves_no_rest(hy, n, repeat):
    """With every class listed nothing is left to be one more outcome, however sum p rounds: the loss is that of the listed classes."""
    torch = _torch()
    rng = np.random.default_rng(n)
    t = 12
    z, ids, teacher, lse = _problem(rng, n, t, n, "f32", 1.0, True)
    if repeat:                                       # a class twice, none left out; another list leaves one out
        ids = np.concatenate([ids, ids[:, :1]], axis=1)
        teacher = np.concatenate([teacher, teacher[:, :1] - 30], axis=1).astype(np.float32)
        ids[1, 3] = ids[1, 2]
    lse = lse + np.float32(1e-6) * rng.integers(-1, 2, t).astype(np.float32)
    r = Run(hy, z, ids, teacher, 1.0, lse, None, "f32")
    d = r.step()
    loss, g = r.loss.double().cpu().numpy(), d.double().cpu().numpy()
    for row in range(t):
        if repeat and row == 1:
            want, grad, _ = P.distill(z[1:2], ids[1:2], teacher[1:2], 1.0, lse[1:2], None)
            assert abs(loss[1] - want[0]) <= 4 * TERM + 2.0 ** -24 * want[0]
            continue
        u = z[row] - z[row].max()
        logq = u - np.log(np.exp(u).sum())
        p = np.zeros(n)
        listed = np.exp(teacher[row].astype(np.float64) - float(lse[row]))
        np.add.at(p, ids[row], listed)
        want = (listed * (teacher[row].astype(np.float64) - float(lse[row]) - logq[ids[row]])).sum()
        assert abs(loss[row] - want) <= 4 * TERM + 2.0 ** -24 * abs(want), (row, loss[row], want)
        assert (np.abs(g[row] - (np.exp(logq) * p.sum() - p)) <= 4 * TERM * (np.exp(logq) + p) + 2.0 ** -24).all()
    once = d.clone()
    r.dZ.fill_(9.0)
    assert torch.equal(r.grad(), once)
