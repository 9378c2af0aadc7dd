"""Distillation loss and gradient on the GPU against the 64-bit statement."""
import numpy as np
import pytest

from tests import w4_plain as P

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


# A term exp2f((z - top) * log2(e) / tau): the difference, the constant and the product are each rounded once, relative 3 * 2^-24 of
# an exponent below 128 in magnitude, so 3 * 128 * ln 2 * 2^-24, plus 2 units of the function itself and the rounding of a
# 32-bit partial sum of at most 2^7 such terms per thread.
TERM = (3 * 128 * 0.6932 + 4 + 128) * 2.0 ** -24


def _problem(rng, n, t, k, kind, tau, tail, spread=3.0):
    z = P.round_to(rng.standard_normal((t, n)) * spread, kind)
    full = z + 0.5 * rng.standard_normal((t, n))
    kk = min(k, n)
    ids = np.full((t, k), -1, dtype=np.int32)
    ids[:, :kk] = np.argsort(-full, axis=1)[:, :kk]
    teacher = np.zeros((t, k), dtype=np.float32)
    teacher[:, :kk] = np.take_along_axis(full, ids[:, :kk].astype(np.int64), 1)
    lse = np.log(np.exp(full / tau - (full / tau).max(1, keepdims=True)).sum(1)) + (full / tau).max(1) if tail else None
    return z, ids, teacher, None if lse is None else lse.astype(np.float32)


class Run:
    def __init__(self, hy, z, ids, teacher, tau, lse, weight, kind, pad=0, shift=0):
        torch = _torch()
        self.hy, self.kind, self.tau = hy, kind, tau
        self.t, self.n = z.shape
        self.k = ids.shape[1]
        dt, self.code = P.kinds()[kind]
        self.ld = self.n + pad
        self.Z = torch.full((self.t * self.ld + shift,), float("nan"), dtype=dt, device="cuda")[shift:].view(self.t, self.ld)
        self.Z[:, :self.n] = torch.from_numpy(z).to(dt).cuda()
        self.dZ = torch.full((self.t * self.ld + shift,), 9.0, dtype=dt, device="cuda")[shift:].view(self.t, self.ld)
        self.ids = torch.from_numpy(np.ascontiguousarray(ids)).cuda()
        self.teacher = torch.from_numpy(np.ascontiguousarray(teacher)).cuda()
        self.lse = None if lse is None else torch.from_numpy(lse).cuda()
        self.weight = None if weight is None else torch.from_numpy(np.asarray(weight, dtype=np.float32)).cuda()
        self.loss = torch.full((self.t,), 3.0, device="cuda")
        self.stats = torch.zeros((self.t, 2), device="cuda")

    def step(self, in_place=False, loss=True, stats=True, grad=True):
        d = (self.Z if in_place else self.dZ) if grad else None
        rc = self.hy.distill_loss(self.code, self.n, self.t, self.Z, self.ld, self.k, self.ids, self.teacher, self.k, self.tau, self.lse, self.weight,
                                  self.loss if loss else None, self.stats if stats else None, d, self.ld)
        _torch().cuda.synchronize()
        assert rc == 0
        return d

    def grad(self):
        rc = self.hy.distill_grad(self.code, self.n, self.t, self.Z, self.ld, self.k, self.ids, self.teacher, self.k, self.tau, self.lse, self.weight,
                                  self.stats, self.dZ, self.ld)
        _torch().cuda.synchronize()
        assert rc == 0
        return self.dZ


def _check(r, z, ids, teacher, tau, lse, weight, d=None):
    want_loss, want, scale = P.distill(z, ids, teacher, tau, lse, weight)
    w = np.ones(r.t) if weight is None else np.abs(weight)
    got = r.loss.double().cpu().numpy()
    tol = P.HALF_STEP["f32"] * np.abs(want_loss) + 2 * TERM * w * 2
    fin = np.isfinite(want_loss)
    assert np.array_equal(got[~fin], want_loss[~fin])
    assert (np.abs(got[fin] - want_loss[fin]) <= tol[fin]).all(), (np.abs(got[fin] - want_loss[fin]) / tol[fin]).max()
    if d is None:
        return
    g = d[:, :r.n].double().cpu().numpy()
    tol = P.HALF_STEP[r.kind] * np.abs(want) + 2 * TERM * scale + P.TINY[r.kind]
    assert np.isfinite(g).all()
    assert (np.abs(g - want) <= tol).all(), (np.abs(g - want) / tol).max()


CASES = [  # n, t, k, kind, tau, tail, pad, shift
    (1, 1, 1, "f32", 1.0, False, 0, 0), (2, 3, 1, "f32", 1.0, True, 0, 0), (7, 4, 7, "f16", 0.7, False, 1, 0), (7, 4, 3, "bf16", 2.0, True, 0, 1),
    (100, 5, 8, "f32", 1.0, True, 3, 0), (1000, 6, 16, "bf16", 2.0, False, 0, 0), (1001, 6, 33, "f16", 1.0, True, 0, 0), (4096, 3, 64, "f32", 4.0, False, 0, 0),
    (8192, 9, 128, "bf16", 1.0, True, 8, 3), (50257, 4, 32, "f16", 1.0, True, 0, 0), (50257, 3, 1024, "f32", 0.5, True, 2, 1), (128000, 3, 64, "bf16", 2.0, False, 0, 0),
    (256000, 2, 50, "bf16", 1.0, True, 0, 5), (131071, 2, 20, "f32", 1.0, False, 0, 0), (1 << 20, 1, 40, "f32", 1.0, True, 0, 0), (300, 700, 5, "bf16", 1.0, True, 0, 0),
]


@pytest.mark.parametrize("n,t,k,kind,tau,tail,pad,shift", CASES)
def test_loss_and_gradient_against_the_definition(hy, n, t, k, kind, tau, tail, pad, shift):
    rng = np.random.default_rng(n + t)
    z, ids, teacher, lse = _problem(rng, n, t, k, kind, tau, tail)
    weight = P.round_to(rng.uniform(0.5, 1.5, t), "f32")
    r = Run(hy, z, ids, teacher, tau, lse, weight, kind, pad, shift)
    d = r.step()
    _check(r, z, ids, teacher, tau, lse, weight, d)
    assert (r.dZ[:, n:] == 9.0).all(), "entries behind the last class were written"
    one = r.dZ.clone()
    loss = r.loss.clone()
    # the gradient from the saved statistics, and in place of the logits, is the same to the bit
    r.dZ.fill_(9.0)
    assert _torch().equal(r.grad(), one)
    r.loss.fill_(0)
    r.step(grad=False)
    assert _torch().equal(r.loss, loss)
    d = r.step(in_place=True)
    assert _torch().equal(d[:, :n], one[:, :n]) and _torch().equal(r.loss, loss)


def test_ragged_lists_and_masked_tokens(hy):
    """Entries of -1 anywhere, lists that are empty, ids out of range, a class listed twice, tokens of weight 0 that hold NaN."""
    rng = np.random.default_rng(2)
    n, t, k = 500, 10, 12
    for tail in (False, True):
        z, ids, teacher, lse = _problem(rng, n, t, k, "f32", 1.5, tail)
        ids[0, :] = -1
        ids[1, ::2] = -1
        ids[2, 3] = n
        ids[2, 4] = 2 ** 31 - 1
        ids[2, 5] = -(2 ** 31)
        ids[3, 7] = ids[3, 2]
        ids[3, 9] = ids[3, 2]
        if tail:
            lse += 1.0                                               # keeps sum p below one with the doubled entries
        weight = np.ones(t)
        weight[[4, 9]] = 0
        spoiled = z.copy()
        spoiled[4, :] = np.nan
        r = Run(hy, spoiled, ids, teacher, 1.5, lse, weight, "f32")
        d = r.step()
        z[4] = 0
        _check(r, z, ids, teacher, 1.5, lse, weight, d)
        assert (d[[4, 9]] == 0).all() and (r.loss[[4, 9]] == 0).all()
        assert np.isnan(r.stats[[4, 9]].cpu().numpy()).all()
        if not tail:
            assert r.loss[0] == 0 and (d[0] == 0).all()


def test_infinite_logits(hy):
    """Masked classes (-inf) get probability 0; a listed class that the student rules out costs infinity with a finite gradient; a
    teacher that rules a class out ignores it; a row without any class left."""
    rng = np.random.default_rng(4)
    n, t, k = 300, 6, 8
    for tail in (False, True):
        z, ids, teacher, lse = _problem(rng, n, t, k, "f32", 1.0, tail)
        free = np.setdiff1d(np.arange(n), ids[0])
        z[0, free[:200]] = -np.inf
        z[1, ids[1, 2]] = -np.inf
        teacher[2, 3] = -np.inf
        z[2, ids[2, 3]] = -np.inf
        z[3, :] = -np.inf
        z[4, np.setdiff1d(np.arange(n), ids[4])] = -np.inf           # only listed classes are left
        low = np.finfo(np.float32).min
        z[5, free[:100]] = low                                       # a mask of the type's lowest value
        r = Run(hy, z, ids, teacher, 1.0, lse, None, "f32")
        d = r.step()
        _check(r, z, ids, teacher, 1.0, lse, None, d)
        assert np.isposinf(r.loss[1].item()) and np.isposinf(r.loss[3].item())
        first = d.clone()
        assert _torch().equal(r.grad(), first)


def test_far_apart_and_nearly_agreeing(hy):
    """Outside mass of e^-60 next to the listed classes, logits of +-1e4, and a student that equals the teacher."""
    rng = np.random.default_rng(6)
    n, k = 2000, 4
    z = P.round_to(rng.standard_normal((4, n)), "f32")
    ids = np.tile(np.array([5, 17, 900, 1999], dtype=np.int32), (4, 1))
    z[0, ids[0]] += 60
    z[1] = P.round_to(z[1] * 3000, "f32")
    z[2, ids[2]] += 20
    teacher = np.take_along_axis(z, ids.astype(np.int64), 1).astype(np.float32)
    teacher[0] -= 50
    lse = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1)
    lse[0] = np.log(np.exp(teacher[0]).sum() + 1e3)
    lse = lse.astype(np.float32)
    r = Run(hy, z, ids, teacher, 1.0, lse, None, "f32")
    d = r.step()
    want_loss, want, scale = P.distill(z, ids, teacher, 1.0, lse, None)
    g = d.double().cpu().numpy()
    # exponents reach 3 * 12000 * 1.44 here: relative 3 * 2^16 * ln 2 * 2^-24 where a term counts at all (exponent > -150)
    assert (np.abs(g - want) <= 2 * TERM * 2 * scale + 1e-37).all()
    assert (np.abs(r.loss.double().cpu().numpy() - want_loss) <= 4 * TERM + 2.0 ** -24 * np.abs(want_loss)).all()


def test_gradient_against_differences_of_the_loss(hy):
    """Central differences of the GPU's own loss, summed over many classes along random directions."""
    torch = _torch()
    rng = np.random.default_rng(9)
    n, t, k = 64, 1, 6
    for tail in (False, True):
        z, ids, teacher, lse = _problem(rng, n, t, k, "f32", 1.3, tail, spread=1.0)
        d = Run(hy, z, ids, teacher, 1.3, lse, None, "f32").step().double().cpu().numpy()[0]
        for _ in range(4):
            direction = rng.standard_normal(n)
            step = 2.0 ** -6
            up, down = [P.round_to(z + s * step * direction, "f32") for s in (1, -1)]
            losses = []
            for zz in (up, down):
                r = Run(hy, zz, ids, teacher, 1.3, lse, None, "f32")
                r.step(grad=False)
                losses.append(r.loss.item())
            # third derivatives of order 1 along a direction of length ~8: step^2 / 6 * 8^3 = 0.02; losses in 32 bits: 1e-6 / 2^-5
            assert abs((losses[0] - losses[1]) - ((up - down)[0] * d).sum()) / (2 * step) < 0.03


def test_captured_and_replayed():
    torch = _torch()
    from hyacinth_b200 import api
    rng = np.random.default_rng(12)
    n, t, k = 3001, 5, 10
    stream = torch.cuda.Stream()
    with api.Hyacin(stream=stream.cuda_stream) as h:
        data = [_problem(rng, n, t, k, "bf16", 1.0, True) for _ in range(2)]
        r = Run(h, *[data[0][0], data[0][1], data[0][2]], 1.0, data[0][3], None, "bf16")
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            r.step()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                assert h.distill_loss(r.code, n, t, r.Z, n, k, r.ids, r.teacher, k, 1.0, r.lse, None, r.loss, r.stats, r.dZ, n) == 0
                assert h.distill_grad(r.code, n, t, r.Z, n, k, r.ids, r.teacher, k, 1.0, r.lse, None, r.stats, r.Z, n) == 0
            for z, ids, teacher, lse in data[::-1]:
                r.Z.copy_(torch.from_numpy(z)); r.ids.copy_(torch.from_numpy(ids)); r.teacher.copy_(torch.from_numpy(teacher)); r.lse.copy_(torch.from_numpy(lse))
                g.replay()
                stream.synchronize()
                _check(r, z, ids, teacher, 1.0, lse, None, r.dZ)
                assert torch.equal(r.Z, r.dZ)
        del g
