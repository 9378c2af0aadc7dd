"""What the 4-bit weight and distillation entry points refuse (checked before anything touches a device), the code layout
of the plain statement, and its gradient against differences."""
import ctypes

import numpy as np
import pytest

from hyacinth_b200 import api
from tests import w4_plain as P

FAKE = 1 << 20          # an address that is never dereferenced: every call below is refused or has nothing to do


def _lib():
    return api.load()


def _quantize(**kw):
    a = dict(wtype=api.F32, m=200, n=3, W=FAKE, ldw=200, seg=64, stype=api.F32, codes=FAKE, ldq=128, scales=FAKE, zeros=None, lds=4, R=None, ldr=0)
    a.update(kw)
    h = api.HyacinHandle()
    return _lib().hyacinB200QuantizeW4(ctypes.byref(h), a["wtype"], a["m"], a["n"], a["W"], a["ldw"], a["seg"], a["stype"], a["codes"],
                                       a["ldq"], a["scales"], a["zeros"], a["lds"], a["R"], a["ldr"])


def _product(**kw):
    a = dict(op=b"T", m=200, n=3, t=2, xtype=api.F16, codes=FAKE, ldq=128, seg=64, scales=FAKE, zeros=None, lds=4, X=FAKE, ldx=200, rank=0,
             U=None, ldu=0, V=None, ldv=0, Y=FAKE, ldy=3)
    a.update(kw)
    h = api.HyacinHandle()
    return _lib().hyacinB200ProductW4(ctypes.byref(h), a["op"], a["m"], a["n"], a["t"], a["xtype"], a["codes"], a["ldq"], a["seg"], a["scales"],
                                      a["zeros"], a["lds"], a["X"], a["ldx"], a["rank"], a["U"], a["ldu"], a["V"], a["ldv"], a["Y"], a["ldy"])


def _loss(**kw):
    a = dict(ztype=api.F16, n=100, t=2, Z=FAKE, ldz=100, k=4, ids=FAKE, teacher=FAKE, ldk=4, tau=1.0, lse=None, weight=None, loss=FAKE, stats=FAKE,
             dZ=None, lddz=0)
    a.update(kw)
    h = api.HyacinHandle()
    return _lib().hyacinB200DistillLoss(ctypes.byref(h), a["ztype"], a["n"], a["t"], a["Z"], a["ldz"], a["k"], a["ids"], a["teacher"], a["ldk"],
                                        a["tau"], a["lse"], a["weight"], a["loss"], a["stats"], a["dZ"], a["lddz"])


def _grad(**kw):
    a = dict(ztype=api.F16, n=100, t=2, Z=FAKE, ldz=100, k=4, ids=FAKE, teacher=FAKE, ldk=4, tau=1.0, lse=None, weight=None, stats=FAKE,
             dZ=FAKE + 4096, lddz=100)
    a.update(kw)
    h = api.HyacinHandle()
    return _lib().hyacinB200DistillGrad(ctypes.byref(h), a["ztype"], a["n"], a["t"], a["Z"], a["ldz"], a["k"], a["ids"], a["teacher"], a["ldk"],
                                        a["tau"], a["lse"], a["weight"], a["stats"], a["dZ"], a["lddz"])


@pytest.mark.parametrize("bad", [dict(wtype=api.F64), dict(stype=api.F32_COMPLEX), dict(m=-1), dict(n=-1), dict(seg=0), dict(seg=48), dict(seg=-32),
                                 dict(W=None), dict(codes=None), dict(scales=None), dict(ldw=199), dict(lds=3), dict(ldq=120), dict(ldq=64),
                                 dict(codes=FAKE + 8), dict(R=FAKE, ldr=199)])
def test_quantize_refuses(bad):
    assert _quantize(**bad) == -1


@pytest.mark.parametrize("bad", [dict(op=b"C"), dict(xtype=api.F64), dict(m=-1), dict(n=-1), dict(t=-1), dict(rank=-1), dict(seg=16), dict(codes=None),
                                 dict(scales=None), dict(X=None), dict(Y=None), dict(ldx=199), dict(ldy=2), dict(lds=3), dict(ldq=64), dict(ldq=132),
                                 dict(codes=FAKE + 4), dict(rank=2), dict(rank=2, U=FAKE, ldu=199, V=FAKE, ldv=3), dict(rank=2, U=FAKE, ldu=200, V=FAKE, ldv=2),
                                 dict(op=b"N", ldx=2), dict(op=b"N", ldx=3, ldy=199)])
def test_product_refuses(bad):
    assert _product(**bad) == -1


DISTILL_BAD = [dict(ztype=api.F64), dict(n=0), dict(n=(1 << 20) + 1, ldz=1 << 21, lddz=1 << 21), dict(t=-1), dict(k=-1), dict(k=1025, ldk=1025), dict(Z=None),
               dict(ldz=99), dict(ids=None), dict(teacher=None), dict(ldk=3), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("nan")), dict(tau=float("inf")),
               dict(dZ=FAKE + 4096, lddz=99), dict(dZ=FAKE, lddz=101)]


@pytest.mark.parametrize("bad", DISTILL_BAD)
def test_distill_refuses(bad):
    assert _loss(**bad) == -1
    assert _grad(**bad) == -1


def test_distill_grad_refuses_missing_buffers():
    assert _grad(stats=None) == -1
    assert _grad(dZ=None) == -1


def test_null_handle_is_refused():
    lib = _lib()
    assert lib.hyacinB200QuantizeW4(None, api.F32, 1, 1, FAKE, 1, 32, api.F32, FAKE, 64, FAKE, None, 1, None, 0) == -1
    assert lib.hyacinB200ProductW4(None, b"T", 1, 1, 1, api.F32, FAKE, 64, 32, FAKE, None, 1, FAKE, 1, 0, None, 0, None, 0, FAKE, 1) == -1
    assert lib.hyacinB200DistillLoss(None, api.F32, 1, 1, FAKE, 1, 0, None, None, 0, 1.0, None, None, FAKE, None, None, 0) == -1


def test_nothing_to_do_is_no_error():
    assert _quantize(m=0) == 0 and _quantize(n=0) == 0
    assert _product(t=0) == 0 and _product(n=0) == 0 and _product(op=b"N", m=0) == 0
    assert _loss(t=0) == 0 and _grad(t=0) == 0


def test_plain_layout_round_trip():
    rng = np.random.default_rng(0)
    assert sorted(P.row_of_nibble()) == list(range(128))
    for m in (1, 31, 32, 127, 128, 129, 300):
        codes = rng.integers(0, 16, (3, m), dtype=np.uint8)
        assert np.array_equal(P.unpack(P.pack(codes, -(-m // 128) * 64 + 16), m), codes)
    # word 4 c + i, nibble p + 4 h: rows 0 and 1 of a block share the lowest halves of word 0
    one = np.zeros((1, 128), dtype=np.uint8)
    one[0, 0], one[0, 1], one[0, 32], one[0, 8] = 1, 2, 3, 4
    word = P.pack(one, 64).view(np.uint32)[0]
    assert word[0] == 1 | (2 << 16) and word[1] == 3 and word[4] == 4


@pytest.mark.parametrize("tail", [False, True])
def test_plain_distillation_gradient_against_differences(tail):
    rng = np.random.default_rng(1)
    n, k, tau = 11, 4, 1.7
    z = rng.standard_normal((1, n)) * 2
    ids = np.array([[3, 7, 3, -1]])                     # one class twice, one entry skipped
    teacher = rng.standard_normal((1, k))
    lse = np.array([np.log(np.exp(teacher[0, :3] / tau).sum()) + 0.4]) if tail else None
    weight = np.array([1.3])
    _, grad, _ = P.distill(z, ids, teacher, tau, lse, weight)
    step = 1e-6                                         # central differences: error ~ step^2 + 1e-16 / step, 1e-9 is ample
    for j in range(n):
        d = np.zeros_like(z)
        d[0, j] = step
        diff = (P.distill(z + d, ids, teacher, tau, lse, weight)[0] - P.distill(z - d, ids, teacher, tau, lse, weight)[0]) / (2 * step)
        assert abs(diff[0] - grad[0, j]) < 2e-9


def test_pointers_off_their_boundary_and_sizes_beyond_the_largest_are_refused():
    for bad in (dict(W=FAKE + 2), dict(wtype=api.F16, W=FAKE + 1), dict(scales=FAKE + 2), dict(R=FAKE + 2, ldr=200), dict(m=0x7fffff80, ldw=0x7fffff80, seg=1 << 20, lds=4096, ldq=1 << 30)):
        assert _quantize(**bad) == -1
    factors = dict(rank=2, U=FAKE, ldu=200, V=FAKE, ldv=3)
    for bad in (dict(X=FAKE + 1), dict(Y=FAKE + 1), dict(scales=FAKE + 1), dict(factors, U=FAKE + 1), dict(factors, V=FAKE + 1), dict(factors, rank=(1 << 20) + 1), dict(t=0x7fffff80)):
        assert _product(**bad) == -1
    for bad in (dict(Z=FAKE + 1), dict(ids=FAKE + 2), dict(teacher=FAKE + 2), dict(lse=FAKE + 1), dict(weight=FAKE + 2), dict(stats=FAKE + 2), dict(dZ=FAKE + 4097, lddz=100)):
        assert _loss(**bad) == -1 and _grad(**bad) == -1
    assert _loss(loss=FAKE + 2) == -1


def test_refusals_name_their_reason(capfd):
    """Each refusal comes from the check of that argument, not from the last one (the handle's device), which stops every call here."""
    def message(call, bad):
        capfd.readouterr()
        assert call(**bad) == -1
        return capfd.readouterr().err

    marks = {f: [m for m in f.pytestmark if m.name == "parametrize"][0].args[1] for f in (test_quantize_refuses, test_product_refuses)}
    calls = [(_quantize, bad) for bad in marks[test_quantize_refuses]] + [(_product, bad) for bad in marks[test_product_refuses]]
    calls += [(call, bad) for bad in DISTILL_BAD for call in (_loss, _grad)] + [(_grad, dict(stats=None)), (_quantize, dict(W=FAKE + 2)), (_product, dict(rank=(1 << 20) + 1))]
    for call, bad in calls:
        err = message(call, bad)
        if bad in (dict(stats=None),):               # found after the device
            continue
        assert "hyacinB200" in err and "another device" not in err, (call.__name__, bad, err)
    import os
    if not os.path.exists("/dev/nvidiactl"):         # no GPU: the calls that are in order get as far as the device
        for call in (_quantize, _product, _loss, _grad):
            assert "another device" in message(call, {})
