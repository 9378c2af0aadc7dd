"""4-bit weight matrices at the ends of their ranges: segments, magnitudes, infinities, rows behind the last one, errors of other calls."""
import numpy as np
import pytest

from tests import w4_plain as P
from tests.test_w4_gpu import _back, _check_product, _dev, _problem, _run_product

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


# ---- segments -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("op,t", [("T", 1), ("T", 20), ("T", 300), ("N", 1), ("N", 20), ("N", 300)])
@pytest.mark.parametrize("m,seg", [(4096, 0x7fffffe0), (200, 0x7fffff80), (33, 0x7fffffe0), (4096, 0x40000000)])
def test_one_scale_per_column_by_the_largest_segments(hy, op, t, m, seg):
    """M + segM beyond 2^31: one segment per column all the same."""
    rng = np.random.default_rng(m + t)
    n = 96
    for kind, zeros in (("bf16", True), ("f16", False), ("f32", True)):
        codes, scales, zp = _problem(rng, m, n, seg, kind, zeros)
        assert scales.shape[1] == 1
        x = P.round_to(rng.standard_normal((t, m if op == "T" else n)), kind)
        got = _run_product(hy, op, m, n, t, kind, seg, codes, scales, zp, x)
        _check_product(got, op, m, n, kind, seg, codes, scales, zp, x)


# ---- the correction apart from the main sum ---------------------------------------------------------------------------
def _correction_only(hy, op, kind, rank, t, exponents, m=512, n=200):
    """All scales zero: Y = second (first^T x).  first and x hold whole numbers below 2^10 and 2^3 times powers of two, so every sum of
    first^T x is a whole number below 2^10 2^3 512 = 2^22 times a power of two, exact in 32 bits."""
    e_first, e_x, e_second = exponents
    rng = np.random.default_rng(rank + t)
    inn = m if op == "T" else n
    codes, scales, _ = _problem(rng, m, n, 128, kind, False)
    scales[:] = 0
    most = 128 if kind == "bf16" else 1024
    first = rng.integers(-most, most, (rank, inn)) * 2.0 ** e_first
    second = rng.integers(-most, most, (rank, n if op == "T" else m)) * 2.0 ** e_second / most
    x = rng.integers(-7, 8, (t, inn)) * 2.0 ** e_x
    for v in (first, second, x):
        assert np.array_equal(P.round_to(v, kind), v)
    u, v = (first, second) if op == "T" else (second, first)
    got = _run_product(hy, op, m, n, t, kind, 128, codes, scales, None, x, u, v)
    mid = x @ first.T
    assert np.abs(mid).max() < 2.0 ** (24 + e_first + e_x)
    want, mag = mid @ second, np.abs(mid) @ np.abs(second)
    # mid in parts of 8 bits: three for half (what is left of second times the third is 2^-24 of the magnitude), two for bfloat16; one
    # rounding by a place of the largest term, 2^-23, for each of at most five addends per entry of the rank (padded to 16) and the
    # joining of the shares; then the rounding of Y
    lost = {"f16": 2.0 ** -23, "bf16": 2.0 ** -15, "f32": 0.0}[kind]
    tol = P.HALF_STEP[kind] * np.abs(want) + (lost + (5 * (-(-rank // 16) * 16) + 32) * 2.0 ** -23) * mag + P.TINY[kind]
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    return mid


@pytest.mark.parametrize("op,t", [("T", 4), ("T", 20), ("T", 200), ("N", 3), ("N", 20), ("N", 200)])
@pytest.mark.parametrize("rank", [1, 16, 40, 64, 100])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_correction_beyond_the_ends_of_its_type(hy, op, t, rank, kind):
    """first^T x above the largest half (65504) and far below the smallest, with a Y that a half holds."""
    mid = _correction_only(hy, op, kind, rank, t, (3, 1, -12))
    assert np.abs(mid).max() > 65504
    mid = _correction_only(hy, op, kind, rank, t, (-24, -8, 9))
    assert np.abs(mid).max() < 2.0 ** -10 and np.median(np.abs(mid)) < 2.0 ** -14


@pytest.mark.parametrize("op,t", [("T", 2), ("T", 20), ("N", 20)])
def test_correction_of_an_infinite_entry_stays_infinite(hy, op, t):
    """An infinite first^T x gives infinities of the second factor's signs where that is not zero."""
    rng = np.random.default_rng(5)
    m, n, rank = 256, 200, 3
    for kind in ("bf16", "f16", "f32"):
        codes, scales, _ = _problem(rng, m, n, 128, kind, False)
        scales[:] = 0
        inn, out = (m, n) if op == "T" else (n, m)
        first, second = np.abs(rng.integers(1, 9, (rank, inn))) * 1.0, P.round_to(rng.standard_normal((rank, out)), kind)
        second[1:] = 0
        first[1:] = 0
        x = np.ones((t, inn))
        first[0, 7] = np.inf
        u, v = (first, second) if op == "T" else (second, first)
        got = _run_product(hy, op, m, n, t, kind, 128, codes, scales, None, x, u, v)
        want = np.where(second[0] != 0, np.inf * np.sign(second[0]), np.nan)
        assert np.array_equal(got, np.tile(want, (t, 1)), equal_nan=True)


# ---- few vectors: nothing but Y is rounded ------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,m,bits", [("f16", 512, 10), ("f16", 500, 10), ("f16", 4096, 7), ("bf16", 512, 7), ("bf16", 4000, 7)])
@pytest.mark.parametrize("seg", [128, 64, 32, 96, 512])
@pytest.mark.parametrize("t,zeros", [(1, False), (3, True), (8, False)])
def test_few_vectors_of_one_sign_are_exact(hy, kind, m, bits, seg, t, zeros):
    """x = 1 + k 2^-bits, scales of 1: every product is a multiple of 2^-bits and every sum of them, at most 15 * 2 * M, a 32-bit
    number, so Y is the exact sum, rounded once."""
    rng = np.random.default_rng(m + seg + t)
    n = 150
    codes, scales, zp = _problem(rng, m, n, seg, kind, zeros)
    scales[:] = 1
    x = 1 + rng.integers(0, 1 << bits, (t, m)) * 2.0 ** -bits
    assert 30 * m * 2 ** bits <= 2 ** 24 and np.array_equal(P.round_to(x, kind), x)
    got = _run_product(hy, "T", m, n, t, kind, seg, codes, scales, zp, x)
    want = x @ P.values(codes, scales, zp, seg).T
    assert np.array_equal(got, P.round_to(want, kind))


@pytest.mark.parametrize("t", [1, 5, 8])
@pytest.mark.parametrize("seg", [32, 64, 128])
def test_few_vectors_with_an_entry_near_the_end_of_the_range(hy, t, seg):
    """One entry of 2^122 beside zeros: fifteen times it is a 32-bit number, and so is every step on the way."""
    rng = np.random.default_rng(t)
    m, n = 384, 48
    codes, scales, zp = _problem(rng, m, n, seg, "bf16", True)
    scales[:] = 2.0 ** -100
    x = np.zeros((t, m))
    x[:, 77] = 2.0 ** 122
    got = _run_product(hy, "T", m, n, t, "bf16", seg, codes, scales, zp, x)
    assert np.array_equal(got, x @ P.values(codes, scales, zp, seg).T)


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("t", [1, 4, 20, 140])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_an_infinite_entry_gives_infinities_of_the_weights_signs(hy, op, t, kind):
    """For every number of vectors the same: infinity times the sign of the weight, NaN where the weight is zero."""
    rng = np.random.default_rng(t)
    m, n, seg = 200, 150, 32
    for zeros in (False, True):
        codes, scales, zp = _problem(rng, m, n, seg, kind, zeros)
        x = P.round_to(rng.standard_normal((t, m if op == "T" else n)), kind)
        x[0, 17] = -np.inf
        got = _run_product(hy, op, m, n, t, kind, seg, codes, scales, zp, x)
        w = P.values(codes, scales, zp, seg)
        w = w[:, 17] if op == "T" else w[17]
        assert np.array_equal(got[0], np.where(w == 0, np.nan, -np.inf * np.sign(w)), equal_nan=True)
        assert np.isfinite(got[1:]).all()


# ---- rows behind the last one ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [1, 8, 9, 20, 200])
@pytest.mark.parametrize("m", [1, 7, 33, 135, 200, 253])
@pytest.mark.parametrize("seg", [32, 128])
def test_rows_behind_the_last_one_do_not_count_whatever_their_scale(hy, t, m, seg):
    """A segment whose weights reach 60000: the stored 0 of a row that does not exist stands for -8 s, beyond the largest half."""
    torch = _torch()
    from hyacinth_b200 import api
    rng = np.random.default_rng(m)
    n = 40
    w = P.round_to(rng.standard_normal((n, m)), "f16")
    w[:, -1] = 60000
    segs, ldq = -(-m // seg), -(-m // 128) * 64
    W = _dev(w, "f16")
    Q = torch.zeros((n, ldq), dtype=torch.uint8, device="cuda")
    S = torch.zeros((n, segs), dtype=torch.float16, device="cuda")
    assert hy.quantize_w4(api.F16, m, n, W, m, seg, api.F16, Q, ldq, S, None, segs, None, 0) == 0
    x = P.round_to(rng.standard_normal((t, m)) * 0.1, "f16")
    X, Y = _dev(x, "f16"), torch.zeros((t, n), dtype=torch.float16, device="cuda")
    assert hy.product_w4("T", m, n, t, api.F16, Q, ldq, seg, S, None, segs, X, m, 0, None, 0, None, 0, Y, n) == 0
    torch.cuda.synchronize()
    _check_product(_back(Y, n), "T", m, n, "f16", seg, P.unpack(Q.cpu().numpy(), m), _back(S, segs), None, x)


# ---- errors of other calls --------------------------------------------------------------------------------------------------
def test_an_earlier_error_is_not_reported_again(hy, capfd):
    """A product whose scratch nobody can allocate (2^20 x 2^29 numbers) returns -3 before anything is launched; the next calls succeed."""
    torch = _torch()
    from hyacinth_b200 import api
    n, m = 4, 128
    W = torch.ones((n, m), device="cuda")
    Q, S = torch.zeros((n, 64), dtype=torch.uint8, device="cuda"), torch.zeros((n, 1), device="cuda")
    Y, loss = torch.zeros((1, n), device="cuda"), torch.zeros(1, device="cuda")
    ids, teacher, stats = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros((1, 1), device="cuda"), torch.zeros((1, 2), device="cuda")

    def fail():
        assert hy.product_w4("N", m, n, 1 << 29, api.F32, Q, 64, 128, S, None, 1, W, m, 1 << 20, W, m, W, n, Y, m) == -3
    calls = [lambda: hy.quantize_w4(api.F32, m, n, W, m, 128, api.F32, Q, 64, S, None, 1, None, 0),
             lambda: hy.quantize_w4(api.F32, m, n, W, m, 96, api.F32, Q, 64, torch.zeros((n, 2), device="cuda"), None, 2, None, 0),
             lambda: hy.product_w4("T", m, n, 1, api.F32, Q, 64, 128, S, None, 1, W, m, 0, None, 0, None, 0, Y, n),
             lambda: hy.product_w4("T", 0, n, 1, api.F32, Q, 64, 128, S, None, 1, W, m, 0, None, 0, None, 0, Y, n),
             lambda: hy.distill_loss(api.F32, n, 1, Y, n, 1, ids, teacher, 1, 1.0, None, None, loss, stats, None, 0),
             lambda: hy.distill_grad(api.F32, n, 1, Y, n, 1, ids, teacher, 1, 1.0, None, None, stats, Y, n)]
    A, V, sv = torch.randn((8, 64), dtype=torch.float64, device="cuda"), torch.zeros((8, 8), dtype=torch.float64, device="cuda"), torch.zeros(8, dtype=torch.float64, device="cuda")
    fit = (lambda: hy.tsvd_fit(1e-6, "N", 64, 8, 8, A, 64, sv, V, 8, 64, api.F64) - 8)
    for call in calls + [fit]:
        fail()
        capfd.readouterr()
        assert call() == 0
        torch.cuda.synchronize()
        assert capfd.readouterr().err == ""


def test_segment_timer_beside_a_captured_call(monkeypatch):
    """A handle with a timer: what is captured into a graph is not timed (its events would have no time), eager calls still are."""
    torch = _torch()
    from hyacinth_b200 import api
    monkeypatch.setenv("HYACIN_CREATE_TIMER", "1")
    n, m = 512, 4096
    W = torch.randn((n, m), device="cuda")
    Q, S = torch.zeros((n, m // 2), dtype=torch.uint8, device="cuda"), torch.zeros((n, m // 128), device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with api.Hyacin(stream=stream.cuda_stream) as h, torch.cuda.stream(stream):
        def call():
            assert h.quantize_w4(api.F32, m, n, W, m, 128, api.F32, Q, m // 2, S, None, m // 128, None, 0) == 0
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call()
        g.replay()
        for _ in range(3):
            call()
        assert h.sync_timer("R")["R"] > 0
        call()
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other, stream=stream):
            call()
        other.replay()
        call()
        assert h.sync_timer("R")["R"] > 0
        del g, other


def test_a_handle_that_was_never_created_is_refused(hy, capfd):
    """Zero-initialised, it names device 0, the current one, but has neither its number of SMs nor a pool."""
    import ctypes
    torch = _torch()
    from hyacinth_b200 import api
    lib, raw = api.load(), api.HyacinHandle()
    h = ctypes.byref(raw)
    W = torch.ones((4, 128), device="cuda")
    Q, S = torch.zeros((4, 64), dtype=torch.uint8, device="cuda"), torch.zeros((4, 1), device="cuda")
    Y, stats = torch.zeros((40, 4), device="cuda"), torch.zeros((40, 2), device="cuda")
    w, q, s, y, st = (t.data_ptr() for t in (W, Q, S, Y, stats))
    assert lib.hyacinB200QuantizeW4(h, api.F32, 128, 4, w, 128, 128, api.F32, q, 64, s, None, 1, None, 0) == -1
    for kind in (api.F32, api.F16):
        for t in (1, 4):
            assert lib.hyacinB200ProductW4(h, b"T", 128, 4, t, kind, q, 64, 128, s, None, 1, w, 128, 0, None, 0, None, 0, y, 4) == -1
    assert lib.hyacinB200DistillLoss(h, api.F32, 4, 1, y, 4, 0, None, None, 0, 1.0, None, None, st, None, None, 0) == -1
    assert lib.hyacinB200DistillGrad(h, api.F32, 4, 1, y, 4, 0, None, None, 0, 1.0, None, None, st, y, 4) == -1
    assert capfd.readouterr().err.count("hyacinCreate") == 7


# ---- the same beside other shapes ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("op,t,rank,m,n", [("T", 20, 7, 501, 203), ("T", 300, 33, 500, 203), ("N", 20, 7, 203, 501), ("N", 300, 65, 203, 500), ("T", 20, 1000, 256, 130),
                                           ("N", 12, 700, 130, 256), ("T", 40, 64, 512, 5000), ("T", 3, 20, 501, 203)])
def test_correction_of_odd_shapes(hy, op, t, rank, m, n):
    """Factors off their alignment, several tiles of tokens, ranks of many steps, more tiles than a cluster shares."""
    for kind in ("f16", "bf16"):
        _correction_only(hy, op, kind, rank, t, (3, 1, -12), m, n)
        _correction_only(hy, op, kind, rank, t, (-24, -8, 9), m, n)


@pytest.mark.parametrize("t", [9, 13, 16])
def test_vectors_beside_a_scattered_table_are_exact(hy, t):
    """Tables whose rows cannot be fetched a block at a time stream up to sixteen vectors, with the same promise."""
    rng = np.random.default_rng(t)
    m, n, seg = 500, 150, 32
    for kind, bits in (("f16", 10), ("bf16", 7)):
        codes, scales, zp = _problem(rng, m, n, seg, kind, True)
        scales[:] = 1
        x = 1 + rng.integers(0, 1 << bits, (t, m)) * 2.0 ** -bits
        got = _run_product(hy, "T", m, n, t, kind, seg, codes, scales, zp, x, pads=(1, 0, 0))
        assert np.array_equal(got, P.round_to(x @ P.values(codes, scales, zp, seg).T, kind))


@pytest.mark.parametrize("op,t", [("T", 20), ("N", 20)])
def test_half_with_a_correction_captured_and_replayed(op, t):
    """The correction's parts, scratch of the call, in two graphs replayed on two streams at once."""
    torch = _torch()
    from hyacinth_b200 import api
    rng = np.random.default_rng(t)
    m, n, rank, seg = 640, 384, 24, 128
    inn, out = (m, n) if op == "T" else (n, m)
    codes, scales, _ = _problem(rng, m, n, seg, "f16", False)
    Q, S = torch.from_numpy(P.pack(codes, m // 2)).cuda(), _dev(scales, "f16")
    u, v = P.round_to(0.1 * rng.standard_normal((rank, m)), "f16"), P.round_to(0.1 * rng.standard_normal((rank, n)), "f16")
    U, V = _dev(u, "f16"), _dev(v, "f16")
    xs = [P.round_to(rng.standard_normal((t, inn)), "f16") for _ in range(2)]
    X, Y = [_dev(x, "f16") for x in xs], [torch.zeros((t, out), dtype=torch.float16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    handles, graphs = [api.Hyacin(stream=s.cuda_stream) for s in streams], []
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[i]):
                assert handles[i].product_w4(op, m, n, t, api.F16, Q, m // 2, seg, S, None, m // seg, X[i], inn, rank, U, m, V, n, Y[i], out) == 0
            graphs.append(g)
    for _ in range(4):
        for y in Y:
            y.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            _check_product(_back(Y[i], out), op, m, n, "f16", seg, codes, scales, None, xs[i], u, v)
    del graphs, g
    for h in handles:
        h.destroy()
