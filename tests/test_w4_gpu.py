"""4-bit weight matrices on the GPU against their 64-bit statement: form, products in both directions, and a run of quantise,
fit of the residual, product and distillation together."""
import numpy as np
import pytest

from tests import w4_plain as P

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def _dev(x, kind, ld=None, fill=float("nan")):
    """(rows, cols) float64 -> device tensor (rows, ld) of the storage type, filled behind the last column."""
    torch = _torch()
    ld = ld or x.shape[1]
    out = torch.full((x.shape[0], ld), fill, dtype=P.kinds()[kind][0], device="cuda")
    out[:, :x.shape[1]] = torch.from_numpy(np.ascontiguousarray(x)).to(P.kinds()[kind][0]).cuda()
    return out


def _back(t, cols):
    return t[:, :cols].double().cpu().numpy()


# ---- form ------------------------------------------------------------------------------------------------------
QCASES = [  # m, n, seg, weight kind, scale kind, zeros, residual, pad
    (1, 1, 32, "f32", "f32", False, True, 0), (31, 2, 32, "bf16", "bf16", True, True, 1), (33, 3, 32, "f16", "f16", False, True, 3),
    (128, 5, 128, "bf16", "bf16", False, False, 0), (129, 4, 64, "f32", "f16", True, True, 2), (255, 7, 96, "f32", "bf16", False, True, 1),
    (300, 3, 256, "f16", "f32", True, True, 0), (700, 9, 1024, "bf16", "f32", True, False, 5), (1000, 33, 160, "f32", "f32", True, True, 0),
    (4096, 16, 128, "bf16", "bf16", True, True, 0), (2049, 11, 32, "f16", "f16", True, True, 7), (640, 21, 64, "bf16", "f16", False, True, 8),
]


@pytest.mark.parametrize("m,n,seg,wkind,skind,zeros,residual,pad", QCASES)
def test_codes_scales_and_residual_are_those_of_the_definition(hy, m, n, seg, wkind, skind, zeros, residual, pad):
    torch = _torch()
    rng = np.random.default_rng(m * 7 + n)
    w = P.round_to(rng.standard_normal((n, m)) * np.exp(rng.standard_normal((n, 1))), wkind)
    w[0, : min(m, seg)] = 0                                           # a segment of zeros
    if n > 2:
        w[1, :] = np.abs(w[1, :])                                     # one-sided: the zero point sits at the border
        w[2, -1] *= 50
        w[2] = P.round_to(w[2], wkind)
    if n > 4:                                                         # exact halves: multiples of half a scale that is a power of two
        w[3, :] = P.round_to(rng.integers(-14, 15, m) * 0.125, wkind)
        w[3, ::seg] = 7 * 0.25
        w[4, m // 2] = np.inf
    segs = -(-m // seg)
    ldq = -(-m // 128) * 64 + 16
    W = _dev(w, wkind, m + pad)
    codes = torch.full((n, ldq), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, segs + 1), 7.0, dtype=P.kinds()[skind][0], device="cuda")
    zp = torch.full((n, segs + 1), 99, dtype=torch.uint8, device="cuda") if zeros else None
    R = torch.full((n, m + 2), 5.0, device="cuda") if residual else None
    rc = hy.quantize_w4(P.kinds()[wkind][1], m, n, W, m + pad, seg, P.kinds()[skind][1], codes, ldq, scales, zp, segs + 1, R, m + 2)
    torch.cuda.synchronize()
    assert rc == 0
    want_codes, want_scales, want_zp = P.quantize(w, seg, skind, zeros)
    got = codes.cpu().numpy()
    assert np.array_equal(got[:, :ldq - 16], P.pack(want_codes, ldq)[:, :ldq - 16])
    assert (got[:, ldq - 16:] == 0xAB).all(), "bytes behind the last block were written"
    assert np.array_equal(_back(scales, segs), want_scales, equal_nan=True)
    assert (scales[:, segs] == 7.0).all()
    if zeros:
        assert np.array_equal(zp[:, :segs].cpu().numpy(), want_zp) and (zp[:, segs] == 99).all()
    if residual:
        # the product of a scale and a code is exact in 64 bits; one rounding to float
        with np.errstate(invalid="ignore"):
            want = w - P.values(want_codes, want_scales, want_zp, seg)
        live = np.isfinite(want)
        have = _back(R, m)
        assert np.isnan(have[~live]).all()
        assert (np.abs(have - want)[live] <= 2.0 ** -24 * np.abs(want[live])).all()
        assert (R[:, m:] == 5.0).all()


# ---- products --------------------------------------------------------------------------------------------------
def _problem(rng, m, n, seg, kind, zeros):
    codes = rng.integers(0, 16, (n, m), dtype=np.uint8)
    segs = -(-m // seg)
    scales = P.round_to(np.exp(rng.standard_normal((n, segs))) * 0.02, kind)
    zp = rng.integers(0, 16, (n, segs), dtype=np.uint8) if zeros else None
    return codes, scales, zp


def _run_product(hy, op, m, n, t, kind, seg, codes, scales, zp, x, u=None, v=None, pads=(0, 0, 0), ldq_extra=0):
    torch = _torch()
    ldq = -(-m // 128) * 64 + ldq_extra
    segs = scales.shape[1]
    out = n if op == "T" else m
    inn = m if op == "T" else n
    packed = P.pack(codes, ldq)
    if m % 128:                                                     # nibbles of rows behind the last are ignored
        full = np.full((n, -(-m // 128) * 128), 15, dtype=np.uint8)
        full[:, :m] = codes
        packed[:, :ldq - ldq_extra] = P.pack(full, ldq)[:, :ldq - ldq_extra]
    dq = torch.from_numpy(packed).cuda()
    ds = _dev(scales, kind, segs + pads[0])
    dz = None
    if zp is not None:
        dz = torch.full((n, segs + pads[0]), 200, dtype=torch.uint8, device="cuda")
        dz[:, :segs] = torch.from_numpy(zp).cuda()
    X = _dev(x, kind, inn + pads[1])
    Y = torch.full((t, out + pads[2]), 77.0, dtype=P.kinds()[kind][0], device="cuda")
    rank = 0 if u is None else u.shape[0]
    U = None if u is None else _dev(u, kind, m + pads[1])
    V = None if v is None else _dev(v, kind, n + pads[2])
    rc = hy.product_w4(op, m, n, t, P.kinds()[kind][1], dq, ldq, seg, ds, dz, segs + pads[0], X, inn + pads[1], rank, U, m + pads[1], V, n + pads[2],
                       Y, out + pads[2])
    torch.cuda.synchronize()
    assert rc == 0 and hy.status() == 0
    assert (Y[:, out:] == 77.0).all(), "rows behind the last were written"
    return _back(Y, out)


def _check_product(got, op, m, n, kind, seg, codes, scales, zp, x, u=None, v=None):
    """|error| <= half a step of the result + what 32-bit sums and 16-bit factors can lose.

    A sum of L products in 32 bits is off by at most 2 L 2^-24 times the sum of the magnitudes, in any order and with
    truncating adders; the matrix pipes add 16 products at once, so no term passes through more than L / 8 + 64 additions.
    The 16-bit types may round each scaled weight once more: half a step of the sum of magnitudes at the very most, but these
    roundings are independent, each uniform in a half step, so eight standard deviations of their sum,
    8 * half_step / sqrt(3) * sqrt(sum (w x)^2), bound them as well."""
    w = P.values(codes, scales, zp, seg)
    a = w if op == "T" else w.T
    want, mag, sq = x @ a.T, np.abs(x) @ np.abs(a).T, (x * x) @ (a * a).T
    terms = a.shape[1]
    if u is not None:
        f, s = (u, v) if op == "T" else (v, u)
        want = want + (x @ f.T) @ s
        mag = mag + (np.abs(x) @ np.abs(f).T) @ np.abs(s)
        terms += u.shape[0] * 8 + terms
    tol = P.HALF_STEP[kind] * np.abs(want) + (terms / 8 + 64) * 2.0 ** -23 * mag + P.TINY[kind]
    if kind != "f32":
        tol += 8 * P.HALF_STEP[kind] / np.sqrt(3) * np.sqrt(sq) * (1 + P.HALF_STEP[kind])
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, f"{worst:.2f} of the tolerance"


PCASES = [  # op, m, n, t, seg, kind, zeros, rank, pads (scales, X/U, Y/V)
    ("T", 1, 1, 1, 32, "f16", False, 0, (0, 0, 0)), ("T", 128, 16, 1, 128, "bf16", False, 0, (0, 0, 0)), ("T", 130, 17, 2, 64, "f16", True, 3, (1, 1, 1)),
    ("T", 1000, 37, 5, 32, "bf16", True, 0, (0, 3, 5)), ("T", 512, 257, 8, 128, "f16", False, 8, (0, 0, 0)), ("T", 4096, 96, 1, 128, "bf16", False, 16, (0, 0, 0)),
    ("T", 777, 130, 9, 96, "f16", True, 0, (0, 1, 0)), ("T", 640, 200, 16, 64, "bf16", False, 0, (2, 8, 0)), ("T", 640, 200, 17, 64, "bf16", True, 5, (0, 0, 1)),
    ("T", 1024, 384, 33, 256, "f16", False, 0, (0, 0, 0)), ("T", 900, 300, 64, 32, "bf16", True, 7, (0, 4, 4)), ("T", 2048, 256, 100, 128, "bf16", False, 32, (0, 0, 0)),
    ("T", 512, 130, 256, 128, "f16", True, 0, (0, 8, 0)), ("T", 320, 140, 300, 64, "bf16", False, 0, (0, 0, 0)), ("T", 8192, 64, 3, 8192, "f16", True, 0, (0, 0, 0)),
    ("T", 300, 75, 1, 32, "f32", True, 2, (0, 0, 0)), ("T", 2048, 130, 4, 128, "f32", False, 0, (1, 1, 1)), ("T", 777, 90, 23, 64, "f32", True, 9, (0, 0, 0)),
    ("N", 1, 1, 1, 32, "f16", False, 0, (0, 0, 0)), ("N", 256, 300, 1, 128, "bf16", False, 0, (0, 0, 0)), ("N", 130, 1001, 2, 64, "f16", True, 4, (1, 1, 1)),
    ("N", 1000, 513, 16, 32, "bf16", True, 0, (0, 5, 3)), ("N", 512, 2048, 64, 64, "f16", True, 32, (0, 0, 0)), ("N", 640, 777, 65, 128, "bf16", False, 0, (0, 7, 0)),
    ("N", 384, 520, 256, 96, "bf16", True, 8, (0, 0, 0)), ("N", 200, 300, 280, 256, "f16", False, 0, (0, 4, 8)), ("N", 257, 400, 1, 32, "f32", True, 0, (0, 0, 0)),
    ("N", 1024, 350, 7, 128, "f32", False, 5, (1, 1, 1)),
    # long x: the streaming kernel's smaller stages, the tensor-core kernel, and what neither takes
    ("T", 16384, 40, 1, 128, "f32", False, 0, (0, 0, 0)), ("T", 30001, 24, 2, 64, "f32", True, 3, (0, 0, 0)), ("T", 16390, 40, 8, 32, "bf16", True, 0, (1, 0, 0)),
    ("T", 20000, 20, 4, 128, "f16", False, 17, (0, 0, 0)), ("T", 16384, 33, 1, 96, "bf16", True, 0, (0, 0, 0)), ("T", 2600, 150, 13, 32, "f16", True, 6, (1, 1, 0)),
    # every shape of the correction: ranks of 16, 32, 64 and others, one and two parts per step
    ("T", 512, 200, 40, 128, "bf16", False, 16, (0, 0, 0)), ("T", 512, 200, 40, 128, "f16", False, 33, (0, 0, 0)), ("T", 512, 200, 129, 128, "bf16", False, 64, (0, 0, 0)),
    ("T", 512, 200, 250, 64, "bf16", True, 70, (0, 1, 1)), ("T", 512, 200, 40, 128, "bf16", False, 150, (0, 0, 0)), ("N", 300, 512, 40, 32, "bf16", False, 90, (0, 0, 0)),
    ("N", 300, 512, 200, 64, "f16", True, 16, (0, 2, 2)), ("N", 5000, 700, 5, 64, "f32", True, 3, (0, 0, 0)), ("N", 200, 16, 1, 64, "f32", False, 0, (0, 0, 0)),
    ("N", 128, 20000, 33, 128, "f32", False, 2, (0, 0, 0)), ("T", 384, 19000, 20, 128, "f16", False, 0, (0, 0, 0)), ("N", 19000, 200, 20, 128, "f16", False, 0, (0, 0, 0)),
]


@pytest.mark.parametrize("op,m,n,t,seg,kind,zeros,rank,pads", PCASES)
def test_product_against_the_definition(hy, op, m, n, t, seg, kind, zeros, rank, pads):
    rng = np.random.default_rng(m + 31 * n + 7 * t)
    codes, scales, zp = _problem(rng, m, n, seg, kind, zeros)
    x = P.round_to(rng.standard_normal((t, m if op == "T" else n)), kind)
    u = P.round_to(0.1 * rng.standard_normal((rank, m)), kind) if rank else None
    v = P.round_to(rng.standard_normal((rank, n)) / np.sqrt(n), kind) if rank else None
    got = _run_product(hy, op, m, n, t, kind, seg, codes, scales, zp, x, u, v, pads, ldq_extra=16 if pads[0] else 0)
    _check_product(got, op, m, n, kind, seg, codes, scales, zp, x, u, v)


def test_product_of_nothing_is_zero(hy):
    """No inputs (M = 0 for 'T', N = 0 for 'N'): the sum over nothing."""
    torch = _torch()
    for op, m, n in (("T", 0, 9), ("N", 9, 0)):
        Y = torch.full((3, 9), 5.0, dtype=torch.float16, device="cuda")
        assert hy.product_w4(op, m, n, 3, P.kinds()["f16"][1], None, 64, 32, None, None, 0, None, 0, 4, None, 0, None, 0, Y, 9) == 0
        torch.cuda.synchronize()
        assert (Y == 0).all()


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("t", [1, 20])
def test_product_leaves_nan_and_infinity_where_they_belong(hy, op, t):
    """A token that holds a NaN or an infinity spoils its own column of Y only, a NaN scale its own outputs only."""
    rng = np.random.default_rng(5)
    m, n, seg = 256, 192, 64
    codes, scales, _ = _problem(rng, m, n, seg, "bf16", False)
    codes[:] = np.where(codes == 8, 9, codes)                        # no zero weight: 0 * inf does not arise
    x = P.round_to(rng.standard_normal((t + 1, m if op == "T" else n)), "bf16")
    clean = _run_product(hy, op, m, n, t + 1, "bf16", seg, codes, scales, None, x)
    x[0, 17] = np.inf
    got = _run_product(hy, op, m, n, t + 1, "bf16", seg, codes, scales, None, x)
    assert not np.isfinite(got[0]).any()
    assert np.array_equal(got[1:], clean[1:])
    scales[3, 1] = np.nan
    got = _run_product(hy, op, m, n, t + 1, "bf16", seg, codes, scales, None, x)
    hit = np.zeros(n if op == "T" else m, dtype=bool)
    if op == "T":
        hit[3] = True
    else:
        hit[64:128] = True
    assert np.isnan(got[1:, hit]).all() and np.array_equal(got[1:, ~hit], clean[1:, ~hit])


def test_product_is_the_same_every_time_and_for_every_alignment(hy):
    """Bit-identical repeats; pointers that are aligned to one element only give the same values as aligned ones."""
    torch = _torch()
    rng = np.random.default_rng(11)
    for op, m, n, t, kind in (("T", 520, 200, 3, "bf16"), ("T", 520, 200, 40, "f16"), ("N", 520, 200, 40, "bf16"), ("T", 520, 200, 3, "f32")):
        codes, scales, zp = _problem(rng, m, n, 64, kind, True)
        inn, out = (m, n) if op == "T" else (n, m)
        x = P.round_to(rng.standard_normal((t, inn)), kind)
        first = _run_product(hy, op, m, n, t, kind, 64, codes, scales, zp, x)
        for _ in range(3):
            assert np.array_equal(first, _run_product(hy, op, m, n, t, kind, 64, codes, scales, zp, x))
        dt, code = P.kinds()[kind]
        flat = torch.zeros(t * (inn + 1) + 1, dtype=dt, device="cuda")
        X = flat[1:].view(t, inn + 1)
        X[:, :inn] = torch.from_numpy(x).to(dt).cuda()
        Y = torch.zeros(t * (out + 1) + 1, dtype=dt, device="cuda")[1:].view(t, out + 1)
        S = torch.zeros(n * 10 + 1, dtype=dt, device="cuda")[1:].view(n, 10)
        S[:, :scales.shape[1]] = torch.from_numpy(scales).to(dt).cuda()
        Z = torch.zeros(n * 10 + 3, dtype=torch.uint8, device="cuda")[3:].view(n, 10)
        Z[:, :scales.shape[1]] = torch.from_numpy(zp).cuda()
        Q = torch.from_numpy(P.pack(codes, -(-m // 128) * 64)).cuda()
        assert hy.product_w4(op, m, n, t, code, Q, Q.shape[1], 64, S, Z, 10, X, inn + 1, 0, None, 0, None, 0, Y, out + 1) == 0
        torch.cuda.synchronize()
        _check_product(_back(Y, out), op, m, n, kind, 64, codes, scales, zp, x)


@pytest.mark.parametrize("op,t,rank", [("T", 1, 4), ("T", 40, 4), ("N", 8, 4)])
def test_product_captured_and_replayed(op, t, rank):
    """A captured call, with its scratch, replayed on new inputs, next to eager calls of the same handle on the same stream, and two
    graphs after each other."""
    torch = _torch()
    from hyacinth_b200 import api
    rng = np.random.default_rng(3)
    m, n, seg, kind = 640, 384, 128, "bf16"
    dt, code = P.kinds()[kind]
    codes, scales, zp = _problem(rng, m, n, seg, kind, True)
    inn, out = (m, n) if op == "T" else (n, m)
    Q, S, Z = torch.from_numpy(P.pack(codes, m // 2)).cuda(), _dev(scales, kind), torch.from_numpy(zp).cuda()
    u, v = P.round_to(0.1 * rng.standard_normal((rank, m)), kind), P.round_to(0.1 * rng.standard_normal((rank, n)), kind)
    U, V = _dev(u, kind), _dev(v, kind)
    stream = torch.cuda.Stream()
    with api.Hyacin(stream=stream.cuda_stream) as h:
        def call(X, Y):
            assert h.product_w4(op, m, n, t, code, Q, m // 2, seg, S, Z, S.shape[1], X, inn, rank, U, m, V, n, Y, out) == 0
        xs = [P.round_to(rng.standard_normal((t, inn)), kind) for _ in range(3)]
        X = [torch.empty((t, inn), dtype=dt, device="cuda") for _ in range(2)]
        Y = [torch.zeros((t, out), dtype=dt, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            call(X[0], Y[0])
            graphs = []
            for i in range(2):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    call(X[i], Y[i])
                graphs.append(g)
            for a, b in ((0, 1), (2, 0)):
                X[0].copy_(_dev(xs[a], kind)); X[1].copy_(_dev(xs[b], kind))
                graphs[0].replay(); graphs[1].replay()
                eager = torch.zeros_like(Y[0])
                call(X[0], eager)
                stream.synchronize()
                _check_product(_back(Y[0], out), op, m, n, kind, seg, codes, scales, zp, xs[a], u, v)
                _check_product(_back(Y[1], out), op, m, n, kind, seg, codes, scales, zp, xs[b], u, v)
                assert torch.equal(eager, Y[0])
        del graphs, g


def test_product_far_into_a_large_matrix(hy):
    """Code offsets beyond 2^32 bytes: the last columns of a matrix with a wide pitch."""
    torch = _torch()
    rng = np.random.default_rng(8)
    m, n, ldq = 256, 70000, 65536                                   # 4.6 GB, of which 128 bytes per column are codes
    codes = rng.integers(0, 16, (n, m), dtype=np.uint8)
    Q = torch.zeros((n, ldq), dtype=torch.uint8, device="cuda")
    Q[:, :128] = torch.from_numpy(P.pack(codes, 128)).cuda()
    scales = P.round_to(np.exp(0.3 * rng.standard_normal((n, 2))), "f16")
    S = _dev(scales, "f16")
    for op, t in (("T", 2), ("T", 20), ("N", 2)):
        inn, out = (m, n) if op == "T" else (n, m)
        x = P.round_to(rng.standard_normal((t, inn)), "f16")
        X, Y = _dev(x, "f16"), torch.zeros((t, out), dtype=torch.float16, device="cuda")
        assert hy.product_w4(op, m, n, t, P.kinds()["f16"][1], Q, ldq, 128, S, None, 2, X, inn, 0, None, 0, None, 0, Y, out) == 0
        torch.cuda.synchronize()
        _check_product(_back(Y, out), op, m, n, "f16", 128, codes, scales, None, x)
    del Q


# ---- a run of them together ------------------------------------------------------------------------------------------
def test_quantise_fit_product_and_distil_together(hy):
    """A head is brought to 4 bits, the residual's basis comes from hyacinTsvdFit, the corrected product gives the logits, the
    distillation loss compares them with the original's, and its gradient goes back through the same product."""
    torch = _torch()
    from hyacinth_b200 import api
    rng = np.random.default_rng(21)
    m, n, t, rank_cap, k = 256, 512, 24, 32, 16
    w = rng.standard_normal((n, m)) * 0.05
    w += (rng.standard_normal((n, 8)) @ rng.standard_normal((8, m))) * 0.02
    W = torch.from_numpy(w).float().cuda()
    Q = torch.zeros((n, m // 2), dtype=torch.uint8, device="cuda")
    S = torch.zeros((n, m // 64), dtype=torch.float32, device="cuda")
    R = torch.zeros((n, m), dtype=torch.float32, device="cuda")
    assert hy.quantize_w4(api.F32, m, n, W, m, 64, api.F32, Q, m // 2, S, None, m // 64, R, m) == 0
    sv = torch.zeros((n,), dtype=torch.float32, device="cuda")
    V = torch.zeros((n, n), dtype=torch.float32, device="cuda")
    r = hy.tsvd_fit(1e-3, "N", m, n, rank_cap, R, m, sv, V, n, m, api.F32)
    assert 0 < r <= rank_cap
    V = V[:r].contiguous()
    U = (V @ R).contiguous()                                          # U = R V, column-major m x r
    x = torch.from_numpy(rng.standard_normal((t, m))).float().cuda()
    Y = torch.zeros((t, n), dtype=torch.float32, device="cuda")
    assert hy.product_w4("T", m, n, t, api.F32, Q, m // 2, 64, S, None, m // 64, x, m, r, U, m, V, n, Y, n) == 0
    torch.cuda.synchronize()
    wq = P.values(P.unpack(Q.cpu().numpy(), m), S.double().cpu().numpy(), None, 64)
    weff = wq + V.double().cpu().numpy().T @ U.double().cpu().numpy()
    assert np.linalg.norm(weff - w) < np.linalg.norm(wq - w), "the correction does not bring the product nearer"
    teacher = x.double().cpu().numpy() @ w.T
    order = np.argsort(-teacher, axis=1)[:, :k]
    ids = torch.from_numpy(order.astype(np.int32)).cuda()
    top = torch.from_numpy(np.take_along_axis(teacher, order, 1)).float().cuda()
    lse = torch.from_numpy(np.log(np.exp(teacher).sum(1))).float().cuda()
    loss, dZ = torch.zeros((t,), device="cuda"), torch.zeros((t, n), device="cuda")
    assert hy.distill_loss(api.F32, n, t, Y, n, k, ids, top, k, 1.0, lse, None, loss, None, dZ, n) == 0
    dX = torch.zeros((t, m), device="cuda")
    assert hy.product_w4("N", m, n, t, api.F32, Q, m // 2, 64, S, None, m // 64, dZ, n, r, U, m, V, n, dX, m) == 0
    torch.cuda.synchronize()
    z = x.double().cpu().numpy() @ weff.T
    args = (order, top.cpu().numpy(), 1.0, lse.cpu().numpy(), None)
    want_loss, want_grad, _ = P.distill(z, *args)
    # logits of magnitude < 20 in 32 bits with sums of < 600 terms: errors below 1e-4, hence losses within 2e-4 absolutely, gradients
    # within 2e-4 of probabilities <= 1
    assert np.abs(loss.cpu().numpy() - want_loss).max() < 2e-4
    assert np.abs(dZ.cpu().numpy() - want_grad).max() < 2e-4
    want_dx = want_grad @ weff
    assert np.abs(dX.cpu().numpy() - want_dx).max() < 2e-4 * np.abs(weff).sum(0).max()
    # the gradient to the input against central differences of the whole chain in 64 bits
    for (a, b) in ((0, 0), (3, 100), (23, 255)):
        xd = x.double().cpu().numpy()
        step = 1e-5
        d = np.zeros_like(xd); d[a, b] = step
        diff = (P.distill((xd + d) @ weff.T, *args)[0][a] - P.distill((xd - d) @ weff.T, *args)[0][a]) / (2 * step)
        assert abs(diff - want_dx[a, b]) < 1e-6


# ---- the ends of the ranges ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("wkind,skind", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("zeros", [False, True])
def test_codes_beside_halves_and_at_the_ends_of_the_range(hy, wkind, skind, zeros):
    """Weights on every half-way point of their scale and on the numbers next to it, for scales of every size: those that lose bits as
    a subnormal number, vanish or overflow among them."""
    torch = _torch()
    rng = np.random.default_rng(5)
    dt, code = P.kinds()[wkind]
    low, high = {"f32": (-149, 125), "f16": (-24, 12), "bf16": (-133, 125)}[wkind]
    seg, n = 64, 4 * (high - low)
    m = 2 * seg + 32
    exponent = low + (np.arange(n) % (high - low))
    s = P.round_to((1 + rng.random(n)), skind) * 2.0 ** exponent                      # a scale with all its bits
    steps = rng.integers(-15, 15, (n, m)) / 2 if not zeros else rng.integers(-10, 20, (n, m)) / 2
    w = P.round_to(steps * s[:, None], wkind)
    t = torch.from_numpy(w).to(dt)
    bits = t.view(torch.int32 if dt == torch.float32 else torch.int16)
    moved = bits + torch.from_numpy(rng.integers(-1, 2, (n, m))).to(bits.dtype)       # up or down a place
    w = torch.where((t != 0) & torch.isfinite(moved.view(dt)), moved.view(dt), t).double().numpy()
    w[:, 0::seg], w[:, 1::seg] = (7 * s)[:, None], (0 * s)[:, None]                    # where these are the extremes the scale is s
    if zeros:
        w[:, 0::seg], w[:, 1::seg] = (10 * s)[:, None], (-5 * s)[:, None]
    w = P.round_to(w, wkind)
    w[~np.isfinite(w)] = 0
    segs = -(-m // seg)
    ldq = -(-m // 128) * 64
    W = _dev(w, wkind)
    codes = torch.zeros((n, ldq), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((n, segs), dtype=P.kinds()[skind][0], device="cuda")
    zp = torch.zeros((n, segs), dtype=torch.uint8, device="cuda") if zeros else None
    assert hy.quantize_w4(code, m, n, W, m, seg, P.kinds()[skind][1], codes, ldq, scales, zp, segs, None, 0) == 0
    torch.cuda.synchronize()
    with np.errstate(over="ignore"):
        want_codes, want_scales, want_zp = P.quantize(w, seg, skind, zeros)
    assert np.array_equal(_back(scales, segs), want_scales, equal_nan=True)
    if zeros:
        assert np.array_equal(zp.cpu().numpy(), want_zp)
    assert np.array_equal(P.unpack(codes.cpu().numpy(), m), want_codes)


@pytest.mark.parametrize("op,rank", [("T", 2), ("N", 0), ("N", 2)])
def test_product_of_more_vectors_than_one_launch_takes(hy, op, rank):
    rng = np.random.default_rng(12)
    m, n, t, kind = (32, 8, (1 << 19) + 300, "bf16") if op == "T" else (8, 32, (1 << 19) + 300, "bf16")
    codes, scales, zp = _problem(rng, m, n, 32, kind, False)
    x = P.round_to(rng.standard_normal((t, m if op == "T" else n)), kind)
    u = P.round_to(0.1 * rng.standard_normal((rank, m)), kind) if rank else None
    v = P.round_to(rng.standard_normal((rank, n)) / np.sqrt(n), kind) if rank else None
    got = _run_product(hy, op, m, n, t, kind, 32, codes, scales, zp, x, u, v)
    _check_product(got, op, m, n, kind, 32, codes, scales, zp, x, u, v)


def test_two_threads_on_two_streams(hy):
    """Two handles used at the same time from two threads give what each gives alone."""
    import threading
    torch = _torch()
    from hyacinth_b200 import api
    rng = np.random.default_rng(14)
    m, n, seg, rank, vocab, k = 1024, 512, 64, 8, 9001, 8
    problems = []
    for kind in ("bf16", "f16"):
        dt, code = P.kinds()[kind]
        W = torch.from_numpy(rng.standard_normal((n, m))).to(dt).cuda()
        U, V = torch.from_numpy(rng.standard_normal((rank, m)) * 0.1).to(dt).cuda(), torch.from_numpy(rng.standard_normal((rank, n))).to(dt).cuda()
        xs = [(op, t, torch.from_numpy(rng.standard_normal((t, m if op == "T" else n))).to(dt).cuda()) for op, t in (("T", 1), ("T", 4), ("T", 40), ("N", 3))]
        Z = torch.from_numpy(3 * rng.standard_normal((6, vocab))).to(dt).cuda()
        ids = torch.from_numpy(rng.integers(0, vocab, (6, k)).astype(np.int32)).cuda()
        teacher = torch.from_numpy(rng.standard_normal((6, k))).float().cuda()
        problems.append((dt, code, W, U, V, xs, Z, ids, teacher))
    torch.cuda.synchronize()

    def run(problem, repeats, out):
        dt, code, W, U, V, xs, Z, ids, teacher = problem
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream), api.Hyacin(stream=stream.cuda_stream) as h:
            for _ in range(repeats):
                Q = torch.zeros((n, m // 2), dtype=torch.uint8, device="cuda")
                S = torch.zeros((n, m // seg), dtype=dt, device="cuda")
                loss = torch.zeros(6, device="cuda")
                dZ = torch.zeros_like(Z)
                results = [Q, S, loss, dZ]
                rc = h.quantize_w4(code, m, n, W, m, seg, code, Q, m // 2, S, None, m // seg, None, 0)
                for op, t, x in xs:
                    inn, wide = (m, n) if op == "T" else (n, m)
                    Y = torch.zeros((t, wide), dtype=dt, device="cuda")
                    rc |= h.product_w4(op, m, n, t, code, Q, m // 2, seg, S, None, m // seg, x, inn, rank, U, m, V, n, Y, wide)
                    results.append(Y)
                rc |= h.distill_loss(code, vocab, 6, Z, vocab, k, ids, teacher, k, 1.5, None, None, loss, None, dZ, vocab)
                stream.synchronize()
                out.append((rc, [r.clone() for r in results]))
            stream.synchronize()

    alone = []
    for problem in problems:
        run(problem, 1, alone)
    together = [[], []]
    threads = [threading.Thread(target=run, args=(problems[i], 15, together[i])) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert hy.status() == 0
    for i in range(2):
        assert alone[i][0] == 0 and len(together[i]) == 15
        for rc, results in together[i]:
            assert rc == 0
            for a, b in zip(alone[i][1], results):
                assert torch.equal(a, b)


@pytest.mark.parametrize("op,m,n,t,seg,zeros,rank,pads", [
    ("T", 33, 1, 25, 32, True, 0, (0, 1, 0)), ("T", 513, 200, 21, 96, False, 33, (1, 3, 1)), ("T", 4096, 300, 64, 128, True, 16, (0, 0, 0)), ("T", 300, 129, 200, 32, False, 0, (0, 0, 0)),
    ("T", 2000, 127, 70, 64, True, 40, (1, 1, 0)), ("N", 1, 40, 5, 32, False, 1, (0, 0, 0)), ("N", 129, 33, 16, 64, True, 0, (1, 1, 0)), ("N", 300, 2000, 65, 32, True, 50, (0, 2, 2)),
    # few outputs and long sums, which several clusters share
    ("N", 200, 20000, 31, 32, True, 9, (0, 1, 1)), ("N", 130, 9001, 3, 64, False, 0, (0, 0, 0)), ("T", 20001, 70, 2, 64, True, 12, (1, 1, 1)), ("T", 16384, 129, 40, 128, False, 0, (0, 0, 0)),
    ("N", 1000, 31, 130, 256, False, 7, (0, 1, 3)), ("N", 128, 4100, 17, 128, True, 0, (0, 0, 0)), ("N", 5000, 64, 4, 64, True, 2, (0, 0, 1)), ("T", 40000, 20, 3, 128, False, 5, (0, 0, 0)),
])
def test_single_precision_of_many_vectors(hy, op, m, n, t, seg, zeros, rank, pads):
    """The tiled kernel: sizes beside its tiles and steps, odd pitches, corrections that end inside a step."""
    rng = np.random.default_rng(m + n + t)
    codes, scales, zp = _problem(rng, m, n, seg, "f32", zeros)
    x = P.round_to(rng.standard_normal((t, m if op == "T" else n)), "f32")
    u = P.round_to(0.1 * rng.standard_normal((rank, m)), "f32") if rank else None
    v = P.round_to(rng.standard_normal((rank, n)) / np.sqrt(n), "f32") if rank else None
    got = _run_product(hy, op, m, n, t, "f32", seg, codes, scales, zp, x, u, v, pads)
    _check_product(got, op, m, n, "f32", seg, codes, scales, zp, x, u, v)


def test_a_handle_of_another_device_is_refused(hy):
    torch = _torch()
    from hyacinth_b200 import api
    W = torch.ones((4, 128), device="cuda")
    Q, S = torch.zeros((4, 64), dtype=torch.uint8, device="cuda"), torch.zeros((4, 1), device="cuda")
    Y, loss = torch.zeros((1, 4), device="cuda"), torch.zeros(1, device="cuda")
    with api.Hyacin(stream=torch.cuda.current_stream().cuda_stream) as h:
        own = h.h.DeviceID
        h.h.DeviceID = own + 1
        try:
            assert h.quantize_w4(api.F32, 128, 4, W, 128, 128, api.F32, Q, 64, S, None, 1, None, 0) == -1
            assert h.product_w4("T", 128, 4, 1, api.F32, Q, 64, 128, S, None, 1, W, 128, 0, None, 0, None, 0, Y, 4) == -1
            assert h.distill_loss(api.F32, 4, 1, Y, 4, 0, None, None, 0, 1.0, None, None, loss, None, None, 0) == -1
        finally:
            h.h.DeviceID = own
        assert h.quantize_w4(api.F32, 128, 4, W, 128, 128, api.F32, Q, 64, S, None, 1, None, 0) == 0
    torch.cuda.synchronize()
    assert torch.equal(S, torch.full_like(S, float(np.float32(1) / np.float32(7))))


@pytest.mark.parametrize("op,m,n,t", [("N", 130, 9001, 3), ("N", 130, 9001, 40), ("T", 9001, 130, 5), ("N", 2000, 300, 2)])
def test_single_precision_captured_and_replayed(op, m, n, t):
    """Its scratch (mid, the shares of several clusters) in two graphs that are replayed on two streams at once."""
    torch = _torch()
    from hyacinth_b200 import api
    rng = np.random.default_rng(t)
    rank = 4
    codes, scales, _ = _problem(rng, m, n, 64, "f32", False)
    inn, out = (m, n) if op == "T" else (n, m)
    ldq = -(-m // 128) * 64
    Q, S = torch.from_numpy(P.pack(codes, ldq)).cuda(), _dev(scales, "f32")
    u, v = P.round_to(0.1 * rng.standard_normal((rank, m)), "f32"), P.round_to(0.1 * rng.standard_normal((rank, n)), "f32")
    U, V = _dev(u, "f32"), _dev(v, "f32")
    xs = [P.round_to(rng.standard_normal((t, inn)), "f32") for _ in range(2)]
    X, Y = [_dev(x, "f32") for x in xs], [torch.zeros((t, out), device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    streams, handles, graphs = [torch.cuda.Stream() for _ in range(2)], [], []
    for i in range(2):
        h = api.Hyacin(stream=streams[i].cuda_stream)
        handles.append(h)

        def call():
            assert h.product_w4(op, m, n, t, api.F32, Q, ldq, 64, S, None, S.shape[1], X[i], inn, rank, U, m, V, n, Y[i], out) == 0
        with torch.cuda.stream(streams[i]):
            call()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[i]):
                call()
            graphs.append(g)
    for _ in range(5):
        for y in Y:
            y.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            _check_product(_back(Y[i], out), op, m, n, "f32", 64, codes, scales, None, xs[i], u, v)
    del graphs, g
    for h in handles:
        h.destroy()
