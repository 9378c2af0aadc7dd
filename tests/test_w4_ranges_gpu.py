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
