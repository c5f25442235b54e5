"""Window attention over finite V whose weighted sums pass FP32's range though their means
do not (tolerances: window_util)."""
import numpy as np
import pytest

from window_util import Case

pytestmark = pytest.mark.gpu
FORMS = {"one row": (None, 0), "rows": ([40], 16), "rows, long tile": ([40], "long")}


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", ["bf16", "mxfp4"])
@pytest.mark.parametrize("signs", ["one", "both"])
def test_means_of_the_largest_values(form, dtype, signs):
    import torch
    import loom_infer_hip as L
    rows, tile = FORMS[form]
    c = Case(71, [90], rows, 4, 2, 50, 3, 16, "NHD", dtype)
    # V up to 2^127 (BF16) or 6 * 2^125 (MXFP4)
    if dtype == "mxfp4":
        codes, scales = c.cache[1]
        scales[:] = 252
        if signs == "one":
            codes &= 0x77
    else:
        v = c.cache[1]
        v[:] = np.sign(v) * 2.0 ** 126 * (1 + np.floor(np.abs(v) * 32) % 128 / 128)
        if signs == "one":
            v[:] = np.abs(v)
    o, lse, *_ = c.reference()
    assert np.isfinite(o).all() and np.abs(o).max() < 2.0 ** 128 * (1 - 2.0 ** -8)
    c.check(*c.run(torch, L, **({} if rows is None else dict(tile_cols=tile))),
            long_tile=tile == "long")
