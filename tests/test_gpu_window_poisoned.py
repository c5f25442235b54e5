"""Window attention over queries or keys that are no numbers: NaN rows, and no more time for
them than a walk and a look at every column."""
import numpy as np
import pytest

from window_util import Case, host

pytestmark = pytest.mark.gpu
FORMS = {"one row": (None, 0), "rows": ([130], 16), "rows, long tile": ([130], "long")}


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", ["bf16", "fp8_e4m3", "mxfp4"])
@pytest.mark.parametrize("what", ["queries", "a first key"])
def test_rows_that_are_no_numbers(what, dtype, form):
    """Finding their columns token by token to the end would take 100 times the command's
    time and more."""
    import torch
    import loom_infer_hip as L
    rows, tile = FORMS[form]
    c = Case(101, [4003], rows, 8, 2, 3000, 3, 16, "NHD", dtype)
    plan = c.plan(L, **({} if rows is None else dict(tile_cols=tile)))

    def best():
        d = c.operands(torch)
        out, lse = c.outputs(torch)
        queue = L.CommandQueue(torch.cuda.current_stream(), 200)
        b = queue.bindings(16)
        args = c.args(L, b, d, out, lse)
        scope = queue.begin(b)
        times = []
        for _ in range(8):
            t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            t0.record()
            for _ in range(4):
                plan.enqueue_into(scope, args)
            t1.record()
            t1.synchronize()
            times.append(t0.elapsed_time(t1))
        scope.finish().wait()
        return min(times), host(out), host(lse)

    usual, *good = best()
    c.check(*good, long_tile=tile == "long")
    if what == "queries":
        c.q[:] = np.nan
    elif dtype == "mxfp4":
        c.cache[0][1][c.indices[0], :, 0] = 255
    else:
        c.cache[0][c.indices[0], :, 0] = 0x7F if dtype == "fp8_e4m3" else np.nan
    this, out, lse = best()
    assert np.isnan(out).all() and np.isnan(lse).all()
    assert this <= 10 * usual, f"{this:.3f} ms against {usual:.3f}"
