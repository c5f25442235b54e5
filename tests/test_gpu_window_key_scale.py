"""Window attention over FP8 pages with a k_scale of 0 or below (tolerances: window_util)."""
import numpy as np
import pytest

import window_util
from window_util import Case, host

pytestmark = pytest.mark.gpu
FORMS = {"one row": (None, 0), "rows": ([130], 16), "rows, long tile": ([130], "long")}
SCALES = [0.0, -0.02, -1e-45]  # (the last leaves nothing of the softmax scale in FP32)


@pytest.fixture(scope="module")
def env():
    import torch
    import loom_infer_hip as L
    return torch, L


def at_scale(c, torch, monkeypatch, scale):
    monkeypatch.setattr(window_util, "K_SCALE", scale)
    return c.operands(torch)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("window,sinks", [(30, 2), (200, 0), (0, 0)])
def test_the_definition(env, monkeypatch, window, sinks, scale, form):
    torch, L = env
    rows, tile = FORMS[form]
    c = Case(81, [333], rows, 4, 2, window, sinks, 16, "NHD", "fp8_e4m3")
    d = at_scale(c, torch, monkeypatch, scale)
    c.check(*c.run(torch, L, d, **({} if rows is None else dict(tile_cols=tile))),
            long_tile=tile == "long")


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", SCALES[:2])
def test_infinite_queries(env, monkeypatch, scale, form):
    """An infinity times 0 is no number, and times a negative scale the other one."""
    torch, L = env
    rows, tile = FORMS[form]
    c = Case(82, [200], rows, 1, 1, 30, 2, 16, "NHD", "fp8_e4m3")
    c.cache[0][..., 0] = 0x38  # 1.0
    c.q[..., 0] = np.inf  # scores of +inf (NaN), or of -inf
    out, lse = c.run(torch, L, at_scale(c, torch, monkeypatch, scale),
                     **({} if rows is None else dict(tile_cols=tile)))
    assert np.isnan(out).all()
    assert np.isnan(lse).all() if scale == 0 else np.isneginf(lse).all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", SCALES[:2])
def test_the_time(env, monkeypatch, scale, form):
    """No slower than a positive scale, but for noise (columns found token by token take
    more than thirty times as long)."""
    torch, L = env
    rows, tile = FORMS[form]
    c = Case(83, [3003], rows, 8, 2, 2000, 3, 16, "NHD", "fp8_e4m3")
    plan = c.plan(L, **({} if rows is None else dict(tile_cols=tile)))

    def best(k_scale):
        d = at_scale(c, torch, monkeypatch, k_scale)
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
        return min(times)

    usual, this = best(0.02), best(scale)
    assert this <= 5 * usual, f"{this:.3f} ms against {usual:.3f}"
