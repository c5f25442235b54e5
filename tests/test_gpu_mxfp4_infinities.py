"""MXFP4 decode where scores are infinite and values are the largest.

A score is -inf here where a finite query meets a key so large that their product
passes FP32; softmax gives such a token no weight.  The tolerances of O and LSE are
those of the finite tokens (test_gpu_mxfp4_decode)."""
import numpy as np
import pytest

import mxfp4_util as mx
from test_gpu_mxfp4_decode import LOG2E, Case, run

pytestmark = pytest.mark.gpu

FORMS = {
    # lens, hq, hkv, page, layout; teams
    "one workgroup each": (([300, 40, 97], 8, 2, 16, "NHD"), 0),
    "tiles of 8 heads": (([333, 64, 5], 32, 2, 32, "HND"), 0),
    "splits": (([1500, 700], 8, 2, 16, "NHD"), 0),
    "splits, tiles of 7": (([1500, 1100], 28, 4, 64, "HND"), 0),
    "balanced": (([300, 500, 64], 8, 2, 16, "NHD"), 13),
    "balanced, tiles of 7": (([800, 33], 28, 4, 64, "HND"), 40),
}


@pytest.fixture(scope="module")
def env():
    import torch

    import loom_infer_hip as L
    return torch, L


def case(env, form):
    """A case whose queries are 2^20 in dim 0, where every key is 0."""
    shape, teams = FORMS[form]
    c = Case(env[0], 130, *shape)
    c.q[:, :, 0] = 2.0 ** 20
    c.k[0][..., 0] &= 0xF0
    return c, teams


def put_key(c, r, t, h, code):
    """Token t's key in request r and kv-head h: `code` * 2^125 in dim 0, else zeros in that
    block of 32."""
    page, row = c.indices[c.indptr[r] + t // c.page], t % c.page
    c.k[0][page, h, row, :16] = 0
    c.k[0][page, h, row, 0] = code
    c.k[1][page, h, row, 0] = 252


def expect(c, out, lse, gone):
    """O and LSE over the tokens that are not in gone[r]."""
    g = c.hq // c.hkv
    for r, n in enumerate(c.lens):
        keep = np.ones(n, bool)
        keep[gone[r]] = False
        k, v = (mx.rows_of(x, c.indptr, c.indices, r, n)[keep] for x in (c.k, c.v))
        ref_o, ref_l = mx.attend(c.q[r], k, v)
        score = max((np.abs(np.ascontiguousarray(k[:, h])) @ np.abs(c.q[r, h * g:(h + 1) * g]).T).max()
                    for h in range(c.hkv))
        off = score * mx.D ** -0.5 * LOG2E * 128 * 2.0 ** -24 + 2.0 ** -20
        bo = 2.0 ** -8 * np.abs(ref_o) + np.abs(v).max() * (2 * off + 2.0 ** -15 + 2.0 ** -20)
        bl = off + 2.0 ** -22 * np.abs(ref_l) + 2.0 ** -20
        assert (np.abs(out[r] - ref_o) <= bo).all() and (np.abs(lse[r] - ref_l) <= bl).all(), r


@pytest.mark.parametrize("form", list(FORMS))
def test_tokens_that_score_minus_infinity(env, form):
    """Runs of them: the first blocks, whole splits and ranges, single ones, all but the
    last token."""
    c, teams = case(env, form)
    gone = []
    for r, n in enumerate(c.lens):
        t = np.arange(n)
        run_ = {0: (t < 70) | ((t > n // 3) & (t < n // 2)) | (t == n - 1),
                1: t < n - 1, 2: t % 5 == 0}[r]
        gone.append(np.flatnonzero(run_))
        for h in range(c.hkv):
            for i in gone[r]:
                put_key(c, r, int(i), h, 0x0F)  # -6 * 2^125 * 2^20
    out, lse, plan = run(env, c, {"teams": teams})
    assert (plan.algorithm == "direct") == (teams == 0)
    expect(c, out, lse, gone)


@pytest.mark.parametrize("form", list(FORMS))
def test_heads_without_a_finite_score(env, form):
    """All -inf: LSE is -inf and O is NaN, as of a softmax over nothing.  One +inf: O and
    LSE are NaN.  Heads and requests beside them keep their bits."""
    c, teams = case(env, form)
    clean = run(env, c, {"teams": teams})
    g = c.hq // c.hkv
    for i in range(c.lens[0]):
        put_key(c, 0, i, 1, 0x0F)
    put_key(c, 1, c.lens[1] // 2, 0, 0x07)
    out, lse, _ = run(env, c, {"teams": teams})
    hit = np.zeros(lse.shape, bool)
    hit[0, g:2 * g] = hit[1, :g] = True
    assert np.isnan(out[hit]).all()
    assert (lse[0, g:2 * g] == -np.inf).all() and np.isnan(lse[1, :g]).all()
    assert np.array_equal(out[~hit], clean[0][~hit]) and np.array_equal(lse[~hit], clean[1][~hit])


@pytest.mark.parametrize("form", list(FORMS))
def test_infinite_queries(env, form):
    """Against keys of one sign: -inf scores throughout, or +inf ones; beside them heads
    with finite queries keep their bits."""
    c, teams = case(env, form)
    clean = run(env, c, {"teams": teams})
    c.k[0][..., 0] |= 0x02  # 1 * 2^scale in dim 0
    c.q[:, :, 0] = 0.0
    c.q[0, 0, 0], c.q[1, 1, 0] = -np.inf, np.inf
    out, lse, _ = run(env, c, {"teams": teams})
    assert np.isnan(out[0, 0]).all() and lse[0, 0] == -np.inf
    assert np.isnan(out[1, 1]).all() and np.isnan(lse[1, 1])
    c.q[0, 0, 0] = c.q[1, 1, 0] = 0.0
    want = run(env, c, {"teams": teams})
    hit = np.zeros(lse.shape, bool)
    hit[0, 0] = hit[1, 1] = True
    assert np.isfinite(want[0]).all() and np.isfinite(clean[0]).all()
    assert np.array_equal(out[~hit], want[0][~hit]) and np.array_equal(lse[~hit], want[1][~hit])


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("form", list(FORMS))
def test_values_up_to_fp32s_range_over_the_tokens(env, form, rising):
    """Weights are at most 1 and O is summed before it is divided: values below 2^128 over
    the request's tokens cannot overflow, of equal scores or of rising ones (whose weights
    come nearest to 1)."""
    c, teams = case(env, form)
    c.k[0][:] = 0
    if rising:  # scores of 7 (log2) below the first block's bound, from the second block on
        c.q[:, :, 0] = mx.bf16_round(np.array(7.9 / LOG2E * mx.D ** 0.5 / 6))
        for r, n in enumerate(c.lens):
            for h in range(c.hkv):
                for i in range(32, n):
                    put_key(c, r, i, h, 0x07)
        c.k[1][..., 0] = 127
    most = max(c.lens)
    c.v[0][:] = 0x77  # 6
    c.v[1][:] = 127 + int(np.floor(np.log2(2.0 ** 128 / (6 * most))))
    v = 6 * 2.0 ** (int(c.v[1].flat[0]) - 127)
    assert v * most < 2.0 ** 128 <= 2 * v * most
    out, lse, _ = run(env, c, {"teams": teams})
    # equal values: O is that value, but for P's 16 bits and the rounding to BF16
    assert (np.abs(out - v) <= v * (2.0 ** -8 + 2.0 ** -15 + 2.0 ** -20)).all()
    assert np.isfinite(lse).all()
