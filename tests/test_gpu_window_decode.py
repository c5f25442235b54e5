"""Window attention of one row per request against the definition in 64 bits
(tolerances: window_util)."""
import numpy as np
import pytest

from window_util import Case, host

pytestmark = pytest.mark.gpu
DTYPES = ["bf16", "fp8_e4m3", "mxfp4"]


@pytest.fixture(scope="module")
def env():
    import torch
    import loom_infer_hip as L
    return torch, L


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,layout", [(16, "NHD"), (32, "HND"), (64, "NHD"), (64, "HND")])
def test_lengths_around_the_window(env, dtype, page, layout):
    """From one token to contexts past the window and the sinks, page ends inside a step."""
    lens = [1, 2, 15, 16, 17, 33, 64, 65, 99, 100, 101, 116, 117, 150, 257, 1000]
    c = Case(1, lens, None, 8, 2, 100, 4, page, layout, dtype)
    c.check(*c.run(*env))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (1, 40), (16, 16), (17, 15), (33, 100),
                                          (128, 0), (1000, 3), (0, 0), (0, 9), (1 << 40, 1 << 40)])
def test_windows_and_sinks(env, dtype, window, sinks):
    c = Case(2, [5, 16, 47, 130, 515], None, 8, 2, window, sinks, 16, "NHD", dtype)
    c.check(*c.run(*env))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (28, 4), (32, 32), (17, 1), (80, 2), (64, 8)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_groups(env, hq, hkv, dtype):
    """Groups of one head, odd ones, and more heads than a tile has columns."""
    c = Case(3, [3, 70, 301], None, hq, hkv, 90, 5, 32, "HND", dtype)
    c.check(*c.run(*env))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,window", [([5000], 4096), ([2600, 40, 1], 2048), ([9000], 0)])
def test_long_windows_of_few_requests(env, dtype, lens, window):
    """Walks that several workgroups share, and more steps than a wave places at once."""
    c = Case(4, lens, None, 8, 2, window, 20, 16, "HND", dtype)
    c.check(*c.run(*env))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_requests(env, dtype):
    c = Case(5, list(np.random.default_rng(5).integers(1, 90, 150)), None, 4, 4, 50, 2, 16, "NHD", dtype)
    c.check(*c.run(*env))


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_given_away(env, dtype):
    """Only the indices of pages that a row sees are read: the others are -1."""
    c = Case(6, [40, 300, 1500], None, 8, 2, 70, 17, 16, "NHD", dtype, freed=True)
    assert (c.indices == -1).sum() > 50
    c.check(*c.run(*env))


@pytest.mark.parametrize("dtype", DTYPES)
def test_aligned_to_four_bytes(env, dtype):
    c = Case(7, [9, 200], None, 8, 2, 64, 4, 16, "NHD", dtype)
    want = c.run(*env)
    got = c.run(*env, offset=4)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("lens", [[700], [33, 260]])
@pytest.mark.parametrize("dtype", ["bf16", "mxfp4", "fp8_e4m3"])
def test_hidden_tokens_have_no_part(env, lens, dtype):
    """NaN and infinities in K and V of tokens that no row sees, the rows of a partly
    visible block and of the last page past the end among them."""
    c = Case(8, lens, None, 8, 2, 50, 5, 16, "NHD", dtype)
    want = c.run(*env)
    for r, n in enumerate(lens):
        slots = range(len(c.indices[c.indptr[r]:c.indptr[r + 1]]) * 16)
        for t in slots:
            if t >= n or c.sinks <= t < n - 50:
                page = c.indices[c.indptr[r] + t // 16]
                for which, cache in enumerate(c.cache):
                    if dtype == "mxfp4":
                        cache[1][page, :, t % 16] = 255
                    elif dtype == "fp8_e4m3":
                        cache[page, :, t % 16] = 0x7F
                    else:
                        cache[page, :, t % 16] = [np.nan, np.inf, -np.inf][(t + which) % 3]
    got = c.run(*env)
    # (a column found token by token is rounded at other places)
    c.check(*got)
    assert np.abs(got[0] - want[0]).max() <= 2 ** -6 * np.abs(want[0]).max()


def test_visible_infinities(env):
    """An infinite V among the visible tokens is the mean's; a score of -inf weighs nothing,
    one of +inf leaves NaN."""
    c = Case(9, [60, 60, 60, 60], None, 4, 1, 40, 2, 16, "NHD", "bf16")
    k, v = c.cache
    slot = lambda r, t: (c.indices[c.indptr[r] + t // 16], 0, t % 16)  # noqa: E731
    v[slot(0, 50)][3] = np.inf
    k[slot(1, 1)][:] = 0
    k[slot(1, 1)][0] = -np.inf
    c.q[1, :, 0] = 1.0
    k[slot(2, 33)][:] = 0
    k[slot(2, 33)][0] = np.inf
    c.q[2, :, 0] = 1.0
    out, lse = c.run(*env)
    assert np.isposinf(out[0, :, 3]).all() and np.isfinite(np.delete(out[0], 3, 1)).all()
    c.check(out, lse, only=[1, 3])
    assert np.isnan(out[2]).all() and np.isnan(lse[2]).all()


def test_every_score_minus_infinity(env):
    c = Case(10, [20], None, 2, 1, 8, 1, 16, "NHD", "bf16")
    c.cache[0][..., 0] = -np.inf
    c.q[..., 0] = 1.0
    out, lse = c.run(*env)
    assert np.isnan(out).all() and np.isneginf(lse).all()


@pytest.mark.parametrize("scale", [0.0, -0.02])
def test_fp8_scales_that_do_not_keep_the_order(env, scale):
    """k_scale 0 (an empty cache's) weighs every token alike."""
    torch, L = env
    import window_util
    c = Case(11, [70, 9], None, 4, 2, 30, 2, 16, "NHD", "fp8_e4m3")
    d = c.operands(torch)
    d["kv_scales"][0] = scale
    saved, window_util.K_SCALE = window_util.K_SCALE, scale
    try:
        c.check(*c.run(torch, L, d))
    finally:
        window_util.K_SCALE = saved


@pytest.mark.parametrize("rows", [None, [1]])
def test_a_normalizer_past_fp32(env, rows):
    """A negative k_scale: weights near FP32's end against the lowest score, whose sum passes
    it, over V of zeros."""
    torch, L = env
    import window_util
    c = Case(19, [32], rows, 1, 1, 0, 0, 16, "NHD", "fp8_e4m3")
    c.q[:] = 0
    c.q[..., 0] = 1
    k, v = c.cache
    k[:] = v[:] = 0
    k[c.indices[0], 0, 0, 0] = 0x50  # 8.0, the other rows' is 0
    scale = np.float32(-127.5 / 8 * np.log(2) * np.sqrt(128))
    d = c.operands(torch)
    d["kv_scales"][0] = float(scale)
    saved, window_util.K_SCALE = window_util.K_SCALE, scale
    try:
        assert window_util.fp8_values()[0x50] == 8.0
        assert abs(c.reference()[1][0, 0] - np.log2(31)) < 1e-6
        for tile in (0,) if rows is None else (16, "long"):
            c.check(*c.run(torch, L, d, **({} if rows is None else dict(tile_cols=tile))),
                    long_tile=tile == "long")
    finally:
        window_util.K_SCALE = saved


def test_scores_far_apart(env):
    """Scores of thousands: one token takes the whole weight."""
    c = Case(12, [300, 45], None, 4, 2, 200, 4, 16, "NHD", "bf16")
    c.q *= 64
    c.check(*c.run(*env))


@pytest.mark.parametrize("what", ["ends", "start", "last", "last_low", "index", "negative", "range"])
def test_bad_tables_leave_rows_untouched(env, what):
    torch, L = env
    c = Case(13, [40, 200, 90], None, 8, 2, 64, 4, 16, "NHD", "bf16")
    want = c.run(torch, L)
    d = c.operands(torch)
    rows = [1]
    if what == "ends":
        d["indptr"][3] -= 1
        rows = [0, 1, 2]
    elif what == "start":
        d["indptr"][0] = 1
        rows = [0, 1, 2]
    elif what == "last":
        d["last"][1] = 17
    elif what == "last_low":
        d["last"][1] = 0
    elif what == "index":
        d["indices"][c.indptr[2] - 1] = c.pool
    elif what == "negative":
        d["indices"][c.indptr[1]] = -1  # a sink's
    elif what == "range":
        d["indptr"][1] = c.indptr[2] + 1
        rows = [1]
    got = c.run(torch, L, d)
    for r in range(3):
        if r in rows:
            assert (got[0][r] == 7).all() and (got[1][r] == 7).all()
        elif what != "range":  # (its first request has another's pages then)
            assert np.array_equal(got[0][r], want[0][r]) and np.array_equal(got[1][r], want[1][r])


def test_capacity_plans_ignore_what_follows(env):
    torch, L = env
    c = Case(14, [40, 200], None, 8, 2, 64, 4, 16, "NHD", "mxfp4")
    want = c.run(torch, L)
    d = c.operands(torch)
    d["indices"] = torch.cat([d["indices"], torch.full((9,), -5, dtype=torch.int32, device="cuda")])
    got = c.run(torch, L, d, capacity=True)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    got = c.run(torch, L, d)
    assert (got[0] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_pages(env, dtype):
    """Pages past 2^32 bytes of the pool."""
    torch, L = env
    row = {"bf16": 256, "fp8_e4m3": 128, "mxfp4": 64}[dtype]
    c = Case(15, [50, 130], None, 8, 2, 60, 4, 64, "HND", dtype)
    want = c.run(torch, L)
    far = (1 << 32) // (64 * 2 * row) + 5
    d = c.operands(torch)
    small, c.pool = c.pool, far + c.pool
    for k in [k for k in d if k[0] in "kv" and k != "kv_scales"]:
        big = torch.zeros(d[k].numel() // small * c.pool, dtype=d[k].dtype, device="cuda")
        big[big.numel() - d[k].numel():] = d[k]
        d[k] = big
    d["indices"] += far
    got = c.run(torch, L, d)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_a_stream_of_its_own(env):
    torch, L = env
    c = Case(16, [70, 2000], None, 8, 2, 1500, 4, 16, "NHD", "bf16")
    want = c.run(torch, L)
    s = torch.cuda.Stream()
    got = c.run(torch, L, stream=s)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeated_and_mixed_commands_on_one_queue(env, dtype):
    """Shared walks leave their queue's words as they found them: the same results command
    after command, two plans and their operands in turn."""
    torch, L = env
    cases = [Case(17, [3000], None, 8, 2, 2048, 4, 16, "NHD", dtype),
             Case(18, [900, 2500], None, 16, 4, 0, 0, 32, "HND", dtype)]
    want = [c.run(torch, L) for c in cases]
    queue = L.CommandQueue(torch.cuda.current_stream(), 100)
    b = queue.bindings(40)
    work = []
    for c in cases:
        o = c.outputs(torch)
        work.append((c.plan(L), c.args(L, b, c.operands(torch), *o), o))
    scope = queue.begin(b)
    for _ in range(10):
        for plan, args, o in work:
            plan.enqueue_into(scope, args)
    scope.finish().wait()
    for (_, _, o), w in zip(work, want):
        assert np.array_equal(host(o[0]), w[0]) and np.array_equal(host(o[1]), w[1])
