"""Window attention of ragged rows against the definition in 64 bits (tolerances:
window_util), on row tiles and on long tiles."""
import numpy as np
import pytest

from window_util import Case, host

pytestmark = pytest.mark.gpu
DTYPES = ["bf16", "fp8_e4m3", "mxfp4"]
TILES = [16, "long"]


@pytest.fixture(scope="module")
def env():
    import torch
    import loom_infer_hip as L
    return torch, L


def check(env, c, tile, **more):
    plan = c.plan(env[1], tile_cols=tile)
    assert plan.algorithm == ("long_tile" if tile == "long" else "row_tile")
    c.check(*c.run(*env, tile_cols=tile, **more), long_tile=tile == "long")


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,layout", [(16, "NHD"), (32, "HND"), (64, "NHD"), (64, "HND")])
def test_ragged_rows(env, tile, dtype, page, layout):
    """Whole prompts, chunks behind prefixes, single rows, requests without rows."""
    c = Case(21, [70, 300, 1, 33, 129, 40], [70, 90, 1, 0, 3, 40], 8, 2, 50, 5, page, layout, dtype)
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (15, 40), (16, 16), (33, 100), (64, 0),
                                          (128, 129), (500, 3), (0, 0), (0, 9), (1 << 40, 1 << 40)])
def test_windows_and_sinks(env, tile, dtype, window, sinks):
    c = Case(22, [515, 47], [160, 47], 4, 1, window, sinks, 16, "NHD", dtype)
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (28, 4), (8, 8), (17, 1), (80, 2), (130, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_groups(env, tile, hq, hkv, dtype):
    """Groups of one head, odd ones, and more heads than a tile has columns."""
    c = Case(23, [37, 170], [5, 41], hq, hkv, 90, 5, 32, "HND", dtype)
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,rows,window", [([5000], [3], 4096), ([2600, 700], [8, 1], 0),
                                              ([4500], [130], 2100)])
def test_long_walks(env, tile, dtype, lens, rows, window):
    """Walks that several workgroups share, and more blocks than are placed at once."""
    c = Case(24, lens, rows, 4, 1, window, 20, 16, "HND", dtype)
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_requests(env, tile, dtype):
    """More requests than a wave holds, some without rows, the last ones too."""
    rng = np.random.default_rng(25)
    lens = rng.integers(1, 120, 150)
    rows = [int(min(n, m)) for n, m in zip(lens, rng.integers(0, 9, 150))]
    rows[0] = rows[-1] = rows[-2] = 0
    c = Case(25, lens, rows, 4, 2, 50, 2, 16, "NHD", dtype)
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_given_away(env, tile, dtype):
    c = Case(26, [40, 300, 1500], [40, 7, 200], 8, 2, 70, 17, 16, "NHD", dtype, freed=True)
    assert (c.indices == -1).sum() > 50
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
def test_large_grids(env, tile):
    """Several rounds of workgroups."""
    c = Case(27, [900, 1300], [900, 700], 16, 4, 200, 4, 16, "NHD", "bf16")
    check(env, c, tile)


@pytest.mark.parametrize("rows", [[1500], [600, 500, 700]])
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_plan_s_own_choice(env, rows, dtype):
    """Enough rows for long tiles of either width."""
    for hq, hkv in ((4, 1), (32, 8)):
        c = Case(28, [n + 41 for n in rows], rows, hq, hkv, 130, 4, 64, "HND", dtype)
        plan = c.plan(env[1])
        c.check(*c.run(*env), long_tile=plan.algorithm == "long_tile")


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_hidden_tokens_have_no_part(env, tile, dtype):
    """NaN and infinities in K and V of one token: rows that do not see it, in its tile and
    its block, keep their results."""
    torch, L = env
    c = Case(29, [300], [200], 4, 2, 50, 5, 16, "NHD", dtype)
    want = c.run(torch, L, tile_cols=tile)
    for t, seen in ((180, range(80, 130)), (3, range(200)), (60, range(10))):
        saved = [[x.copy() for x in s] if dtype == "mxfp4" else s.copy() for s in c.cache]
        page = c.indices[t // 16]
        for which, cache in enumerate(c.cache):
            if dtype == "mxfp4":
                cache[1][page, :, t % 16] = 255
            elif dtype == "fp8_e4m3":
                cache[page, :, t % 16] = 0x7F
            else:
                cache[page, :, t % 16] = [np.nan, np.inf][which]
        got = c.run(torch, L, tile_cols=tile)
        rest = [i for i in range(200) if i not in seen]
        if rest:
            c.check(*got, long_tile=tile == "long", only=rest)
        assert np.isnan(got[0][list(seen)]).any(-1).all() and np.isnan(got[1][list(seen)]).all()
        c.cache = saved
    again = c.run(torch, L, tile_cols=tile)
    assert np.array_equal(again[0], want[0]) and np.array_equal(again[1], want[1])


@pytest.mark.parametrize("tile", TILES)
def test_visible_infinities(env, tile):
    c = Case(30, [90], [90], 2, 1, 40, 2, 16, "NHD", "bf16")
    c.cache[1][c.indices[3], 0, 2, 5] = np.inf  # token 50
    out, lse = c.run(*env, tile_cols=tile)
    seen = list(range(50, 90))
    assert np.isposinf(out[seen][..., 5]).all()
    c.check(out, lse, long_tile=tile == "long", only=[i for i in range(90) if i not in seen])
    assert np.isfinite(np.delete(out[seen], 5, 2)).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_apart(env, tile, dtype):
    c = Case(31, [300, 45], [120, 45], 4, 2, 100, 4, 16, "NHD", dtype)
    c.q *= 64
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
def test_rising_scores(env, tile):
    """Every block's scores above the last one's by far: the reference moves each time."""
    c = Case(32, [400], [70], 2, 1, 0, 0, 16, "NHD", "bf16")
    k = c.cache[0]
    for t in range(400):
        k[c.indices[t // 16], 0, t % 16] = np.sign(c.q[0, 0]) * (t // 8) / 4
    c.q = np.sign(c.q[:1, :1]) * np.ones_like(c.q)
    check(env, c, tile)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("what", ["qo_start", "qo_end", "qo_falls", "ends", "last", "index", "short"])
def test_bad_tables_leave_rows_untouched(env, tile, what):
    torch, L = env
    c = Case(33, [60, 200, 90, 30], [20, 70, 33, 30], 8, 2, 64, 4, 16, "NHD", "bf16")
    want = c.run(torch, L, tile_cols=tile)
    d = c.operands(torch)
    qo = np.concatenate([[0], np.cumsum(c.rows)])
    bad = {1}
    if what == "qo_start":
        d["qo"][0] = 1
        bad = {0, 1, 2, 3}
    elif what == "qo_end":
        d["qo"][4] -= 1
        bad = {0, 1, 2, 3}
    elif what == "qo_falls":  # rows belong to the requests before the first malformed range
        d["qo"][2] = 10
        bad = {1, 2, 3}
    elif what == "ends":
        d["indptr"][4] += 1
        bad = {0, 1, 2, 3}
    elif what == "last":
        d["last"][1] = 0
    elif what == "index":
        d["indices"][c.indptr[1] + 7] = c.pool
    elif what == "short":  # more rows than tokens
        d["indptr"][1] = c.indptr[2] - 1
        d["indices"][c.indptr[1]:c.indptr[2]] = 0
        bad = {1}
    got = c.run(torch, L, d, tile_cols=tile)
    for r in range(4):
        s = slice(qo[r], qo[r + 1])
        if r in bad:
            assert (got[0][s] == 7).all() and (got[1][s] == 7).all(), r
        elif not (what == "short" and r == 0):  # (that one has more tokens then)
            assert np.array_equal(got[0][s], want[0][s]) and np.array_equal(got[1][s], want[1][s])


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_aligned_to_four_bytes(env, tile, dtype):
    c = Case(34, [90, 200], [90, 50], 8, 2, 64, 4, 16, "NHD", dtype)
    want = c.run(*env, tile_cols=tile)
    got = c.run(*env, offset=4, tile_cols=tile)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_far_pages(env, tile, dtype):
    """Pages past 2^32 bytes of the pool."""
    torch, L = env
    row = {"bf16": 256, "fp8_e4m3": 128, "mxfp4": 64}[dtype]
    c = Case(35, [50, 330], [50, 60], 8, 2, 60, 4, 64, "NHD", dtype)
    want = c.run(torch, L, tile_cols=tile)
    far = (1 << 32) // (64 * 2 * row) + 5
    d = c.operands(torch)
    small, c.pool = c.pool, far + c.pool
    for k in [k for k in d if k[0] in "kv" and k != "kv_scales"]:
        big = torch.zeros(d[k].numel() // small * c.pool, dtype=d[k].dtype, device="cuda")
        big[big.numel() - d[k].numel():] = d[k]
        d[k] = big
    d["indices"] += far
    got = c.run(torch, L, d, tile_cols=tile)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_repeated_commands(env, tile, dtype):
    """The same results command after command, on a stream of its own."""
    torch, L = env
    c = Case(36, [3000, 2200], [9, 4], 8, 2, 2048, 4, 16, "NHD", dtype)
    want = c.run(torch, L, tile_cols=tile)
    stream = torch.cuda.Stream()
    d, (out, lse) = c.operands(torch), c.outputs(torch)
    torch.cuda.synchronize()
    queue = L.CommandQueue(stream, 20)
    b = queue.bindings(16)
    plan, args = c.plan(L, tile_cols=tile), c.args(L, b, d, out, lse)
    scope = queue.begin(b)
    for _ in range(20):
        plan.enqueue_into(scope, args)
    scope.finish().wait()
    assert np.array_equal(host(out), want[0]) and np.array_equal(host(lse), want[1])
