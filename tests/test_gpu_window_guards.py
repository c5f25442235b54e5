"""Window attention's device guards where walks are shared by several workgroups, and in the
search among more requests than a wave holds (tolerances: window_util)."""
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


class Runs:
    """Commands of case `c` one after another on one queue."""

    def __init__(self, env, c, **plan):
        self.torch, self.L = env
        self.c, self.plan = c, c.plan(self.L, **plan)
        self.queue = self.L.CommandQueue(self.torch.cuda.current_stream(), 20)

    def __call__(self, d):
        out, lse = self.c.outputs(self.torch)
        self.torch.cuda.synchronize()
        b = self.queue.bindings(16)
        args = self.c.args(self.L, b, d, out, lse)
        scope = self.queue.begin(b)
        self.plan.enqueue_into(scope, args)
        scope.finish().wait()
        return host(out), host(lse)


def same(a, b, rows):
    return all(np.array_equal(x[rows], y[rows]) for x, y in zip(a, b))


def untouched(got, rows):
    return all((x[rows] == 7).all() for x in got)


@pytest.mark.parametrize("what", ["index", "sink", "last", "range", "ends"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [None, [5, 9]])
def test_bad_requests_of_shared_walks(env, rows, dtype, what):
    """A refused request's workgroups count at no word: the queue's next command, and the
    one behind it, are right."""
    torch, L = env
    window = 2500 if what == "sink" else 0
    c = Case(91, [3000, 4100], rows, 8, 2, window, 4, 16, "NHD", dtype)
    run = Runs(env, c)
    good = run(c.operands(torch))
    c.check(*good)
    n0 = c.rows[0]
    d = c.operands(torch)
    bad = [slice(0, n0)]
    if what == "index":  # the last page of the first request
        d["indices"][int(c.indptr[1]) - 1] = c.pool
    elif what == "sink":
        d["indices"][0] = -1
    elif what == "last":
        d["last"][0] = 17
    elif what == "range":  # no page of its own
        d["indptr"][1] = 0
    else:
        d["indptr"][2] -= 1
        bad.append(slice(n0, None))
    for _ in range(2):
        got = run(d)
        for rows_ in bad:
            assert untouched(got, rows_)
        if what in ("index", "sink", "last"):
            assert same(got, good, slice(n0, None))
        assert same(run(c.operands(torch)), good, slice(None))


def many(dtype):
    """150 requests, some without rows, the first and the last two among them."""
    rng = np.random.default_rng(92)
    lens = rng.integers(1, 120, 150)
    rows = [int(min(n, m)) for n, m in zip(lens, rng.integers(0, 9, 150))]
    rows[0] = rows[-1] = rows[-2] = 0
    rows[70], rows[71] = min(4, int(lens[70])), 0
    return Case(92, lens, rows, 4, 2, 50, 2, 16, "NHD", dtype)


@pytest.mark.parametrize("what", ["qo_falls", "qo_start", "qo_end", "ends", "index", "last", "short"])
@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", ["bf16", "mxfp4"])
def test_bad_tables_of_many_requests(env, dtype, tile, what):
    torch, L = env
    c = many(dtype)
    good = c.run(torch, L, tile_cols=tile)
    c.check(*good, long_tile=tile == "long")
    qo = np.concatenate([[0], np.cumsum(c.rows)])
    d = c.operands(torch)
    r = 70
    mine, rest = slice(qo[r], qo[r + 1]), [slice(0, qo[r]), slice(qo[r + 1], None)]
    if what == "qo_falls":  # rows from the first falling range on
        d["qo"][r + 1] = int(qo[r]) - 1
        mine, rest = slice(qo[r], None), [slice(0, qo[r])]
    elif what in ("qo_start", "qo_end", "ends"):
        if what == "ends":
            d["indptr"][150] += 1
        else:
            d["qo"][0 if what == "qo_start" else 150] += 1
        mine, rest = slice(0, None), []
    elif what == "index":
        d["indices"][int(c.indptr[r + 1]) - 1] = -1
    elif what == "last":
        d["last"][r] = 0
    elif what == "short":  # no page left: fewer tokens than rows
        d["indptr"][r + 1] = int(c.indptr[r])
        rest = [slice(0, qo[r]), slice(qo[r + 2], None)]  # (the next one has its pages)
    got = c.run(torch, L, d, tile_cols=tile)
    assert untouched(got, mine)
    for s in rest:
        assert same(got, good, s)
