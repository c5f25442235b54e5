"""Page tables of the MXFP4 commands that are longer than what is in use: capacity plans
ignore whatever lies behind indptr[B], other plans write nothing; and decode plans whose
bound is far above their tokens."""
import numpy as np
import pytest

import mxfp4_util as mx
from test_gpu_mxfp4_append import Append, rows_wanted, same_bits
from test_gpu_mxfp4_decode import Case, check, dev, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch

    import loom_infer_hip as L
    return torch, L


def longer(env, indices, entries, pool):
    """The table in front of entries that name no page."""
    rng = np.random.default_rng(entries)
    junk = rng.choice([-1, pool, 2 ** 31 - 1, -2 ** 31], entries - len(indices))
    return dev(env[0], np.concatenate([indices, junk]).astype(np.int32))


FORMS = {
    # lens, hq, hkv, page, layout; entries of the table; teams; algorithm; whether it splits
    "whole table in registers": (([40, 90, 33], 8, 2, 16, "NHD"), 15, 0, "direct", False),
    "all its entries": (([17, 1, 64], 8, 8, 32, "HND"), 128, 0, "direct", True),
    "table in memory": (([50] * 40, 4, 1, 16, "NHD"), 300, 0, "direct", False),
    "splits": (([900, 20], 28, 4, 16, "NHD"), 200, 0, "direct", True),
    "balanced": (([70, 35, 128], 8, 2, 64, "HND"), 90, 16, "balanced_split_kv", True),
}


@pytest.mark.parametrize("form", list(FORMS))
def test_decode_over_a_capacity_table(env, form):
    shape, entries, teams, algorithm, splits = FORMS[form]
    c = Case(env[0], 120, *shape)
    x = c.device()
    x[6] = longer(env, c.indices, entries, c.pool)
    opts = {"teams": teams, "max_total_pages": entries}
    out, lse, plan = run(env, c, {**opts, "indices_capacity": True}, operands=x)
    assert plan.algorithm == algorithm and (plan.info.state_slots > 0) == splits
    check(c, out, lse)
    # without the flag the table's length has to be indptr[B]
    out, lse, _ = run(env, c, opts, operands=x, fill=7.0)
    assert (out == 7.0).all() and (lse == 7.0).all()
    # a table that is shorter than indptr[B]
    x[6] = dev(env[0], c.indices[:-1])
    out, lse, _ = run(env, c, {**opts, "indices_capacity": True}, operands=x, fill=7.0)
    assert (out == 7.0).all() and (lse == 7.0).all()


@pytest.mark.parametrize("times", [1, 4, 64, 700])
@pytest.mark.parametrize("shape", [
    ([200], 32, 8, 16, "NHD"),
    ([1, 333, 64], 28, 4, 32, "HND"),
    ([5], 64, 64, 64, "NHD"),
])
def test_decode_plans_bounded_above_their_tokens(env, shape, times):
    """Splits and teams are planned from the bound: most of them get no block here."""
    c = Case(env[0], 121, *shape)
    bound = times * len(c.indices)
    out, lse, _ = run(env, c, {"max_total_pages": bound})
    check(c, out, lse)
    x = c.device()
    x[6] = longer(env, c.indices, bound, c.pool) if bound > len(c.indices) else x[6]
    got = run(env, c, {"max_total_pages": bound, "indices_capacity": True}, operands=x)
    assert np.array_equal(got[0], out) and np.array_equal(got[1], lse)
    # an invalid page keeps its request's sentinels, however many splits it has
    r = len(c.lens) - 1
    x[6][int(c.indptr[r])] = c.pool
    got = run(env, c, {"max_total_pages": bound, "indices_capacity": True}, operands=x, fill=7.0)
    assert (got[0][r] == 7.0).all() and (got[1][r] == 7.0).all()
    assert np.array_equal(got[0][:r], out[:r]) and np.array_equal(got[1][:r], lse[:r])


def read(env, c, counts, table, capacity):
    torch, L = env
    nnz = int(sum(counts))
    plan = L.PrefillProvider.load(0).plan_paged_kv_read(
        L.PagedKvReadSpec(len(c.lens), nnz, c.pool, c.hkv, kv_layout=c.layout,
                          kv_page_size=c.page), indices_capacity=capacity)
    x = c.device()[1:]
    x[5] = table
    out = [torch.full((nnz * c.hkv * mx.D,), 7.0, dtype=torch.bfloat16, device="cuda")
           for _ in range(2)]
    queue = L.CommandQueue(torch.cuda.current_stream(), 2)
    b = queue.bindings(10)
    kv = dev(torch, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    h = [b.bind_read(t) for t in (*x, kv)] + [b.bind_read_write(t).write() for t in out]
    scope = queue.begin(b)
    plan.enqueue_into(scope, L.PagedKvReadArgs(*h))
    scope.finish().wait()
    return [t.view(torch.int16).cpu().numpy().view(np.uint16).reshape(nnz, c.hkv, mx.D)
            for t in out]


@pytest.mark.parametrize("batch", [3, 70])
def test_read_back_over_a_capacity_table(env, batch):
    rng = np.random.default_rng(batch + 1)
    c = Case(env[0], 122, [int(n) for n in rng.integers(1, 60, batch)], 3, 3, 16, "HND")
    table = longer(env, c.indices, len(c.indices) + 50, c.pool)
    want = rows_wanted(c, [0] * batch, c.lens, sum(c.lens))
    for got, w in zip(read(env, c, c.lens, table, True), want):
        assert same_bits(got, w)
    for capacity, t in ((False, table), (True, dev(env[0], c.indices[:-1]))):
        for got in read(env, c, c.lens, t, capacity):
            assert (mx.bf16_values(got) == 7.0).all()


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16", "fp8_e4m3"])
@pytest.mark.parametrize("form", ["every workgroup validates", "chunks", "a token per wave",
                                  "two launches"])
def test_append_over_a_capacity_table(env, form, dtype):
    torch, L = env
    rows = {"every workgroup validates": [3, 2], "a token per wave": [900, 600]}.get(form, [90, 60])
    a = Append(env, 123, [rows[0] + 19, rows[1]], rows, 8, 2, dtype=dtype)
    flags = L.PLAN_APPEND_TWO_LAUNCH if form == "two launches" else 0
    entries = len(a.indices) + 60

    def table(x):
        x["page_indices"] = longer(env, a.indices, entries, a.pool)
    a.check(a.run(flags=flags | L.PLAN_PAGE_INDICES_CAPACITY, change=table))

    def short(x):
        x["page_indices"] = dev(torch, a.indices[:-1])
    for f, change in ((0, table), (L.PLAN_PAGE_INDICES_CAPACITY, short)):
        got = a.run(flags=flags | f, change=change)
        assert (mx.bf16_values(got["query_output"]) == 7.0).all()
        assert np.array_equal(got["key_pages"], a.pages[0])
        assert np.array_equal(got["value_pages"], a.pages[1])


def test_append_over_a_capacity_table_of_many_entries(env):
    """More entries than a command takes whose workgroups all validate."""
    a = Append(env, 124, [30, 5], [4, 1], 8, 2)

    def table(x):
        x["page_indices"] = longer(env, a.indices, 5000, a.pool)
    a.check(a.run(flags=env[1].PLAN_PAGE_INDICES_CAPACITY, change=table))
