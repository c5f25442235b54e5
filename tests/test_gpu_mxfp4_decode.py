"""Paged decode over MXFP4 pages against attention in 64 bits over the values that the
pages hold.

Tolerances.  The codes become BF16 exactly, so errors come from the command's own
arithmetic.  A score is a sum of 128 exact products in FP32: it is off by at most
128 * 2^-24 of the sum of the products' magnitudes (times softmax scale and log2 e),
which moves LSE by as much and every weight by that fraction.  A weight keeps 16
bits (2^-15 after two truncations), and O is rounded once to BF16 (2^-8 of it).
v_exp_f32 and v_log_f32 are good to about 2^-22 of their results.
"""
import numpy as np
import pytest

import mxfp4_util as mx

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


@pytest.fixture(scope="module")
def env():
    import torch
    import loom_infer_hip as L
    return torch, L


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def dev_bf16(torch, values):
    return dev(torch, mx.bf16_bits(values).view(np.int16)).view(torch.bfloat16)


def host_bf16(torch, t):
    return mx.bf16_values(t.view(torch.int16).cpu().numpy().view(np.uint16))


class Case:
    """A cache, a table and queries; host copies in 64 bits and device operands."""

    def __init__(self, torch, seed, lens, hq, hkv, page=16, layout="NHD", spare=3):
        rng = np.random.default_rng(seed)
        self.torch, self.lens, self.hq, self.hkv = torch, lens, hq, hkv
        self.page, self.layout = page, layout
        self.pool, self.indptr, self.indices, self.last = mx.table(rng, lens, page, spare)
        self.k = mx.random_cache(rng, self.pool, page, hkv)
        self.v = mx.random_cache(rng, self.pool, page, hkv)
        self.q = mx.bf16_round(rng.standard_normal((len(lens), hq, mx.D)))

    def device(self, offset=0):
        t = self.torch

        def put(a):  # `offset` bytes past an aligned start
            b = t.empty(a.nbytes + 16, dtype=t.uint8, device="cuda")
            w = b[offset:offset + a.nbytes]
            w.copy_(dev(t, a).view(t.uint8).flatten())
            return w

        q = put(mx.bf16_bits(self.q)).view(t.bfloat16)
        kp, vp = (put(mx.in_layout(c[0], self.layout)) for c in (self.k, self.v))
        ks, vs = (put(c[1]) for c in (self.k, self.v))
        return [q, kp, vp, ks, vs, *(dev(t, a) for a in (self.indptr, self.indices, self.last))]

    def reference(self):
        o, l = [], []
        for r, n in enumerate(self.lens):
            k, v = (mx.rows_of(c, self.indptr, self.indices, r, n) for c in (self.k, self.v))
            a, b = mx.attend(self.q[r], k, v)
            o.append(a)
            l.append(b)
        return np.array(o), np.array(l)

    def bounds(self, ref_o, ref_l):
        """How far O and LSE may be off (see the module's text)."""
        score = vmax = 0.0
        for r, n in enumerate(self.lens):
            k, v = (mx.rows_of(c, self.indptr, self.indices, r, n) for c in (self.k, self.v))
            g = self.hq // self.hkv
            for h in range(self.hkv):
                heads = np.abs(self.q[r, h * g:(h + 1) * g])
                score = max(score, (np.abs(np.ascontiguousarray(k[:, h])) @ heads.T).max())
            vmax = max(vmax, np.abs(v).max())
        off = score * mx.D ** -0.5 * LOG2E * 128 * 2.0 ** -24 + 2.0 ** -20
        return (2.0 ** -8 * np.abs(ref_o) + vmax * (2 * off + 2.0 ** -15 + 2.0 ** -20),
                off + 2.0 ** -22 * np.abs(ref_l) + 2.0 ** -20)


def run(env, c, plan_opts=None, workspace=False, offset=0, operands=None, fill=float("nan")):
    torch, L = env
    spec = L.Bf16PagedBatchDecodeSpec(len(c.lens), c.pool, c.hq, c.hkv, kv_layout=c.layout,
                                      kv_dtype="mxfp4", kv_page_size=c.page)
    plan = L.DecodeProvider.load(0).plan_bf16_paged_batch(spec, **(plan_opts or {}))
    queue = L.CommandQueue(torch.cuda.current_stream(), 4)
    x = operands or c.device(offset)
    out = torch.full((spec.output_numel,), fill, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((spec.lse_numel,), fill, device="cuda")
    b = queue.bindings(11)
    h = [b.bind_read(t) for t in x] + [b.bind_read_write(t) for t in (out, lse)]
    ws = None
    if workspace:
        ws = b.bind_read_write(torch.full((plan.workspace_bytes,), 0xFF, dtype=torch.uint8,
                                          device="cuda")).write()
    scope = queue.begin(b)
    plan.enqueue_into(scope, L.Mxfp4PagedBatchDecodeArgs(*h[:8], h[8].write(), h[9].write(), ws))
    scope.finish().wait()
    shape = (len(c.lens), c.hq)
    return host_bf16(torch, out).reshape(*shape, mx.D), lse.cpu().numpy().reshape(shape), plan


def check(c, out, lse):
    ref_o, ref_l = c.reference()
    bo, bl = c.bounds(ref_o, ref_l)
    assert np.isfinite(out).all() and np.isfinite(lse).all()
    assert (np.abs(out - ref_o) <= bo).all(), (np.abs(out - ref_o) / bo).max()
    assert (np.abs(lse - ref_l) <= bl).all(), (np.abs(lse - ref_l) / bl).max()


SHAPES = [
    # lens, hq, hkv, page, layout
    ([1], 1, 1, 16, "NHD"),
    ([1, 2, 15, 16, 17], 8, 8, 16, "NHD"),
    ([33, 1, 64, 31], 16, 4, 16, "HND"),
    ([200], 32, 8, 32, "NHD"),
    ([63, 65, 1], 28, 4, 64, "HND"),
    ([127, 48, 129], 8, 1, 32, "HND"),
    ([5], 12, 4, 64, "NHD"),
    ([100, 7], 22, 2, 16, "NHD"),  # 11 heads per kv-head: two tiles, the second of 3
    ([700, 1, 333], 16, 2, 16, "NHD"),
]


@pytest.mark.parametrize("teams", [0, 1, 3, 64])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_decode_matches_64_bits(env, shape, teams):
    lens, hq, hkv, page, layout = SHAPES[shape]
    c = Case(env[0], 100 + shape, lens, hq, hkv, page, layout)
    out, lse, plan = run(env, c, {"teams": teams}, workspace=shape % 2 == 1)
    if teams:
        assert plan.algorithm == "balanced_split_kv"
    check(c, out, lse)


@pytest.mark.parametrize("seed", range(6))
def test_random_tables(env, seed):
    rng = np.random.default_rng(900 + seed)
    B = int(rng.integers(1, 9))
    hkv = int(rng.choice([1, 2, 3, 8]))
    hq = hkv * int(rng.choice([1, 2, 4, 7, 8, 16]))
    lens = [int(np.exp(rng.uniform(0, np.log(1500)))) for _ in range(B)]
    c = Case(env[0], seed, lens, hq, hkv, int(rng.choice([16, 32, 64])),
             ["NHD", "HND"][seed % 2])
    out, lse, _ = run(env, c)
    check(c, out, lse)


def test_more_requests_than_one_scan_block(env):
    """Batches past 256 and 512 requests take the table from memory."""
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(1, 40, 600)]
    c = Case(env[0], 6, lens, 4, 2)
    out, lse, _ = run(env, c)
    check(c, out, lse)


@pytest.mark.parametrize("teams", [0, 37, 2000])
@pytest.mark.parametrize("batch", [64, 65, 300, 600, 1300])
def test_many_requests(env, batch, teams):
    """Balanced commands keep the list of up to 64 requests in registers, of up to 512 in
    LDS, and of more in steps of 2, 4, ... requests; among them requests that no team
    starts with, and (invalid last-page lengths) some without blocks."""
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(1, 100, batch)]
    c = Case(env[0], 6, lens, 4, 2)
    out, lse, _ = run(env, c, {"teams": teams})
    check(c, out, lse)
    x = c.device()
    broken = sorted(set(int(r) for r in rng.integers(0, batch, 7)) | {0, batch - 1})
    x[7][env[0].tensor(broken, device="cuda")] = 0
    got, got_l, _ = run(env, c, {"teams": teams}, operands=x, fill=7.0)
    for r in range(batch):
        if r in broken:
            assert (got[r] == 7.0).all() and (got_l[r] == 7.0).all()
    whole = [r for r in range(batch) if r not in broken]
    ref_o, ref_l = c.reference()
    bo, bl = c.bounds(ref_o, ref_l)
    assert (np.abs(got - ref_o) <= bo)[whole].all() and (np.abs(got_l - ref_l) <= bl)[whole].all()


@pytest.mark.parametrize("shape", [
    # lens, hq, hkv, page, layout: the planner's three forms at their sizes
    ([5000], 8, 8, 16, "NHD"),                   # direct, split over many workgroups
    ([5200, 5100], 32, 32, 16, "NHD"),           # direct, two kv-heads per workgroup
    ([5200, 5100], 32, 32, 64, "HND"),           # direct, one
    ([300] * 40, 64, 32, 32, "NHD"),             # direct, two, not split
    ([17000, 16500], 64, 32, 64, "HND"),         # balanced
    ([33333], 32, 32, 32, "NHD"),                # balanced, one request in every team
])
def test_planned_forms(env, shape):
    lens, hq, hkv, page, layout = shape
    c = Case(env[0], 77, lens, hq, hkv, page, layout)
    out, lse, plan = run(env, c)
    rows = c.pool * page * hkv
    assert plan.algorithm == ("direct" if rows <= 1 << 20 else "balanced_split_kv")
    check(c, out, lse)


@pytest.mark.parametrize("teams", [0, 40])
@pytest.mark.parametrize("shape", [
    ([50, 3], 128, 1, 16, "NHD"),   # 16 tiles of 8 heads
    ([70, 33], 17, 17, 32, "NHD"),  # an odd number of kv-heads: one per wave
    ([41], 27, 3, 64, "HND"),       # 9 heads per kv-head: the second tile of one
    ([600, 90], 64, 64, 16, "NHD"),
])
def test_head_layouts(env, shape, teams):
    c = Case(env[0], 78, *shape)
    out, lse, _ = run(env, c, {"teams": teams})
    check(c, out, lse)


def test_the_largest_batch(env):
    """65536 requests of 1 to 40 tokens; one in 61 compared."""
    rng = np.random.default_rng(79)
    lens = [int(n) for n in rng.integers(1, 41, 65536)]
    c = Case(env[0], 80, lens, 1, 1)
    for opts in ({}, {"teams": 333}):
        out, lse, _ = run(env, c, opts)
        assert np.isfinite(out).all() and np.isfinite(lse).all()
        part = Case.__new__(Case)
        part.__dict__.update(c.__dict__)
        some = list(range(0, 65536, 61)) + [65535]
        part.lens, part.q = [lens[r] for r in some], c.q[some]
        pages = [c.indices[c.indptr[r]:c.indptr[r + 1]] for r in some]
        part.indptr = np.concatenate([[0], np.cumsum([len(p) for p in pages])]).astype(np.int32)
        part.indices = np.concatenate(pages)
        check(part, out[some], lse[some])


def test_two_queues_at_once(env):
    """Split commands of two queues on two streams, submitted without waiting."""
    torch, L = env
    cases = [Case(torch, 81, [1200, 900], 8, 2), Case(torch, 82, [2500], 32, 8, 32, "HND")]
    torch.cuda.synchronize()
    flight = []
    for c in cases:
        spec = L.Bf16PagedBatchDecodeSpec(len(c.lens), c.pool, c.hq, c.hkv, kv_layout=c.layout,
                                          kv_dtype="mxfp4", kv_page_size=c.page)
        plan = L.DecodeProvider.load(0).plan_bf16_paged_batch(spec)
        assert plan.workspace_bytes > 256
        queue = L.CommandQueue(torch.cuda.Stream(), 64)
        queue.reserve_workspace(plan.workspace_bytes)
        b = queue.bindings(10)
        out = torch.full((spec.output_numel,), float("nan"), dtype=torch.bfloat16, device="cuda")
        lse = torch.full((spec.lse_numel,), float("nan"), device="cuda")
        torch.cuda.synchronize()
        h = [b.bind_read(t) for t in c.device()] + [b.bind_read_write(t).write()
                                                    for t in (out, lse)]
        flight.append((c, plan, queue, queue.begin(b), L.Mxfp4PagedBatchDecodeArgs(*h), out, lse))
    torch.cuda.synchronize()
    for _ in range(50):
        for _, plan, _, scope, args, _, _ in flight:
            plan.enqueue_into(scope, args)
    for _, _, _, scope, _, _, _ in flight:
        scope.finish().wait()
    for c, _, _, _, _, out, lse in flight:
        shape = (len(c.lens), c.hq)
        check(c, host_bf16(torch, out).reshape(*shape, mx.D), lse.cpu().numpy().reshape(shape))


@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_pages_past_32_bit_offsets(env, layout):
    """Codes of 4.6 GB for K and for V, of which the last pages are in use."""
    torch, L = env
    c = Case(torch, 83, [100, 1], 16, 8, 64, layout)
    x = c.device()
    pool = 140000
    for i, width in ((1, 64), (2, 64), (3, 4), (4, 4)):
        size = 64 * 8 * width
        big = torch.empty(pool * size, dtype=torch.uint8, device="cuda")
        big[-c.pool * size:] = x[i]
        x[i] = big
    x[6] = x[6] + (pool - c.pool)
    far = Case.__new__(Case)
    far.__dict__.update(c.__dict__)
    far.pool = pool
    for teams in (0, 3):
        out, lse, _ = run(env, far, {"teams": teams, "max_total_pages": len(c.indices)},
                          operands=x)
        check(c, out, lse)


def test_results_repeat_bit_for_bit(env):
    c = Case(env[0], 7, [1000, 3, 517], 16, 4, 32, "HND")
    a, b = run(env, c), run(env, c, workspace=True)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("teams", [0, 5])
def test_four_byte_alignment(env, teams):
    c = Case(env[0], 8, [77, 16, 1], 8, 2)
    a, b = run(env, c, {"teams": teams}), run(env, c, {"teams": teams}, offset=4)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("teams", [0, 4])
def test_rows_behind_the_last_token_and_other_pages_are_not_read(env, teams):
    """NaN scales in every row that belongs to no token change nothing."""
    c = Case(env[0], 9, [21, 1, 64, 50], 8, 2, 32)
    want = run(env, c, {"teams": teams})
    used = np.zeros((c.pool, c.page), bool)
    for r, n in enumerate(c.lens):
        for t in range(n):
            used[c.indices[c.indptr[r] + t // c.page], t % c.page] = True
    for cache in (c.k, c.v):
        cache[0].swapaxes(1, 2)[~used] = 0x77
        cache[1].swapaxes(1, 2)[~used] = 255
    got = run(env, c, {"teams": teams})
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("teams", [0, 4])
def test_nan_blocks(env, teams):
    """A NaN block of V reaches its 32 dims of its request and kv-head, one of K
    the whole heads; nothing else."""
    c = Case(env[0], 10, [40, 90, 33], 8, 2)
    clean = run(env, c, {"teams": teams})
    page, row = c.indices[c.indptr[1] + 3], 5
    c.v[1][page, 1, row, 2] = 255
    out, lse, _ = run(env, c, {"teams": teams})
    hit = np.zeros(out.shape, bool)
    hit[1, 4:, 64:96] = True
    assert np.isnan(out[hit]).all()
    assert np.array_equal(out[~hit], clean[0][~hit]) and np.array_equal(lse, clean[1])
    c.k[1][page, 0, row, 0] = 255
    out, lse, _ = run(env, c, {"teams": teams})
    hit[1, :4] = True
    assert np.isnan(out[hit]).all() and np.array_equal(out[~hit], clean[0][~hit])
    assert np.isnan(lse[1, :4]).all()
    lse[1, :4] = clean[1][1, :4]
    assert np.array_equal(lse, clean[1])


def test_smallest_and_largest_scales(env):
    c = Case(env[0], 11, [50, 3], 8, 2)
    rng = np.random.default_rng(12)
    c.k[1][:] = rng.choice([0, 1, 60, 125, 127], c.k[1].shape)
    c.v[1][:] = rng.choice([100, 127, 140], c.v[1].shape)
    out, lse, _ = run(env, c)
    check(c, out, lse)
    c.v[1][:] = 252  # values up to 6 * 2^125
    c.v[0][:] &= 0x33  # no value above 1.5, so that no sum passes FP32
    out, _, _ = run(env, c)
    ref, _ = c.reference()
    assert (np.abs(out - ref) <= 2.0 ** -7 * np.abs(ref).max()).all()


@pytest.mark.parametrize("teams", [0, 4])
def test_invalid_page_index_keeps_the_requests_sentinels(env, teams):
    torch, _ = env
    c = Case(env[0], 13, [40, 90, 33], 8, 2)
    want = run(env, c, {"teams": teams})
    for wrong in (c.pool, -1, 2 ** 31 - 1):
        x = c.device()
        x[6][int(c.indptr[1]) + 2] = wrong
        out, lse, _ = run(env, c, {"teams": teams}, operands=x, fill=7.0)
        assert (out[1] == 7.0).all() and (lse[1] == 7.0).all()
        for r in (0, 2):
            assert np.array_equal(out[r], want[0][r]) and np.array_equal(lse[r], want[1][r])


@pytest.mark.parametrize("teams", [0, 4])
def test_invalid_tables_write_nothing(env, teams):
    c = Case(env[0], 14, [40, 90], 8, 2)
    for at, value in ((0, 1), (2, 10 ** 6)):
        x = c.device()
        x[5][at] = value
        out, lse, _ = run(env, c, {"teams": teams}, operands=x, fill=7.0)
        assert (out == 7.0).all() and (lse == 7.0).all()
    x = c.device()
    x[7][0] = c.page + 1
    out, lse, _ = run(env, c, {"teams": teams}, operands=x, fill=7.0)
    assert (out[0] == 7.0).all() and np.isfinite(out[1]).all() and (out[1] != 7.0).any()


SPLIT = [
    # lens, hq, hkv, page, layout: plans that split every request over 4 to 64 workgroups
    ([900], 32, 8, 16, "NHD"),
    ([1500, 1, 1000], 28, 4, 32, "HND"),
    ([40000], 4, 1, 64, "NHD"),
    ([70000], 22, 2, 64, "HND"),
    ([11000], 32, 32, 16, "NHD"),  # two kv-heads per workgroup
]


@pytest.mark.parametrize("shape", range(len(SPLIT)))
def test_split_requests_on_one_queue(env, shape):
    """Commands one after another on one queue, whose arrival words each leaves zero: a
    valid one, one with an invalid page index in one split, one of another plan, and the
    first again, in one scope and in a graph that is replayed."""
    torch, L = env
    c = Case(torch, 90 + shape, *SPLIT[shape])
    other = Case(torch, 95, [1000, 950], 8, 2)
    bad = c.device()
    bad[6][len(c.indices) // 3] = c.pool
    commands = [(c, c.device()), (c, bad), (other, other.device()), (c, c.device())]
    plans = {}
    for case in (c, other):
        spec = L.Bf16PagedBatchDecodeSpec(len(case.lens), case.pool, case.hq, case.hkv,
                                          kv_layout=case.layout, kv_dtype="mxfp4",
                                          kv_page_size=case.page)
        plans[case] = L.DecodeProvider.load(0).plan_bf16_paged_batch(spec)
        assert plans[case].algorithm == "direct" and plans[case].workspace_bytes > 256
    outs = [(torch.empty(case.q.size, dtype=torch.bfloat16, device="cuda"),
             torch.empty(case.q.size // mx.D, device="cuda")) for case, _ in commands]

    def enqueue(b, scope, handles):
        for (case, _), h in zip(commands, handles):
            plans[case].enqueue_into(scope, L.Mxfp4PagedBatchDecodeArgs(
                *h[:8], h[8].write(), h[9].write()))

    def bind(b):
        return [[b.bind_read(t) for t in x] + [b.bind_read_write(t) for t in o]
                for (_, x), o in zip(commands, outs)]

    def fill():
        for o in outs:
            for t in o:
                t.fill_(7.0)
        torch.cuda.synchronize()

    def verify(want=[]):
        got = []
        for (case, x), (o, l) in zip(commands, outs):
            shape = (len(case.lens), case.hq)
            o, l = host_bf16(torch, o).reshape(*shape, mx.D), l.cpu().numpy().reshape(shape)
            if x is bad:
                assert (o[0] == 7.0).all() and (l[0] == 7.0).all()
            elif not want:
                check(case, o, l)
            got.append((o, l))
        want[:] = want or got
        assert all(np.array_equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))

    queue = L.CommandQueue(torch.cuda.current_stream(), 8)
    b = queue.bindings(48)
    h = bind(b)
    fill()
    scope = queue.begin(b)
    enqueue(b, scope, h)
    scope.finish().wait()
    verify()
    gq = L.GraphQueue(0, 8)
    gq.reserve_workspace(max(p.workspace_bytes for p in plans.values()))
    b = gq.bindings(48)
    h = bind(b)
    fill()
    graph = gq.capture(b, lambda s: enqueue(b, s, h)).instantiate()
    for _ in range(3):
        graph.launch().wait()
        verify()
        fill()


def test_split_command_in_a_callers_capture(env):
    """Captured by the caller into a graph of its own, whose replays the queue does not
    order, a split command counts its workgroups in its workspace, which may hold
    anything; the queue's own commands go on between the replays."""
    torch, L = env
    c = Case(torch, 96, [900, 1300], 8, 2)
    x = c.device()
    spec = L.Bf16PagedBatchDecodeSpec(2, c.pool, 8, 2, kv_dtype="mxfp4")
    plan = L.DecodeProvider.load(0).plan_bf16_paged_batch(spec)
    assert plan.algorithm == "direct" and plan.workspace_bytes > 256
    stream = torch.cuda.Stream()
    outs = [(torch.empty(c.q.size, dtype=torch.bfloat16, device="cuda"),
             torch.empty(c.q.size // mx.D, device="cuda")) for _ in range(2)]
    works = [torch.full((plan.workspace_bytes,), 0xFF, dtype=torch.uint8, device="cuda")
             for _ in range(2)]
    queues = [L.CommandQueue(stream, 4) for _ in range(2)]
    torch.cuda.synchronize()

    def bind(i):
        b = queues[i].bindings(11)
        h = [b.bind_read(t) for t in x] + [b.bind_read_write(t).write()
                                           for t in (*outs[i], works[i])]
        return b, L.Mxfp4PagedBatchDecodeArgs(*h)
    b, args = bind(0)
    scope = queues[0].begin(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        plan.enqueue_into(scope, args)
    scope.finish().wait()
    for _ in range(3):
        for t in (*outs[0], *outs[1]):
            t.fill_(float("nan"))
        works[0].random_(0, 256)
        torch.cuda.synchronize()
        graph.replay()
        b, args = bind(1)
        scope = queues[1].begin(b)
        plan.enqueue_into(scope, args)
        scope.finish().wait()
        torch.cuda.synchronize()
        for o, l in outs:
            check(c, host_bf16(torch, o).reshape(2, 8, mx.D), l.cpu().numpy().reshape(2, 8))


def test_capacity_table_in_a_graph(env):
    """One captured command over a capacity table, replayed as the table grows, with
    eager work between the replays."""
    torch, L = env
    c = Case(env[0], 15, [70, 35, 128], 8, 2, spare=8)
    need = int(c.indptr[-1])
    x = c.device()
    cap = torch.zeros(need + 8, dtype=torch.int32, device="cuda")
    cap[:need] = x[6]
    x[6] = cap
    spec = L.Bf16PagedBatchDecodeSpec(3, c.pool, 8, 2, kv_dtype="mxfp4")
    plan = L.DecodeProvider.load(0).plan_bf16_paged_batch(spec, teams=16, indices_capacity=True)
    gq = L.GraphQueue(0, 2)
    gq.reserve_workspace(plan.workspace_bytes)
    out = torch.zeros(spec.output_numel, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(spec.lse_numel, device="cuda")
    b = gq.bindings(10)
    h = [b.bind_read(t) for t in x]
    o, l = b.bind_read_write(out), b.bind_read_write(lse)
    torch.cuda.synchronize()
    graph = gq.capture(b, lambda s: plan.enqueue_into(
        s, L.Mxfp4PagedBatchDecodeArgs(*h, o.write(), l.write()))).instantiate()
    spare = [p for p in range(c.pool) if p not in set(c.indices.tolist())]
    for step in range(4):
        graph.launch().wait()
        check(c, host_bf16(torch, out).reshape(3, 8, mx.D), lse.cpu().numpy().reshape(3, 8))
        out.zero_()
        # request 2 gets one more page of 9 rows
        c.lens[2] += 9 if c.lens[2] % 16 == 0 else 16
        if len(c.indices) < -(-c.lens[2] // 16) + int(c.indptr[2]):
            c.indices = np.append(c.indices, np.int32(spare.pop()))
            c.indptr[3] += 1
        c.last[2] = c.lens[2] - (c.indptr[3] - c.indptr[2] - 1) * 16
        cap[:len(c.indices)] = dev(torch, c.indices)
        x[5].copy_(dev(torch, c.indptr))
        x[7].copy_(dev(torch, c.last))
        torch.cuda.synchronize()
