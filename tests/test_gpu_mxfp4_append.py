"""The normed append (norms of the query and key heads, rotation, paged write) and the
read back of MXFP4 pages, against 64 bits.

Tolerances.  Codes and scales of MXFP4 rows have to be equal: keys are computed in 64
bits and rounded once.  Q and BF16 keys are computed in FP32 and rounded once: half a
BF16 step (2^-8 of the value) plus FP32's own error, some roundings of 2^-24 of the
row's largest term (the norm's sum of 128 squares: 8 in a lane, 4 additions across
lanes, a root, a quotient, two products, the rotation's two; 24 in all).  An FP8 key may
be a step off where FP32 moves it over a border: values differ by at most one E4M3
step (2^-3 of the value, 2^-9 of the scale near zero) there.
"""
import numpy as np
import pytest

import mxfp4_util as mx
from test_gpu_mxfp4_decode import Case, check as check_decode, dev, dev_bf16, host_bf16

pytestmark = pytest.mark.gpu
THETA, EPS = 1e6, 1e-6


@pytest.fixture(scope="module")
def env():
    import torch
    import loom_infer_hip as L
    return torch, L


class Append:
    """Explicit tokens (or one per request) over a random table."""

    def __init__(self, env, seed, lens, rows, hq, hkv, page=16, layout="NHD", dtype="mxfp4",
                 norm=True, explicit=True):
        self.torch, self.L = env
        rng = np.random.default_rng(seed)
        self.lens, self.hq, self.hkv, self.page, self.layout = lens, hq, hkv, page, layout
        self.dtype, self.norm, self.explicit = dtype, norm, explicit
        self.pool, self.indptr, self.indices, self.last = mx.table(rng, lens, page)
        req = np.repeat(np.arange(len(lens)), rows)
        pos = np.concatenate([np.arange(n - k, n) for n, k in zip(lens, rows)])
        order = rng.permutation(len(req)) if explicit else np.arange(len(req))
        self.req, self.pos = req[order].astype(np.int32), pos[order].astype(np.int32)
        T = self.T = len(req)
        self.q = mx.bf16_round(rng.standard_normal((T, hq, mx.D)) * 3)
        self.k = mx.bf16_round(rng.standard_normal((T, hkv, mx.D))
                               * np.exp(rng.standard_normal((hkv, mx.D))))
        self.v = mx.bf16_round(rng.standard_normal((T, hkv, mx.D)))
        self.qw, self.kw = (mx.bf16_round(1 + 0.3 * rng.standard_normal(mx.D)) for _ in range(2))
        n = self.pool * page * hkv
        if dtype == "mxfp4":
            self.pages = [rng.integers(0, 256, n * 64, dtype=np.uint8) for _ in range(2)]
            self.scales = [rng.integers(0, 255, n * 4, dtype=np.uint8) for _ in range(2)]
        elif dtype == "bf16":
            self.pages = [rng.integers(0, 1 << 15, n * mx.D, dtype=np.uint16) for _ in range(2)]
        else:
            self.pages = [rng.integers(0, 120, n * mx.D, dtype=np.uint8) for _ in range(2)]
        self.kv_scales = np.array([0.031, 0.017], np.float32)

    def spec(self, **kw):
        return self.L.NormRopePagedKvAppendSpec(
            self.T, len(self.lens), self.pool, self.hq, self.hkv, kv_layout=self.layout,
            kv_dtype=self.dtype, kv_page_size=self.page, rope_theta=THETA,
            norm_eps=EPS if self.norm else None, explicit_tokens=self.explicit, **kw)

    def operands(self):
        t = self.torch
        x = {"query": dev_bf16(t, self.q), "key": dev_bf16(t, self.k), "value": dev_bf16(t, self.v),
             "page_indptr": dev(t, self.indptr), "page_indices": dev(t, self.indices),
             "last_page_len": dev(t, self.last)}
        if self.explicit:
            x |= {"batch_indices": dev(t, self.req), "positions": dev(t, self.pos)}
        if self.norm:
            x |= {"query_norm": dev_bf16(t, self.qw), "key_norm": dev_bf16(t, self.kw)}
        if self.dtype == "fp8_e4m3":
            x["kv_scales"] = dev(t, self.kv_scales)
        y = {"query_output": t.full((self.T * self.hq * mx.D,), 7.0, dtype=t.bfloat16, device="cuda")}
        for name, p in zip(("key_pages", "value_pages"), self.pages):
            y[name] = dev(t, p.view(np.int16)).view(t.bfloat16) if self.dtype == "bf16" else dev(t, p)
        if self.dtype == "mxfp4":
            for name, p in zip(("key_scales", "value_scales"), self.scales):
                y[name] = dev(t, p)
        return x, y

    def run(self, flags=0, workspace=False, change=None, odd_output=False):
        t = self.torch
        plan = self.L.RopeProvider.load(0).plan_norm_paged_append(self.spec(), flags=flags)
        queue = self.L.CommandQueue(t.cuda.current_stream(), 4)
        x, y = self.operands()
        if change:
            change(x)
        if odd_output:  # the rotated queries one element past an aligned start
            y["query_output"] = t.full((y["query_output"].numel() + 1,), 7.0, dtype=t.bfloat16,
                                       device="cuda")[1:]
        if workspace:
            y["workspace"] = t.zeros(plan.workspace_bytes, dtype=t.uint8, device="cuda")
        b = queue.bindings(20)
        h = {k: b.bind_read(v) for k, v in x.items()}
        h |= {k: b.bind_read_write(v).write() for k, v in y.items()}
        scope = queue.begin(b)
        plan.enqueue_into(scope, self.L.NormRopePagedKvAppendArgs(**h))
        scope.finish().wait()
        return {k: (v.view(t.int16).cpu().numpy().view(np.uint16) if v.dtype == t.bfloat16
                    else v.cpu().numpy()) for k, v in y.items()}

    def slot(self, t):
        p = int(self.pos[t])
        return int(self.indices[self.indptr[self.req[t]] + p // self.page]), p % self.page

    def place(self, pages, width, rows):
        """`rows` [T, hkv, width] scattered over a copy of `pages` (codes or values)."""
        shape = ((self.pool, self.page, self.hkv, width) if self.layout == "NHD"
                 else (self.pool, self.hkv, self.page, width))
        a = pages.copy().reshape(shape)
        for t in range(self.T):
            p, o = self.slot(t)
            if self.layout == "NHD":
                a[p, o] = rows[t]
            else:
                a[p, :, o] = rows[t]
        return a.reshape(-1)

    def place_scales(self, scales, rows):
        a = scales.copy().reshape(self.pool, self.hkv, self.page, 4)
        for t in range(self.T):
            p, o = self.slot(t)
            a[p, :, o] = rows[t]
        return a.reshape(-1)

    def exact(self):
        w = (self.qw, self.kw) if self.norm else (None, None)
        return (mx.norm_rotate(self.q, w[0], self.pos, EPS, THETA),
                mx.norm_rotate(self.k, w[1], self.pos, EPS, THETA))

    def bound32(self, x, w, ref):
        """Half a BF16 step and FP32's error (see the module's text)."""
        if self.norm:
            x = np.abs(x) / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * np.abs(w)
        pair = np.abs(x) + np.abs(np.roll(x, 64, -1))
        return 2.0 ** -8 * np.abs(ref) + 24 * 2.0 ** -24 * pair + 1e-40

    def check(self, got):
        q, k = self.exact()
        qo = mx.bf16_values(got["query_output"]).reshape(q.shape)
        assert (np.abs(qo - q) <= self.bound32(self.q, self.qw, q)).all()
        if self.dtype == "mxfp4":
            for rows, pages, scales, name in ((k, self.pages[0], self.scales[0], "key"),
                                              (self.v, self.pages[1], self.scales[1], "value")):
                c, s = mx.quantise(rows)
                assert np.array_equal(got[name + "_scales"], self.place_scales(scales, s))
                assert np.array_equal(got[name + "_pages"], self.place(pages, 64, c))
        elif self.dtype == "bf16":
            assert np.array_equal(got["value_pages"],
                                  self.place(self.pages[1], mx.D, mx.bf16_bits(self.v)))
            # slots without a token keep their bits, whatever they are
            new = self.place(np.zeros(len(self.pages[0]), bool), mx.D, np.ones(k.shape, bool))
            assert np.array_equal(got["key_pages"][~new], self.pages[0][~new])
            want = self.place(np.zeros(len(new)), mx.D, k)[new]
            tol = self.place(np.zeros(len(new)), mx.D, self.bound32(self.k, self.kw, k))[new]
            assert (np.abs(mx.bf16_values(got["key_pages"][new]) - want) <= tol).all()
        else:
            e4m3 = self.torch.arange(256, dtype=self.torch.uint8).view(
                self.torch.float8_e4m3fn).double().numpy()
            for rows, old, s, name in ((k, self.pages[0], self.kv_scales[0], "key_pages"),
                                       (self.v, self.pages[1], self.kv_scales[1], "value_pages")):
                u = np.clip(rows / np.float64(s), -448, 448)
                want = self.place(e4m3[old], mx.D, u)
                # half a step, and a whole one where FP32 moves a key over a border
                step = np.where(np.abs(u) < 2.0 ** -6, 2.0 ** -9, np.abs(u) * 2.0 ** -3)
                tol = self.place(np.zeros(len(want)), mx.D, step * 0.51)
                assert (np.abs(e4m3[got[name]] - want) <= tol).all()


SHAPES = [
    # lens, rows, hq, hkv, page, layout
    ([1], [1], 1, 1, 16, "NHD"),
    ([5, 40, 17], [5, 3, 1], 8, 2, 16, "NHD"),
    ([16, 33, 64], [16, 20, 9], 28, 4, 32, "HND"),
    ([130, 90], [100, 90], 16, 4, 64, "HND"),
    ([200, 7, 65], [70, 7, 64], 64, 8, 16, "NHD"),
]


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype", ["mxfp4", "bf16", "fp8_e4m3"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_append_matches_64_bits(env, shape, dtype, norm):
    lens, rows, hq, hkv, page, layout = SHAPES[shape]
    a = Append(env, 40 + shape, lens, rows, hq, hkv, page, layout, dtype, norm)
    a.check(a.run(workspace=shape % 2 == 0))


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype", ["mxfp4", "bf16", "fp8_e4m3"])
@pytest.mark.parametrize("heads", [(1, 1), (6, 3), (28, 4), (40, 10)])
def test_commands_of_many_tokens(env, heads, dtype, norm):
    """A token per wave: heads that do not fill a wave's 4 rows, a last workgroup that is
    not full, the one-launch and the two-launch form alike."""
    rows = [700, 1, 699, 33]
    a = Append(env, 60, [711, 5, 699, 90], rows, *heads, dtype=dtype, norm=norm)
    got = a.run()
    a.check(got)
    if heads == (6, 3):
        two = a.run(flags=env[1].PLAN_APPEND_TWO_LAUNCH)
        assert all(np.array_equal(got[k], two[k]) for k in got)


@pytest.mark.parametrize("rows", [3, 90, 1300])
def test_rows_on_two_byte_boundaries(env, rows):
    """The append's operands need no alignment beyond their elements'."""
    torch = env[0]
    a = Append(env, 65, [rows + 9], [rows], 6, 3)
    plain = a.run()

    def shift(x):
        for n in ("query", "key", "value", "query_norm", "key_norm"):
            b = torch.empty(x[n].numel() + 9, dtype=torch.bfloat16, device="cuda")
            b[1:1 + x[n].numel()] = x[n].flatten()
            x[n] = b[1:1 + x[n].numel()]
    a.check(plain)
    got = a.run(change=shift, odd_output=True)
    assert all(np.array_equal(got[k], plain[k]) for k in got)


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
def test_many_tokens_of_many_requests(env, dtype):
    rng = np.random.default_rng(61)
    lens = [int(n) for n in rng.integers(1, 40, 1501)]
    a = Append(env, 62, lens, [1] * 1501, 4, 1, dtype=dtype, explicit=False)
    a.check(a.run())


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
def test_many_tokens_with_one_slot_twice_write_nothing(env, dtype):
    a = Append(env, 63, [800, 700], [800, 700], 4, 2, 32, dtype=dtype)

    def twice(x):
        x["positions"][1499] = x["positions"][802]
    for change in (twice, lambda x: x["positions"].__setitem__(3, 800)):
        got = a.run(change=change)
        assert (mx.bf16_values(got["query_output"]) == 7.0).all()
        assert np.array_equal(got["key_pages"], a.pages[0])
        assert np.array_equal(got["value_pages"], a.pages[1])


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
@pytest.mark.parametrize("batch", [1, 6, 100])
def test_one_token_per_request(env, batch, dtype):
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in rng.integers(1, 90, batch)]
    a = Append(env, 3, lens, [1] * batch, 16, 2, 16, "NHD", dtype, explicit=False)
    a.check(a.run())


def test_two_launch_form(env):
    a = Append(env, 4, [100, 50], [80, 50], 8, 2)
    one, two = a.run(), a.run(flags=env[1].PLAN_APPEND_TWO_LAUNCH)
    a.check(two)
    assert all(np.array_equal(one[k], two[k]) for k in one)


def test_far_positions(env):
    """Positions near 2^20 keep their phase (the angle is a 64-bit product)."""
    n = (1 << 20) + 11
    a = Append(env, 5, [n], [12], 4, 1, 64, "HND")
    a.check(a.run())


@pytest.mark.parametrize("norm", [True, False])
def test_ties_and_special_rows(env, norm):
    """At position 0 without norms keys reach the quantiser as they are: ties go to the
    even code, blocks of zeros, subnormals and the largest values get the clamped
    scales, and a block with a NaN or an infinity becomes NaN alone."""
    a = Append(env, 6, [1] * 8, [1] * 8, 2, 2, norm=norm)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.5, 4, 0, -0.25, -5, -2.5, -0.0])
    for row in (a.k, a.v):
        row[0] = np.tile(ties, 8)
        row[1] = 0.0
        row[2] = -0.0
        row[3, :, ::3] = 2.0 ** -130
        row[3, :, 1::3] = 2.0 ** -126
        row[3, :, 2::3] = -(2.0 ** -127)
        if not norm:
            row[4, :, :64] = float(2 ** 128 - 2 ** 120)
        row[5, 0, 40] = np.nan
        row[6, 1, 100] = -np.inf
        row[7] *= 2.0 ** np.arange(-64, 64)
    if norm:  # a NaN or an infinity reaches its whole head through the sum
        a.k[5:7] = a.v[4]
    with np.errstate(invalid="ignore", over="ignore"):
        a.check(a.run())


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
@pytest.mark.parametrize("rows", [3, 90])
def test_invalid_metadata_writes_nothing(env, rows, dtype):
    def wrong(name, at, value):
        def change(x):
            x[name][at] = value
        return change

    a = Append(env, 7, [95, 120], [rows, rows], 8, 2, dtype=dtype)
    for change in (wrong("page_indices", 2, a.pool), wrong("page_indices", 0, -1),
                   wrong("page_indptr", 0, 1), wrong("last_page_len", 1, 17),
                   wrong("positions", 1, 10 ** 6), wrong("positions", 0, -1),
                   wrong("batch_indices", 0, 2)):
        got = a.run(change=change)
        assert (mx.bf16_values(got["query_output"]) == 7.0).all()
        assert np.array_equal(got["key_pages"], a.pages[0])
        assert np.array_equal(got["value_pages"], a.pages[1])
        if dtype == "mxfp4":
            assert np.array_equal(got["key_scales"], a.scales[0])
            assert np.array_equal(got["value_scales"], a.scales[1])

    def twice(x):  # two tokens with one slot
        x["positions"][1] = x["positions"][0]
        x["batch_indices"][1] = x["batch_indices"][0]
    got = a.run(change=twice)
    assert np.array_equal(got["key_pages"], a.pages[0])


# ---- read back ----------------------------------------------------------------------
def read(env, c, starts, counts, nnz=None, indptr=None, change=None, give_start=True):
    torch, L = env
    kv = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32) if indptr is None else indptr
    nnz = int(kv[-1]) if nnz is None else nnz
    spec = L.PagedKvReadSpec(len(c.lens), nnz, c.pool, c.hkv, kv_layout=c.layout, kv_page_size=c.page)
    plan = L.PrefillProvider.load(0).plan_paged_kv_read(spec)
    x = c.device()[1:]
    if change:
        change(x)
    k, v = (torch.full((spec.output_numel,), 7.0, dtype=torch.bfloat16, device="cuda")
            for _ in range(2))
    queue = L.CommandQueue(torch.cuda.current_stream(), 2)
    b = queue.bindings(11)
    h = [b.bind_read(t) for t in x] + [b.bind_read(dev(torch, kv))]
    o = [b.bind_read_write(t).write() for t in (k, v)]
    s = b.bind_read(dev(torch, np.asarray(starts, np.int32))) if give_start else None
    scope = queue.begin(b)
    plan.enqueue_into(scope, L.PagedKvReadArgs(*h, *o, kv_start=s))
    scope.finish().wait()
    return [t.view(torch.int16).cpu().numpy().view(np.uint16).reshape(nnz, c.hkv, mx.D)
            for t in (k, v)]


def same_bits(got, want):
    """Equal BF16 values, NaN for NaN."""
    got = mx.bf16_values(got)
    return np.array_equal(got, want, equal_nan=True)


def rows_wanted(c, starts, counts, nnz):
    out = []
    for cache in (c.k, c.v):
        rows = [mx.rows_of(cache, c.indptr, c.indices, r, n)[s:s + k]
                for r, (n, s, k) in enumerate(zip(c.lens, starts, counts))]
        rows = np.concatenate(rows)
        out.append(np.concatenate([mx.bf16_round(rows),
                                   np.full((nnz - len(rows), *rows.shape[1:]), 7.0)]))
    return out


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("hkv", [1, 3, 8])
def test_read_back_is_exact(env, hkv, page, layout):
    c = Case(env[0], hkv + page, [1, 100, 33, 17, 64], hkv, hkv, page, layout)
    rng = np.random.default_rng(1)
    for cache in (c.k, c.v):  # every scale: 0 (2^-127) to 252, NaN; 253 and 254 may pass BF16
        cache[1][:] = rng.integers(0, 256, cache[1].shape)
    starts, counts = [0, 3, 33, 5, 1], [1, 97, 0, 7, 63]
    nnz = sum(counts) + 5  # rows behind the last request stay as they were
    for got, want in zip(read(env, c, starts, counts, nnz), rows_wanted(c, starts, counts, nnz)):
        assert same_bits(got, want)


def test_read_back_of_many_requests(env):
    rng = np.random.default_rng(2)
    lens = [int(n) for n in rng.integers(1, 20, 5000)]
    c = Case(env[0], 3, lens, 1, 1)
    counts = [int(rng.integers(0, n + 1)) * int(rng.random() < 0.3) for n in lens]
    counts[100:400] = [0] * 300  # more empty requests than one round of the search holds
    starts = [n - k for n, k in zip(lens, counts)]
    nnz = sum(counts)
    for got, want in zip(read(env, c, starts, counts), rows_wanted(c, starts, counts, nnz)):
        assert same_bits(got, want)


@pytest.mark.parametrize("hkv", [1, 5, 70])
@pytest.mark.parametrize("batch", [1, 62, 63, 64, 65, 127, 200])
def test_read_back_over_batches(env, batch, hkv):
    """Around the 64 requests whose table words one wave holds, with empty ones between;
    1 to 64 output rows per workgroup."""
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in rng.integers(1, 24, batch)]
    c = Case(env[0], batch, lens, hkv, hkv, 16, "HND")
    counts = [int(rng.integers(0, n + 1)) * int(rng.random() < 0.6) for n in lens]
    counts[-1] = 1
    starts = [int(rng.integers(0, n - k + 1)) for n, k in zip(lens, counts)]
    nnz = sum(counts)
    for got, want in zip(read(env, c, starts, counts), rows_wanted(c, starts, counts, nnz)):
        assert same_bits(got, want)


def test_read_back_from_the_first_token_without_starts(env):
    c = Case(env[0], 4, [40, 20], 2, 2)
    for got, want in zip(read(env, c, [], [9, 20], give_start=False),
                         rows_wanted(c, [0, 0], [9, 20], 29)):
        assert same_bits(got, want)


def test_read_back_guards(env):
    c = Case(env[0], 5, [40, 20, 30], 2, 2)
    starts, counts = [0, 0, 0], [40, 20, 30]
    good = rows_wanted(c, starts, counts, 90)

    def untouched(rows, **kw):
        for got, want in zip(read(env, c, kw.pop("starts", starts), counts, **kw), good):
            want = want.copy()
            want[rows] = 7.0
            assert same_bits(got, want)

    everything = slice(0, 90)
    untouched(slice(40, 60), starts=[0, 1, 0])  # one row past the request's tokens
    untouched(slice(40, 60), starts=[0, -1, 0])
    untouched(slice(0, 40), starts=[2 ** 31 - 1, 0, 0])
    untouched(everything, indptr=np.array([1, 40, 60, 90], np.int32))
    untouched(everything, indptr=np.array([0, 40, 60, 91], np.int32), nnz=90)

    def put(i, at, value):
        def change(x):
            x[i][at] = value
        return change
    untouched(slice(16, 32), change=put(5, 1, c.pool))  # one page of request 0
    untouched(slice(16, 32), change=put(5, 1, -5))
    untouched(slice(40, 60), change=put(6, 1, 0))
    untouched(slice(40, 60), change=put(6, 1, 17))
    untouched(everything, change=put(4, 0, 1))
    untouched(everything, change=put(4, 3, 10 ** 6))


@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_pages_past_32_bit_offsets(env, layout):
    """Codes of 4.6 GB for K and for V: tokens appended to the last page and read back."""
    torch, L = env
    pool, page, hkv, lens = 140000, 64, 8, [70, 3]
    codes = [torch.full((pool * page * hkv * 64,), 0x55, dtype=torch.uint8, device="cuda")
             for _ in range(2)]
    scales = [torch.full((pool * page * hkv * 4,), 99, dtype=torch.uint8, device="cuda")
              for _ in range(2)]
    rng = np.random.default_rng(64)
    k, v = (mx.bf16_round(rng.standard_normal((73, hkv, mx.D))) for _ in range(2))
    q = torch.zeros(73 * hkv * mx.D, dtype=torch.bfloat16, device="cuda")
    table = [dev(torch, np.array(t, np.int32)) for t in
             ([0, 2, 3], [pool - 2, pool - 3, pool - 1], [6, 3])]
    form = dict(kv_layout=layout, kv_page_size=page, kv_dtype="mxfp4")
    aplan = L.RopeProvider.load(0).plan_norm_paged_append(L.NormRopePagedKvAppendSpec(
        73, 2, pool, hkv, hkv, rope_theta=THETA, **form))
    rplan = L.PrefillProvider.load(0).plan_paged_kv_read(L.PagedKvReadSpec(2, 73, pool, hkv, **form))
    queue = L.CommandQueue(torch.cuda.current_stream(), 4)
    b = queue.bindings(24)
    req, pos = np.repeat([0, 1], lens), np.concatenate([np.arange(n) for n in lens])
    r = b.bind_read
    hq, hk, hv, hr, hp, *ht, hkv_ = (r(t) for t in (
        q, dev_bf16(torch, k).flatten(), dev_bf16(torch, v).flatten(),
        dev(torch, req.astype(np.int32)), dev(torch, pos.astype(np.int32)), *table,
        dev(torch, np.array([0, 70, 73], np.int32))))
    pages = [b.bind_read_write(t) for t in (*codes, *scales)]
    qo, ko, vo = (torch.zeros_like(q) for _ in range(3))
    hqo, hko, hvo = (b.bind_read_write(t).write() for t in (qo, ko, vo))
    scope = queue.begin(b)
    aplan.enqueue_into(scope, L.NormRopePagedKvAppendArgs(
        hq, hk, hv, *ht, hqo, pages[0].write(), pages[1].write(), hr, hp,
        key_scales=pages[2].write(), value_scales=pages[3].write()))
    rplan.enqueue_into(scope, L.PagedKvReadArgs(*(p.read() for p in pages), *ht, hkv_, hko, hvo))
    scope.finish().wait()
    for got, rows in ((ko, mx.norm_rotate(k, None, pos, EPS, THETA)), (vo, v)):
        assert np.array_equal(host_bf16(torch, got).reshape(73, hkv, mx.D),
                              mx.values(*mx.quantise(rows)))
    for t in (*codes, *scales):  # nothing before those pages
        assert (t[:1 << 20] == t[0]).all() and t[0] in (0x55, 99)


# ---- together -------------------------------------------------------------------------
def test_append_decode_and_read_back_in_one_graph(env):
    """A decode step over an MXFP4 cache as a captured graph (normed append, decode), its
    cache read back in the same graph, replayed with new inputs and eager work between."""
    torch, L = env
    lens, hq, hkv, page = [33, 70, 1, 129], 16, 4, 32
    c = Case(torch, 20, lens, hq, hkv, page, "HND")
    x = c.device()
    q, kp, vp, ks, vs, ip, ix, ln = x
    B = len(lens)
    nk, nv = (torch.zeros(B * hkv * mx.D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rng = np.random.default_rng(21)
    qw, kw = (mx.bf16_round(1 + 0.3 * rng.standard_normal(mx.D)) for _ in range(2))
    form = dict(kv_layout="HND", kv_dtype="mxfp4", kv_page_size=page)
    aplan = L.RopeProvider.load(0).plan_norm_paged_append(L.NormRopePagedKvAppendSpec(
        B, B, c.pool, hq, hkv, rope_theta=THETA, norm_eps=EPS, explicit_tokens=False, **form))
    dplan = L.DecodeProvider.load(0).plan_bf16_paged_batch(
        L.Bf16PagedBatchDecodeSpec(B, c.pool, hq, hkv, **form))
    n = sum(lens)
    rplan = L.PrefillProvider.load(0).plan_paged_kv_read(L.PagedKvReadSpec(B, n, c.pool, hkv, **form))
    bf = dict(dtype=torch.bfloat16, device="cuda")
    qr, o, lse = torch.zeros(B * hq * mx.D, **bf), torch.zeros(B * hq * mx.D, **bf), \
        torch.zeros(B * hq, device="cuda")
    rk, rv = torch.zeros(n * hkv * mx.D, **bf), torch.zeros(n * hkv * mx.D, **bf)
    gq = L.GraphQueue(0, 3)
    gq.reserve_workspace(dplan.workspace_bytes)
    b = gq.bindings(24)
    kv = dev(torch, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    hq_, hnk, hnv, hip, hix, hln, hkvp, hqw, hkw = (b.bind_read(t) for t in (
        q, nk, nv, ip, ix, ln, kv, dev_bf16(torch, qw), dev_bf16(torch, kw)))
    hkp, hvp, hks, hvs, hqr, ho, hl, hrk, hrv = (b.bind_read_write(t) for t in (
        kp, vp, ks, vs, qr, o, lse, rk, rv))

    def step(scope):
        aplan.enqueue_into(scope, L.NormRopePagedKvAppendArgs(
            hq_, hnk, hnv, hip, hix, hln, hqr.write(), hkp.write(), hvp.write(), query_norm=hqw,
            key_norm=hkw, key_scales=hks.write(), value_scales=hvs.write()))
        dplan.enqueue_into(scope, L.Mxfp4PagedBatchDecodeArgs(
            hqr.read(), hkp.read(), hvp.read(), hks.read(), hvs.read(), hip, hix, hln, ho.write(),
            hl.write()))
        rplan.enqueue_into(scope, L.PagedKvReadArgs(
            hkp.read(), hvp.read(), hks.read(), hvs.read(), hip, hix, hln, hkvp, hrk.write(),
            hrv.write()))
    torch.cuda.synchronize()
    graph = gq.capture(b, step).instantiate()
    pos = np.array(lens) - 1
    for i in range(3):
        new_q, new_k, new_v = (mx.bf16_round(rng.standard_normal((B, h, mx.D)))
                               for h in (hq, hkv, hkv))
        for t, a in ((q, new_q), (nk, new_k), (nv, new_v)):
            t.copy_(dev_bf16(torch, a).flatten())
        torch.cuda.synchronize()
        graph.launch().wait()
        # the host's copy of the cache takes the same rows
        for cache, rows in ((c.k, mx.norm_rotate(new_k, kw, pos, EPS, THETA)), (c.v, new_v)):
            codes, scales = mx.quantise(rows)
            for r in range(B):
                page_, off = c.indices[c.indptr[r] + pos[r] // page], pos[r] % page
                cache[0][page_, :, off], cache[1][page_, :, off] = codes[r], scales[r]
        c.q = host_bf16(torch, qr).reshape(B, hq, mx.D)
        check_decode(c, host_bf16(torch, o).reshape(B, hq, mx.D), lse.cpu().numpy().reshape(B, hq))
        for got, cache in ((rk, c.k), (rv, c.v)):
            want = np.concatenate([mx.rows_of(cache, c.indptr, c.indices, r, m)
                                   for r, m in enumerate(lens)])
            assert np.array_equal(host_bf16(torch, got).reshape(want.shape), want)
        o.zero_()


def test_chunk_over_a_read_back_prefix(env):
    """A chunk of a prompt behind an MXFP4 prefix: append the chunk, read the whole
    context back, and run the ragged prefill over it."""
    torch, L = env
    lens, rows, hq, hkv = [90, 40], [20, 40], 8, 2
    a = Append(env, 30, lens, rows, hq, hkv)
    a.pages = [p for p in a.pages]
    for s in a.scales:
        s[:] = np.random.default_rng(31).integers(123, 128, s.shape)
    got = a.run()
    a.check(got)
    c = Case(torch, 0, lens, hq, hkv)
    c.pool, c.indptr, c.indices, c.last = a.pool, a.indptr, a.indices, a.last
    head_major = lambda p: np.ascontiguousarray(  # noqa: E731
        p.reshape(a.pool, a.page, hkv, 64).swapaxes(1, 2))
    c.k = (head_major(got["key_pages"]), got["key_scales"].reshape(a.pool, hkv, a.page, 4))
    c.v = (head_major(got["value_pages"]), got["value_scales"].reshape(a.pool, hkv, a.page, 4))
    k, v = read(env, c, [0, 0], lens)
    order = np.lexsort((a.pos, a.req))
    q = mx.bf16_values(got["query_output"]).reshape(a.T, hq, mx.D)[order]
    from gpu_util import RaggedRunner
    r = RaggedRunner(L, 2, a.T, sum(lens), hq, hkv)
    out, lse = r.run(mx.bf16_bits(q).ravel(), k.ravel(), v.ravel(), [0, 20, 60], [0, 90, 130])
    out = mx.bf16_values(out).reshape(a.T, hq, mx.D)
    at = 0
    for i, (n, m) in enumerate(zip(lens, rows)):
        kk, vv = (mx.rows_of(x, c.indptr, c.indices, i, n) for x in (c.k, c.v))
        for j in range(m):
            e = n - m + j + 1
            ref, ref_l = mx.attend(q[at], kk[:e], vv[:e])
            # the ragged prefill's own: weights of 16 bits or more, O rounded to BF16
            assert np.abs(out[at] - ref).max() <= 2.0 ** -8 * np.abs(ref).max() + 2e-3
            assert np.abs(lse.reshape(a.T, hq)[at] - ref_l).max() <= 1e-3
            at += 1
