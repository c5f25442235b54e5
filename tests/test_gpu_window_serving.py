"""Window attention among other commands: behind the appends that write its cache, in
captured graphs, on two queues at once, in every kernel that a plan chooses, and what it
refuses on the host."""
import ctypes as C

import numpy as np
import pytest

import mxfp4_util as mx
from window_util import Case, host

pytestmark = pytest.mark.gpu
DTYPES = ["bf16", "fp8_e4m3", "mxfp4"]


@pytest.fixture(scope="module")
def env():
    import torch
    import loom_infer_hip as L
    return torch, L


class Command:
    """A command of case `c`, bound on `queue`."""

    def __init__(self, env, queue, c, **plan):
        torch, L = env
        self.c, self.plan = c, c.plan(L, **plan)
        self.bindings = queue.bindings(16)
        self.out, self.lse = c.outputs(torch)
        self.args = c.args(L, self.bindings, c.operands(torch), self.out, self.lse)

    def enqueue(self, scope):
        self.plan.enqueue_into(scope, self.args)

    def fill(self):
        for t in (self.out, self.lse):
            t.fill_(float("nan"))

    def check(self):
        self.c.check(host(self.out), host(self.lse), self.plan.algorithm == "long_tile")


# Cases whose plans choose each kernel: (rows or None, lens, hq, hkv, window), and what the
# plan reports: columns and threads per workgroup.  (The chip's 256 CUs set the borders.)
def tiles(b, n, rows=None, hq=8, hkv=8, window=40):
    return ([rows] * b if rows else None), [n] * b, hq, hkv, window


KERNELS = {
    "16 columns, 8 waves": (*tiles(3, 200, window=120), 16, 512),
    "16 columns, 4 waves, few steps": (*tiles(3, 150), 16, 256),
    "16 columns, 4 waves, windows": (*tiles(40, 90), 16, 256),
    "16 columns, 4 waves, whole": (*tiles(70, 60, window=0), 16, 256),
    "32 columns, 8 waves": (*tiles(24, 190, 28, window=0), 32, 512),
    "32 columns, 4 waves": (*tiles(33, 70, 21), 32, 256),
    "one row, 32 columns, 8 waves": (*tiles(200, 140, hq=32, hkv=1, window=0), 32, 512),
    "one row, 32 columns, 4 waves": (*tiles(500, 20, hq=32, hkv=1), 32, 256),
    "32 columns, long walks that differ": (*tiles(2, 1100, 700, window=0), 32, 512),
    "64 columns, 2 groups": (*tiles(40, 100, 70), 64, 256),
    "64 columns, 4 groups": (*tiles(1, 1500, 1400), 64, 512),
    "64 columns, 4 groups, long walks that differ": (*tiles(2, 1200, 1050, window=0), 64, 512),
    "128 columns, 1 group": (*tiles(16, 300, 260, 16, 16), 128, 256),
    "128 columns, 2 groups": (*tiles(16, 300, 260, 16, 16, window=0), 128, 512),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kernel", list(KERNELS))
def test_every_kernel(env, kernel, dtype):
    torch, L = env
    rows, lens, hq, hkv, window, cols, threads = KERNELS[kernel]
    c = Case(41, lens, rows, hq, hkv, window, 3, 16, "NHD", dtype)
    if dtype == "mxfp4":  # other borders
        cols, threads = {"64 columns, 2 groups": (128, 512),
                         "64 columns, 4 groups, long walks that differ": (32, 256)}.get(
                             kernel, (cols, threads))
    info = c.plan(L).info
    assert (info.tile_cols, info.block_threads) == (cols, threads)
    c.check(*c.run(torch, L), long_tile=cols > 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_walks_of_a_chunk_are_shared(env, dtype):
    """Few tiles of a grid that has room for more, contexts that differ."""
    c = Case(42, [2600, 2100, 1500, 4000, 2300, 2047, 1999, 2500], [8] * 8, 4, 1, 0, 0, 16, "NHD", dtype)
    c.check(*c.run(*env))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [None, [5, 3]])
def test_captured_beside_the_queues_own_commands(env, dtype, rows):
    """A caller's capture uses none of the queue's memory, though its walks would be shared:
    it may be replayed on any stream, beside the queue's shared commands."""
    torch, L = env
    stream, beside = torch.cuda.Stream(), torch.cuda.Stream()
    queue = L.CommandQueue(stream, 64)
    captured = Command(env, queue, Case(43, [3000, 2200], rows, 8, 2, 2048, 4, 16, "NHD", dtype))
    other = Command(env, queue, Case(44, [2500, 4000], rows, 8, 2, 0, 0, 32, "HND", dtype))
    torch.cuda.synchronize()
    held = queue.workspace_bytes
    scope = queue.begin(captured.bindings)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        captured.enqueue(scope)
    scope.finish().wait()
    assert queue.workspace_bytes == held
    for _ in range(3):
        captured.fill()
        other.fill()
        torch.cuda.synchronize()
        scope = queue.begin(other.bindings)
        for _ in range(4):
            with torch.cuda.stream(beside):
                graph.replay()
            other.enqueue(scope)
        scope.finish().wait()
        torch.cuda.synchronize()
        captured.check()
        other.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_graph_of_shared_walks(env, dtype):
    """A graph queue's own capture has words and states of its private queue: every replay
    is the eager command's, whatever runs between."""
    torch, L = env
    c = Case(47, [5000, 3100, 700], None, 8, 2, 0, 0, 16, "HND", dtype)
    want = c.run(torch, L)
    gq = L.GraphQueue(0, 2)
    b = gq.bindings(16)
    out, lse = c.outputs(torch)
    plan, args = c.plan(L), c.args(L, b, c.operands(torch), out, lse)
    torch.cuda.synchronize()
    graph = gq.capture(b, lambda scope: (plan.enqueue_into(scope, args),
                                         plan.enqueue_into(scope, args))).instantiate()
    for i in range(4):
        out.fill_(7.0)
        lse.fill_(7.0)
        torch.cuda.synchronize()
        graph.launch().wait()
        assert np.array_equal(host(out), want[0]) and np.array_equal(host(lse), want[1])
        if i == 1:
            graph.set_replay_mode("hip_graph_launch")
        c.run(torch, L)


def test_two_queues_at_once(env):
    """Shared walks on two streams: each queue has words and states of its own."""
    torch, L = env
    queues = [L.CommandQueue(torch.cuda.Stream(), 40) for _ in range(2)]
    work = [Command(env, q, Case(45 + i, [3000, 1700 + i], None, 8, 2, 0, 0, 16, "NHD", "bf16"))
            for i, q in enumerate(queues)]
    torch.cuda.synchronize()
    scopes = [q.begin(w.bindings) for q, w in zip(queues, work)]
    for _ in range(20):
        for w, s in zip(work, scopes):
            w.enqueue(s)
    for s in scopes:
        s.finish().wait()
    for w in work:
        w.check()


@pytest.mark.parametrize("dtype", ["bf16", "mxfp4"])
def test_a_serving_step(env, dtype):
    """A chunk of new rows, then steps of single tokens: the append writes the cache, and
    window attention reads what it wrote; the single tokens' step is one captured graph,
    replayed with new inputs."""
    torch, L = env
    lens, rows, hq, hkv, page, theta, eps = [130, 45, 70], [30, 45, 1], 8, 2, 32, 1e4, 1e-6
    c = Case(46, lens, rows, hq, hkv, 50, 5, page, "HND", dtype)
    c.last = c.last.copy()
    B = len(lens)
    d = c.operands(torch)
    form = dict(kv_layout="HND", kv_dtype=dtype, kv_page_size=page)
    rng = np.random.default_rng(47)
    qw, kw = (mx.bf16_round(1 + 0.3 * rng.standard_normal(mx.D)) for _ in range(2))

    def bf16(x):
        return torch.from_numpy(mx.bf16_bits(x).view(np.int16).copy()).cuda().view(torch.bfloat16)

    def ints(x):
        return torch.from_numpy(np.asarray(x, np.int32)).cuda()

    weights = {"query_norm": bf16(qw), "key_norm": bf16(kw)}

    def new(req, pos):
        """New rows, and the cache's own copy of what the append writes."""
        q, k, v = (mx.bf16_round(rng.standard_normal((len(req), h, mx.D))) for h in (hq, hkv, hkv))
        exact = mx.norm_rotate(k, kw, pos, eps, theta), v
        for which, x in enumerate(exact):
            for i, (r, p) in enumerate(zip(req, pos)):
                slot = c.indices[c.indptr[r] + p // page], slice(None), p % page
                if dtype == "mxfp4":
                    c.cache[which][0][slot], c.cache[which][1][slot] = mx.quantise(x[i])
                else:
                    c.cache[which][slot] = mx.bf16_round(x[i])
        return q, k, v

    def take_pages():
        """BF16 rounds K's FP32 to its own nearest: the pages as the append left them."""
        if dtype == "bf16":
            for which, name in enumerate("kv"):
                got = mx.bf16_values(d[name].view(torch.int16).cpu().numpy().view(np.uint16))
                got = got.reshape(c.cache[which].shape)
                assert np.abs(got - c.cache[which]).max() <= 2.0 ** -7 * np.abs(got).max()
                c.cache[which][:] = got

    def append(b, T, x, explicit):
        plan = L.RopeProvider.load(0).plan_norm_paged_append(L.NormRopePagedKvAppendSpec(
            T, B, c.pool, hq, hkv, rope_theta=theta, norm_eps=eps, explicit_tokens=explicit, **form))
        names = ["query", "key", "value", "query_norm", "key_norm"]
        names += ["batch_indices", "positions"] if explicit else []
        h = {n: b.bind_read(x[n]) for n in names}
        h |= {k: handles[n] for k, n in (("page_indptr", "indptr"), ("page_indices", "indices"),
                                         ("last_page_len", "last"))}
        h |= {"key_pages": handles["k"].write(), "value_pages": handles["v"].write()}
        if dtype == "mxfp4":
            h |= {"key_scales": handles["k_mx"].write(), "value_scales": handles["v_mx"].write()}
        rotated = b.bind_read_write(x["query_output"])
        return plan, L.NormRopePagedKvAppendArgs(query_output=rotated.write(), **h), rotated

    def bind(b, names):
        return {n: b.bind_read_write(t) if n[0] in "kv" else b.bind_read(t)
                for n, t in d.items() if n in names}

    def window_args(rotated, out, lse, qo=None):
        more = {} if dtype == "bf16" else dict(key_scales=handles["k_mx"].read(),
                                               value_scales=handles["v_mx"].read())
        return L.WindowPagedAttentionArgs(
            rotated.read(), handles["k"].read(), handles["v"].read(), handles["indptr"],
            handles["indices"], handles["last"], out, lse, qo_indptr=qo, **more)

    cached = ("k", "v", "k_mx", "v_mx", "indptr", "indices", "last")
    # the chunk
    req = np.repeat(np.arange(B), rows)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, rows)])
    q, k, v = new(req, pos)
    queue = L.CommandQueue(torch.cuda.current_stream(), 4)
    b = queue.bindings(32)
    handles = bind(b, cached)
    x = dict(query=bf16(q), key=bf16(k), value=bf16(v), batch_indices=ints(req), positions=ints(pos),
             query_output=torch.zeros(len(req) * hq * mx.D, dtype=torch.bfloat16, device="cuda"), **weights)
    plan, args, rotated = append(b, len(req), x, True)
    out, lse = c.outputs(torch)
    attend = c.plan(L)
    wargs = window_args(rotated, b.bind_read_write(out).write(), b.bind_read_write(lse).write(),
                        b.bind_read(d["qo"]))
    torch.cuda.synchronize()
    scope = queue.begin(b)
    plan.enqueue_into(scope, args)
    attend.enqueue_into(scope, wargs)
    scope.finish().wait()
    take_pages()
    c.q = host(x["query_output"]).reshape(-1, hq, mx.D)
    c.check(host(out), host(lse), attend.algorithm == "long_tile")
    # single tokens, as a graph: the tables say one token more before each replay
    c.single, c.rows, c.nnz = True, [1] * B, B
    gq = L.GraphQueue(0, 2)
    b = gq.bindings(32)
    handles = bind(b, cached)
    x = {n: torch.zeros(B * h * mx.D, dtype=torch.bfloat16, device="cuda")
         for n, h in (("query", hq), ("key", hkv), ("value", hkv), ("query_output", hq))} | weights
    plan, args, rotated = append(b, B, x, False)
    out, lse = c.outputs(torch)
    attend = c.plan(L)
    wargs = window_args(rotated, b.bind_read_write(out).write(), b.bind_read_write(lse).write())
    torch.cuda.synchronize()
    graph = gq.capture(b, lambda scope: (plan.enqueue_into(scope, args),
                                         attend.enqueue_into(scope, wargs))).instantiate()
    for _ in range(4):
        c.lens = [n + 1 for n in c.lens]  # (within the last pages)
        c.last += 1
        assert c.last.max() <= page
        for name, a in zip(("query", "key", "value"), new(range(B), np.array(c.lens) - 1)):
            x[name].copy_(bf16(a).flatten())
        d["last"].copy_(ints(c.last))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.launch().wait()
        take_pages()
        c.q = host(x["query_output"]).reshape(B, hq, mx.D)
        c.check(host(out), host(lse))


# ---- refusals ---------------------------------------------------------------------
SHAPE = dict(lens=[20, 40], hq=8, hkv=2, window=16, sinks=2)


def refused_command(env, dtype, rows, variant, operand, change):
    torch, L = env
    c = Case(48, rows=rows, dtype=dtype, **SHAPE)
    d, (out, lse) = c.operands(torch), c.outputs(torch)
    x = dict(d, out=out, lse=lse)
    change(x)
    queue = L.CommandQueue(torch.cuda.current_stream(), 4)
    b = queue.bindings(16)
    args = c.args(L, b, {k: v for k, v in x.items() if k not in ("out", "lse")}, x["out"], x["lse"])
    plan = c.plan(L)
    torch.cuda.synchronize()
    scope = queue.begin(b)
    with pytest.raises(L.LoomError) as e:
        plan.enqueue_into(scope, args)
    assert (e.value.variant, e.value.operand) == (variant, operand), e.value
    scope.finish().wait()
    for t in (out, lse):
        assert (host(t) == 7).all()


OPERANDS = {"q": "Q", "k": "K_pages", "v": "V_pages", "indptr": "page_indptr", "last": "last_page_len",
            "out": "O", "lse": "LSE", "qo": "qo_indptr", "kv_scales": "kv_scales", "k_mx": "K_scales",
            "v_mx": "V_scales"}


@pytest.mark.parametrize("name", list(OPERANDS))
@pytest.mark.parametrize("more", [-1, 1])
def test_operands_of_a_wrong_length(env, name, more):
    torch = env[0]
    dtype = {"kv_scales": "fp8_e4m3", "k_mx": "mxfp4", "v_mx": "mxfp4"}.get(name, "bf16")

    def change(x):
        t = x[name].flatten()
        x[name] = t[:-1].clone() if more < 0 else torch.cat([t, t[:1]])
    refused_command(env, dtype, [3, 9], "LengthMismatch", OPERANDS[name], change)


@pytest.mark.parametrize("dtype", DTYPES)
def test_page_indices_too_short(env, dtype):
    def change(x):
        x["indices"] = x["indices"][:1].clone()
    refused_command(env, dtype, None, "PageIndicesTooShort", "page_indices", change)


@pytest.mark.parametrize("name,dtype", [("q", "bf16"), ("k", "bf16"), ("v", "fp8_e4m3"), ("k_mx", "mxfp4"),
                                        ("out", "bf16")])
def test_operands_off_a_four_byte_boundary(env, name, dtype):
    torch = env[0]

    def change(x):
        t = x[name].flatten()
        x[name] = torch.cat([t[:1], t])[1:] if t.element_size() == 2 else torch.cat([t[:2], t])[2:]
    refused_command(env, dtype, [3, 9], "MisalignedBuffer", OPERANDS[name], change)


@pytest.mark.parametrize("scale", [0.0, -0.1, float("inf"), float("nan"), 3e38])
@pytest.mark.parametrize("rows", [None, [3, 9]])
def test_plans_refuse_scales(env, scale, rows):
    L = env[1]
    c = Case(49, rows=rows, **SHAPE)
    spec = c.spec(L)
    spec._c.paged.softmax_scale = scale
    with pytest.raises(L.PlanError) as e:
        (L.DecodeProvider.load(0).plan_window_paged_batch if rows is None
         else L.PrefillProvider.load(0).plan_window_paged)(spec)
    assert (e.value.variant, e.value.operand) == ("InvalidOption", "softmax_scale")


def test_plans_refuse_the_other_form(env):
    L = env[1]
    for rows, plan in ((None, L.PrefillProvider.load(0).plan_window_paged),
                       ([3, 9], L.DecodeProvider.load(0).plan_window_paged_batch)):
        with pytest.raises(L.PlanError) as e:
            plan(Case(50, rows=rows, **SHAPE).spec(L))
        assert e.value.variant == "InvalidOption"


@pytest.mark.parametrize("shape", [dict(rows=1 << 26, batch_size=1, num_query_heads=32, num_kv_heads=8),
                                   dict(rows=1 << 24, batch_size=1 << 24, num_query_heads=64,
                                        num_kv_heads=64, explicit_rows=False),
                                   dict(rows=5, batch_size=5, num_query_heads=4098, num_kv_heads=4098)])
def test_plans_refuse_what_a_launch_cannot_hold(env, shape):
    L = env[1]
    spec = L.WindowPagedAttentionSpec(max_num_pages=9, **shape)
    with pytest.raises(L.PlanError) as e:
        (L.PrefillProvider.load(0).plan_window_paged if spec.explicit_rows
         else L.DecodeProvider.load(0).plan_window_paged_batch)(spec)
    assert e.value.variant == "StateCountOutOfRange"


def test_flags_of_another_form(env):
    L = env[1]
    from loom_infer_hip import _ffi
    lib, out, err = L.lib(), C.c_void_p(), _ffi.Error()
    one, many = Case(51, rows=None, **SHAPE).spec(L), Case(51, rows=[3, 9], **SHAPE).spec(L)
    decode, prefill = L.DecodeProvider.load(0), L.PrefillProvider.load(0)
    for flags in (1 << 1, 1 << 2, 1 << 3, 1 << 31):
        assert lib.loom_decode_provider_plan_window_paged_batch(
            decode._p, C.byref(one._c), flags, C.byref(out), C.byref(err)) == 75 and not out.value
    for flags in (1 << 2, 1 << 1 | 1 << 3, 1 << 31):  # both tiles, among others
        assert lib.loom_prefill_provider_plan_window_paged(
            prefill._p, C.byref(many._c), flags, C.byref(out), C.byref(err)) == 75 and not out.value
