"""What the commands over an MXFP4 cache refuse on the host, before anything is launched:
operands of a wrong length, type or alignment, missing ones, and another command's plan.
Every refused command leaves its outputs, and its queue, as they were."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, POOL, HQ, HKV, P, T = 2, 5, 8, 2, 16, 3
D = 128


@pytest.fixture(scope="module")
def env():
    import torch

    import loom_infer_hip as L
    return torch, L


def numbers(torch):
    """Every operand of the three commands, valid."""
    bf = dict(dtype=torch.bfloat16, device="cuda")
    u8 = dict(dtype=torch.uint8, device="cuda")
    x = {"query": torch.ones(B * HQ * D, **bf), "output": torch.full((B * HQ * D,), 7.0, **bf),
         "lse": torch.full((B * HQ,), 7.0, device="cuda"),
         "tokens_query": torch.ones(T * HQ * D, **bf), "key": torch.ones(T * HKV * D, **bf),
         "value": torch.ones(T * HKV * D, **bf),
         "query_output": torch.full((T * HQ * D,), 7.0, **bf),
         "query_norm": torch.ones(D, **bf), "key_norm": torch.ones(D, **bf),
         "read_key": torch.full((20 * HKV * D,), 7.0, **bf),
         "read_value": torch.full((20 * HKV * D,), 7.0, **bf)}
    for n in ("key", "value"):
        x[n + "_pages"] = torch.zeros(POOL * P * HKV * 64, **u8)
        x[n + "_scales"] = torch.full((POOL * HKV * P * 4,), 127, **u8)
    for n, v in (("page_indptr", [0, 1, 3]), ("page_indices", [4, 0, 2]), ("last_page_len", [7, 9]),
                 ("batch_indices", [0, 1, 1]), ("positions", [6, 23, 24]), ("kv_indptr", [0, 5, 20]),
                 ("kv_start", [1, 4])):
        x[n] = torch.tensor(v, dtype=torch.int32, device="cuda")
    return x


WRITTEN = ("output", "lse", "query_output", "read_key", "read_value")


def plans(L):
    form = dict(kv_dtype="mxfp4")
    return {
        "decode": L.DecodeProvider.load(0).plan_bf16_paged_batch(
            L.Bf16PagedBatchDecodeSpec(B, POOL, HQ, HKV, **form)),
        "append": L.RopeProvider.load(0).plan_norm_paged_append(
            L.NormRopePagedKvAppendSpec(T, B, POOL, HQ, HKV, norm_eps=1e-6, **form)),
        "read": L.PrefillProvider.load(0).plan_paged_kv_read(
            L.PagedKvReadSpec(B, 20, POOL, HKV, **form)),
    }


NAMES = {  # argument: the operand's name in errors
    "decode": dict(query="Q", key_pages="K_pages", value_pages="V_pages", key_scales="K_scales",
                   value_scales="V_scales", page_indptr="page_indptr",
                   last_page_len="last_page_len", output="O", lse="LSE"),
    "append": dict(tokens_query="query", key="key", value="value", batch_indices="batch_indices",
                   positions="positions", page_indptr="page_indptr", last_page_len="last_page_len",
                   query_norm="query_norm", key_norm="key_norm", query_output="query_output",
                   key_pages="key_pages", value_pages="value_pages", key_scales="key_scales",
                   value_scales="value_scales"),
    "read": dict(key_pages="K_pages", value_pages="V_pages", key_scales="K_scales",
                 value_scales="V_scales", page_indptr="page_indptr", last_page_len="last_page_len",
                 kv_indptr="kv_indptr", kv_start="kv_start", read_key="K", read_value="V"),
}


def command(L, op, b, x):
    """The command's arguments over the tensors of `x`."""
    r, w = (lambda n: b.bind_read(x[n])), (lambda n: b.bind_read_write(x[n]).write())
    table = ("page_indptr", "page_indices", "last_page_len")
    if op == "decode":
        return L.Mxfp4PagedBatchDecodeArgs(
            *(r(n) for n in ("query", "key_pages", "value_pages", "key_scales", "value_scales")),
            *(r(n) for n in table), w("output"), w("lse"))
    if op == "append":
        return L.NormRopePagedKvAppendArgs(
            r("tokens_query"), r("key"), r("value"), *(r(n) for n in table), w("query_output"),
            w("key_pages"), w("value_pages"), r("batch_indices"), r("positions"), r("query_norm"),
            r("key_norm"), w("key_scales"), w("value_scales"))
    return L.PagedKvReadArgs(
        *(r(n) for n in ("key_pages", "value_pages", "key_scales", "value_scales")),
        *(r(n) for n in table), r("kv_indptr"), w("read_key"), w("read_value"), r("kv_start"))


def refused(env, op, x, plan=None, args=None):
    """The error of the command over `x`; a valid command goes through afterwards."""
    torch, L = env
    p = plans(L)
    queue = L.CommandQueue(torch.cuda.current_stream(), 4)
    b = queue.bindings(20)
    a = args(b) if args else command(L, op, b, x)
    scope = queue.begin(b)
    with pytest.raises(L.LoomError) as e:
        p[plan or op].enqueue_into(scope, a)
    scope.finish().wait()
    for n in WRITTEN:
        assert (x[n] == 7.0).all(), n
    good = numbers(torch)
    b = queue.bindings(20)
    a = command(L, op, b, good)
    scope = queue.begin(b)
    p[op].enqueue_into(scope, a)
    scope.finish().wait()
    changed = {"decode": "output", "append": "query_output", "read": "read_key"}[op]
    assert (good[changed] != 7.0).all()
    return e.value


@pytest.mark.parametrize("op", list(NAMES))
def test_lengths(env, op):
    torch, _ = env
    for n, name in NAMES[op].items():
        x = numbers(torch)
        x[n] = x[n][:-1]
        e = refused(env, op, x)
        assert (e.variant, e.operand) == ("LengthMismatch", name), n
    x = numbers(torch)
    x["page_indices"] = x["page_indices"][:1]
    assert refused(env, op, x).variant == "PageIndicesTooShort"


@pytest.mark.parametrize("op", list(NAMES))
def test_element_types(env, op):
    torch, _ = env
    for n in NAMES[op]:
        x = numbers(torch)
        other = torch.float32 if x[n].dtype == torch.int32 else torch.int32
        x[n] = torch.zeros(x[n].numel(), dtype=other, device="cuda")
        if n in WRITTEN:
            x[n].fill_(7)
        refused(env, op, x)


@pytest.mark.parametrize("op", ["decode", "read"])
def test_alignment(env, op):
    torch, _ = env
    for n, name in NAMES[op].items():
        x = numbers(torch)
        t = x[n]
        if t.element_size() > 2:
            continue
        b = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")
        b[1:1 + t.numel()] = t
        x[n] = b[1:1 + t.numel()]
        e = refused(env, op, x)
        assert (e.variant, e.operand) == ("MisalignedBuffer", name), n


def test_missing_operands(env):
    """Norm weights, scales or explicit tokens that the plan needs."""
    torch, L = env
    import dataclasses
    x = numbers(torch)
    for n in ("query_norm", "key_norm", "key_scales", "value_scales", "batch_indices", "positions"):
        refused(env, "append", x, args=lambda b: dataclasses.replace(
            command(L, "append", b, x), **{n: None}))


def test_other_commands_plans(env):
    """An enqueue form refuses a plan over other pages, and a plan of another append."""
    torch, L = env
    x = numbers(torch)
    bf = dict(dtype=torch.bfloat16, device="cuda")
    pages = [torch.zeros(POOL * P * HKV * D, **bf) for _ in range(2)]

    def bf16_decode(b):
        r = b.bind_read
        return L.Bf16PagedBatchDecodeArgs(
            r(x["query"]), r(pages[0]), r(pages[1]), r(x["page_indptr"]), r(x["page_indices"]),
            r(x["last_page_len"]), b.bind_read_write(x["output"]).write(),
            b.bind_read_write(x["lse"]).write())
    refused(env, "decode", x, args=bf16_decode)

    def bf16_append(b):
        r = b.bind_read
        return L.Bf16RopePagedKvAppendTokensArgs(
            r(x["tokens_query"]), r(x["key"]), r(x["value"]), r(x["batch_indices"]),
            r(x["positions"]), r(x["page_indptr"]), r(x["page_indices"]), r(x["last_page_len"]),
            b.bind_read_write(x["query_output"]).write(), b.bind_read_write(pages[0]).write(),
            b.bind_read_write(pages[1]).write())
    refused(env, "append", x, args=bf16_append)
    # the MXFP4 forms over plans of BF16 pages
    queue = L.CommandQueue(torch.cuda.current_stream(), 4)
    others = {
        "decode": L.DecodeProvider.load(0).plan_bf16_paged_batch(
            L.Bf16PagedBatchDecodeSpec(B, POOL, HQ, HKV)),
        "append": L.RopeProvider.load(0).plan_bf16_paged_append_tokens(
            L.Bf16RopePagedKvAppendTokensSpec(T, B, POOL, HQ, HKV)),
    }
    for op, plan in others.items():
        b = queue.bindings(20)
        a = command(L, op, b, x)
        scope = queue.begin(b)
        with pytest.raises(L.LoomError):
            plan.enqueue_into(scope, a)
        scope.finish().wait()
    for n in WRITTEN:
        assert (x[n] == 7.0).all(), n


def test_plans(env):
    """What only a plan can refuse."""
    torch, L = env
    with pytest.raises(L.LoomError) as e:  # the reference-shaped append writes no scales
        L.RopeProvider.load(0).plan_bf16_paged_append_tokens(
            L.Bf16RopePagedKvAppendTokensSpec(T, B, POOL, HQ, HKV, kv_dtype="mxfp4"))
    assert e.value.operand == "kv_dtype"
    with pytest.raises(L.PlanError):  # more requests than a command takes
        L.DecodeProvider.load(0).plan_bf16_paged_batch(
            L.Bf16PagedBatchDecodeSpec(65537, 70000, 1, 1, kv_dtype="mxfp4"))
    with pytest.raises(L.PlanError):  # a merge of more threads than a launch holds
        L.DecodeProvider.load(0).plan_bf16_paged_batch(
            L.Bf16PagedBatchDecodeSpec(65536, 70000, 1024, 1, kv_dtype="mxfp4"), teams=7)
    with pytest.raises(L.PlanError):
        L.PrefillProvider.load(0).plan_paged_kv_read(L.PagedKvReadSpec(1, 1, 4, 4097))
    import ctypes as C
    out, err = C.c_void_p(), L._ffi.Error()
    spec = L.PagedKvReadSpec(1, 1, 4, 4)
    for flags in (2, 1 << 20):
        assert L.lib().loom_prefill_provider_plan_paged_kv_read(
            L.PrefillProvider.load(0)._p, C.byref(spec._c), flags, C.byref(out), C.byref(err)) != 0
        assert err.operand == b"flags" and not out.value
    with pytest.raises(L.PlanError) as e:
        L.RopeProvider.load(0).plan_norm_paged_append(
            L.NormRopePagedKvAppendSpec(T, B, POOL, HQ, HKV), flags=1 << 20)
    assert e.value.operand == "flags"


def test_one_tensor_for_two_operands(env):
    """K and V pages, or an output that is also read, in one buffer."""
    torch, L = env
    x = numbers(torch)
    x["value_pages"] = x["key_pages"]
    queue = L.CommandQueue(torch.cuda.current_stream(), 4)
    with pytest.raises(L.LoomError):
        command(L, "append", queue.bindings(20), x)
