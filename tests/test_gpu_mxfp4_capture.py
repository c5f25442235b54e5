"""MXFP4 decode commands without a workspace of their own, captured by the caller into a
graph of its own.  Such a graph may be replayed on any stream, beside the queue's own
commands, so it uses none of the queue's memory: nothing has to be reserved for it, and
neither side changes the other's results."""
import numpy as np
import pytest

import mxfp4_util as mx
from test_gpu_mxfp4_decode import Case, check, host_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch

    import loom_infer_hip as L
    return torch, L


class Command:
    """A decode command of case `c`, bound on `queue`."""

    def __init__(self, env, queue, c, **plan):
        torch, L = env
        self.torch, self.c = torch, c
        spec = L.Bf16PagedBatchDecodeSpec(len(c.lens), c.pool, c.hq, c.hkv, kv_layout=c.layout,
                                          kv_dtype="mxfp4", kv_page_size=c.page)
        self.plan = L.DecodeProvider.load(0).plan_bf16_paged_batch(spec, **plan)
        self.out = torch.empty(c.q.size, dtype=torch.bfloat16, device="cuda")
        self.lse = torch.empty(c.q.size // mx.D, device="cuda")
        self.bindings = queue.bindings(10)
        b = self.bindings
        self.args = L.Mxfp4PagedBatchDecodeArgs(
            *(b.bind_read(t) for t in c.device()),
            *(b.bind_read_write(t).write() for t in (self.out, self.lse)))

    def fill(self):
        for t in (self.out, self.lse):
            t.fill_(float("nan"))

    def check(self):
        n = (len(self.c.lens), self.c.hq)
        check(self.c, host_bf16(self.torch, self.out).reshape(*n, mx.D),
              self.lse.cpu().numpy().reshape(n))


FORMS = {
    # lens, hq, hkv, page, layout; teams; the plan's algorithm
    "split": (([900, 1300], 8, 2, 16, "NHD"), 0, "direct"),
    "split, pairs of kv-heads": (([11000], 32, 32, 16, "NHD"), 0, "direct"),
    "one workgroup each": (([20, 40, 33], 16, 4, 32, "HND"), 0, "direct"),
    "balanced": (([333, 1, 700, 90], 28, 4, 64, "HND"), 16, "balanced_split_kv"),
    "balanced, pairs": (([500, 70], 64, 64, 16, "NHD"), 9, "balanced_split_kv"),
    "balanced by its rows": (([5000], 8, 8, 16, "NHD"), 0, "balanced_split_kv"),
}


@pytest.mark.parametrize("form", list(FORMS))
def test_captured_beside_the_queues_own_commands(env, form):
    torch, L = env
    shape, teams, algorithm = FORMS[form]
    c = Case(torch, 110, *shape)
    if form == "balanced by its rows":
        c.pool += 9000  # the bound that a plan takes from its pool
        more = np.zeros((9000, *c.k[0].shape[1:]), np.uint8)
        c.k, c.v = ((np.concatenate([a, more]), np.concatenate([s, more[..., :4]])) for a, s in (c.k, c.v))
    stream = torch.cuda.Stream()
    queue = L.CommandQueue(stream, 64)
    captured = Command(env, queue, c, teams=teams)
    assert captured.plan.algorithm == algorithm
    torch.cuda.synchronize()
    scope = queue.begin(captured.bindings)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        captured.plan.enqueue_into(scope, captured.args)
    scope.finish().wait()
    # the queue's own: a split command and a balanced one, which use its workspace
    others = [Command(env, queue, Case(torch, 111, [1500, 1000], 28, 4)),
              Command(env, queue, Case(torch, 112, [400, 900, 70], 8, 2), teams=24)]
    assert [o.plan.algorithm for o in others] == ["direct", "balanced_split_kv"]
    queue.reserve_workspace(max(o.plan.workspace_bytes for o in others))
    beside = torch.cuda.Stream()
    for overlap in (False, True, True):
        for o in (captured, *others):
            o.fill()
        torch.cuda.synchronize()
        with torch.cuda.stream(beside if overlap else stream):
            graph.replay()
        if not overlap:
            torch.cuda.synchronize()
            captured.check()
        for o in others:
            scope = queue.begin(o.bindings)
            for _ in range(4):
                if overlap:
                    with torch.cuda.stream(beside):
                        graph.replay()
                o.plan.enqueue_into(scope, o.args)
            scope.finish().wait()
        torch.cuda.synchronize()
        for o in (captured, *others):
            o.check()


def test_the_queues_workspace_stays_as_it_is(env):
    """A captured command reserves nothing, and one of one workgroup per request needs none
    eager either."""
    torch, L = env
    stream = torch.cuda.Stream()
    queue = L.CommandQueue(stream, 8)
    held = queue.workspace_bytes
    split = Command(env, queue, Case(torch, 113, [1200], 8, 2))
    short = Command(env, queue, Case(torch, 114, [30, 9], 8, 2))
    assert split.plan.workspace_bytes > 256 and short.plan.info.state_slots == 0
    torch.cuda.synchronize()
    for o in (split, short):
        scope = queue.begin(o.bindings)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            o.plan.enqueue_into(scope, o.args)
        scope.finish().wait()
        o.fill()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        o.check()
    scope = queue.begin(short.bindings)
    short.fill()
    torch.cuda.synchronize()
    short.plan.enqueue_into(scope, short.args)
    scope.finish().wait()
    short.check()
    assert queue.workspace_bytes == held
