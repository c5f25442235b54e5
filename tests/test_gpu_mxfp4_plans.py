"""MXFP4 decode plans: the limits of a launch, and the softmax scale."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    import torch  # noqa: F401  (its HIP runtime first)

    import loom_infer_hip as L
    return L


def plan(L, batch, hq, hkv, pages, **options):
    return L.DecodeProvider.load(0).plan_bf16_paged_batch(
        L.Bf16PagedBatchDecodeSpec(batch, pages, hq, hkv, kv_dtype="mxfp4"), **options)


def test_direct_plans_hold_fewer_than_2_32_threads(L):
    """Workgroups of 512 threads, one per request and tile of 8 query heads."""
    with pytest.raises(L.PlanError) as e:  # 65536 * 128 = 2^23 of them
        plan(L, 65536, 1024, 1, 65536)
    assert e.value.variant == "StateCountOutOfRange"
    p = plan(L, 65536, 1016, 1, 65536)
    assert p.algorithm == "direct" and p.info.grid_blocks == 65536 * 127
    with pytest.raises(L.PlanError):  # one request of as many tiles
        plan(L, 1, 8 << 23, 1, 1)


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, float("inf"), float("nan")])
@pytest.mark.parametrize("teams", [0, 4])
def test_softmax_scales_that_do_not_keep_the_scores_order_are_refused(L, scale, teams):
    """A scale set by hand in the spec: the kernels find the largest score before they
    scale it."""
    spec = L.Bf16PagedBatchDecodeSpec(2, 9, 8, 2, kv_dtype="mxfp4")
    spec._c.softmax_scale = scale
    with pytest.raises(L.PlanError) as e:
        L.DecodeProvider.load(0).plan_bf16_paged_batch(spec, teams=teams)
    assert (e.value.variant, e.value.operand) == ("InvalidOption", "softmax_scale")


@pytest.mark.parametrize("teams", [0, 4])
def test_other_softmax_scales(L, teams):
    import numpy as np
    import torch

    import mxfp4_util as mx
    from test_gpu_mxfp4_decode import Case, host_bf16
    c = Case(torch, 140, [40, 90, 33], 8, 2)
    spec = L.Bf16PagedBatchDecodeSpec(3, c.pool, 8, 2, kv_dtype="mxfp4")
    spec._c.softmax_scale = 2.0 ** -5
    plan = L.DecodeProvider.load(0).plan_bf16_paged_batch(spec, teams=teams)
    queue = L.CommandQueue(torch.cuda.current_stream(), 1)
    out = torch.zeros(c.q.size, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(c.q.size // mx.D, device="cuda")
    b = queue.bindings(10)
    args = L.Mxfp4PagedBatchDecodeArgs(*(b.bind_read(t) for t in c.device()),
                                       *(b.bind_read_write(t).write() for t in (out, lse)))
    scope = queue.begin(b)
    plan.enqueue_into(scope, args)
    scope.finish().wait()
    # the tolerances of test_gpu_mxfp4_decode, which bound the larger scale of 128^-0.5
    bo, bl = c.bounds(np.zeros(1), np.zeros(1))
    out, lse = host_bf16(torch, out).reshape(3, 8, mx.D), lse.cpu().numpy().reshape(3, 8)
    for r, n in enumerate(c.lens):
        k, v = (mx.rows_of(x, c.indptr, c.indices, r, n) for x in (c.k, c.v))
        ref_o, ref_l = mx.attend(c.q[r], k, v, 2.0 ** -5)
        assert (np.abs(out[r] - ref_o) <= bo + 2.0 ** -8 * np.abs(ref_o)).all()
        assert (np.abs(lse[r] - ref_l) <= bl + 2.0 ** -22 * np.abs(ref_l)).all()
