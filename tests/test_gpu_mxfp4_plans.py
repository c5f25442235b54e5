"""MXFP4 decode plans at the limits of a launch (plans only: nothing is launched)."""
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
