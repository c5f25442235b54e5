"""Window attention's plans at the border of what a launch holds."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    import loom_infer_hip as L
    return L


def plan(L, batch, heads, dtype):
    return L.DecodeProvider.load(0).plan_window_paged_batch(L.WindowPagedAttentionSpec(
        batch, batch, batch, heads, heads, window=16, kv_dtype=dtype, explicit_rows=False))


def test_mxfp4_grids_count_what_is_launched(L):
    """2^24 workgroups of 256 threads are 2^32 threads.  Over MXFP4 pages with an even number
    of kv-heads the launch is a multiple of 16 workgroups, so of 2^24 all but the last 16 are
    plans."""
    assert plan(L, (1 << 23) - 8, 2, "mxfp4").info.block_threads == 256
    for batch in ((1 << 23) - 7, (1 << 23) - 1):
        with pytest.raises(L.PlanError) as e:
            plan(L, batch, 2, "mxfp4")
        assert e.value.variant == "StateCountOutOfRange"


def test_other_grids_are_launched_as_they_are(L):
    for batch, heads, dtype in (((1 << 23) - 1, 2, "bf16"), ((1 << 23) - 1, 2, "fp8_e4m3"),
                                ((1 << 24) - 1, 1, "mxfp4")):
        info = plan(L, batch, heads, dtype).info
        assert info.grid_blocks * info.block_threads == (1 << 32) - 256 * heads
