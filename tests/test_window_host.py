"""CPU tests of window attention's contract."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L():
    import loom_infer_hip as L
    L.lib()
    return L


def spec(L, rows=5, batch=2, pool=7, hq=8, hkv=2, **kw):
    return L.WindowPagedAttentionSpec(rows, batch, pool, hq, hkv, **kw)


def test_the_spec_holds_what_it_was_given(L):
    s = spec(L, window=1 << 40, sinks=3, kv_dtype="mxfp4", kv_layout="HND", kv_page_size=64)
    assert (s.rows, s.batch_size, s.window, s.sinks, s.explicit_rows) == (5, 2, 1 << 40, 3, True)
    assert s.paged.page_size == 64 and s.query_numel == 5 * 8 * 128 and s.lse_numel == 40


def test_one_row_per_request(L):
    assert not spec(L, rows=2, explicit_rows=False).explicit_rows
    with pytest.raises(L.ContractError) as e:
        spec(L, rows=3, explicit_rows=False)
    assert (e.value.variant, e.value.operand) == ("LengthMismatch", "rows")


@pytest.mark.parametrize("kw,variant", [
    (dict(rows=0), "ZeroDimension"), (dict(batch=0), "ZeroDimension"),
    (dict(hq=7), "InvalidHeadMapping"), (dict(head_dim=64), "UnsupportedHeadDimension"),
    (dict(kv_page_size=48), "UnsupportedPageSize"), (dict(rows=1 << 62), "ElementCountOverflow")])
def test_refused_shapes(L, kw, variant):
    with pytest.raises(L.ContractError) as e:
        spec(L, **kw)
    assert e.value.variant == variant


@pytest.mark.parametrize("name", ["window", "sinks", "rows"])
def test_numbers_that_no_64_bits_hold(L, name):
    for n in (-1, 1 << 64):
        with pytest.raises(ValueError):
            spec(L, **{name: n})


def test_an_embedded_spec_is_checked_again(L):
    from loom_infer_hip import _ffi
    p = L.Bf16PagedBatchDecodeSpec(2, 7, 8, 2)
    p._c.kv_dtype = 9
    out, err = _ffi.WindowAttentionSpec(), _ffi.Error()
    rc = L.lib().loom_window_attention_spec_new(C.byref(p._c), 2, 0, 0, 0, C.byref(out), C.byref(err))
    assert rc == 75 and err.code == 75


def test_null_arguments(L):
    from loom_infer_hip import _ffi
    err = _ffi.Error()
    lib = L.lib()
    assert lib.loom_window_attention_spec_new(None, 1, 0, 0, 0, None, C.byref(err)) == 59
    assert lib.loom_window_attention_enqueue(None, None, None, C.byref(err)) == 59
    out = C.c_void_p()
    for plan in (lib.loom_decode_provider_plan_window_paged_batch,
                 lib.loom_prefill_provider_plan_window_paged):
        assert plan(None, None, 0, C.byref(out), C.byref(err)) == 59
    lib.loom_window_attention_plan_free(None)
    lib.loom_window_attention_plan_get_info(None, None)
