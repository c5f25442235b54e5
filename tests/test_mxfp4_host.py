"""CPU tests of the MXFP4 cache's contracts, and of the 64-bit forms that the GPU tests
compare with."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import mxfp4_util as mx


@pytest.fixture(scope="module")
def L():
    import loom_infer_hip as L
    L.lib()
    return L


def test_decode_spec_over_mxfp4_pages(L):
    s = L.Bf16PagedBatchDecodeSpec(3, 7, 8, 2, kv_dtype="mxfp4", kv_layout="HND", kv_page_size=32)
    assert (s.kv_dtype, s.kv_layout, s.page_size) == ("mxfp4", "HND", 32)
    assert s.kv_pages_numel == 7 * 32 * 2 * 64 and s.mx_scales_numel == 7 * 32 * 2 * 4
    assert L.Bf16PagedBatchDecodeSpec(3, 7, 8, 2).kv_pages_numel == 7 * 16 * 2 * 128


def test_other_operations_refuse_mxfp4_pages(L):
    with pytest.raises(L.PlanError) as e:
        L.Bf16PagedPrefillSpec(1, 4, 4, 8, 2, kv_dtype="mxfp4")
    assert (e.value.variant, e.value.operand) == ("InvalidOption", "kv_dtype")
    out, err = L._ffi.PagedDecodeSpec(), L._ffi.Error()
    s = L.Bf16PagedBatchDecodeSpec(1, 4, 8, 2)
    rc = L.lib().loom_paged_decode_spec_with_kv_dtype(C.byref(s._c), 3, C.byref(out), C.byref(err))
    assert rc == 75 and err.operand == b"kv_dtype"


def test_norm_append_spec(L):
    s = L.NormRopePagedKvAppendSpec(5, 2, 7, 8, 2, kv_dtype="mxfp4", kv_page_size=64,
                                    rope_theta=1e6, norm_eps=1e-6)
    assert (s.tokens, s.batch_size, s.rope_theta, s.explicit_tokens) == (5, 2, 1e6, True)
    assert s.norm_eps == np.float32(1e-6) and s.mx_scales_numel == 7 * 64 * 2 * 4
    assert s.query_numel == 5 * 8 * 128 and s.key_numel == 5 * 2 * 128
    assert L.NormRopePagedKvAppendSpec(2, 2, 7, 8, 2, explicit_tokens=False).norm_eps is None

    def refused(variant, tokens=5, **kw):
        with pytest.raises(L.ContractError) as e:
            L.NormRopePagedKvAppendSpec(tokens, 2, 7, 8, 2, **kw)
        assert e.value.variant == variant, e.value.variant
    refused("ZeroDimension", tokens=0)
    refused("UnsupportedAppendTokenCount", tokens=8193)
    refused("LengthMismatch", tokens=3, explicit_tokens=False)
    for theta in (1.0, 0.0, -5.0, float("inf"), float("nan")):
        refused("InvalidRopeTheta", rope_theta=theta)
    for eps in (0.0, -1e-6, float("inf"), float("nan")):
        refused("InvalidEpsilon", norm_eps=eps)
    refused("UnsupportedHeadDimension", head_dim=64)
    refused("UnsupportedPageSize", kv_page_size=48)


def test_read_spec(L):
    s = L.PagedKvReadSpec(2, 100, 7, 3, kv_page_size=32)
    assert (s.nnz_kv, s.output_numel) == (100, 100 * 3 * 128)
    assert s.kv_pages_numel == 7 * 32 * 3 * 64
    for dtype in ("bf16", "fp8_e4m3"):
        with pytest.raises(L.PlanError) as e:
            L.PagedKvReadSpec(2, 100, 7, 3, kv_dtype=dtype)
        assert (e.value.variant, e.value.operand) == ("InvalidOption", "kv_dtype")
    for n, variant in ((0, "ZeroDimension"), (2 ** 31, "ElementCountOverflow")):
        with pytest.raises(L.ContractError) as e:
            L.PagedKvReadSpec(2, n, 7, 3)
        assert e.value.variant == variant


def test_null_arguments(L):
    err = L._ffi.Error()
    lib = L.lib()
    for fn, args in ((lib.loom_norm_rope_append_spec_new, (None, 1, 1, 1e4, 0.0, None)),
                     (lib.loom_paged_kv_read_spec_new, (None, 1, None)),
                     (lib.loom_rope_provider_plan_norm_paged_append, (None, None, 0, None)),
                     (lib.loom_prefill_provider_plan_paged_kv_read, (None, None, 0, None)),
                     (lib.loom_paged_decode_enqueue_mxfp4, (None, None, None)),
                     (lib.loom_norm_rope_append_enqueue, (None, None, None)),
                     (lib.loom_paged_kv_read_enqueue, (None, None, None))):
        assert fn(*args, C.byref(err)) == 59, fn.__name__
        assert fn(*args, None) == 59


def test_quantiser_of_the_tests():
    """Every code comes back as itself, and codes are the nearest of all sixteen."""
    v = np.tile(mx.GRID, 16)
    codes, scales = mx.quantise(v)
    assert np.array_equal(mx.values(codes, scales), v) and (scales == 127).all()
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)) * np.exp(rng.standard_normal((50, 1)) * 10)
    got = mx.values(*mx.quantise(x)).reshape(-1, 32)
    b = x.reshape(-1, 32)
    e = np.floor(np.log2(np.abs(b).max(1))) - 2
    grid = np.concatenate([mx.GRID, -mx.GRID])
    every = np.abs(b[:, :, None] - grid * (2.0 ** e)[:, None, None]).min(-1)
    assert np.array_equal(np.abs(b - got), every)


def test_bf16_rounding_of_the_tests():
    import torch
    rng = np.random.default_rng(1)
    x = rng.standard_normal(10000) * np.exp2(rng.uniform(-140, 127, 10000))
    want = torch.from_numpy(x.astype(np.float32)).to(torch.bfloat16).double().numpy()
    assert np.array_equal(mx.bf16_round(x.astype(np.float32).astype(np.float64)), want)
    assert np.array_equal(mx.bf16_values(mx.bf16_bits(want)), want)


def test_kernels_keep_out_of_scratch_memory(tmp_path):
    """An array, or the argument struct, that a kernel indexes with a choice between two
    fields would live in scratch memory: twice the time of a small append."""
    from test_kernel_lds import LIB, READELF, code_objects
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    seen = 0
    for i, image in enumerate(code_objects(open(LIB, "rb").read())):
        path = tmp_path / f"{i}.elf"
        path.write_bytes(image)
        notes = subprocess.run([READELF, "--notes", str(path)], check=True, capture_output=True,
                               text=True).stdout
        for k in re.split(r"^\s+- \.agpr_count", notes, flags=re.M)[1:]:
            name = re.search(r"^ {4}\.name:\s+(\S+)", k, flags=re.M).group(1)
            if re.search("mx4_decode|append|kv_read", name):
                seen += 1
                assert re.search(r"\.private_segment_fixed_size:\s+0$", k, flags=re.M), name
    assert seen > 20
