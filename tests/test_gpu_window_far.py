"""Window attention at far positions: contexts of 2^30 tokens and more, whose pages behind
the window are given away.  A row sees the same tokens as in a short context with the same
pages at either end, so the short one's definition is the long one's (tolerances:
window_util)."""
import pytest

from window_util import Case

pytestmark = pytest.mark.gpu
DTYPES = ["bf16", "fp8_e4m3", "mxfp4"]
FORMS = {"one row": (None, 0), "rows": ([7], 16), "rows, long tile": ([7], "long")}


@pytest.fixture(scope="module")
def env():
    import torch
    import loom_infer_hip as L
    return torch, L


def check(env, c, form, length):
    """Case `c`'s single request, made `length` tokens long by pages between its sinks and
    its windows that nobody holds."""
    torch, L = env
    n, page = c.lens[0], c.page
    gap, rest = divmod(length - n, page)
    assert rest == 0 and gap > 0
    held = -(-c.sinks // page)  # the sinks' pages
    assert n - c.rows[0] + 1 - c.window >= held * page
    d = c.operands(torch)
    far = torch.full((gap,), -1, dtype=torch.int32, device="cuda")
    d["indices"] = torch.cat([d["indices"][:held], far, d["indices"][held:]])
    d["indptr"][1] = d["indices"].numel()
    tile = FORMS[form][1]
    plan = {} if c.single else dict(tile_cols=tile)
    c.check(*c.run(torch, L, d, **plan), long_tile=tile == "long")


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(70, 0), (100, 4), (1000, 17)])
@pytest.mark.parametrize("length", [(1 << 30) + 37, (1 << 30) + 64 * 40 + 5, (1 << 31) - 64])
def test_positions_past_2_30(env, length, window, sinks, dtype, form):
    """Windows over token 2^30, past it, and up to the last page of 64 rows that 31 bits
    count."""
    c = Case(61, [64 * 20 + length % 64], FORMS[form][0], 8, 2, window, sinks, 64, "HND", dtype)
    check(env, c, form, length)


@pytest.mark.parametrize("form", ["one row", "rows", "rows, long tile"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sinks", [0, 4, 17])
def test_the_last_position(env, sinks, dtype, form):
    """The last token that a table of 16-row pages holds, walks of an odd number of blocks
    and of an even one: behind the last block a pair's second half would begin at
    2^31 - 16 and end at 2^31."""
    c = Case(62, [16 * 9], FORMS[form][0] and [1], 8, 2, 40, sinks, 16, "NHD", dtype)
    check(env, c, form, (1 << 31) - 16)
