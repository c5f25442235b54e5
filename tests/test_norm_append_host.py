"""CPU tests of the normed append's contract."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def L():
    import loom_infer_hip as L
    L.lib()
    return L


def spec(L, eps):
    return L.NormRopePagedKvAppendSpec(5, 2, 7, 8, 2, norm_eps=eps)


@pytest.mark.parametrize("eps", [1e-46, 1e-50, 5e-324, np.float64(1e-60)])
def test_epsilons_that_fp32_takes_for_zero_are_refused(L, eps):
    """A 32-bit 0 means "no norms": such an epsilon would leave the heads unnormed."""
    with pytest.raises(L.ContractError) as e:
        spec(L, eps)
    assert e.value.variant == "InvalidEpsilon"


@pytest.mark.parametrize("eps", [1e-45, 1e-38, 1e-12, 1.0])
def test_the_smallest_epsilons_norm(L, eps):
    assert spec(L, eps).norm_eps == np.float32(eps) > 0


def test_no_epsilon_means_no_norms(L):
    assert spec(L, None).norm_eps is None
