"""hip.group_norm on maps whose slices begin with pixels far from the rest: the deviations from a slice's first pixel are then large, and a variance
taken as a difference of their sums would be off by the slice's length times an fp32 step (8e-4 of the deviation at the first shape below).
Bounds as in test_group_norm_gpu.py: a chain of additions a thread, a tree of joins."""
import pytest
import torch

from tests.test_group_norm_gpu import check, hip, reference  # noqa: F401 (hip: the fixture)

pytestmark = pytest.mark.gpu


def normal(shape, mean, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") + mean).to(dtype)


@pytest.mark.parametrize("shape,groups,mean", [((600, 128, 128, 16), 2, 300.0), ((1100, 64, 64, 64), 8, 1000.0), ((1, 540, 960, 64), 8, 1000.0), ((2, 40, 33, 200), 5, 1000.0)])
def test_a_first_pixel_far_from_the_rest(hip, shape, groups, mean):  # noqa: F811
    x = normal(shape, mean)
    x[:, 0, 0] = 1.0
    got = hip.group_norm(x, groups)
    for i in range(0, shape[0], 200):
        check(got[i:i + 200], *reference(x[i:i + 200], groups, None, None, 1e-5, "none"))
    assert torch.equal(got, hip.group_norm(x, groups)), "two runs differ"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("shape,groups", [((3, 97, 131, 24), 3), ((1, 270, 480, 96), 8), ((700, 30, 41, 8), 1)])
def test_a_border_of_zeros(hip, shape, groups, dtype):  # noqa: F811
    x = normal(shape, 200.0, dtype, 1)
    x[:, 0], x[:, -1], x[:, :, 0], x[:, :, -1] = 0, 0, 0, 0
    gamma, beta = normal(shape[3:], 1.0, seed=2), normal(shape[3:], 0.0, seed=3)
    check(hip.group_norm(x, groups, gamma, beta, act=hip.ACT_RELU), *reference(x, groups, gamma, beta, 1e-5, "relu"))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_first_pixel_that_is_not_finite(hip, value):  # noqa: F811
    x = normal((2, 90, 70, 32), 0.0)
    x[1, 0, 0, 9] = value
    y = hip.group_norm(x, 4)
    assert y[1, ..., 8:16].isnan().all() and torch.isfinite(y[0]).all() and torch.isfinite(y[1, ..., :8]).all() and torch.isfinite(y[1, ..., 16:]).all()
