"""hip.group_norm against its definition in 64 bits.

Bound per element: half a step of the output type, plus the fp32 arithmetic.  A sum is a chain of at most `chain` additions in a thread and a
tree of a few dozen joins, so mean and variance are off by at most (chain + 64) 2^-24 of the deviations they sum; x - mean is rounded
relative to the larger of the two; the activations change at most 1.13 times as fast as their argument and are evaluated to 16 steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "lrelu", "sigmoid", "tanh", "gelu", "silu"]


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from propainter_amd import hip as h
    h.lib()
    return h


def act64(y, act):
    return {"none": lambda: y, "relu": lambda: y.clamp_min(0), "lrelu": lambda: torch.where(y < 0, y * 0.1, y), "sigmoid": lambda: torch.sigmoid(y),
            "tanh": lambda: torch.tanh(y), "gelu": lambda: y * torch.special.ndtr(y), "silu": lambda: y * torch.sigmoid(y)}[act]()


def reference(x, groups, gamma, beta, eps, act):
    """(y, bound of its error without the output's own rounding) in 64 bits"""
    N, H, W, C = x.shape
    v = x.double().reshape(N, H * W, groups, C // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdim=True)
    xhat = (v - mean) / torch.sqrt(var + eps)
    g = gamma.double() if gamma is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    b = beta.double() if beta is not None else torch.zeros(C, dtype=torch.float64, device=x.device)
    z = xhat.reshape(N, H, W, C) * g + b
    far = (mean.abs() / torch.sqrt(var + eps)).expand(N, H * W, groups, C // groups).reshape(N, H, W, C)
    chain = H * W / max(1, 256 // (C // 8)) + 64
    bound = 2.0 ** -24 * ((chain + 8) * (1 + xhat.reshape(N, H, W, C).abs()) * g.abs() + 4 * far * g.abs() + 4 * b.abs())
    y = act64(z, act)
    return y, 1.13 * bound + 16 * 2.0 ** -24 * (1 + y.abs())


def check(got, ref, bound):
    err = (got.double() - ref).abs()
    lim = bound + torch.finfo(got.dtype).eps / 2 * ref.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    worst = (err / lim).max().item()
    assert torch.isfinite(got).all() and worst <= 1, f"error {worst:.3f} times its bound (max {err.max().item():.3e})"


def make(shape, dtype, seed=0, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, H, W, C = shape
    x = torch.randn(shape, generator=g, device="cuda") * (0.5 + torch.rand(C, generator=g, device="cuda")) + shift * torch.randn(C, generator=g, device="cuda")
    return x.to(dtype), 1 + 0.2 * torch.randn(C, generator=g, device="cuda"), 0.2 * torch.randn(C, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("shape,groups", [((1, 1, 1, 8), 1), ((2, 1, 1, 64), 8), ((1, 5, 7, 24), 8), ((3, 9, 13, 40), 5), ((2, 30, 54, 128), 8), ((1, 33, 65, 96), 8),
                                          ((2, 17, 31, 64), 64), ((1, 3, 129, 640), 32), ((2, 6, 10, 2048), 2048), ((1, 7, 5, 2040), 3), ((1, 200, 190, 16), 2),
                                          ((5, 61, 67, 72), 1), ((2, 300, 301, 8), 8), ((1, 90, 160, 256), 16), ((300, 4, 4, 32), 4), ((2, 36, 126, 600), 1), ((1, 20, 130, 2048), 2),
                                          ((3, 50, 40, 1024), 4)])
def test_shapes(hip, shape, groups, dtype):
    x, gamma, beta = make(shape, dtype)
    got = hip.group_norm(x, groups, gamma, beta, act=hip.ACT_RELU)
    check(got, *reference(x, groups, gamma, beta, 1e-5, "relu"))
    assert torch.equal(got, hip.group_norm(x, groups, gamma, beta, act=hip.ACT_RELU)), "two runs differ"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((2, 11, 9, 48), 6), ((1, 150, 140, 48), 4)])
def test_activations_and_missing_parameters(hip, shape, groups, act, dtype):
    x, gamma, beta = make(shape, dtype, 1)
    code = getattr(hip, "ACT_" + act.upper())
    for gm, bt in ((gamma, beta), (None, beta), (gamma, None), (None, None)):
        got = hip.group_norm(x, groups, gm, bt, eps=1e-3, act=code, act_param=0.1)
        check(got, *reference(x, groups, gm, bt, 1e-3, act))


@pytest.mark.parametrize("shape,groups", [((2, 9, 7, 32), 4), ((1, 160, 130, 24), 3)])
def test_a_mean_far_from_zero_keeps_the_variance(hip, shape, groups):
    x, gamma, beta = make(shape, torch.float32, 2)
    x = x + 1000.0
    check(hip.group_norm(x, groups, gamma, beta), *reference(x, groups, gamma, beta, 1e-5, "none"))


def test_constant_groups_and_zero_eps(hip):
    x = torch.full((2, 5, 6, 16), 3.25, device="cuda")
    beta = torch.arange(16, device="cuda").float()
    got = hip.group_norm(x, 2, None, beta)
    assert torch.equal(got, beta.expand(2, 5, 6, 16))
    y, _, _ = make((1, 8, 8, 16), torch.float32, 3)
    check(hip.group_norm(y, 2, None, beta, eps=0.0), *reference(y, 2, None, beta, 0.0, "none"))


@pytest.mark.parametrize("H,W", [(6, 7), (120, 200)])
def test_nan_and_infinity_stay_in_their_group(hip, H, W):
    x, gamma, beta = make((2, H, W, 32), torch.float16, 4)
    clean = hip.group_norm(x, 4, gamma, beta, act=hip.ACT_RELU)
    bad = x.clone()
    bad[1, 3, 2, 9] = float("nan")
    bad[0, 0, 0, 31] = float("inf")
    got = hip.group_norm(bad, 4, gamma, beta, act=hip.ACT_RELU)
    assert torch.isnan(got[1, :, :, 8:16]).all() and torch.isnan(got[0, :, :, 24:]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[1, :, :, 8:16] = False
    keep[0, :, :, 24:] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("H,W", [(9, 6), (130, 170)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_channel_windows_and_in_place(hip, H, W, dtype):
    x, gamma, beta = make((2, H, W, 40), dtype, 5)
    wide = torch.full((2, H, W, 72), 7.0, dtype=dtype, device="cuda")
    wide[..., 16:56] = x
    want = hip.group_norm(x, 5, gamma, beta, act=hip.ACT_SILU)
    out = torch.full((2, H, W, 64), -3.0, dtype=dtype, device="cuda")
    r = hip.group_norm(wide, 5, gamma, beta, act=hip.ACT_SILU, out=out, x_choff=16, C_=40, out_choff=8)
    assert r is out and torch.equal(out[..., 8:48], want)
    assert (out[..., :8] == -3).all() and (out[..., 48:] == -3).all() and (wide[..., :16] == 7).all() and (wide[..., 56:] == 7).all()
    hip.group_norm(wide, 5, gamma, beta, act=hip.ACT_SILU, out=wide, x_choff=16, C_=40, out_choff=16)
    assert torch.equal(wide[..., 16:56], want) and (wide[..., :16] == 7).all() and (wide[..., 56:] == 7).all()
    with pytest.raises(ValueError):
        hip.group_norm(wide, 5, gamma, beta, out=wide, x_choff=16, C_=40, out_choff=24)


def test_an_image_does_not_depend_on_the_others(hip):
    x, gamma, beta = make((3, 40, 50, 64), torch.float16, 6)
    y = hip.group_norm(x, 8, gamma, beta)
    alone = hip.group_norm(x[1:2].contiguous(), 8, gamma, beta)
    check(alone, *reference(x[1:2], 8, gamma, beta, 1e-5, "none"))
    check(y, *reference(x, 8, gamma, beta, 1e-5, "none"))
    assert hip.group_norm(x[:0].contiguous(), 8, gamma, beta).shape == (0, 40, 50, 64)


def test_offsets_past_32_bits(hip):
    """the second image of a wide buffer starts behind 2^31 elements"""
    x = torch.zeros((2, 1024, 1056, 1024), dtype=torch.float16, device="cuda")
    small, gamma, beta = make((1, 1024, 1056, 8), torch.float16, 7)
    x[1, :, :, 1016:] = small[0]
    out = torch.empty((2, 1024, 1056, 8), dtype=torch.float16, device="cuda")
    hip.group_norm(x, 2, gamma, beta, out=out, x_choff=1016, C_=8)
    check(out[1:], *reference(small, 2, gamma, beta, 1e-5, "none"))
    del x


def test_another_stream_and_a_graph(hip):
    x, gamma, beta = make((2, 64, 72, 64), torch.float16, 8)
    want = hip.group_norm(x, 8, gamma, beta, act=hip.ACT_RELU)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = hip.group_norm(x, 8, gamma, beta, act=hip.ACT_RELU)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            kept = hip.group_norm(x, 8, gamma, beta, act=hip.ACT_RELU)
    s.synchronize()
    assert torch.equal(got, want)
    for i in range(3):
        x.copy_(make((2, 64, 72, 64), torch.float16, 9 + i)[0])
        want = hip.group_norm(x, 8, gamma, beta, act=hip.ACT_RELU)
        kept.fill_(-1)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want), i
