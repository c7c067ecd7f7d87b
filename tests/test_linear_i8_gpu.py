"""hip.quantize_tokens and conv.Int8Linear against their definitions.

Codes are whole numbers and have to be equal; a scale is one rounded quotient.  A product's sum is exact: its conversion, the two scales and
the bias are four roundings to fp32, so an output is within 4 * 2^-24 of |product| + |bias|, an activation within 1.13 times that plus 16
steps of its own, and the output's rounding adds half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from propainter_amd import hip as h
    h.lib()
    return h


@pytest.fixture(scope="module")
def conv(hip):
    from propainter_amd import conv as c
    return c


def codes64(x):
    """codes by the definition: the real quotient by the fp32 scale, ties to even"""
    s = (x.double().abs().amax(1) / 127).float()
    q = torch.round(x.double() / torch.where(s > 0, s, torch.ones_like(s)).double()[:, None])
    return q.clamp(-127, 127).to(torch.int8), s


def rand(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda") * torch.exp(torch.randn((shape[0], 1), generator=g, device="cuda"))
    return x.to(dtype)


def check_codes(hip, x):
    q, s = hip.quantize_tokens(x)
    K = x.shape[-1]
    wq, ws = codes64(x.reshape(-1, K))
    assert q.shape == (wq.shape[0], (K + 63) // 64 * 64) and q.dtype == torch.int8 and s.dtype == torch.float32
    assert torch.equal(s, ws), (s - ws).abs().max()
    assert torch.equal(q[:, :K], wq), (q[:, :K] != wq).sum()
    assert not q[:, K:].any()
    return q, s


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 5), (45, 512), (7, 1000), (64, 1024), (5, 1025), (130, 1960), (9, 2048), (3, 2056), (6, 4096), (2, 5001), (3, 8192), (2, 16384),
                                    (2, 16392), (1, 20003), (1, 131072), (1000, 8), (3, 61), (66000, 16), (700, 1023), (300, 4099), (9, 3), (33, 16390)])
def test_codes(hip, rows, K, dtype):
    check_codes(hip, rand((rows, K), dtype, rows + K))


def test_ties_go_to_even_codes(hip):
    """scale 1: quotients at and next to every half; scale 3: the quotient by the reciprocal misses ties"""
    for s in (1.0, 3.0, 0.7):
        n = torch.arange(-126, 127, device="cuda", dtype=torch.float64)
        ties = ((n + 0.5) * float(torch.tensor(s))).float()
        x = torch.cat([torch.tensor([127.0 * s], device="cuda"), ties, torch.nextafter(ties, ties + 1), torch.nextafter(ties, ties - 1), (n * s).float()])[None]
        check_codes(hip, x)
    x = torch.cat([torch.tensor([127.0], device="cuda"), torch.arange(-126.5, 127, 1.0, device="cuda")])[None]
    q, s = hip.quantize_tokens(x)
    assert s.item() == 1.0 and (q[0, 1:x.shape[1]] % 2 == 0).all()


def test_rows_of_zeros_tiny_and_huge_values(hip):
    for v in (1e-45, 1e-44, 3e-43, 1e-40, 1.1754944e-38, 1e-30, 1e30, 3.4028235e38):
        x = torch.tensor([[v, -v, v / 2, v / 3, 0.0, -v / 5]], device="cuda")
        check_codes(hip, x)
    q, s = check_codes(hip, torch.zeros((3, 70), device="cuda", dtype=torch.float16))
    assert not q.any() and not s.any()
    check_codes(hip, torch.tensor([[6e-8, -6e-8, 0.0, 1.2e-7], [65504.0, -1.0, 300.0, 258.0]], device="cuda", dtype=torch.float16))


@pytest.mark.parametrize("K", [70, 512, 3000])
def test_rows_that_are_not_finite_have_no_scale(hip, K):
    x = rand((5, K), torch.float16, 3)
    good_q, good_s = hip.quantize_tokens(x)
    x[1, K - 1] = float("nan")
    x[3, 0] = float("-inf")
    q, s = hip.quantize_tokens(x)
    assert torch.isnan(s[[1, 3]]).all() and not q[[1, 3]].any()
    assert torch.equal(q[[0, 2, 4]], good_q[[0, 2, 4]]) and torch.equal(s[[0, 2, 4]], good_s[[0, 2, 4]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_of_a_wider_buffer(hip, dtype):
    buf = rand((33, 1003), dtype, 4)
    for a, b in ((0, 512), (8, 520), (3, 515), (1, 1003)):
        check_codes(hip, buf[:, a:b])
    check_codes(hip, buf[0, 5:100])
    check_codes(hip, rand((24, 96), dtype, 5).view(2, 3, 4, 96))
    assert hip.quantize_tokens(buf[:0])[0].shape == (0, 1024)
    check_codes(hip, buf[1:2].expand(4, 1003))


def act64(y, act):
    return {"none": lambda: y, "relu": lambda: y.clamp_min(0), "lrelu": lambda: torch.where(y < 0, y * 0.2, y), "sigmoid": lambda: torch.sigmoid(y),
            "tanh": lambda: torch.tanh(y), "gelu": lambda: y * torch.special.ndtr(y), "silu": lambda: y * torch.sigmoid(y)}[act]()


def reference(q, s, wq, ws, bias, act):
    p = (q.double() @ wq.double().t()) * s.double()[:, None] * ws.double()[None, :]
    b = bias.double() if bias is not None else torch.zeros_like(ws).double()
    y = act64(p + b, act)
    bound = 4 * 2.0 ** -24 * (p.abs() + b.abs())
    return y, bound if act == "none" else 1.13 * bound + 16 * 2.0 ** -24 * (1 + y.abs())


def check(got, ref, bound):
    err = (got.double() - ref).abs()
    lim = bound + torch.finfo(got.dtype).eps / 2 * ref.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    worst = (err / lim).max().item()
    assert torch.isfinite(got).all() and worst <= 1, f"error {worst:.3f} times its bound (max {err.max().item():.3e})"


def layer_of(conv, N, K, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wq = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    ws = (0.5 + torch.rand(N, generator=g, device="cuda")) / (64 * K ** 0.5)
    b = torch.randn(N, generator=g, device="cuda") if bias else None
    return conv.Int8Linear.from_codes(wq, ws, b), wq, ws, b


SIZES = [(1, 1, 1), (1, 64, 64), (1, 4096, 512), (2, 100, 30), (3, 1960, 512), (5, 512, 17), (16, 512, 1536), (17, 640, 100), (31, 65, 64), (32, 256, 257), (45, 512, 1536),
         (64, 1000, 65), (65, 128, 48), (100, 192, 1000), (127, 512, 130), (129, 320, 200), (200, 2048, 384), (256, 256, 256), (257, 300, 511), (333, 4100, 72), (513, 576, 640),
         (1025, 64, 24), (2500, 200, 264), (3400, 330, 450), (900, 70, 2000), (70, 1000, 12000), (300, 16384, 16), (20, 130, 9000), (1100, 1000, 1030)]
# weights kept in registers (K <= 256, K <= 512, odd channel blocks), 128 x 256 tiles, 256 x 256 tiles
LARGE = [(49200, 200, 200), (17000, 500, 1000), (50000, 65, 70), (25001, 512, 520), (4200, 600, 2100), (8200, 1960, 770), (8100, 6200, 4100)]


@pytest.mark.parametrize("odt", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(hip, conv, M, K, N, odt):
    layer, wq, ws, b = layer_of(conv, N, K, M + K + N)
    q, s = hip.quantize_tokens(rand((M, K), torch.float16, M))
    got = layer.product(q, s, out_dtype=odt)
    assert got.shape == (M, N) and got.dtype == odt
    check(got, *reference(q[:, :K], s, wq, ws, b, "none"))
    assert torch.equal(got, layer.product(q, s, out_dtype=odt)), "two runs differ"


@pytest.mark.parametrize("M,K,N", LARGE)
def test_large_products(hip, conv, M, K, N):
    layer, wq, ws, b = layer_of(conv, N, K, M + K + N)
    q, s = hip.quantize_tokens(rand((M, K), torch.float16, M))
    for odt in (torch.float16, torch.float32):
        got = layer.product(q, s, act="relu", out_dtype=odt)
        for a in range(0, M, 8192):
            check(got[a:a + 8192], *reference(q[a:a + 8192, :K], s[a:a + 8192], wq, ws, b, "relu"))


@pytest.mark.parametrize("dtype,odt", [(torch.float16, torch.float16), (torch.float32, torch.float16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("M,K,N", [(1, 512, 100), (2, 1030, 512), (1, 4097, 70), (2, 4096, 33), (1, 8192, 64), (3, 64, 64), (4, 4096, 70), (16, 1024, 40), (1, 16384, 70), (1, 16383, 64), (15, 1000, 33), (16, 1025, 64), (5, 7, 3), (7, 4096, 192), (16, 100, 65), (45, 512, 1536), (700, 1960, 136), (1, 20000, 32), (900, 253, 787), (40, 1021, 35), (17, 512, 1536), (33, 2188, 70), (100, 64, 100), (23, 9000, 30),
                                   (400, 300, 20), (16, 512, 17000), (1000, 65, 64), (9, 16384, 20)])
def test_layer_on_float_tokens(hip, conv, M, K, N, dtype, odt):
    layer, wq, ws, b = layer_of(conv, N, K, 5)
    x = rand((M, K), dtype, 6)
    got = layer(x, out_dtype=odt)
    q, s = codes64(x)
    check(got, *reference(q, s, wq, ws, b, "none"))
    y = x.clone()
    y[M // 2, K - 1] = float("inf")
    got2 = layer(y, out_dtype=odt)
    assert torch.isnan(got2[M // 2]).all() and torch.equal(got2[:M // 2], got[:M // 2]) and torch.equal(got2[M // 2 + 1:], got[M // 2 + 1:])


@pytest.mark.parametrize("act", ["none", "relu", "lrelu", "sigmoid", "tanh", "gelu", "silu"])
@pytest.mark.parametrize("M", [1, 20, 300])
def test_activations_and_no_bias(hip, conv, M, act):
    for bias in (True, False):
        layer, wq, ws, b = layer_of(conv, 130, 256, 7, bias)
        q, s = hip.quantize_tokens(rand((M, 256), torch.float16, 8))
        for odt in (torch.float32, torch.float16):
            check(layer.product(q, s, act=act, act_param=0.2, out_dtype=odt), *reference(q, s, wq, ws, b, act))


def test_extreme_codes_do_not_overflow(hip, conv):
    K = 131072
    wq = torch.full((3, K), -127, dtype=torch.int8, device="cuda")
    wq[1] = 127
    layer = conv.Int8Linear.from_codes(wq, torch.ones(3, device="cuda"))
    for M in (1, 40, 260):
        q = torch.full((M, K), 127, dtype=torch.int8, device="cuda")
        got = layer.product(q, torch.ones(M, device="cuda"), out_dtype=torch.float32)
        want = 127.0 * 127.0 * K
        assert (got[:, 1].double() - want).abs().max() <= want * 2.0 ** -24 and torch.equal(got[:, 0], -got[:, 1])


@pytest.mark.parametrize("M", [1, 9, 200])
def test_output_windows(hip, conv, M):
    layer, wq, ws, b = layer_of(conv, 72, 128, 9)
    q, s = hip.quantize_tokens(rand((M, 128), torch.float16, 10))
    want = layer.product(q, s)
    for width, off in ((72, 0), (200, 64), (200, 3), (101, 8)):
        out = torch.full((M, width), 5.0, dtype=torch.float16, device="cuda")
        r = layer.product(q, s, out=out[:, off:off + 72])
        assert torch.equal(out[:, off:off + 72], want) and (out[:, :off] == 5).all() and (out[:, off + 72:] == 5).all() and r.data_ptr() == out[:, off:].data_ptr()


def test_weights_are_quantised_as_tokens_are(hip, conv):
    w = rand((130, 300), torch.float32, 11).cpu()
    bias = torch.randn(130)
    layer = conv.Int8Linear(w, bias)
    wq, ws = codes64(w.cuda())
    x = rand((2, 3 * 300), torch.float16, 12).view(2, 3, 300)
    got = layer(x, act="gelu")
    assert got.shape == (2, 3, 130) and got.dtype == torch.float16
    q, s = codes64(x.reshape(6, 300))
    check(got.view(6, 130), *reference(q, s, wq, ws, bias.cuda(), "gelu"))
    assert layer(x[:0]).shape == (0, 3, 130)


def test_another_stream_and_two_graphs(hip, conv):
    """graphs of a single token and of many tokens, replayed in turn with eager calls in between"""
    layer, wq, ws, b = layer_of(conv, 192, 640, 13)
    xs = [rand((1, 640), torch.float16, 14), rand((150, 640), torch.float16, 15)]
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs, kept = [], []
    with torch.cuda.stream(s):
        for x, w in zip(xs, want):
            assert torch.equal(layer(x), w)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                kept.append(layer(x))
            graphs.append(g)
    s.synchronize()
    for i in range(3):
        for x in xs:
            x.copy_(rand(tuple(x.shape), torch.float16, 20 + i))
        want = [layer(x) for x in xs]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(k, w) for k, w in zip(kept, want)), i
