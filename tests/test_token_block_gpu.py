"""The token operators as one run: group norm -> 8-bit projections -> attention of row bands over their image's pooled tokens -> 8-bit
projection, each stage against its definition on the stage before, eagerly and as a replayed graph; and shared-prefix attention against
sparse_window_attention, whose masked windows are such a batch (pooled tokens = prefix, own and rolled tokens = suffix)."""
import pytest
import torch

from tests import test_group_norm_gpu as gn
from tests import test_linear_i8_gpu as li
from tests import test_prefix_attention_gpu as pa

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from propainter_amd import hip as h
    h.lib()
    return h


class Block:
    """C channels in `heads` heads of 64; bands of `band` rows attend to themselves and to the 4x4-pooled tokens of their image"""

    def __init__(self, hip, C, heads, band, seed=0):
        from propainter_amd import conv
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
        self.hip, self.C, self.heads, self.band = hip, C, heads, band
        self.gamma, self.beta = (1 + 0.1 * r(C)).cuda(), (0.1 * r(C)).cuda()
        self.qkv = conv.Int8Linear(r(3 * C, C) / C ** 0.5, 0.1 * r(3 * C))
        self.proj = conv.Int8Linear(r(C, C) / C ** 0.5, 0.1 * r(C))
        self.pool_w, self.pool_b = torch.full((C, 4, 4), 1 / 16, device="cuda"), torch.zeros(C, device="cuda")

    def __call__(self, x):
        """every stage's output, in order"""
        hip, C = self.hip, self.C
        N, H, W, _ = x.shape
        y = hip.group_norm(x, 8, self.gamma, self.beta, act=hip.ACT_SILU)
        pooled = hip.depthwise_pool(y, self.pool_w, self.pool_b).view(N, -1, C)
        codes, scale = hip.quantize_tokens(y)
        t = self.qkv.product(codes, scale).view(N * H // self.band, self.band * W, 3, self.heads, 64)
        s = self.qkv(pooled).view(N, -1, 3, self.heads, 64)
        a = hip.shared_prefix_attention(t[:, :, 0], s[:, :, 1], s[:, :, 2], t[:, :, 1], t[:, :, 2])
        z = self.proj(a.view(N, H, W, C), out_dtype=torch.float32)
        return y, pooled, codes, scale, t, s, a, z


@pytest.mark.parametrize("N,H,W,C,band", [(2, 12, 20, 128, 4), (3, 8, 9, 64, 2), (1, 16, 12, 192, 16), (5, 4, 4, 64, 1)])
def test_block(hip, N, H, W, C, band):
    heads = C // 64
    block = Block(hip, C, heads, band)
    x = gn.make((N, H, W, C), torch.float16, 1)[0]
    y, pooled, codes, scale, t, s, a, z = block(x)
    gn.check(y, *gn.reference(x, 8, block.gamma, block.beta, 1e-5, "silu"))
    wq, ws = li.codes64(y.view(-1, C))
    assert torch.equal(codes[:, :C], wq) and torch.equal(scale, ws)
    plain = {"qkv": (block.qkv, y.view(-1, C), t.reshape(-1, 3 * C)), "pooled": (block.qkv, pooled.reshape(-1, C), s.reshape(-1, 3 * C)), "proj": (block.proj, a.view(-1, C), z.view(-1, C))}
    g = torch.Generator().manual_seed(0)
    r = lambda *q: torch.randn(q, generator=g)  # noqa: E731
    r(C), r(C)
    weights = {}
    for name, n in (("qkv", 3 * C), ("proj", C)):
        w = (r(n, C) / C ** 0.5).cuda()
        weights[name] = (*li.codes64(w), (0.1 * r(n)).cuda())
    for name, (layer, src, got) in plain.items():
        wc, wsc, b = weights["proj" if name == "proj" else "qkv"]
        q, sc = li.codes64(src)
        li.check(got, *li.reference(q, sc, wc, wsc, b, "none"))
    P, S, B = s.shape[1], t.shape[1], t.shape[0]
    ref, bound = pa.reference({"q": t[:, :, 0], "pk": s[:, :, 1], "pv": s[:, :, 2], "k": t[:, :, 1], "v": t[:, :, 2]}, [P] * N, [S] * B, False, 0.125)
    pa.check(a, ref, bound)

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        block(x)
        with torch.cuda.graph(graph, stream=stream):
            kept = block(x)
    stream.synchronize()
    for i in range(3):
        x.copy_(gn.make((N, H, W, C), torch.float16, 2 + i)[0])
        want = block(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(k, w) for k, w in zip(kept, want)), i


@pytest.mark.parametrize("T,tind", [(3, [0, 2]), (2, [0, 1])])
def test_masked_windows_are_a_batch_behind_their_pooled_tokens(hip, T, tind):
    Hp, Wp, C, heads, P = 10, 18, 512, 4, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((1, T, Hp, Wp, C), generator=g, device="cuda").half() for _ in range(3))
    pk, pv = (torch.randn((1, T, P, C), generator=g, device="cuda").half() for _ in range(2))
    own, rolled = (torch.from_numpy(t).cuda() for t in hip.window_tables(Hp, Wp))
    nW = own.shape[0]
    ti = torch.tensor(tind, dtype=torch.int32, device="cuda")
    want = hip.sparse_window_attention(q, k, v, pk, pv, own, rolled, ti, torch.ones((1, nW), device="cuda"), heads=heads).view(T, Hp * Wp, heads, 128)
    flat = lambda t: t.view(T, Hp * Wp, heads, 128)  # noqa: E731
    rows = torch.cat([own, rolled], 1).long()                                             # [nW, 193]
    qs = flat(q)[:, own.long()].permute(1, 0, 2, 3, 4).reshape(nW, T * 45, heads, 128)
    ks, vs = (flat(t)[tind][:, rows].permute(1, 0, 2, 3, 4).reshape(nW, -1, heads, 128) for t in (k, v))
    ps, us = (t[0, tind].reshape(1, -1, heads, 128) for t in (pk, pv))
    got = hip.shared_prefix_attention(qs, ps, us, ks, vs)
    ref, bound = pa.reference({"q": qs, "pk": ps, "pv": us, "k": ks, "v": vs}, [ps.shape[1]], [ks.shape[1]] * nW, False, 128 ** -0.5)
    pa.check(got, ref, bound)
    there = want[:, own.long()].permute(1, 0, 2, 3, 4).reshape(nW, T * 45, heads, 128)
    pa.check(there, ref, bound)


def test_outputs_over_inputs_are_refused(hip):
    from propainter_amd import conv
    x = torch.randn(64, 256, device="cuda", dtype=torch.float16)
    layer = conv.Int8Linear(torch.randn(128, 256), None)
    with pytest.raises(ValueError, match="overlaps"):
        layer(x, out=x)
    with pytest.raises(ValueError, match="overlaps"):
        layer(x[:1], out=x[:1, 64:])
    both = torch.randn(64, 384, device="cuda", dtype=torch.float16)      # side by side in one buffer
    want = layer(both[:, :256].clone())
    layer(both[:, :256], out=both[:, 256:])
    assert torch.equal(both[:, 256:], want)
    with pytest.raises(ValueError, match="overlaps"):
        layer(both[:, :256], out=both[:, 248:])
    for bad in (torch.empty(64, device="cuda", dtype=torch.float16), torch.empty(63, 128, device="cuda", dtype=torch.float16)):
        with pytest.raises(ValueError, match="out must be"):
            layer(x, out=bad)
    q = torch.randn(2, 3, 2, 64, device="cuda", dtype=torch.float16)
    kv = torch.randn(2, 2, 5, 2, 64, device="cuda", dtype=torch.float16)
    for out in (q, kv[0][:, :3]):
        with pytest.raises(ValueError, match="overlaps"):
            hip.shared_prefix_attention(q, None, None, kv[0], kv[1], out=out)
    m = torch.randn(5, 6, 6, 16, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="overlaps"):
        hip.group_norm(m[:4], 4, out=m[1:])
