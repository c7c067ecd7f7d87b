"""hip.shared_prefix_attention against softmax attention in 64 bits.

Bound per output: a weight of the softmax is off by its own rounding (fp16 operands are multiplied by weights rounded to fp16: 2^-11 of the
weight, 2^-25 of the largest one below fp16's normal range), by the fp32 error of its score ((D + 8) 2^-24 of sum |q k| scale, twice: the
maximum's score counts too) and of the sum of the weights (at most keys + 64 additions); the outputs are weighted means of the values, so the
error is at most that share of the weighted mean of |v|; the output's rounding adds half a step of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from propainter_amd import hip as h
    h.lib()
    return h


def make(B, G, Lq, Hq, Hkv, D, P, S, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return {"q": (1.5 * r(B, Lq, Hq, D)).to(dtype), "pk": r(G, P, Hkv, D) if P else None, "pv": r(G, P, Hkv, D) if P else None,
            "k": r(B, S, Hkv, D) if S else None, "v": r(B, S, Hkv, D) if S else None}


def reference(t, plens, lens, causal, scale):
    """(output, bound without the output's rounding) in 64 bits, one sequence at a time"""
    q = t["q"]
    B, Lq, Hq, D = q.shape
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    G = t["pk"].shape[0] if t["pk"] is not None else 1
    for b in range(B):
        g = b // (B // G)
        ks, vs, np_, ns = [], [], 0, 0
        if t["pk"] is not None:
            np_ = plens[g]
            ks.append(t["pk"][g, :np_])
            vs.append(t["pv"][g, :np_])
        if t["k"] is not None:
            ns = lens[b]
            ks.append(t["k"][b, :ns])
            vs.append(t["v"][b, :ns])
        n = np_ + ns
        if n == 0:
            continue
        rep = Hq // ks[0].shape[1]
        k = torch.cat(ks).double().repeat_interleave(rep, 1).permute(1, 0, 2)        # [Hq, n, D]
        v = torch.cat(vs).double().repeat_interleave(rep, 1).permute(1, 0, 2)
        qb = q[b].double().permute(1, 0, 2)                                           # [Hq, Lq, D]
        s = (qb @ k.transpose(1, 2).contiguous()) * scale
        size = (qb.abs() @ k.abs().transpose(1, 2).contiguous()) * abs(scale)
        if causal:
            j = torch.arange(n, device=q.device)
            hide = (j[None, :] >= np_) & (j[None, :] - np_ > torch.arange(Lq, device=q.device)[:, None] + ns - Lq)
            s = s.masked_fill(hide[None], -math.inf)
        m = s.amax(2, keepdim=True)
        e = torch.exp(s - m.masked_fill(m == -math.inf, 0))
        total = e.sum(2, keepdim=True)
        a = e / total.masked_fill(total == 0, 1)
        o = a @ v
        rel = 2 * 2.0 ** -24 * ((D + 8) * size.amax(2, keepdim=True) + n + 64)
        bd = (a @ v.abs()) * rel
        if q.dtype == torch.float16:
            bd = bd + (a @ v.abs()) * 2.0 ** -11 + 2.0 ** -25 * ((s > -math.inf).double() @ v.abs()) / total.masked_fill(total == 0, 1)
        out[b], bound[b] = o.permute(1, 0, 2), bd.permute(1, 0, 2)
    return out, bound


def check(got, ref, bound):
    err = (got.double() - ref).abs()
    lim = bound + torch.finfo(got.dtype).eps / 2 * ref.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    worst = (err / lim).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1, f"error {worst:.3f} times its bound (max {err.max().item():.3e})"


def lens_of(n, most, seed):
    g = torch.Generator().manual_seed(seed)
    v = torch.randint(0, most + 1, (n,), generator=g)
    if n > 1:
        v[0], v[-1] = most, 0
    return v.to(torch.int32)


def run(hip, t, plens, lens, causal=False, scale=None, **kw):
    dev = t["q"].device
    return hip.shared_prefix_attention(t["q"], t["pk"], t["pv"], t["k"], t["v"], prefix_lens=None if plens is None else torch.tensor(plens, dtype=torch.int32, device=dev),
                                       lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev), causal=causal, scale=scale, **kw)


#        B  G  Lq  Hq Hkv D    P    S
CASES = [(1, 1, 1, 1, 1, 64, 1, 1), (1, 1, 1, 1, 1, 128, 0, 1), (1, 1, 1, 2, 1, 64, 1, 0), (3, 1, 1, 4, 4, 128, 405, 193), (2, 1, 1, 8, 2, 64, 63, 65), (5, 1, 1, 16, 2, 128, 128, 127),
         (4, 2, 1, 8, 8, 64, 129, 30), (6, 3, 2, 8, 1, 128, 300, 77), (8, 1, 4, 16, 2, 64, 1000, 200), (2, 2, 3, 6, 2, 128, 64, 64), (7, 1, 5, 3, 1, 64, 31, 33), (3, 1, 16, 4, 4, 128, 200, 100),
         (2, 1, 17, 4, 2, 128, 65, 129), (2, 1, 45, 4, 4, 128, 405, 193), (4, 1, 33, 8, 1, 64, 256, 40), (2, 1, 64, 2, 2, 128, 192, 64), (1, 1, 130, 2, 1, 128, 70, 300), (3, 1, 129, 1, 1, 64, 17, 5),
         (2, 1, 300, 2, 2, 128, 500, 700), (12, 1, 1, 32, 8, 128, 2100, 260), (1, 1, 1, 4, 1, 128, 5000, 1), (1, 1, 1, 32, 32, 128, 16, 3000), (40, 1, 1, 4, 4, 64, 700, 3), (2, 1, 1, 64, 1, 128, 33, 65),
         (2, 1, 200, 4, 1, 64, 1, 1), (9, 3, 20, 6, 3, 64, 130, 250)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", CASES, ids=[str(c) for c in CASES])
def test_ragged_batches(hip, size, causal, dtype):
    B, G, Lq, Hq, Hkv, D, P, S = size
    t = make(*size, dtype)
    plens, lens = lens_of(G, P, 1).tolist(), lens_of(B, S, 2).tolist()
    if G == 1:
        plens = [max(0, P - 1)] if P > 1 else [P]
    got = run(hip, t, plens, lens, causal)
    check(got, *reference(t, plens, lens, causal, D ** -0.5))
    assert torch.equal(got, run(hip, t, plens, lens, causal)), "two runs differ"
    full = run(hip, t, None, None, causal, scale=0.3)
    check(full, *reference(t, [P] * G, [S] * B, causal, 0.3))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,Lq,Hq,Hkv,P,S", [(3, 1, 4, 2, 100, 90), (2, 40, 4, 2, 100, 90), (2, 150, 2, 2, 70, 70), (20, 1, 8, 1, 900, 20)])
def test_what_lies_behind_the_lengths_is_not_used(hip, B, Lq, Hq, Hkv, P, S, dtype):
    t = make(B, 1, Lq, Hq, Hkv, 128, P, S, dtype, 3)
    plens, lens = [P - 33], [S - 1 - 17 * (i % 3) for i in range(B)]
    want = run(hip, t, plens, lens)
    for bad in (float("nan"), float("inf"), -float("inf")):
        u = {k: v.clone() for k, v in t.items()}
        u["pk"][0, plens[0]:] = bad
        u["pv"][0, plens[0]:] = bad
        for b in range(B):
            u["k"][b, lens[b]:] = bad
            u["v"][b, lens[b]:] = bad
        assert torch.equal(run(hip, u, plens, lens), want)
    assert torch.equal(run(hip, t, [P + 1000], [S + 5] * B), run(hip, t, None, None))
    assert not run(hip, t, [-3], [-1] * B).any()


@pytest.mark.parametrize("Lq", [1, 40, 140])
def test_a_causal_call_hides_later_keys(hip, Lq):
    """queries that see nothing of the suffix, values that are not finite behind the last visible key, and no prefix: rows without keys"""
    t = make(2, 1, Lq, 4, 2, 128, 80, 200, torch.float16, 4)
    lens = [max(1, Lq // 2), 200]
    want = run(hip, t, [80], lens, True)
    check(want, *reference(t, [80], lens, True, 128 ** -0.5))
    u = {k: v.clone() for k, v in t.items()}
    u["v"][0, lens[0] - 1] = float("nan")
    got = run(hip, u, [80], lens, True)
    assert torch.isnan(got[0, Lq - 1]).all() and torch.equal(got[1], want[1])
    nothing = run(hip, dict(t, pk=None, pv=None), None, lens, True)
    hidden = max(0, Lq - lens[0])
    assert not nothing[0, :hidden].any() and (nothing[0, hidden:].abs().sum(-1) > 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_large_scores_and_one_dominant_key(hip, dtype):
    for Lq in (1, 70):
        t = make(2, 1, Lq, 4, 4, 64, 100, 100, dtype, 5)
        t["q"] = t["q"] * 40
        check(run(hip, t, None, None), *reference(t, [100], [100] * 2, False, 64 ** -0.5))
        t["k"][:, 60] = t["k"][:, 60] * 30
        check(run(hip, t, None, None), *reference(t, [100], [100] * 2, False, 64 ** -0.5))
        check(run(hip, t, None, None, scale=-0.125), *reference(t, [100], [100] * 2, False, -0.125))
        z = run(hip, t, None, None, scale=0.0)
        mean = (t["pv"].double().sum(1) + t["v"].double().sum(1)) / 200
        assert (z.double() - mean[:, None]).abs().max() < (2e-3 if dtype == torch.float16 else 1e-5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("Lq,P,S", [(1, 150, 40), (30, 150, 40), (140, 90, 200)])
def test_strides_of_fused_and_transposed_buffers(hip, Lq, P, S, dtype):
    B, H, D = 3, 4, 64
    t = make(B, 1, Lq, H, H, D, P, S, dtype, 6)
    want = run(hip, t, [P], [S, S - 7, 1])
    u = dict(t)
    u["q"] = torch.cat([t["q"], t["q"], t["q"]], -1).view(B, Lq, H, 3 * D)[..., D:2 * D]
    fused = torch.empty(B, S, 3 * H * D, dtype=dtype, device="cuda")
    fused[..., H * D:2 * H * D] = t["k"].reshape(B, S, H * D)
    fused[..., 2 * H * D:] = t["v"].reshape(B, S, H * D)
    u["k"], u["v"] = fused[..., H * D:2 * H * D].view(B, S, H, D), fused[..., 2 * H * D:].view(B, S, H, D)
    u["pk"] = t["pk"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    out = torch.full((B, H, Lq, D), 9.0, dtype=dtype, device="cuda").permute(0, 2, 1, 3)
    assert torch.equal(run(hip, u, [P], [S, S - 7, 1], out=out), want) and torch.equal(out, want)
    one = dict(t, k=t["k"][:1].expand(B, S, H, D), v=t["v"][:1].expand(B, S, H, D))
    check(run(hip, one, None, None), *reference(one, [P], [S] * B, False, D ** -0.5))


def test_the_shared_prefix_is_what_a_copy_for_each_sequence_is(hip):
    """B sequences behind one prefix = the same sequences with the prefix copied in front of each suffix"""
    t = make(6, 1, 2, 8, 2, 128, 333, 70, torch.float16, 7)
    a = run(hip, t, None, None)
    k, v = torch.cat([t["pk"].expand(6, -1, -1, -1), t["k"]], 1), torch.cat([t["pv"].expand(6, -1, -1, -1), t["v"]], 1)
    b = hip.shared_prefix_attention(t["q"], None, None, k, v)
    ref, bound = reference(t, [333], [70] * 6, False, 128 ** -0.5)
    check(a, ref, bound)
    check(b, ref, bound)


def test_offsets_past_32_bits(hip):
    """a suffix cache of more than 2^31 elements: the last sequence, and the last keys of a long one"""
    B, S, H, D = 2, 70000, 128, 128
    k = torch.zeros(B, S, H, D, dtype=torch.float16, device="cuda")
    v = torch.zeros(B, S, H, D, dtype=torch.float16, device="cuda")
    q = torch.randn(B, 1, H, D, device="cuda").half()
    k[:, S - 3:] = torch.randn(B, 3, H, D, device="cuda").half() * 4
    v[:, S - 3:] = torch.randn(B, 3, H, D, device="cuda").half()
    got = hip.shared_prefix_attention(q, None, None, k, v)
    s = torch.einsum("bhd,bjhd->bhj", q[:, 0].double(), k[:, S - 3:].double()) * D ** -0.5
    m = s.amax(2, keepdim=True).clamp_min(0)
    e = torch.exp(s - m)
    want = torch.einsum("bhj,bjhd->bhd", e, v[:, S - 3:].double()) / (e.sum(2) + (S - 3) * torch.exp(-m[..., 0]))[..., None]
    assert (got[:, 0].double() - want).abs().max() <= 2e-3 * v.abs().max()
    del k, v


def test_no_sequences_no_queries_no_keys(hip):
    t = make(2, 1, 3, 4, 2, 64, 5, 6, torch.float16)
    assert hip.shared_prefix_attention(t["q"][:0], t["pk"], t["pv"], t["k"][:0], t["v"][:0]).shape == (0, 3, 4, 64)
    assert hip.shared_prefix_attention(t["q"][:, :0], t["pk"], t["pv"], t["k"], t["v"]).shape == (2, 0, 4, 64)
    assert not hip.shared_prefix_attention(t["q"], None, None, None, None).any()
    assert not hip.shared_prefix_attention(t["q"], t["pk"][:, :0], t["pv"][:, :0], t["k"][:, :0], t["v"][:, :0]).any()


def test_another_stream_and_two_graphs(hip):
    """a graph of single tokens (with scratch memory) and one of long rows share nothing: replayed in turn, and next to an eager call"""
    sets = [make(8, 1, 1, 8, 2, 128, 900, 100, torch.float16, 8), make(2, 1, 150, 4, 4, 128, 100, 100, torch.float16, 9)]
    lens = [torch.tensor([100 - 9 * i for i in range(8)], dtype=torch.int32, device="cuda"), torch.tensor([100, 3], dtype=torch.int32, device="cuda")]
    call = lambda t, n: hip.shared_prefix_attention(t["q"], t["pk"], t["pv"], t["k"], t["v"], lens=n)  # noqa: E731
    want = [call(t, n) for t, n in zip(sets, lens)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs, kept = [], []
    with torch.cuda.stream(s):
        for t, n, w in zip(sets, lens, want):
            assert torch.equal(call(t, n), w)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                kept.append(call(t, n))
            graphs.append(g)
    s.synchronize()
    for i in range(3):
        for t in sets:
            t["q"].copy_(torch.randn_like(t["q"]))
        lens[0].copy_(torch.randint(0, 101, (8,)))
        want = [call(t, n) for t, n in zip(sets, lens)]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(k, w) for k, w in zip(kept, want)), i
