"""hip.shared_prefix_attention where the softmax' range is wide: weights far below the largest one that count because they are many, and scores
whose fp32 neighbours lie far apart.

First bound: fp16 weights are held to 2^-11 of themselves and 2^-39 of the largest one (scores are exact here: one channel, small integers);
n + 64 additions in fp32.  Second: products of powers of two are exact, keys of the same score weigh the same and a key behind by more than 200
weighs nothing, so the output is a mean of at most n values: n 2^-24 of the mean size.  fp16 weights are rounded once as operands and not in their
sum (sum round(w) v / sum w: at most 2^-11 of the mean size more; below 2^20 a score leaves the weights' common factor no power of two)."""
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


def places(n, S):
    """n keys as prefix alone, suffix alone, and both"""
    return [(n, 0), (0, n), (n - S, S)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,Lq,Hq,Hkv,D,n,S,gap", [(1, 1, 1, 1, 64, 1 << 20, 300, 24), (1, 1, 8, 1, 128, 200_000, 5000, 22), (1, 70, 2, 2, 64, 400_000, 100, 23), (8, 1, 4, 1, 64, 150_000, 40, 21)])
def test_many_small_weights_count(hip, B, Lq, Hq, Hkv, D, n, S, gap, dtype):
    """one key leads the others by a factor of 2^(gap + 1/2): its value is 0, theirs 1"""
    for P, own in places(n, S):
        q = torch.zeros(B, Lq, Hq, D, device="cuda", dtype=dtype)
        q[..., 0] = 1
        k = lambda *s: torch.zeros(*s, Hkv, D, device="cuda", dtype=dtype)  # noqa: E731
        pk, ks = (k(1, P) if P else None), (k(B, own) if own else None)
        pv, vs = (None if pk is None else torch.ones_like(pk)), (None if ks is None else torch.ones_like(ks))
        lead_k, lead_v = (pk[:, P // 3], pv[:, P // 3]) if P else (ks[:, own // 3], vs[:, own // 3])
        lead_k[..., 0], lead_v[...] = 2, 0
        got = hip.shared_prefix_attention(q, pk, pv, ks, vs, scale=(gap + 0.5) * math.log(2) / 2).double()
        tail = (P + own - 1) * 2.0 ** -(gap + 0.5)
        want = tail / (1 + tail)
        rel = (n + 64 + gap) * 2.0 ** -24 + (2.0 ** -11 + 2.0 ** -39 * 2.0 ** (gap + 0.5) if dtype == torch.float16 else 0)
        lim = want * rel + want * torch.finfo(dtype).eps / 2 + 2.0 ** -25
        assert (got - want).abs().max().item() <= lim, ((got - want).abs().max().item(), want, lim)


@pytest.mark.parametrize("dtype,size", [(t, sign * 2.0 ** e) for t, e in ((torch.float16, 11), (torch.float16, 15), (torch.float32, 11), (torch.float32, 15), (torch.float32, 60),
                                                                           (torch.float32, 63)) for sign in (1, -1)])
@pytest.mark.parametrize("B,Lq,Hq,Hkv,D,P,S", [(1, 1, 1, 1, 64, 0, 64), (3, 1, 4, 2, 128, 500, 12), (2, 90, 2, 2, 64, 200, 56), (64, 1, 8, 1, 128, 4000, 96), (2, 40, 4, 4, 128, 0, 128)])
def test_scores_far_from_zero(hip, B, Lq, Hq, Hkv, D, P, S, dtype, size):
    n = P + S
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, Hkv, D, generator=g, device="cuda").to(dtype)  # noqa: E731
    q = torch.zeros(B, Lq, Hq, D, device="cuda", dtype=dtype)
    q[..., 0] = abs(size)
    k = lambda *s: torch.zeros(*s, Hkv, D, device="cuda", dtype=dtype)  # noqa: E731
    pk, pv, ks, vs = (k(1, P), r(1, P), k(B, S), r(B, S)) if P else (None, None, k(B, S), r(B, S))
    for t in (pk, ks):
        if t is not None:
            t[..., 0] = size
    # every key the same score: the mean of all values
    got = hip.shared_prefix_attention(q, pk, pv, ks, vs).double()
    rep = Hq // Hkv
    mean = lambda v: v.double().repeat_interleave(rep, 2)  # noqa: E731
    every = mean(vs) if P == 0 else torch.cat([mean(pv).expand(B, -1, -1, -1), mean(vs)], 1)
    lim = every.abs().mean(1, keepdim=True) * ((n + 64) * 2.0 ** -24 + (2.0 ** -11 if dtype == torch.float16 else 0)) + every.mean(1, keepdim=True).abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25
    assert ((got - every.mean(1, keepdim=True)).abs() <= lim).all()
    # four of them lead by a last place of the keys' type: the mean of those
    lead = [0, S // 4, S // 2, S - 1]
    ks[:, lead, :, 0] = size * (1 + torch.finfo(dtype).eps) if size > 0 else size * (1 - torch.finfo(dtype).eps / 2)
    if abs(size) ** 2 * D ** -0.5 * torch.finfo(dtype).eps / 2 > 200:
        got = hip.shared_prefix_attention(q, pk, pv, ks, vs).double()
        four = mean(vs[:, lead]).mean(1, keepdim=True)
        lim = mean(vs[:, lead]).abs().mean(1, keepdim=True) * (80 * 2.0 ** -24 + (2.0 ** -11 if dtype == torch.float16 else 0)) + four.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25
        assert ((got - four).abs() <= lim).all()


def test_more_rows_to_join_than_one_launch_has_waves(hip):
    """2^26 rows, each the join of one prefix key and one suffix key"""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    B, Hq, D = 1 << 21, 32, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    r = lambda *s: torch.randn(*s, D, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
    q, pk, pv, k, v = r(B, 1, Hq), r(1, 1, 1), r(1, 1, 1), r(B, 1, 1), r(B, 1, 1)
    out = torch.full_like(q, float("nan"))
    hip.shared_prefix_attention(q, pk, pv, k, v, out=out)
    for s in (slice(0, 2000), slice(B // 4 - 1000, B // 4 + 1000), slice(B // 2 - 1000, B // 2 + 1000), slice(B - 2000, B)):
        q64, k64, v64 = (t[s].double() for t in (q, k, v))
        d = ((q64 * k64).sum(-1) - (q64 * pk.double()).sum(-1)) * D ** -0.5
        w = torch.sigmoid(d)[..., None]
        want, size = w * v64 + (1 - w) * pv.double(), w * v64.abs() + (1 - w) * pv.double().abs()
        scores = ((q64 * k64).abs().sum(-1) + (q64 * pk.double()).abs().sum(-1))[..., None] * D ** -0.5
        lim = size * (2.0 ** -11 + 2.0 ** -24 * (2 * (D + 8) * scores + 70)) + want.abs() * 2.0 ** -11 + 2.0 ** -25
        assert ((out[s].double() - want).abs() <= lim).all()
