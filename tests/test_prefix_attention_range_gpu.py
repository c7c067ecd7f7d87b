"""hip.shared_prefix_attention where weights far below the largest one count because they are many.

Bound: fp16 weights are held to 2^-11 of themselves and 2^-39 of the largest one (scores are exact here: one channel, small integers);
n + 64 additions in fp32."""
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
