"""Outputs that lie beside an operator's inputs in one buffer: the same bytes as with a buffer of their own, the inputs left as they were."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from propainter_amd import hip as h
    h.lib()
    return h


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,P", [(3, 1, 0), (2, 5, 300), (2, 70, 40)])
def test_attention_into_a_slot_of_the_queries_buffer(hip, B, L, P, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    buf, prefix = r(B, L, 4, 2, 64), r(2, 1, P, 2, 64)
    pk, pv = (prefix[0], prefix[1]) if P else (None, None)
    q, k, v, out = buf.unbind(2)
    before = buf.clone()
    want = hip.shared_prefix_attention(q.clone(), pk, pv, k.clone(), v.clone())
    assert hip.shared_prefix_attention(q, pk, pv, k, v, out=out) is out
    assert torch.equal(out, want) and torch.equal(buf[:, :, :3], before[:, :, :3])
    with pytest.raises(ValueError, match="overlaps"):
        hip.shared_prefix_attention(q, pk, pv, k, v, out=v)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("N,H,W,C,groups", [(2, 9, 11, 32, 4), (1, 150, 160, 64, 8), (3, 70, 90, 24, 3)])
def test_group_norm_into_the_channels_beside_its_input(hip, N, H, W, C, groups, dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    buf = torch.randn(N, H, W, 2 * C + 16, generator=g, device="cuda").to(dtype)
    before = buf.clone()
    for x_at, out_at in ((8, C + 16), (C + 8, 8), (8, 8)):
        buf.copy_(before)
        want = hip.group_norm(before[..., x_at:x_at + C].contiguous(), groups)
        hip.group_norm(buf, groups, out=buf, x_choff=x_at, C_=C, out_choff=out_at)
        assert torch.equal(buf[..., out_at:out_at + C], want)
        before_out = before.clone()
        before_out[..., out_at:out_at + C] = want
        assert torch.equal(buf, before_out)
    with pytest.raises(ValueError, match="overlaps"):
        hip.group_norm(buf, groups, out=buf, x_choff=8, C_=C, out_choff=C)
