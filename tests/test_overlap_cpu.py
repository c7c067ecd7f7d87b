"""Which outputs share memory with an input (hip._overlap) against the sets of their bytes.  No GPU: addresses are compared, nothing is read."""
import random

import pytest
import torch

from propainter_amd import hip


def offsets(t, base):
    idx = torch.zeros((), dtype=torch.long)
    for n, s in zip(t.shape, t.stride()):
        idx = idx[..., None] + torch.arange(n) * s
    first = t.data_ptr() - base + idx.reshape(-1) * t.element_size()
    return set((first[:, None] + torch.arange(t.element_size())).reshape(-1).tolist())


def view(rng, buf):
    """a random strided view of one of its types"""
    t = buf.view(rng.choice([torch.int8, torch.float16, torch.float32]))
    dims = rng.randint(0, 4)
    shape, stride = [], []
    for _ in range(dims):
        shape.append(rng.choice([1, 1, 2, 3, 5]))
        stride.append(rng.choice([0, 1, 2, 3, 8, 12, 16, 24, 40]))
    span = sum((n - 1) * s for n, s in zip(shape, stride)) + 1
    return torch.as_strided(t, shape, stride, rng.randint(0, t.numel() - span)) if span <= t.numel() else view(rng, buf)


def test_random_views():
    rng, buf = random.Random(3), torch.zeros(640, dtype=torch.int8)
    got = {True: 0, False: 0}
    for _ in range(3000):
        a, b = view(rng, buf), view(rng, buf)
        want = bool(offsets(a, buf.data_ptr()) & offsets(b, buf.data_ptr()))
        assert hip._overlap(a, b) == want == hip._overlap(b, a), (a.shape, a.stride(), b.shape, b.stride())
        got[want] += 1
    assert min(got.values()) > 200


def test_slots_of_one_buffer():
    qkv = torch.zeros(2, 7, 3, 4, 64, dtype=torch.float16)
    for i in range(3):
        for j in range(3):
            assert hip._overlap(qkv[:, :, i], qkv[:, :, j]) == (i == j)
    assert hip._overlap(qkv[:, :, 0, 1:], qkv[:, :, 0, :2]) and not hip._overlap(qkv[:, :, 0, :2], qkv[:, :, 0, 2:]) and not hip._overlap(qkv[0, :, 1], qkv[1:, :, 1])
    m = torch.zeros(2, 5, 6, 48)
    assert not hip._overlap(m[..., :16], m[..., 16:]) and hip._overlap(m[..., :24], m[..., 16:]) and not hip._overlap(m[..., :0], m)
    big = torch.zeros(1).expand(1 << 20, 1 << 10, 64)
    assert hip._overlap(big, big[:1]) and not hip._overlap(big, m)


def test_the_refusal_names_who_refuses():
    x = torch.zeros(4, 8)
    hip._refuse_overlap("op", x[:2], x[2:], None)
    with pytest.raises(ValueError, match="op: out overlaps an input"):
        hip._refuse_overlap("op", x[:2], None, x[1:])
