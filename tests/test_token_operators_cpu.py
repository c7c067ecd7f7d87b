"""Group norm, 8-bit linear layer, shared-prefix attention: what the C entries refuse before any launch, sizes of workspaces and layouts, and
the wrappers' refusal of CPU tensors.  No GPU: the pointers are addresses that nothing reads."""
import ctypes as C

import pytest
import torch

from propainter_amd import conv, hip

A = 0x1000          # a 16-byte aligned address
ARG, DTYPE, ALIGN, WORK = -1, -2, -3, -4


@pytest.fixture(scope="module")
def L():
    return hip.lib()


def ptr(v):
    return C.c_void_p(v)


def gn(L, inp=A, out=A, ws=A, cs=64, co=0, ocs=64, oco=0, N=1, H=4, W=4, Cc=64, G=8, eps=1e-5, act=0, dt=1):
    i = C.c_int
    return L.pp_group_norm(ptr(inp), i(cs), i(co), ptr(out), i(ocs), i(oco), None, None, ptr(ws), i(N), i(H), i(W), i(Cc), i(G), C.c_float(eps), i(act),
                           C.c_float(0), i(dt), None)


@pytest.mark.parametrize("kw,rc", [(dict(inp=0), ARG), (dict(out=0), ARG), (dict(ws=0, H=400, W=400), WORK), (dict(N=0), ARG), (dict(H=0), ARG), (dict(N=70000), ARG), (dict(H=1 << 20, W=1 << 20), ARG),
                                   (dict(Cc=60, G=4), ARG), (dict(G=7), ARG), (dict(G=0), ARG), (dict(Cc=2056, G=8, cs=4096, ocs=4096), ARG), (dict(act=7), ARG), (dict(act=-1), ARG),
                                   (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG), (dict(dt=2), DTYPE), (dict(cs=56), ARG), (dict(co=8), ARG), (dict(oco=-8), ARG),
                                   (dict(cs=68, co=4), ALIGN), (dict(cs=100), ALIGN), (dict(inp=A + 8), ALIGN), (dict(out=A + 4), ALIGN), (dict(ws=A + 4), ALIGN)])
def test_group_norm_refuses(L, kw, rc):
    assert gn(L, **kw) == rc and L.pp_last_error_string().startswith(b"pp_group_norm")


def test_group_norm_workspace(L):
    f = lambda *a: L.pp_group_norm_workspace_floats(*[C.c_int(v) for v in a])  # noqa: E731
    assert f(1, 4, 4, 64, 8) >= 0 and f(16, 540, 960, 64, 64) < 1 << 24
    for bad in ((0, 4, 4, 64, 8), (1, 4, 4, 60, 4), (1, 4, 4, 64, 7), (1, 4, 4, 4096, 8), (1, 1 << 16, 1 << 16, 8, 1)):
        assert f(*bad) < 0


def quant(L, x=A, xrs=128, q=A, qrs=128, s=A, rows=4, K=100, dt=1):
    return L.pp_quantize_tokens(ptr(x), C.c_int64(xrs), ptr(q), C.c_int64(qrs), ptr(s), C.c_int64(rows), C.c_int(K), C.c_int(dt), None)


@pytest.mark.parametrize("kw,rc", [(dict(x=0), ARG), (dict(q=0), ARG), (dict(s=0), ARG), (dict(rows=-1), ARG), (dict(K=0), ARG), (dict(K=131073), ARG), (dict(dt=2), DTYPE), (dict(qrs=100), ARG),
                                   (dict(qrs=136), ALIGN), (dict(q=A + 8), ALIGN), (dict(x=A + 1), ALIGN), (dict(xrs=-1), ARG), (dict(rows=0), 0)])
def test_quantize_tokens_refuses(L, kw, rc):
    assert quant(L, **kw) == rc


def test_row_and_weight_bytes(L):
    assert [L.pp_i8_row_bytes(C.c_int(k)) for k in (1, 64, 65, 1960, 131072, 0, -5, 131073)] == [64, 64, 128, 1984, 131072, ARG, ARG, ARG]
    f = lambda n, k: L.pp_linear_i8_weight_bytes(C.c_int(n), C.c_int(k))  # noqa: E731
    assert f(1, 1) >= 64 and f(64, 64) >= 4096 and f(4194240, 131072) >= 4194240 * 131072 and f(0, 64) == ARG and f(5, 0) == ARG and f(4194241, 64) == ARG


def lin(L, q=A, qrs=128, xs=A, w=A, ws=A, out=A, ors=80, M=4, N=80, K=100, act=0, odt=1):
    return L.pp_linear_i8(ptr(q), C.c_int64(qrs), ptr(xs), ptr(w), ptr(ws), None, ptr(out), C.c_int64(ors), C.c_int64(M), C.c_int(N), C.c_int(K), C.c_int(act),
                          C.c_float(0), C.c_int(odt), None)


@pytest.mark.parametrize("kw,rc", [(dict(q=0), ARG), (dict(xs=0), ARG), (dict(w=0), ARG), (dict(ws=0), ARG), (dict(out=0), ARG), (dict(M=-1), ARG), (dict(M=(1 << 30) + 1), ARG), (dict(N=0), ARG),
                                   (dict(K=0), ARG), (dict(act=7), ARG), (dict(odt=2), DTYPE), (dict(qrs=112), ARG), (dict(qrs=136), ALIGN), (dict(q=A + 4), ALIGN), (dict(w=A + 8), ALIGN),
                                   (dict(out=A + 1), ALIGN), (dict(ors=79), ARG), (dict(M=0), 0)])
def test_linear_i8_refuses(L, kw, rc):
    assert lin(L, **kw) == rc


def tokens(L, x=A, xrs=100, xdt=1, w=A, ws=A, out=A, ors=80, M=4000, N=80, K=100, act=0, odt=1, work=A, wb=1 << 20):
    return L.pp_linear_i8_tokens(ptr(x), C.c_int64(xrs), C.c_int(xdt), ptr(w), ptr(ws), None, ptr(out), C.c_int64(ors), C.c_int64(M), C.c_int(N), C.c_int(K), C.c_int(act),
                                 C.c_float(0), C.c_int(odt), ptr(work), C.c_int64(wb), None)


@pytest.mark.parametrize("kw,rc", [(dict(x=0), ARG), (dict(w=0), ARG), (dict(ws=0), ARG), (dict(out=0), ARG), (dict(M=-1), ARG), (dict(N=0), ARG), (dict(K=0), ARG), (dict(act=9), ARG),
                                   (dict(xdt=2), DTYPE), (dict(odt=5), DTYPE), (dict(xrs=-4), ARG), (dict(x=A + 1), ALIGN), (dict(w=A + 8), ALIGN), (dict(ors=79), ARG), (dict(work=0), WORK),
                                   (dict(wb=4000 * 132 - 1), WORK), (dict(work=A + 4), WORK), (dict(M=0), 0)])
def test_linear_i8_tokens_refuses(L, kw, rc):
    assert tokens(L, **kw) == rc


def test_linear_i8_tokens_workspace(L):
    f = lambda m, k, n=80: L.pp_linear_i8_tokens_workspace_bytes(C.c_int64(m), C.c_int(n), C.c_int(k))  # noqa: E731
    assert f(0, 64) == 0 and f(4000, 100) == 4000 * 132 and f(40, 100) == 0 and f(40, 100, 50000) == 40 * 132 and f(1, 100, 0) == ARG and f(1, 100, 4194241) == ARG and f(-1, 64) == ARG and f(1, 0) == ARG and f(1000, 131072) == 1000 * 131076


def test_linear_i8_pack_refuses(L):
    f = lambda q=A, rs=100, w=A, N=5, K=100: L.pp_linear_i8_pack(ptr(q), C.c_int64(rs), ptr(w), C.c_int(N), C.c_int(K), None)  # noqa: E731
    assert f(q=0) == ARG and f(w=0) == ARG and f(rs=99) == ARG and f(N=0) == ARG and f(K=0) == ARG and f(w=A + 8) == ALIGN


def attn_args(B=4, G=2, Lq=3, Hq=8, Hkv=2, D=64, P=10, S=12, dtype=1, **kw):
    a = hip.PrefixAttnArgs()
    a.dtype, a.B, a.G, a.Lq, a.Hq, a.Hkv, a.D, a.P, a.S, a.scale = dtype, B, G, Lq, Hq, Hkv, D, P, S, 0.125
    for name, n, H in (("q", Lq, Hq), ("out", Lq, Hq), ("pk", P, Hkv), ("pv", P, Hkv), ("k", S, Hkv), ("v", S, Hkv)):
        setattr(a, name, A)
        getattr(a, name + "_stride")[:] = (max(n, 1) * H * D, H * D, D)
    a.work, a.work_bytes = A, 1 << 40
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [(dict(dtype=2), DTYPE), (dict(D=96), ARG), (dict(B=-1), ARG), (dict(G=0), ARG), (dict(G=3), ARG), (dict(Hq=7), ARG), (dict(Hkv=0), ARG), (dict(P=-1), ARG),
                                   (dict(S=-1), ARG), (dict(B=1 << 20, Lq=1 << 12), ARG), (dict(S=1 << 30, P=1 << 30), ARG), (dict(causal=2), ARG), (dict(scale=float("inf")), ARG),
                                   (dict(scale=float("nan")), ARG), (dict(q=0), ARG), (dict(out=0), ARG), (dict(pk=0), ARG), (dict(pv=0), ARG), (dict(k=0), ARG), (dict(v=0), ARG),
                                   (dict(q=A + 8), ALIGN), (dict(v=A + 8), ALIGN), (dict(q_stride=(1536, 512, 60)), ALIGN), (dict(k_stride=(1536, 56, 64)), ARG), (dict(k_stride=(1536, 0, 64)), ARG),
                                   (dict(k_stride=(-1536, 128, 64)), ALIGN), (dict(pk_stride=(1280, 1 << 23, 64)), ARG), (dict(out_stride=(0, 512, 64)), ARG),
                                   (dict(out_stride=(1536, 512, 0)), ARG), (dict(B=0, G=1), 0), (dict(Lq=0), 0)])
def test_shared_prefix_attention_refuses(L, kw, rc):
    a = attn_args(**kw)
    assert L.pp_shared_prefix_attention(C.byref(a), None) == rc, L.pp_last_error_string()


def test_shared_prefix_attention_workspace(L):
    f = lambda **kw: L.pp_shared_prefix_attention_workspace_bytes(C.byref(attn_args(**kw)))  # noqa: E731
    assert f() >= 0 and f(D=80) == ARG and f(dtype=7) == DTYPE
    big = dict(B=64, G=1, Lq=1, Hq=32, Hkv=8, D=128, P=8192, S=1024)
    need = f(**big)
    assert 0 <= need < 1 << 30
    if need:
        assert L.pp_shared_prefix_attention(C.byref(attn_args(work_bytes=need - 1, **big)), None) == WORK
        assert L.pp_shared_prefix_attention(C.byref(attn_args(work=0, **big)), None) == WORK
        assert L.pp_shared_prefix_attention(C.byref(attn_args(work=A + 8, **big)), None) == WORK


def test_struct_size(L):
    assert L.pp_sizeof_prefix_attn_args() == C.sizeof(hip.PrefixAttnArgs)


def test_wrappers_need_gpu_tensors():
    x = torch.zeros(1, 2, 2, 8)
    for call in (lambda: hip.group_norm(x, 1), lambda: hip.quantize_tokens(x), lambda: hip.linear_i8_pack(torch.zeros(4, 64, dtype=torch.int8)),
                 lambda: hip.linear_i8(torch.zeros(1, 64, dtype=torch.int8), torch.zeros(1), torch.zeros(4096, dtype=torch.int8), torch.zeros(4), None, 4, 64),
                 lambda: hip.shared_prefix_attention(torch.zeros(1, 1, 1, 64), None, None, None, None), lambda: conv.Int8Linear(torch.zeros(4, 8), device="cpu")):
        with pytest.raises(RuntimeError, match="GPU|HIP"):
            call()
