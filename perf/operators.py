"""Performance cases of the group norm, the 8-bit linear layer and the shared-prefix attention.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, 64 where a rounding decides about a whole
number), or, where `own` is set, through the package's own entry points; `exact` computes it once more in 64 bits.

The operators, with their arguments as the package's entry points have them:

group_norm         y = act((x - mean) / sqrt(var + eps) * gamma + beta) over an NHWC map; mean and (biased) variance per image and
                   group of C / groups consecutive channels.
quantize_tokens    per row: scale = max|x| / 127 rounded to fp32; code = x / scale rounded to the nearest integer, ties to even
                   (scale 0: code 0).  The codes' rows are padded with zeros to a multiple of 64.
linear_i8          y[m, n] = act(sum_k xq[m, k] wq[n, k] * xs[m] * ws[n] + bias[n]) of quantised rows and quantised output channels.
prefix_attention   softmax(scale * q k^T) v for B sequences of Lq queries each over the keys of a prefix that the B / G sequences of a
                   group share and their own suffix keys (lens[b] of S).  Query i of a causal call sees the suffix keys up to
                   lens[b] - Lq + i.  Query head h reads key head h // (Hq / Hkv).  A query without keys gives zeros.
"""
import math

import torch

own = False

F16, F32 = "float16", "float32"
EPS = 1e-5


def listed():
    return [
        # group norm of a feature encoder: the 1/8 map of one 432x240 frame (latency), the half-resolution map of four 720x1280 frames,
        # the quarter-resolution fp32 map of two 1080x1920 frames (12 channels a group)
        gn("gn_240p_eighth", 1, 30, 54, 128, 8, "relu", F16),
        gn("gn_720p_half", 4, 360, 640, 64, 8, "relu", F16),
        gn("gn_1080p_quarter_f32", 2, 270, 480, 96, 8, "relu", F32),
        # codes of the 45 tokens of one attention window; of the feed-forward activations (width 1960) of a 17-frame 720x1280 window
        quant("quant_window", 45, 512, F16),
        quant("quant_ffn_720p", 110160, 1960, F16),
        # one token through a square layer (the weights' bytes count); the query | key | value projection of a 17-frame window from fp16
        # tokens; the largest: a square product whose codes are in hand (several layers read the same tokens)
        linear("lin_token", 1, 4096, 4096, "none", F16, F16, False),
        linear("lin_qkv_720p", 110160, 512, 1536, "none", F16, F16, False),
        linear("lin_square", 8192, 8192, 8192, "none", F16, F16, True),
        # a few single-token sequences behind the pooled tokens of one frame (latency); a batch of single tokens behind a long prefix; a
        # draft of four tokens a sequence in fp32; 24 attention windows of a 17-frame 720x1280 clip behind the pooled tokens of 6 key frames
        attn("attn_small", 4, 1, 1, 4, 4, 128, 405, 193, True, False, F16),
        attn("attn_decode", 64, 1, 1, 32, 8, 128, 8192, 1024, True, False, F16),
        attn("attn_draft_f32", 16, 2, 4, 16, 2, 64, 4096, 512, True, True, F32),
        attn("attn_windows_720p", 24, 1, 765, 4, 4, 128, 2430, 1158, False, False, F16),
    ]


def gn(name, N, H, W, C, groups, act, dtype):
    return {"name": name, "op": "group_norm", "N": N, "H": H, "W": W, "C": C, "groups": groups, "act": act, "dtype": dtype}


def quant(name, rows, K, dtype):
    return {"name": name, "op": "quantize_tokens", "rows": rows, "K": K, "dtype": dtype}


def linear(name, M, K, N, act, dtype, out_dtype, codes):
    return {"name": name, "op": "linear_i8", "M": M, "K": K, "N": N, "act": act, "dtype": dtype, "out_dtype": out_dtype, "codes": codes}


def attn(name, B, G, Lq, Hq, Hkv, D, P, S, ragged, causal, dtype):
    return {"name": name, "op": "prefix_attention", "B": B, "G": G, "Lq": Lq, "Hq": Hq, "Hkv": Hkv, "D": D, "P": P, "S": S, "ragged": ragged,
            "causal": causal, "dtype": dtype}


def spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group_norm", "quantize_tokens", "linear_i8", "linear_i8", "prefix_attention", "prefix_attention"])
    if op == "group_norm":
        C = 8 * spread(rng, 1, 80)
        groups = rng.choice([g for g in (1, 2, 4, 8, 16, 32, 64) if C % g == 0])
        H, W = spread(rng, 4, 540), spread(rng, 4, 960)
        N = spread(rng, 1, 16)
        while N * H * W * C > 60_000_000:
            N, H, W = max(1, N // 2), max(1, H * 3 // 4), max(1, W * 3 // 4)
        c = gn("", N, H, W, C, groups, rng.choice(["none", "relu", "silu", "gelu"]), rng.choice([F16, F16, F32]))
    elif op == "quantize_tokens":
        K = spread(rng, 8, 16384)
        c = quant("", spread(rng, 1, min(150_000, 200_000_000 // K)), K, rng.choice([F16, F16, F32]))
    elif op == "linear_i8":
        K, N = spread(rng, 32, 8192), spread(rng, 8, 8192)
        M = spread(rng, 1, min(120_000, 8192 ** 3 // 4 // (K * N), 200_000_000 // max(K, N)))
        c = linear("", M, K, N, rng.choice(["none", "none", "relu", "gelu"]), rng.choice([F16, F16, F32]), rng.choice([F16, F16, F32]), rng.random() < 0.5)
    else:
        Hkv, rep, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8]), rng.choice([64, 128, 128])
        G, Lq = rng.choice([1, 1, 1, 2, 3]), rng.choice([1, 1, 1, spread(rng, 2, 8), spread(rng, 16, 800)])
        B = G * spread(rng, 1, 96 if Lq < 16 else 24)
        P, S = spread(rng, 1, 16384 if Lq < 16 else 4096), spread(rng, 1, 2048)
        while B * Lq * Hkv * rep * (P + S) > 250_000_000:
            P, S, Lq = max(1, P * 3 // 4), max(1, S * 3 // 4), max(1, Lq * 3 // 4)
        c = attn("", B, G, Lq, Hkv * rep, Hkv, D, P, S, rng.random() < 0.7, rng.random() < 0.5, rng.choice([F16, F16, F16, F32]))
    del c["name"]
    return c


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = generator(seed)
    dt = getattr(torch, case.get("dtype", F32))
    if case["op"] == "group_norm":
        N, H, W, C = case["N"], case["H"], case["W"], case["C"]
        # a convolution's output: channels of different means and spreads
        x = normal(g, N, H, W, C) * (0.5 + torch.rand(C, generator=g, device="cuda")) + normal(g, C)
        return {"case": case, "x": x.to(dt), "gamma": 1 + 0.2 * normal(g, C), "beta": 0.2 * normal(g, C)}
    if case["op"] == "quantize_tokens":
        return {"case": case, "x": tokens(g, case["rows"], case["K"]).to(dt)}
    if case["op"] == "linear_i8":
        M, K, N = case["M"], case["K"], case["N"]
        x = tokens(g, M, K).to(dt)
        wq, ws = quantized(normal(g, N, K) / math.sqrt(K))
        s = {"case": case, "wq": wq, "ws": ws, "bias": 0.1 * normal(g, N)}
        if case["codes"]:
            q, s["xs"] = quantized(x)
            s["xq"] = padded(q)
        else:
            s["x"] = x
        if own:
            from propainter_amd import conv
            s["layer"] = conv.Int8Linear.from_codes(wq, ws, s["bias"])
        return s
    B, G, Lq, Hq, Hkv, D, P, S = (case[k] for k in ("B", "G", "Lq", "Hq", "Hkv", "D", "P", "S"))
    s = {"case": case, "q": 1.5 * normal(g, B, Lq, Hq, D), "pk": normal(g, G, P, Hkv, D), "pv": normal(g, G, P, Hkv, D),
         "k": normal(g, B, S, Hkv, D), "v": normal(g, B, S, Hkv, D)}
    s = {k: v if k == "case" else v.to(dt) for k, v in s.items()}
    lens, plens = lengths(case)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")[torch.randperm(B, generator=g, device="cuda")]
    s["plens"] = torch.tensor(plens, dtype=torch.int32, device="cuda")[torch.randperm(G, generator=g, device="cuda")]
    return s


def tokens(g, rows, K):
    """Token rows of different magnitudes, a few large values among them."""
    x = normal(g, rows, K) * torch.exp(0.5 * normal(g, rows, 1))
    return x + x * (x.abs() > 3) * 2


def lengths(case):
    """The suffix lengths of the sequences and the prefix lengths of the groups, in some order: the same ones for every seed."""
    B, G, P, S = case["B"], case["G"], case["P"], case["S"]
    if not case["ragged"]:
        return [S] * B, [P] * G
    return [1 + (S - 1) * (i + 1) // B for i in range(B)], [P - (P // 2) * i // G for i in range(G)]


def padded(q):
    return torch.nn.functional.pad(q, (0, -q.shape[1] % 64))


def quantized(x):
    """Codes and scales of rows: the scale is rounded to fp32 once, and the quotient by that scale is taken in 64 bits, where no rounding
    makes or hides a tie."""
    s = (x.abs().amax(1).double() / 127).float()
    q = torch.round(x.double() / torch.where(s > 0, s, 1.0).double()[:, None])
    return q.to(torch.int8), s


def activation(y, act):
    if act == "relu":
        return y * (y > 0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def run(state):
    case = state["case"]
    if own:
        from propainter_amd import hip
        if case["op"] == "group_norm":
            return hip.group_norm(state["x"], case["groups"], state["gamma"], state["beta"], eps=EPS, act=getattr(hip, "ACT_" + case["act"].upper()))
        if case["op"] == "quantize_tokens":
            return hip.quantize_tokens(state["x"])
        if case["op"] == "linear_i8":
            odt = getattr(torch, case["out_dtype"])
            if case["codes"]:
                return state["layer"].product(state["xq"], state["xs"], act=case["act"], out_dtype=odt)
            return state["layer"](state["x"], act=case["act"], out_dtype=odt)
        return hip.shared_prefix_attention(state["q"], state["pk"], state["pv"], state["k"], state["v"], prefix_lens=state["plens"], lens=state["lens"],
                                           causal=case["causal"])
    if case["op"] == "group_norm":
        return plain_group_norm(state)
    if case["op"] == "quantize_tokens":
        q, s = quantized(state["x"])
        return padded(q), s
    if case["op"] == "linear_i8":
        q, s = (state["xq"][:, :case["K"]], state["xs"]) if case["codes"] else quantized(state["x"])
        y = torch.matmul(q.float(), state["wq"].float().t()) * s[:, None] * state["ws"] + state["bias"]
        return activation(y, case["act"]).to(getattr(torch, case["out_dtype"]))
    return plain_attention(state)


def plain_group_norm(state):
    case, x = state["case"], state["x"]
    N, H, W, C, G = (case[k] for k in ("N", "H", "W", "C", "groups"))
    y = x.float().view(N, H * W, G, C // G)
    y = y - y.mean((1, 3), keepdim=True)
    y = y / torch.sqrt((y * y).mean((1, 3), keepdim=True) + EPS)
    return activation(y.view(N, H, W, C) * state["gamma"] + state["beta"], case["act"]).to(x.dtype)


def plain_attention(state):
    case = state["case"]
    B, G, Lq, Hq, Hkv, D, P, S = (case[k] for k in ("B", "G", "Lq", "Hq", "Hkv", "D", "P", "S"))
    rep, n = Hq // Hkv, B // G
    q = state["q"].float().view(B, Lq, Hkv, rep, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Lq * rep, D) / math.sqrt(D)
    heads = lambda t: t.float().permute(0, 2, 1, 3).contiguous()  # noqa: E731
    pk, pv, k, v = heads(state["pk"]), heads(state["pv"]), heads(state["k"]), heads(state["v"])
    rows = lambda t, w: t.reshape(G, n, Hkv, Lq * rep, w).permute(0, 2, 1, 3, 4).reshape(G, Hkv, n * Lq * rep, w)  # noqa: E731
    back = lambda t, w: t.view(G, Hkv, n, Lq * rep, w).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Lq * rep, w)  # noqa: E731
    sp = back(torch.matmul(rows(q, D), pk.transpose(2, 3).contiguous()), P)
    ss = torch.matmul(q, k.transpose(2, 3).contiguous())
    at = torch.arange(max(P, S), device=q.device)
    seen = state["lens"].view(B, 1) - (Lq - 1 - torch.arange(Lq, device=q.device).view(1, Lq)) if case["causal"] else state["lens"].view(B, 1).expand(B, Lq)
    seen = seen.repeat_interleave(rep, 1).view(B, 1, Lq * rep, 1)
    sp = sp.masked_fill(at[:P] >= state["plens"].repeat_interleave(n).view(B, 1, 1, 1), -math.inf)
    ss = ss.masked_fill(at[:S] >= seen, -math.inf)
    top = torch.maximum(sp.amax(3, keepdim=True), ss.amax(3, keepdim=True)).clamp_min(-1e30)
    sp, ss = torch.exp(sp - top), torch.exp(ss - top)
    total = sp.sum(3, keepdim=True) + ss.sum(3, keepdim=True)
    out = (back(torch.matmul(rows(sp, P), pv), D) + torch.matmul(ss, v)) / torch.where(total > 0, total, 1.0)
    return out.view(B, Hkv, Lq, rep, D).permute(0, 2, 1, 3, 4).reshape(B, Lq, Hq, D).to(state["q"].dtype)


def size(name):
    return 2 if name == F16 else 4


def work(case):
    if case["op"] == "group_norm":
        n = case["N"] * case["H"] * case["W"] * case["C"]
        return {"bytes": 2 * n * size(case["dtype"]) + 8 * case["C"], "flops": 8 * n}
    if case["op"] == "quantize_tokens":
        n = case["rows"] * case["K"]
        return {"bytes": n * (size(case["dtype"]) + 1) + 4 * case["rows"], "flops": 4 * n}
    if case["op"] == "linear_i8":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * (1 if case["codes"] else size(case["dtype"])) + N * K + M * N * size(case["out_dtype"]) + 4 * M * case["codes"] + 8 * N,
                "flops": 2 * M * K * N}
    B, G, Lq, Hq, Hkv, D = (case[k] for k in ("B", "G", "Lq", "Hq", "Hkv", "D"))
    lens, plens = lengths(case)
    own_pairs = sum(sum(min(n, max(0, n - Lq + 1 + i)) for i in range(Lq)) if case["causal"] else n * Lq for n in lens)
    pairs = own_pairs + sum(plens) * (B // G) * Lq
    return {"bytes": size(case["dtype"]) * D * (2 * B * Lq * Hq + 2 * Hkv * (sum(lens) + sum(plens))), "flops": 4 * D * Hq * pairs}


def exact(case, seed):
    """The operator's definition in 64 bits."""
    with torch.no_grad():
        s = prepare(case, seed)
        if case["op"] == "group_norm":
            return exact_group_norm(case, s)
        if case["op"] == "quantize_tokens":
            return exact_codes(s["x"], case["K"])
        if case["op"] == "linear_i8":
            return exact_linear(case, s)
        return exact_attention(case, s)


def exact_group_norm(case, s):
    each = []
    step = case["C"] // case["groups"]
    for image in s["x"]:
        parts = []
        for c in range(0, case["C"], step):
            x = image[:, :, c:c + step].double()
            var, mean = torch.var_mean(x, correction=0)
            parts.append((x - mean) * torch.rsqrt(var + EPS) * s["gamma"][c:c + step].double() + s["beta"][c:c + step].double())
        each.append(torch.cat(parts, 2))
    return exact_activation(torch.stack(each), case["act"])


def exact_activation(y, act):
    if act == "relu":
        return y.clamp_min(0)
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return y * torch.special.ndtr(y)
    return y


def exact_codes(x, K):
    x = x.double()
    scale = x.abs().max(dim=1).values / 127.0
    held = scale.float().double()
    ratio = torch.where(held[:, None] > 0, x / held[:, None], torch.zeros_like(x))
    low = torch.floor(ratio)
    up = (ratio - low > 0.5) | ((ratio - low == 0.5) & (low % 2 == 1))
    codes = torch.zeros(x.shape[0], (K + 63) // 64 * 64, dtype=torch.int8, device=x.device)
    codes[:, :K] = (low + up).to(torch.int8)
    return codes, scale


def exact_linear(case, s):
    K, N = case["K"], case["N"]
    if case["codes"]:
        codes, scale = s["xq"][:, :K], s["xs"]
    else:
        codes, scale = exact_codes(s["x"], K)
        codes, scale = codes[:, :K], scale.float()
    rows = []
    for at in range(0, codes.shape[0], 16384):
        y = codes[at:at + 16384].double() @ s["wq"].double().t()
        y = y * (scale[at:at + 16384].double()[:, None] * s["ws"].double()[None, :]) + s["bias"].double()
        rows.append(exact_activation(y, case["act"]))
    return torch.cat(rows)


def exact_attention(case, s):
    B, G, Lq, Hq, Hkv, D = (case[k] for k in ("B", "G", "Lq", "Hq", "Hkv", "D"))
    out = torch.zeros(B, Lq, Hq, D, dtype=torch.float64, device=s["q"].device)
    lens, plens = s["lens"].tolist(), s["plens"].tolist()
    for b in range(B):
        g = b // (B // G)
        k = torch.cat([s["pk"][g, :plens[g]], s["k"][b, :lens[b]]]).double().repeat_interleave(Hq // Hkv, 1)
        v = torch.cat([s["pv"][g, :plens[g]], s["v"][b, :lens[b]]]).double().repeat_interleave(Hq // Hkv, 1)
        logits = torch.bmm(s["q"][b].double().transpose(0, 1), k.permute(1, 2, 0)) * D ** -0.5
        if case["causal"]:
            at = torch.arange(k.shape[0], device=k.device) - plens[g]
            last = torch.arange(Lq, device=k.device)[:, None] + (lens[b] - Lq)
            logits = logits.masked_fill((at >= 0) & (at > last), -math.inf)
        top = logits.amax(2, keepdim=True)
        p = torch.exp(logits - top.masked_fill(top == -math.inf, 0.0))
        total = p.sum(2, keepdim=True)
        out[b] = (torch.bmm(p, v.transpose(0, 1)) / total.masked_fill(total == 0, 1.0)).transpose(0, 1)
    return out
