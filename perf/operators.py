"""Measured cases of the token operators: norms of queries and keys with the position rotation, attention over key
ranges (documents, prefixes, causal, capped or distance-biased scores) with its gradient, attention of new tokens over
a cache, and a shared projection with the low-rank adapters of many requests.

``run`` computes a case either in elementary torch operations in 32 bits (``own = False``) or through this package's
calls (``own = True``); ``exact`` computes it from the definition in 64 bits.
"""
import math

import torch

own = False

_BF, _F32, _F64 = torch.bfloat16, torch.float32, torch.float64
_DT = {"bf16": _BF, "f32": _F32}


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # eight requests, one new token each, before the attention over their caches: the call's latency counts
        dict(name="norm_rope_tokens", op="norm_rope", dtype="bf16", B=8, N=1, heads=20, kv_heads=5, D=64, axes=1, rot=64,
             interleaved=False, train=False),
        # a training batch of 64 x 64 token grids (rows and columns rotate half of the channels each), gradient included
        dict(name="norm_rope_grid_train", op="norm_rope", dtype="bf16", B=4, N=4096, heads=20, kv_heads=20, D=64, axes=2, rot=64,
             interleaved=False, train=True),
        # fp32 mode, an odd token count, neighbouring channels rotated together, a third of the head left unrotated
        dict(name="norm_rope_f32_train", op="norm_rope", dtype="f32", B=3, N=1021, heads=8, kv_heads=8, D=80, axes=1, rot=48,
             interleaved=True, train=True),
        # a short prompt of one request: latency
        dict(name="attn_prompt", op="attn", B=1, N=77, heads=8, kv_heads=2, D=64, mask="causal", docs=1, cap=30.0, bias=False,
             train=False),
        # images of several aspect ratios packed into one row of tokens, every image attends to itself
        dict(name="attn_packed_images", op="attn", B=1, N=9001, heads=10, kv_heads=10, D=64, mask="docs", docs=7, cap=0.0,
             bias=False, train=False),
        # a training step over packed ragged sequences with shared key heads and capped scores
        dict(name="attn_packed_train", op="attn", B=2, N=2111, heads=20, kv_heads=5, D=64, mask="causal_docs", docs=5, cap=20.0,
             bias=False, train=True),
        # a training step whose first 1000 tokens (the condition) are seen by all, scores falling off with the distance
        dict(name="attn_prefix_train", op="attn", B=2, N=4096, heads=8, kv_heads=8, D=80, mask="prefix", docs=1, cap=0.0,
             bias=True, train=True),
        # one request with a long cache, one new token: the split over the keys has to fill the chip
        dict(name="cache_one_request", op="cache", B=1, new=1, cap_rows=16384, longest=16000, heads=20, kv_heads=5, D=64, cap=0.0,
             bias=False),
        # many requests of different lengths: the bandwidth of the cache counts
        dict(name="cache_many_requests", op="cache", B=64, new=1, cap_rows=8192, longest=8191, heads=20, kv_heads=5, D=64,
             cap=30.0, bias=False),
        # one new token of each of 16 requests through a projection, seven adapters among them, some requests without
        dict(name="adapters_tokens", op="adapters", requests=16, rows=1, K=1280, N=1280, adapters=7, rank=16),
        # a few odd short prompts, wide output
        dict(name="adapters_prompts", op="adapters", requests=5, rows=77, K=640, N=5120, adapters=3, rank=8),
        # eight images of 32 x 32 tokens, each with an adapter of its own, through the stacked q / k / v projection
        dict(name="adapters_images", op="adapters", requests=8, rows=1024, K=1280, N=3840, adapters=8, rank=32),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(("norm_rope", "attn", "attn", "cache", "adapters"))
    kv = rng.choice((1, 2, 4, 5, 8))
    if op == "norm_rope":
        D = rng.choice((32, 40, 64, 80, 128, 160))
        axes = rng.choice((1, 1, 2))
        c = dict(op=op, dtype=rng.choice(("bf16", "bf16", "f32")), B=rng.randint(1, 4), N=_log(rng, 1, 4000), kv_heads=kv,
                 heads=kv * rng.choice((1, 1, 2, 4)), D=D, axes=axes, rot=rng.choice((D, D, D // 16 * 8)),
                 interleaved=rng.random() < 0.3, train=rng.random() < 0.5)
        c["heads"] = min(c["heads"], 20 // kv * kv)
        return c
    if op == "attn":
        N = _log(rng, 2, 4000)
        heads = kv * rng.choice((1, 2, 4))
        heads = max(kv, min(heads, int(1.2e8 / (N * N)) // kv * kv))
        return dict(op=op, B=1 if N > 1500 else rng.randint(1, 4), N=N, heads=heads, kv_heads=kv, D=rng.choice((32, 40, 64, 80, 128, 160)),
                    mask=rng.choice(("full", "causal", "docs", "causal_docs", "prefix", "window")), docs=rng.randint(1, max(1, min(9, N // 2))),
                    cap=rng.choice((0.0, 0.0, 15.0, 50.0)), bias=rng.random() < 0.3, train=rng.random() < 0.6)
    if op == "cache":
        rows = _log(rng, 64, 16000)
        return dict(op=op, B=max(1, min(_log(rng, 1, 64), 500000 // rows)), new=rng.choice((1, 1, 1, 2, 5)), cap_rows=rows,
                    longest=max(8, rows - rng.randint(0, rows // 2)), heads=kv * rng.choice((1, 2, 4, 8)), kv_heads=kv,
                    D=rng.choice((32, 40, 64, 80, 128, 160)), cap=rng.choice((0.0, 0.0, 30.0)), bias=rng.random() < 0.3)
    rows = _log(rng, 1, 1024)
    return dict(op=op, requests=rng.randint(1, 8) if rows > 1 else rng.randint(1, 48), rows=rows, K=rng.choice((320, 640, 1280, 2560)),
                N=rng.choice((320, 640, 1280, 1920, 3840)), adapters=rng.randint(1, 8), rank=rng.choice((4, 8, 16, 32, 64)))


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def _dev():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _offsets(c):
    """cumulative token counts of the packed documents of a row; with more than one document, a sixteenth of the row is
    padding behind the last"""
    n = c["docs"]
    used = c["N"] - c["N"] // 16 if n > 1 else c["N"]
    w = [(7 * i) % 5 + 1 for i in range(n)]
    at, off = 0, [0]
    for x in w:
        at += x
        off.append(used * at // sum(w))
    return off


def _prefix(c):
    return min(c["N"], 1000 if c["N"] > 2000 else c["N"] // 3)


_WINDOW = 300


def _row_ranges(c):
    """per query token: the first visible key and the one behind the last (equal: none)"""
    off, N = _offsets(c), c["N"]
    first, behind = [0] * N, [0] * N
    for a, b in zip(off, off[1:]):
        for i in range(a, b):
            first[i], behind[i] = a, b
    if c["mask"] in ("full", "prefix", "causal", "window"):
        first, behind = [0] * N, [N] * N
    if c["mask"] == "prefix":
        behind = [max(i + 1, _prefix(c)) for i in range(N)]
    if c["mask"] in ("causal", "window"):
        behind = [i + 1 for i in range(N)]
    if c["mask"] == "window":
        first = [max(0, i + 1 - _WINDOW) for i in range(N)]
    if c["mask"] == "causal_docs":
        behind = [min(b, i + 1) if b else 0 for i, b in enumerate(behind)]
    return first, behind


def _lens(c):
    """tokens in each request's cache, the new ones included: the first request's is the longest"""
    B = c["B"]
    return [max(c["new"], c["longest"] - (c["longest"] * ((37 * b) % max(B, 2))) // (max(B, 2) + 3)) for b in range(B)]


def _scale(c):
    return 1.0 / math.sqrt(c["D"])


def prepare(case, seed):
    c, dev = case, _dev()
    g = torch.Generator(device=dev).manual_seed(int(seed))
    s = {"case": c}

    def rnd(*shape, dtype=_BF, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale + shift).to(dtype)

    if c["op"] == "norm_rope":
        dt, B, N, H, Hk, D = _DT[c["dtype"]], c["B"], c["N"], c["heads"], c["kv_heads"], c["D"]
        s["q"], s["k"] = rnd(B, N, H * D, dtype=dt, scale=1.5), rnd(B, N, Hk * D, dtype=dt, scale=0.7)
        s["wq"], s["wk"] = rnd(D, dtype=dt, scale=0.1, shift=1.0), rnd(D, dtype=dt, scale=0.1, shift=1.0)
        F = c["rot"] // 2 // c["axes"]
        side = math.isqrt(max(1, N - 1)) + 1
        far = side if c["axes"] == 2 else 32768
        inv = 10000.0 ** (-torch.arange(F, device=dev, dtype=_F64) / F)
        ang = torch.arange(far, device=dev, dtype=_F64)[:, None] * inv
        s["table"] = torch.stack((ang.cos(), ang.sin()), -1).to(_F32).contiguous()
        i = torch.arange(N, device=dev)
        if c["axes"] == 2:
            pos = torch.stack((i // side, i % side), -1).expand(B, N, 2)
        else:
            start = torch.randint(0, far - N + 1, (B, 1), generator=g, device=dev)
            pos = (start + i).unsqueeze(-1)
        s["pos"] = pos.to(torch.int32).contiguous()
        if c["train"]:
            s["gq"], s["gk"] = rnd(B, N, H * D, dtype=dt), rnd(B, N, Hk * D, dtype=dt)
            for n in ("q", "k", "wq", "wk"):
                s[n].requires_grad_(True)
    elif c["op"] == "attn":
        B, N, H, Hk, D = c["B"], c["N"], c["heads"], c["kv_heads"], c["D"]
        s["q"], s["k"], s["v"] = rnd(B, N, H * D, scale=2.0), rnd(B, N, Hk * D), rnd(B, N, Hk * D)
        s["ranges"] = torch.tensor(_row_ranges(c), dtype=torch.int32).t().to(dev).expand(B, N, 2).contiguous()
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=dev, dtype=_F32) / H) if c["bias"] else None
        if c["train"]:
            s["g"] = rnd(B, N, H * D)
            for n in ("q", "k", "v"):
                s[n].requires_grad_(True)
    elif c["op"] == "cache":
        B, H, Hk, D = c["B"], c["heads"], c["kv_heads"], c["D"]
        s["q"] = rnd(B, c["new"], H * D, scale=2.0)
        s["k"], s["v"] = rnd(B, c["cap_rows"], Hk * D), rnd(B, c["cap_rows"], Hk * D)
        s["lens"] = torch.tensor([min(n, c["cap_rows"]) for n in _lens(c)], dtype=torch.int32, device=dev)
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=dev, dtype=_F32) / H) if c["bias"] else None
    else:
        K, N, r, n = c["K"], c["N"], c["rank"], c["adapters"]
        s["x"] = rnd(c["requests"], c["rows"], K)
        s["w"], s["b"] = rnd(N, K, scale=K ** -0.5), rnd(N, dtype=_F32)
        s["down"], s["up"] = rnd(n, r, K, scale=K ** -0.5), rnd(n, N, r, scale=r ** -0.5)
        s["scaling"] = torch.rand(n, generator=g, device=dev) + 0.5
        # every fifth request has no adapter; the others take them in turn, from a start that the seed moves
        pick = (torch.arange(c["requests"], device=dev) + torch.randint(0, n, (1,), generator=g, device=dev)) % n
        s["index"] = torch.where(torch.arange(c["requests"], device=dev) % 5 == 4, -1, pick).to(torch.int32)
    return s


# ----------------------------------------------------------------------------------------------------------------
# plain forms, 32 bits
# ----------------------------------------------------------------------------------------------------------------
def _rotation(s):
    """cosine and sine of each token's pairs, [B, N, 1, rot / 2]"""
    t = s["table"][s["pos"].long()]                      # [B, N, axes, F, 2]
    t = t.reshape(*t.shape[:2], 1, -1, 2)
    return t[..., 0], t[..., 1]


def _rotate(x, cos, sin, rot, interleaved):
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return y


_EPS = 1e-6


def _plain_norm_rope(x, w, s, grad):
    c, D = s["case"], s["case"]["D"]
    cos, sin = _rotation(s)
    xf, wf = x.detach().float().unflatten(-1, (-1, D)), w.detach().float()
    rstd = torch.rsqrt(xf.square().mean(-1, keepdim=True) + _EPS)
    xh = xf * rstd
    y = _rotate(xh * wf, cos, sin, c["rot"], c["interleaved"]).flatten(-2).to(x.dtype)
    if grad is None:
        return (y,)
    gy = _rotate(grad.float().unflatten(-1, (-1, D)), cos, -sin, c["rot"], c["interleaved"])
    dw = (gy * xh).sum((0, 1, 2))
    gx = gy * wf
    dx = rstd * (gx - xh * (gx * xh).mean(-1, keepdim=True))
    return y, dx.flatten(-2).to(x.dtype), dw.to(w.dtype)


def _heads(x, D, group=1):
    """[B, N, H * D] -> f32 [B, H * group, N, D]"""
    x = x.detach().float().unflatten(-1, (-1, D)).transpose(1, 2)
    return x.repeat_interleave(group, 1) if group > 1 else x.contiguous()


def _rows(x, dtype):
    return x.transpose(1, 2).flatten(-2).to(dtype)


def _plain_scores(q, k, c, seen, dist, slopes):
    """masked scores, and the derivative of the capped ones"""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(_scale(c))
    d = None
    if c["cap"]:
        t = torch.tanh(x / c["cap"])
        d = 1.0 - t * t
        x = t * c["cap"]
    if slopes is not None:
        x = x - slopes[:, None, None] * dist
    return x.masked_fill(~seen, -math.inf), d


def _plain_softmax(x):
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    z = e.sum(-1, keepdim=True)
    return e / torch.where(z == 0, 1.0, z)


def _plain_attn(s):
    c, D = s["case"], s["case"]["D"]
    group = c["heads"] // c["kv_heads"]
    j = torch.arange(c["N"], device=s["q"].device)
    seen = ((j >= s["ranges"][..., :1]) & (j < s["ranges"][..., 1:]))[:, None]
    q, k, v = _heads(s["q"], D), _heads(s["k"], D, group), _heads(s["v"], D, group)
    x, d = _plain_scores(q, k, c, seen, (j[:, None] - j).abs().float(), s["slopes"])
    p = _plain_softmax(x)
    del x
    o = torch.matmul(p, v)
    if not c["train"]:
        return {"o": _rows(o, _BF)}
    g = _heads(s["g"], D)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), g)
    dx = torch.matmul(g, v.transpose(-1, -2).contiguous())
    dx = p * (dx - (g * o).sum(-1, keepdim=True)) * _scale(c)
    if d is not None:
        dx = dx * d
    dq = torch.matmul(dx, k)
    dk = torch.matmul(dx.transpose(-1, -2).contiguous(), q)
    dk, dv = (t.unflatten(1, (-1, group)).sum(2) for t in (dk, dv))
    return {"o": _rows(o, _BF), "dq": _rows(dq, _BF), "dk": _rows(dk, _BF), "dv": _rows(dv, _BF)}


def _plain_cache(s):
    c, D = s["case"], s["case"]["D"]
    group = c["heads"] // c["kv_heads"]
    j = torch.arange(c["cap_rows"], device=s["q"].device)
    at = s["lens"].long()[:, None] - c["new"] + torch.arange(c["new"], device=j.device)      # position of each new token
    seen = (j <= at[..., None])[:, None]
    q, k, v = _heads(s["q"], D), _heads(s["k"], D, group), _heads(s["v"], D, group)
    x, _ = _plain_scores(q, k, c, seen, (at[:, None, :, None] - j).abs().float(), s["slopes"])
    return {"o": _rows(torch.matmul(_plain_softmax(x), v), _BF)}


def _plain_adapters(s):
    x = s["x"].float()
    use = (s["index"] >= 0).float() * s["scaling"][s["index"].clamp(min=0).long()]
    down, up = s["down"].float()[s["index"].clamp(min=0).long()], s["up"].float()[s["index"].clamp(min=0).long()]
    y = torch.matmul(x, s["w"].float().t().contiguous()) + s["b"]
    t = torch.matmul(x, down.transpose(-1, -2).contiguous()) * use[:, None, None]
    return {"y": (y + torch.matmul(t, up.transpose(-1, -2).contiguous())).to(_BF)}


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def _run_own(s):
    from lbm_amd import ops
    from lbm_amd.models import layers
    c = s["case"]
    if c["op"] == "norm_rope":
        y = layers.qk_norm_rope(s["q"], s["k"], c["D"], s["wq"], s["wk"], s["table"], s["pos"], eps=_EPS, interleaved=c["interleaved"])
        if not c["train"]:
            return {"q": y[0], "k": y[1]}
        dq, dk, dwq, dwk = torch.autograd.grad(y, (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return {"q": y[0], "k": y[1], "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if c["op"] == "attn":
        o = layers.ranged_attention(s["q"], s["k"], s["v"], c["heads"], c["kv_heads"], c["D"], s["ranges"], cap=c["cap"], slopes=s["slopes"])
        if not c["train"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["g"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "cache":
        return {"o": ops.cached_attn(s["q"], s["k"], s["v"], s["lens"], c["heads"], c["kv_heads"], c["D"], cap=c["cap"], slopes=s["slopes"])}
    return {"y": ops.linear_adapters(s["x"], ops.pack_linear_weight(s["w"], s["b"]), s["down"], s["up"], s["index"], s["scaling"])}


def run(state):
    s = state
    if own:
        return _run_own(s)
    with torch.no_grad():
        op = s["case"]["op"]
        if op == "norm_rope":
            q, k = _plain_norm_rope(s["q"], s["wq"], s, s.get("gq")), _plain_norm_rope(s["k"], s["wk"], s, s.get("gk"))
            out = {"q": q[0], "k": k[0]}
            if s["case"]["train"]:
                out.update(dq=q[1], dk=k[1], dwq=q[2], dwk=k[2])
            return out
        return {"attn": _plain_attn, "cache": _plain_cache, "adapters": _plain_adapters}[op](s)


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "norm_rope":
        e = 2 if c["dtype"] == "bf16" else 4
        n = c["B"] * c["N"] * (c["heads"] + c["kv_heads"]) * c["D"]
        tokens = c["B"] * c["N"]
        side = math.isqrt(max(1, c["N"] - 1)) + 1
        table = min(tokens, side if c["axes"] == 2 else tokens) * c["rot"] // c["axes"] * 4
        # forward: read and write q, k; with the gradient: read them and the output gradients again, write theirs
        return {"bytes": n * e * (5 if c["train"] else 2) + tokens * 4 * c["axes"] + table, "flops": n * (25 if c["train"] else 8)}
    if c["op"] == "attn":
        first, behind = _row_ranges(c)
        pairs = c["B"] * sum(max(0, b - a) for a, b in zip(first, behind))
        q, k = c["B"] * c["N"] * c["heads"] * c["D"] * 2, c["B"] * c["N"] * c["kv_heads"] * c["D"] * 2
        one = 2.0 * pairs * c["heads"] * c["D"]
        if c["train"]:      # forward two products, backward five; q, k, v, o, its gradient in, three gradients and o out
            return {"bytes": 4 * q + 4 * k + c["B"] * c["N"] * 8, "flops": 7 * one}
        return {"bytes": 2 * q + 2 * k + c["B"] * c["N"] * 8, "flops": 2 * one}
    if c["op"] == "cache":
        rows = sum(min(n, c["cap_rows"]) for n in _lens(c))
        return {"bytes": rows * c["kv_heads"] * c["D"] * 4 + 4 * c["B"] * c["new"] * c["heads"] * c["D"],
                "flops": 4.0 * rows * c["new"] * c["heads"] * c["D"]}
    T, K, N, r = c["requests"] * c["rows"], c["K"], c["N"], c["rank"]
    with_one = T * (c["requests"] - c["requests"] // 5) / c["requests"]
    used = min(c["adapters"], c["requests"] - c["requests"] // 5)
    return {"bytes": 2 * (T * K + N * K + T * N + used * r * (K + N)) + 4 * N, "flops": 2.0 * T * K * N + 2.0 * with_one * r * (K + N)}


# ----------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def _exact_norm_rope(s):
    c, D = s["case"], s["case"]["D"]
    half, per = c["rot"] // 2, c["rot"] // 2 // c["axes"]
    # every pair as one complex number times a unit one; the angle's cosine and sine are inputs (the table)
    axis = torch.arange(half, device=s["pos"].device) // per
    unit = torch.view_as_complex(s["table"].double())[s["pos"].long()[..., axis], torch.arange(half, device=axis.device) % per][:, :, None]
    lo = torch.arange(half, device=axis.device) * (2 if c["interleaved"] else 1)
    hi = lo + (1 if c["interleaved"] else half)
    rest = torch.arange(c["rot"], D, device=axis.device)
    order = torch.cat((lo, hi, rest))
    leaves = [s[n].detach().double().requires_grad_(c["train"]) for n in ("q", "k", "wq", "wk")]
    out = []
    for x, w in ((leaves[0], leaves[2]), (leaves[1], leaves[3])):
        x = x.view(*x.shape[:2], -1, D)
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + _EPS) * w
        z = torch.complex(y[..., lo], y[..., hi]) * unit
        y = torch.cat((z.real, z.imag, y[..., rest]), -1)[..., torch.argsort(order)]
        out.append(y.reshape(*y.shape[:2], -1))
    if not c["train"]:
        return {"q": out[0], "k": out[1]}
    d = torch.autograd.grad(out, leaves, (s["gq"].double(), s["gk"].double()))
    return {"q": out[0].detach(), "k": out[1].detach(), "dq": d[0], "dk": d[1], "dwq": d[2], "dwk": d[3]}


def _exact_attn_row(c, q, k, v, slopes, at, seen):
    """one request: q [n, H, D], k / v [N, Hk, D] in 64 bits, ``at`` the new tokens' positions, ``seen`` [n, N]"""
    n, H, D = q.shape
    Hk = k.shape[1]
    qg = q.reshape(n, Hk, H // Hk, D).permute(1, 2, 0, 3).reshape(Hk, -1, D)                    # heads of a group stacked as rows
    x = torch.bmm(qg, k.permute(1, 2, 0).contiguous()).reshape(H, n, -1) / math.sqrt(D)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if slopes is not None:
        j = torch.arange(k.shape[0], device=q.device)
        x = x - slopes.double()[:, None, None] * (at[:, None] - j).abs()
    x = torch.where(seen, x, torch.full_like(x, -1e300))
    p = torch.softmax(x, -1) * seen.any(-1)[:, None]
    o = torch.bmm(p.reshape(Hk, -1, p.shape[-1]), v.permute(1, 0, 2).contiguous()).reshape(H, n, D)
    return o.permute(1, 0, 2)


def _exact_attn(s):
    c, D = s["case"], s["case"]["D"]
    N, dev = c["N"], s["q"].device
    i = torch.arange(N, device=dev)
    doc = torch.full((N,), -1, device=dev)
    for n, (a, b) in enumerate(zip(_offsets(c), _offsets(c)[1:])):
        doc[a:b] = n
    seen = {"full": lambda: torch.ones(N, N, dtype=torch.bool, device=dev),
            "causal": lambda: i <= i[:, None],
            "window": lambda: (i <= i[:, None]) & (i[:, None] - i < _WINDOW),
            "prefix": lambda: (i <= i[:, None]) | (i < _prefix(c)),
            "docs": lambda: (doc[:, None] == doc) & (doc >= 0),
            "causal_docs": lambda: (doc[:, None] == doc) & (doc >= 0) & (i <= i[:, None])}[c["mask"]]()
    got = []
    for b in range(c["B"]):
        q, k, v = (s[n][b].detach().double().view(N, -1, D).requires_grad_(c["train"]) for n in ("q", "k", "v"))
        o = _exact_attn_row(c, q, k, v, s["slopes"], i, seen)
        d = torch.autograd.grad(o, (q, k, v), s["g"][b].double().view(N, -1, D)) if c["train"] else ()
        got.append([t.detach().reshape(N, -1) for t in (o, *d)])
    return {n: torch.stack(t) for n, t in zip(("o", "dq", "dk", "dv"), zip(*got))}


def _exact_cache(s):
    c, D = s["case"], s["case"]["D"]
    out = []
    for b in range(c["B"]):
        n = int(s["lens"][b])
        at = torch.arange(n - c["new"], n, device=s["q"].device)
        q, k, v = s["q"][b].double().view(-1, c["heads"], D), s["k"][b, :n].double().view(n, -1, D), s["v"][b, :n].double().view(n, -1, D)
        out.append(_exact_attn_row(c, q, k, v, s["slopes"], at, torch.arange(n, device=at.device) <= at[:, None]).reshape(c["new"], -1))
    return {"o": torch.stack(out)}


def _exact_adapters(s):
    w, out = s["w"].double().t().contiguous(), []
    for x, a in zip(s["x"].double(), s["index"].tolist()):
        y = x @ w + s["b"].double()
        if a >= 0:      # the adapter as the change of the weight that it stands for
            y = y + x @ (s["scaling"][a].double() * (s["up"][a].double() @ s["down"][a].double())).t().contiguous()
        out.append(y)
    return {"y": torch.stack(out)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "attn": _exact_attn, "cache": _exact_cache, "adapters": _exact_adapters}[case["op"]](s)
