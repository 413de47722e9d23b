"""Attention over key ranges (ops.ranged_attn, its backward, layers.ranged_attention, ops.key_ranges) and over a cache
(ops.cached_attn) against the definition in 64 bits.

Tolerances, element by element.  Roundings to bf16 are off by at most half a step, H = 2^-8 of the value: of each probability
before P V (adds H sum p|v|), of each dS before dS K and dS^T Q, of P before P^T dO, and of each output.  The exponent of a
probability is a f32 sum of D products, mapped by a few f32 operations: its error is below (D + 32) * 2^-24 * (1 + the sum of
the products' magnitudes, or the cap, or the bias), which is at most E = 2^-12 for the inputs here (sums of magnitudes below
100), and a probability is off by twice that (its own and the row sum's).  delta = dO.o is taken from the rounded o: it is off by
at most sum |dO| times o's tolerance."""
import math

import pytest
import torch

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
H8, E = 2.0 ** -8, 2.0 ** -12


def heads_of(x, D, group=1):
    x = x.double().unflatten(-1, (-1, D)).transpose(1, 2)
    return x.repeat_interleave(group, 1)


def rows_of(x):
    return x.transpose(1, 2).flatten(-2)


def definition(q, k, v, H, Hk, D, seen, pos, scale, cap, slopes, g=None):
    """outputs, gradients and their tolerances in 64 bits; seen [B, Nq, Nk], pos [B, Nq]"""
    group = H // Hk
    q, k, v = heads_of(q, D), heads_of(k, D, group), heads_of(v, D, group)
    x = q @ k.transpose(-1, -2) * scale
    fac = torch.ones_like(x)
    if cap:
        t = torch.tanh(x / cap)
        x, fac = cap * t, 1 - t * t
    if slopes is not None:
        x = x - slopes.double()[:, None, None] * (pos[:, None, :, None] - torch.arange(k.shape[2])).abs()
    seen = seen[:, None]
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True) if x.shape[-1] else x.new_zeros(*x.shape[:-1], 1)
    p = torch.exp(x - m.masked_fill(m == -math.inf, 0.0)).masked_fill(~seen, 0.0)
    z = p.sum(-1, keepdim=True)
    p = p / z.masked_fill(z == 0, 1.0)
    o = p @ v
    to = (H8 + 2 * E) * (p @ v.abs()) + H8 * o.abs() + 1e-30
    out = {"o": (rows_of(o), rows_of(to))}
    if g is None:
        return out
    g = heads_of(g, D)
    dp, delta = g @ v.transpose(-1, -2), (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * fac
    tds = (H8 + 4 * E) * ds.abs() + p * fac * (g.abs() * to).sum(-1, keepdim=True) + 4 * E * p * (dp.abs() + delta.abs())
    fold = lambda t: t.unflatten(1, (-1, group)).sum(2)  # noqa: E731
    dq, tq = ds @ k * scale, tds @ k.abs() * scale
    dk, tk = fold(ds.transpose(-1, -2) @ q) * scale, fold(tds.transpose(-1, -2) @ q.abs()) * scale
    dv, tv = fold(p.transpose(-1, -2) @ g), fold(((H8 + 2 * E) * p).transpose(-1, -2) @ g.abs())
    for n, d, t in (("dq", dq, tq), ("dk", dk, tk), ("dv", dv, tv)):
        out[n] = rows_of(d), rows_of(t + H8 * d.abs() + 1e-30)
    return out


def check(name, got, want):
    ref, tol = want
    off = (got.double().cpu() - ref).abs()
    assert bool((off <= tol).all()), (name, float((off / tol).max()))


def ranges_of(kind, B, Nq, Nk, gen):
    i = torch.arange(Nq) + Nk - Nq
    lo, hi = torch.zeros(B, Nq, dtype=torch.long), torch.full((B, Nq), Nk)
    if kind == "causal":
        hi = (i + 1).clamp(0, Nk).expand(B, Nq)
    elif kind == "window":
        lo, hi = (i - 6).clamp(min=0).expand(B, Nq), (i + 1).clamp(0, Nk).expand(B, Nq)
    elif kind == "random":          # any intervals, in no order, a fifth of them empty or upside down
        lo, hi = torch.randint(0, Nk + 1, (B, Nq), generator=gen), torch.randint(0, Nk + 1, (B, Nq), generator=gen)
        flip = torch.rand(B, Nq, generator=gen) < 0.8
        lo, hi = torch.where(flip, torch.minimum(lo, hi), lo), torch.where(flip, torch.maximum(lo, hi), hi)
    elif kind == "docs":
        cut = max(1, Nk // 3)
        lo = (i // cut * cut).expand(B, Nq)
        hi = (i // cut * cut + cut).clamp(max=Nk).expand(B, Nq)
    elif kind == "beyond":          # clipped to the keys
        lo, hi = torch.full((B, Nq), -7), torch.full((B, Nq), 2 ** 31 - 1)
    return torch.stack((lo, hi), -1).to(I32).contiguous()


def seen_by(ranges, Nk):
    j = torch.arange(Nk)
    return (j >= ranges[..., :1]) & (j < ranges[..., 1:])


def make(seed, B, Nq, Nk, H, Hk, D):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    return r(B, Nq, H * D), r(B, Nk, Hk * D), r(B, Nk, Hk * D), r(B, Nq, H * D), g


CASES = [  # B, Nq, Nk, H, Hk, D, mask, cap, bias
    (1, 1, 1, 1, 1, 64, "none", 0.0, False),
    (2, 2, 2, 2, 1, 64, "causal", 0.0, False),
    (1, 31, 31, 2, 2, 64, "causal", 5.0, False),
    (1, 63, 63, 1, 1, 64, "none", 0.0, True),
    (1, 64, 64, 2, 1, 64, "causal", 0.0, True),
    (2, 65, 65, 4, 2, 64, "docs", 0.0, False),
    (1, 127, 127, 2, 2, 64, "random", 3.0, True),
    (1, 129, 129, 2, 2, 64, "window", 0.0, False),
    (2, 333, 333, 4, 1, 64, "random", 0.0, False),
    (1, 300, 300, 6, 2, 64, "beyond", 0.0, False),
    (1, 5, 200, 2, 2, 64, "causal", 0.0, True),          # the last queries of a longer row of keys
    (1, 200, 5, 2, 1, 64, "causal", 0.0, False),         # queries in front of the first key see nothing
    (1, 130, 77, 2, 2, 64, "none", 2.0, False),
    (1, 77, 130, 3, 3, 8, "random", 0.0, False),
    (1, 77, 77, 2, 2, 32, "causal", 0.0, True),
    (2, 129, 129, 2, 1, 40, "docs", 4.0, False),
    (1, 150, 150, 2, 2, 72, "random", 0.0, True),
    (1, 200, 200, 4, 2, 80, "causal", 0.0, False),
    (1, 140, 140, 2, 1, 96, "random", 0.0, False),
    (1, 200, 200, 2, 2, 128, "causal", 3.0, False),
    (1, 135, 135, 2, 1, 136, "random", 0.0, False),
    (1, 200, 200, 2, 1, 160, "docs", 0.0, True),
    (1, 700, 700, 2, 1, 64, "causal", 0.0, False),       # the keys' gradients in several parts
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(cuda, case):
    from lbm_amd import ops
    B, Nq, Nk, H, Hk, D, mask, cap, bias = case
    q, k, v, g, gen = make(1, B, Nq, Nk, H, Hk, D)
    ranges = None if mask == "none" else ranges_of(mask, B, Nq, Nk, gen)
    slopes = 2.0 ** -torch.arange(1, H + 1, dtype=F32) if bias else None
    seen = torch.ones(B, Nq, Nk, dtype=torch.bool) if ranges is None else seen_by(ranges, Nk)
    pos = (torch.arange(Nq) + Nk - Nq).expand(B, Nq)
    want = definition(q, k, v, H, Hk, D, seen, pos, D ** -0.5, cap, slopes, g)
    dev = [None if t is None else t.to(cuda) for t in (q, k, v, g, ranges, slopes)]
    kw = dict(cap=cap, slopes=dev[5])
    o, lse = ops.ranged_attn(*dev[:3], H, Hk, D, dev[4], return_lse=True, **kw)
    check("o", o, want["o"])
    assert torch.equal(o, ops.ranged_attn(*dev[:3], H, Hk, D, dev[4], **kw))
    assert torch.equal(torch.isinf(lse).cpu(), ~seen.any(-1)[:, None].expand(B, H, Nq))
    grads = ops.ranged_attn_bwd(*dev[:3], o, dev[3], lse, H, Hk, D, dev[4], **kw)
    for n, x in zip(("dq", "dk", "dv"), grads):
        check(n, x, want[n])
    for a, b in zip(grads, ops.ranged_attn_bwd(*dev[:3], o, dev[3], lse, H, Hk, D, dev[4], **kw)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk,H,D,mask,times", [
    (700, 4200, 2, 64, "random", (1, 30, 70)),           # 24, 720 and 1680 workgroups
    (700, 4200, 2, 64, "docs", (1, 30, 70)),
    (300, 4300, 2, 40, "causal", (1, 50)),
    (300, 4200, 2, 96, "docs", (1, 50)),
    (260, 4200, 1, 128, "random", (1, 90, 170)),
    (260, 4200, 1, 160, "random", (1, 90)),
    (200, 4200, 2, 32, "random", (1, 100)),
])
def test_ranked_workgroups_over_long_rows(cuda, Nq, Nk, H, D, mask, times):
    """with few heads against the definition; the same heads many times over take other workgroups in another order, and each of
    them has the same bits (the keys' gradients are cut into other parts: against the definition again)"""
    from lbm_amd import ops
    q, k, v, g, gen = make(9, 1, Nq, Nk, H, H, D)
    ranges = ranges_of(mask, 1, Nq, Nk, gen)
    want = definition(q, k, v, H, H, D, seen_by(ranges, Nk), (torch.arange(Nq) + Nk - Nq).expand(1, Nq), D ** -0.5, 0.0, None, g)
    q, k, v, g, ranges = (t.to(cuda) for t in (q, k, v, g, ranges))
    first = None
    for n in times:
        a, b, c, d = (t.repeat(1, 1, n) for t in (q, k, v, g))
        o, lse, rest = ops.ranged_attn(a, b, c, n * H, n * H, D, ranges, return_lse=True, return_rest=True)
        got = (o,) + ops.ranged_attn_bwd(a, b, c, o, d, lse, n * H, n * H, D, ranges, rest=rest)
        first = first or got
        for name, x, y in zip(("o", "dq", "dk", "dv"), got, first):
            for part in (x[..., :H * D], x[..., -H * D:]):
                check(name, part, want[name])
            if name in ("o", "dq"):
                assert torch.equal(x, y.repeat(1, 1, n)), (name, n)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [40, 64, 128, 160])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_at_places_that_are_not_seen(cuda, D, value):
    """padding between and behind documents, and later tokens under a causal mask, may hold anything"""
    from lbm_amd import ops
    B, N, H, Hk = 1, 200, 2, 1
    q, k, v, g, _ = make(2, B, N, N, H, Hk, D)
    ranges = torch.zeros(B, N, 2, dtype=I32)
    pad = torch.zeros(N, dtype=torch.bool)
    for a, b, end in ((0, 45, 50), (50, 120, 130), (130, 190, 200)):
        for i in range(a, b):
            ranges[0, i] = torch.tensor([a, i + 1])
        pad[b:end] = True
    clean = [t.clone() for t in (q, k, v, g)]
    for t in clean:
        t[:, pad] = 0
    for t in (q, k, v, g):
        t[:, pad] = value
    slopes = torch.tensor([0.5, 0.25])
    seen = seen_by(ranges, N)
    want = definition(*clean[:3], H, Hk, D, seen, torch.arange(N).expand(B, N), D ** -0.5, 9.0, slopes, clean[3])
    dev = [t.to(cuda) for t in (q, k, v, g, ranges, slopes)]
    o, lse = ops.ranged_attn(*dev[:3], H, Hk, D, dev[4], cap=9.0, slopes=dev[5], return_lse=True)
    check("o", o, want["o"])
    assert bool((o[:, pad.to(cuda)] == 0).all())
    grads = ops.ranged_attn_bwd(*dev[:3], o, dev[3], lse, H, Hk, D, dev[4], cap=9.0, slopes=dev[5])
    for n, x in zip(("dq", "dk", "dv"), grads):
        check(n, x, want[n])
        assert bool((x[:, pad.to(cuda)] == 0).all()), n

    # one bad value at a place that later rows see: rows in front of it keep their results, rows that see it are not finite
    q, k, v, g = clean
    v2, k2, g2 = v.clone(), k.clone(), g.clone()
    v2[0, 60, 3] = value
    o2 = ops.ranged_attn(q.to(cuda), k.to(cuda), v2.to(cuda), H, Hk, D, dev[4])
    ref = definition(q, k, v, H, Hk, D, seen, torch.arange(N).expand(B, N), D ** -0.5, 0.0, None)["o"]
    o2 = o2.cpu().view(B, N, H, D)
    hit = torch.zeros(B, N, H, D, dtype=torch.bool)
    hit[:, 60:120, :, 3] = True
    assert not bool(torch.isfinite(o2[hit]).any())
    off = (o2.double() - ref[0].view(B, N, H, D)).abs()
    assert bool((off <= ref[1].view(B, N, H, D))[~hit].all())
    # a key of NaN: only rows that see it
    k2[0, 60] = float("nan")
    o3 = ops.ranged_attn(q.to(cuda), k2.to(cuda), v.to(cuda), H, Hk, D, dev[4]).cpu().view(B, N, H, D)
    hit[:, 60:120] = True
    assert bool(torch.isnan(o3[hit]).all()) and bool((o3.double() - ref[0].view(B, N, H, D)).abs()[~hit].le(ref[1].view(B, N, H, D)[~hit]).all())
    # a bad output gradient of one row reaches the keys it sees, and no other
    good = ops.ranged_attn(q.to(cuda), k.to(cuda), v.to(cuda), H, Hk, D, dev[4], return_lse=True)
    g2[0, 60] = value
    dq, dk, dv = (x.cpu() for x in ops.ranged_attn_bwd(q.to(cuda), k.to(cuda), v.to(cuda), good[0], g2.to(cuda), good[1], H, Hk, D, dev[4]))
    rows = torch.arange(N)
    reach = (rows >= 50) & (rows <= 60)
    assert not bool(torch.isfinite(dv[0, reach]).any()) and bool(torch.isfinite(dv[0, ~reach]).all()) and bool(torch.isfinite(dk[0, ~reach]).all())
    assert bool(torch.isfinite(dq[0, rows != 60]).all())


@pytest.mark.gpu
def test_windows_of_a_packed_projection_and_broadcast_keys(cuda):
    from lbm_amd import ops
    B, N, H, Hk, D = 2, 130, 4, 2, 64
    q, k, v, g, gen = make(3, B, N, N, H, Hk, D)
    packed = torch.cat((k, q, v), -1).to(cuda)
    pk, pq, pv = packed.split((Hk * D, H * D, Hk * D), -1)
    ranges = ranges_of("random", B, N, N, gen).to(cuda)
    o, lse = ops.ranged_attn(q.to(cuda), k.to(cuda), v.to(cuda), H, Hk, D, ranges, return_lse=True)
    o2, lse2 = ops.ranged_attn(pq, pk, pv, H, Hk, D, ranges, return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    wide = torch.zeros(B, N, 2 * H * D, dtype=BF, device=cuda)
    wide[..., H * D:] = g.to(cuda)
    for a, b in zip(ops.ranged_attn_bwd(q.to(cuda), k.to(cuda), v.to(cuda), o, g.to(cuda), lse, H, Hk, D, ranges),
                    ops.ranged_attn_bwd(pq, pk, pv, o, wide[..., H * D:], lse, H, Hk, D, ranges)):
        assert torch.equal(a, b)
    # one set of keys for the whole batch
    o3 = ops.ranged_attn(pq, pk[:1].expand(B, N, -1), pv[:1].expand(B, N, -1), H, Hk, D, ranges)
    o4 = ops.ranged_attn(pq, pk[:1].repeat(B, 1, 1), pv[:1].repeat(B, 1, 1), H, Hk, D, ranges)
    assert torch.equal(o3, o4)


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["none", "causal", "docs"])
def test_slopes_that_favour_far_keys(cuda, mask):
    """a negative slope: scores grow with the distance, far beyond exp2's range for a row that is not there (300 rows end inside a
    tile), and the softmax's maximum alone keeps the others finite"""
    from lbm_amd import ops
    N, H, D = 300, 2, 64
    q, k, v, g, gen = make(11, 1, N, N, H, H, D)
    ranges = None if mask == "none" else ranges_of(mask, 1, N, N, gen)
    seen = torch.ones(1, N, N, dtype=torch.bool) if ranges is None else seen_by(ranges, N)
    slopes = torch.tensor([-1.0, -0.25])
    want = definition(q, k, v, H, H, D, seen, torch.arange(N).expand(1, N), D ** -0.5, 0.0, slopes, g)
    q, k, v, g, slopes = (t.to(cuda) for t in (q, k, v, g, slopes))
    ranges = None if ranges is None else ranges.to(cuda)
    o, lse = ops.ranged_attn(q, k, v, H, H, D, ranges, slopes=slopes, return_lse=True)
    check("o", o, want["o"])
    for n, x in zip(("dq", "dk", "dv"), ops.ranged_attn_bwd(q, k, v, o, g, lse, H, H, D, ranges, slopes=slopes)):
        check(n, x, want[n])


@pytest.mark.gpu
def test_no_queries_no_keys(cuda):
    from lbm_amd import ops
    q, k, v, g, _ = make(4, 2, 9, 6, 2, 1, 64)
    q, k, v, g = (t.to(cuda) for t in (q, k, v, g))
    o, lse = ops.ranged_attn(q, k[:, :0], v[:, :0], 2, 1, 64, return_lse=True)
    assert bool((o == 0).all()) and bool(torch.isinf(lse).all())
    dq, dk, dv = ops.ranged_attn_bwd(q, k[:, :0], v[:, :0], o, g, lse, 2, 1, 64)
    assert bool((dq == 0).all()) and dk.shape == (2, 0, 64)
    o, lse = ops.ranged_attn(q[:, :0], k, v, 2, 1, 64, return_lse=True)
    dq, dk, dv = ops.ranged_attn_bwd(q[:, :0], k, v, o, g[:, :0], lse, 2, 1, 64)
    assert dq.shape == (2, 0, 128) and bool((dk == 0).all()) and bool((dv == 0).all())
    assert ops.ranged_attn(q[:0], k[:0], v[:0], 2, 1, 64).shape == (0, 9, 128)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """2^31 elements between the first and the last key row of a wide packed buffer: byte and element offsets pass 32 bits"""
    from lbm_amd import ops
    N, W, D = 300_000, 8192, 64
    buf = torch.zeros(1, N, W, dtype=BF, device=cuda)
    g = torch.Generator().manual_seed(5)
    kv = torch.randn(1, 100, 2 * D, generator=g).to(BF)
    buf[:, N - 100:, W - 2 * D:] = kv.to(cuda)
    q = torch.randn(1, 3, 2 * D, generator=g).to(BF)
    k, v = buf[..., W - 2 * D:W - D], buf[..., W - D:]
    ranges = torch.tensor([[[N - 100, N], [N - 50, N - 3], [N - 1, N]]], dtype=I32)
    local = (ranges - (N - 100)).clamp(min=0)
    do = torch.randn(1, 3, 2 * D, generator=g).to(BF)
    want = definition(q, kv[..., :D], kv[..., D:], 2, 1, D, seen_by(local, 100), torch.zeros(1, 3), D ** -0.5, 0.0, None, do)
    o, lse = ops.ranged_attn(q.to(cuda), k, v, 2, 1, D, ranges.to(cuda), return_lse=True)
    check("o", o, want["o"])
    dq, dk, dv = ops.ranged_attn_bwd(q.to(cuda), k, v, o, do.to(cuda), lse, 2, 1, D, ranges.to(cuda))
    check("dq", dq, want["dq"])
    check("dk", dk[:, N - 100:], want["dk"])
    check("dv", dv[:, N - 100:], want["dv"])
    assert bool((dk[:, :N - 100] == 0).all())
    lens = torch.tensor([N], dtype=I32, device=cuda)
    seen = seen_by(torch.tensor([[[0, 98], [0, 99], [0, 100]]]), 100)
    want = definition(q, kv[..., :D], kv[..., D:], 2, 1, D, seen & (torch.arange(100) >= torch.tensor([48, 49, 50])[:, None]), torch.zeros(1, 3), D ** -0.5, 0.0, None)
    check("o", ops.cached_attn(q.to(cuda), k, v, lens, 2, 1, D, window=50), want["o"])


@pytest.mark.gpu
def test_autograd_against_differences_and_scalar_gradients(cuda):
    """central differences of the 64-bit definition along random directions (their own error is below 1e-6 of the value);
    the kernel's gradients may be off by the sum of their tolerances times the direction"""
    from lbm_amd.models import layers
    B, N, H, Hk, D = 1, 90, 4, 2, 64
    q, k, v, g, gen = make(6, B, N, N, H, Hk, D)
    ranges = ranges_of("causal", B, N, N, gen)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625])
    seen, pos = seen_by(ranges, N), torch.arange(N).expand(B, N)
    leaves = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    o = layers.ranged_attention(*leaves, H, Hk, D, ranges.to(cuda), cap=4.0, slopes=slopes.to(cuda))
    grads = torch.autograd.grad(o, leaves, g.to(cuda))
    want = definition(q, k, v, H, Hk, D, seen, pos, D ** -0.5, 4.0, slopes, g)
    base = [t.double() for t in (q, k, v)]

    def value(q, k, v):
        return float((definition(q, k, v, H, Hk, D, seen, pos, D ** -0.5, 4.0, slopes)["o"][0] * g.double()).sum())
    h = 1e-4
    for i, (n, x) in enumerate(zip(("dq", "dk", "dv"), grads)):
        u = torch.randn(base[i].shape, generator=gen, dtype=F64)
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * u, base[i] - h * u
        diff = (value(*up) - value(*dn)) / (2 * h)
        room = float((want[n][1] * u.abs()).sum()) + 1e-5 * float((want[n][0] * u).abs().sum())
        assert abs(float((x.double().cpu() * u).sum()) - diff) <= room, n
    layers.ranged_attention(*leaves, H, Hk, D, ranges.to(cuda)).float().sum().backward()
    assert all(bool(torch.isfinite(t.grad).all()) for t in leaves)
    with torch.no_grad():
        assert not layers.ranged_attention(*leaves, H, Hk, D).requires_grad
    with pytest.raises(NotImplementedError, match="slopes"):
        layers.ranged_attention(*leaves, H, Hk, D, slopes=slopes.to(cuda).requires_grad_(True))


@pytest.mark.gpu
def test_graph_replay_and_side_stream(cuda):
    from lbm_amd import ops
    B, N, H, Hk, D = 1, 300, 4, 2, 64
    q, k, v, g, gen = make(7, B, N, N, H, Hk, D)
    q, k, v, g = (t.to(cuda) for t in (q, k, v, g))
    docs = torch.tensor([0, 90, 200, 290], dtype=I32, device=cuda)
    lens = torch.tensor([300], dtype=I32, device=cuda)

    def all_of():
        r = ops.key_ranges(B, N, causal=True, documents=docs)
        o, lse = ops.ranged_attn(q, k, v, H, Hk, D, r, cap=5.0, return_lse=True)
        return (o, lse) + ops.ranged_attn_bwd(q, k, v, o, g, lse, H, Hk, D, r, cap=5.0) + (ops.cached_attn(q[:, :2], k, v, lens, H, Hk, D),)
    all_of()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_of()
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(BF))
        docs[1] = 50 + 20 * n
        lens[0] = 300 - 100 * n
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, all_of()):
            assert torch.equal(a, b), n
    want = all_of()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


# ---- ranges --------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk", [(1, 1), (50, 50), (7, 60), (60, 7)])
@pytest.mark.parametrize("kind", ["full", "causal", "window", "docs", "causal_docs", "prefix", "prefix_docs", "lens", "causal_lens", "docs_per_row"])
def test_key_ranges(cuda, Nq, Nk, kind):
    from lbm_amd import ops
    B = 3
    docs = torch.tensor([[2, 2, 9, 30, 33], [0, 1, 1, 1, 40], [5, 5, 5, 5, 5]], dtype=I32)
    lens = torch.tensor([0, 6, 1000], dtype=I32)
    prefix = torch.tensor([0, 4, 1000], dtype=I32)
    kw, one = {}, docs[0]
    if "docs" in kind:
        kw["documents"] = docs if kind == "docs_per_row" else one
    if kind.startswith("causal") or kind.startswith("prefix") or kind == "window":
        kw["causal"] = True
    if kind.startswith("prefix"):
        kw["prefix"] = prefix
    if kind == "window":
        kw["window"] = 5
    if "lens" in kind:
        kw["lens"] = lens
    got = ops.key_ranges(B, Nq, Nk, **{n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in kw.items()}, device=cuda).cpu()
    p, j = torch.arange(Nq) + Nk - Nq, torch.arange(Nk)
    for b in range(B):
        seen = torch.ones(Nq, Nk, dtype=torch.bool) & (p >= 0)[:, None]
        start = torch.zeros(Nq, dtype=torch.long)
        if "documents" in kw:
            off = (docs[b] if kind == "docs_per_row" else one).tolist()
            doc = lambda x: torch.tensor([next((n for n in range(4) if off[n] <= t < off[n + 1]), -1) for t in x.tolist()])  # noqa: E731
            dp, dj = doc(p), doc(j)
            seen &= (dp[:, None] == dj) & (dp >= 0)[:, None]
            start = torch.tensor([off[n] if n >= 0 else 0 for n in dp.tolist()])
        if kw.get("causal"):
            late = j > p[:, None]
            if "prefix" in kw:
                late &= j >= (start + int(prefix[b]))[:, None]
            seen &= ~late
        if "window" in kw:
            seen &= j > p[:, None] - 5
        if "lens" in kw:
            seen &= j < int(lens[b])
        assert torch.equal(seen_by(got[b], Nk), seen), b
        assert bool((got[b] >= 0).all()) and bool((got[b] <= Nk).all())


# ---- cache ---------------------------------------------------------------------------------------------------------
CACHE = [  # B, n, rows, H, Hk, D, lens, cap, bias, window
    (1, 1, 1, 1, 1, 64, [1], 0.0, False, 0),
    (3, 1, 40, 4, 2, 64, [0, 1, 40], 0.0, False, 0),
    (2, 1, 700, 8, 1, 64, [700, 33], 4.0, True, 0),
    (2, 1, 3000, 20, 5, 64, [2999, 517], 0.0, False, 0),         # several parts, one of them short
    (2, 3, 900, 4, 2, 64, [900, 2], 0.0, True, 0),               # a token in front of the cache's start
    (1, 5, 600, 40, 5, 64, [599], 3.0, False, 0),                # 40 rows per key head: two row blocks
    (2, 1, 2000, 4, 4, 64, [1999, 1024], 0.0, False, 100),
    (2, 4, 2000, 4, 4, 64, [1999, 3], 0.0, False, 7),
    (2, 1, 300, 2, 2, 8, [300, 129], 0.0, False, 0),
    (2, 1, 300, 4, 2, 32, [300, 129], 0.0, True, 0),
    (1, 2, 300, 8, 8, 40, [257], 0.0, False, 0),
    (1, 1, 1500, 8, 2, 80, [1490], 2.0, False, 0),
    (1, 2, 1500, 4, 2, 128, [1500], 0.0, True, 0),
    (2, 1, 1500, 4, 1, 160, [1500, 8], 0.0, False, 0),
    (2, 1, 64, 2, 1, 64, [5000, -3], 0.0, False, 0),             # lengths outside the cache are clipped
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CACHE, ids=lambda c: "-".join(map(str, c)))
def test_cache(cuda, case):
    from lbm_amd import ops
    B, n, rows, H, Hk, D, lens, cap, bias, window = case
    q, k, v, _, gen = make(8, B, n, rows, H, Hk, D)
    slopes = 2.0 ** -torch.arange(1, H + 1, dtype=F32) / 8 if bias else None
    real = torch.tensor([min(max(x, 0), rows) for x in lens])
    j = torch.arange(rows)
    pos = real[:, None] - n + torch.arange(n)
    seen = j <= pos[..., None]
    if window:
        seen &= j > pos[..., None] - window
    want = definition(q, k, v, H, Hk, D, seen, pos, D ** -0.5, cap, slopes)["o"]
    behind = j >= real[:, None]
    k[behind], v[behind] = float("nan"), float("inf")            # rows behind the last token are not read
    # both caches as columns of one wider buffer
    both = torch.full((B, rows, 2 * Hk * D + 24), float("nan"), dtype=BF)
    both[..., :Hk * D], both[..., Hk * D + 8:2 * Hk * D + 8] = k, v
    both = both.to(cuda)
    ks, vs = both[..., :Hk * D], both[..., Hk * D + 8:2 * Hk * D + 8]
    ln = torch.tensor(lens, dtype=I32, device=cuda)
    args = (ln, H, Hk, D)
    kw = dict(cap=cap, slopes=None if slopes is None else slopes.to(cuda), window=window)
    o = ops.cached_attn(q.to(cuda), ks, vs, *args, **kw)
    check("o", o, want)
    assert torch.equal(o, ops.cached_attn(q.to(cuda), k.to(cuda), v.to(cuda), *args, **kw))
    assert bool((o.cpu()[~seen.any(-1)] == 0).all())


@pytest.mark.gpu
def test_cache_agrees_with_the_whole_row_and_hides_later_tokens(cuda):
    from lbm_amd import ops
    B, n, H, Hk, D = 2, 6, 4, 2, 64
    q, k, v, _, _ = make(9, B, n, 500, H, Hk, D)
    lens = torch.tensor([500, 260], dtype=I32)
    v[0, 497, 2], k[1, 257] = float("nan"), float("inf")         # the third newest token of each request
    o = ops.cached_attn(q.to(cuda), k.to(cuda), v.to(cuda), lens.to(cuda), H, Hk, D).cpu()
    assert bool(torch.isfinite(o[0, :3]).all()) and bool(torch.isnan(o[0, 3:].view(3, H, D)[:, :2, 2]).all())
    assert bool(torch.isfinite(o[1, :3]).all()) and not bool(torch.isfinite(o[1, 3:]).any())
    v[0, 497, 2], k[1, 257] = 0.0, 0.0
    want = definition(q, k, v, H, Hk, D, torch.arange(500) <= (lens[:, None] - n + torch.arange(n))[..., None],
                      lens[:, None] - n + torch.arange(n), D ** -0.5, 0.0, None)["o"]
    for b in range(B):
        L = int(lens[b])
        r = ops.key_ranges(1, n, L, causal=True, device=cuda)
        check("row", ops.ranged_attn(q[b:b + 1].to(cuda), k[b:b + 1, :L].to(cuda), v[b:b + 1, :L].to(cuda), H, Hk, D, r),
              [t[b:b + 1] for t in want])
    check("cache", ops.cached_attn(q.to(cuda), k.to(cuda), v.to(cuda), lens.to(cuda), H, Hk, D), want)
    assert ops.cached_attn(q[:, :0].to(cuda), k.to(cuda), v.to(cuda), lens.to(cuda), H, Hk, D).shape == (2, 0, H * D)
    assert bool((ops.cached_attn(q.to(cuda), k[:, :0].to(cuda), v[:, :0].to(cuda), lens.to(cuda), H, Hk, D) == 0).all())


# ---- refusals ------------------------------------------------------------------------------------------------------
def _ranged():
    return dict(q=torch.zeros(2, 5, 128, dtype=BF), k=torch.zeros(2, 7, 64, dtype=BF), v=torch.zeros(2, 7, 64, dtype=BF), heads=2, kv_heads=1,
                head_dim=64, ranges=torch.zeros(2, 5, 2, dtype=I32))


REFUSED = [
    (dict(q=torch.zeros(2, 5, 128)), "float32"),
    (dict(k=torch.zeros(2, 7, 64, dtype=torch.half)), "float16"),
    (dict(q=torch.zeros(5, 128, dtype=BF)), "expected"),
    (dict(k=torch.zeros(3, 7, 64, dtype=BF)), "expected"),
    (dict(v=torch.zeros(2, 8, 64, dtype=BF)), "k "),
    (dict(heads=3), "channels"),
    (dict(heads=0), "heads"),
    (dict(heads=2, kv_heads=3), "over 3 key heads"),
    (dict(head_dim=12), "head_dim 12"),
    (dict(head_dim=168), "head_dim 168"),
    (dict(q=torch.zeros(2, 128, 5, dtype=BF).transpose(1, 2)), "adjacent"),
    (dict(k=torch.zeros(2, 7, 65, dtype=BF)[..., 1:]), "16 bytes"),
    (dict(ranges=torch.zeros(2, 5, 2, dtype=torch.long)), "ranges"),
    (dict(ranges=torch.zeros(2, 7, 2, dtype=I32)), "ranges"),
    (dict(ranges=torch.zeros(2, 2, 5, dtype=I32).transpose(1, 2)), "ranges"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(cap=-1.0), "cap"), (dict(cap=float("inf")), "cap"),
    (dict(slopes=torch.zeros(3)), "slopes"), (dict(slopes=torch.zeros(2, dtype=BF)), "slopes"),
]


@pytest.mark.parametrize("change,text", REFUSED, ids=range(len(REFUSED)))
def test_refusals(change, text):
    from lbm_amd import ops
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.ranged_attn(**_ranged())
    with pytest.raises(ValueError, match=text):
        ops.ranged_attn(**{**_ranged(), **change})
    if not any(n in change for n in ("ranges",)):
        a = {**_ranged(), **change}
        a.pop("ranges")
        a["k_cache"], a["v_cache"], a["lens"] = a.pop("k"), a.pop("v"), torch.zeros(2, dtype=I32)
        with pytest.raises(ValueError, match=text.replace("k ", "k_cache ")):
            ops.cached_attn(**a)


def test_refusals_of_the_backward_the_cache_and_the_ranges():
    from lbm_amd import ops
    a = _ranged()
    b = dict(a, o=torch.zeros(2, 5, 128, dtype=BF), do=torch.zeros(2, 5, 128, dtype=BF), lse=torch.zeros(2, 2, 5))
    c = dict(q=a["q"], k_cache=a["k"], v_cache=a["v"], lens=torch.zeros(2, dtype=I32), heads=2, kv_heads=1, head_dim=64)
    for change, text in ((dict(lens=torch.zeros(2, dtype=torch.long)), "lens"), (dict(lens=torch.zeros(3, dtype=I32)), "lens"), (dict(window=-1), "window")):
        with pytest.raises(ValueError, match=text):
            ops.cached_attn(**{**c, **change})
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.ranged_attn_bwd(**b)
    one = torch.zeros(3, dtype=I32)
    for kw, text in ((dict(window=3), "causal"), (dict(prefix=one), "causal"), (dict(causal=True, window=2, prefix=one), "no interval"),
                     (dict(lens=one[:2]), "lens"), (dict(lens=one.long()), "lens"), (dict(documents=one[:1]), "documents"),
                     (dict(documents=torch.zeros(2, 4, dtype=I32)), "documents"), (dict(window=-1), "window")):
        with pytest.raises(ValueError, match=text):
            ops.key_ranges(3, 5, **kw)


def test_entry_points_refuse_what_their_kernels_do_not_take():
    import ctypes
    from lbm_amd import _C

    def ranged(**kw):
        d = _C.RangedAttnDesc()
        base = dict(q=4096, k=4096, v=4096, o=4096, dout=4096, dq=4096, dk=4096, dv=4096, lse=4096, scratch=4096, B=1, H=2, Hk=1, Nq=4, Nk=4, D=64,
                    ldq=128, ldk=64, ldv=64, ldo=128, ldg=128, scale=0.125)
        base.update(kw)
        for n, x in base.items():
            setattr(d, n, x)
        return ctypes.byref(d)

    def cached(**kw):
        d = _C.CachedAttnDesc()
        base = dict(q=4096, k=4096, v=4096, o=4096, lens=4096, scratch=4096, B=1, H=2, Hk=1, n=1, cap_rows=4096, D=64, ldq=128, ldk=64, ldv=64, scale=0.125)
        base.update(kw)
        for n, x in base.items():
            setattr(d, n, x)
        return ctypes.byref(d)
    both = (dict(D=12), dict(D=168), dict(H=3, Hk=2), dict(H=0), dict(B=-1), dict(scale=0.0), dict(cap=-1.0), dict(q=0), dict(k=4104), dict(ldq=120),
            dict(ldk=56), dict(ldv=68), dict(ldk=1 << 24), dict(sk=-64), dict(sk=4), dict(slopes=4097))
    for bad in both + (dict(ranges=4100), dict(Nq=1 << 30), dict(Nk=-1), dict(ldo=64)):
        assert _C.lib.lbmk_ranged_attn(ranged(**bad), None) == 1, bad
        assert _C.lib.lbmk_ranged_attn_bwd(ranged(**bad), None) == 1, bad
    for bad in (dict(lse=0), dict(scratch=0), dict(scratch=4104), dict(dout=0), dict(dq=0), dict(dk=4100), dict(ldg=64)):
        assert _C.lib.lbmk_ranged_attn_bwd(ranged(**bad), None) == 1, bad
    for bad in both + (dict(lens=0), dict(lens=4097), dict(n=-1), dict(window=-1), dict(scratch=0), dict(cap_rows=1 << 30)):
        assert _C.lib.lbmk_cached_attn(cached(**bad), None) == 1, bad
    assert _C.lib.lbmk_key_ranges(None, None, 0, 0, None, None, 1, 1, 1, 0, 0, None) == 1
    assert _C.lib.lbmk_key_ranges(4096, 4096, 0, 0, None, None, 1, 1, 1, 0, 0, None) == 1
