"""Attention over key ranges and over a cache at the edges of what their arguments allow, against the definition in 64 bits
(that of test_ranged_attn_gpu, with its tolerances)."""
import ctypes
import math

import pytest
import torch

from test_ranged_attn_gpu import BF, F32, I32, check, definition, make, ranges_of, seen_by


# ---- caps ----------------------------------------------------------------------------------------------------------
# A capped score is off by a few f32 roundings of itself whatever the cap is (cap tanh(x / cap) is x for a cap that is far from the
# scores), so the tolerances hold with the E = 2^-12 that they have without a cap: the products' magnitudes of a row sum to below 100.
@pytest.mark.gpu
@pytest.mark.parametrize("cap", [100.0, 200.0, 1e4, 1e5, 1e6, 1e30])
@pytest.mark.parametrize("D,bias,train", [(64, False, True), (64, True, True), (40, False, True), (128, False, False), (80, True, False), (160, False, True),
                                          (96, False, False), (32, False, False)])
def test_large_caps(cuda, cap, D, bias, train):
    from lbm_amd import ops
    B, N, H, Hk = 2, 150, 4, 2
    q, k, v, g, gen = make(21, B, N, N, H, Hk, D)
    ranges = ranges_of("causal", B, N, N, gen)
    slopes = 2.0 ** -torch.arange(1, H + 1, dtype=F32) if bias else None
    seen, pos = seen_by(ranges, N), torch.arange(N).expand(B, N)
    want = definition(q, k, v, H, Hk, D, seen, pos, D ** -0.5, cap, slopes, g)
    q, k, v, g, ranges = (t.to(cuda) for t in (q, k, v, g, ranges))
    kw = dict(cap=cap, slopes=None if slopes is None else slopes.to(cuda))
    o, lse = ops.ranged_attn(q, k, v, H, Hk, D, ranges, return_lse=True, **kw)
    check("o", o, want["o"])
    if train:
        for n, x in zip(("dq", "dk", "dv"), ops.ranged_attn_bwd(q, k, v, o, g, lse, H, Hk, D, ranges, **kw)):
            check(n, x, want[n])
    last = torch.full((B,), N, dtype=I32, device=cuda)
    check("cache", ops.cached_attn(q[:, -3:], k, v, last, H, Hk, D, **kw), [t[:, -3:] for t in want["o"]])


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [4.0, 50.0, 128.0, 129.0])
def test_both_sides_of_a_cap(cuda, cap):
    """scores far below, around and far above the cap in one call: every key is a multiple of one direction, queries and values
    are few, so a row's weights are known in 64 bits.  A score's error is below 1.5e-5 cap / 50 log2 units (half a step of the largest
    intermediate, 1.44 cap, a few times over) plus 2^-20 of itself: with caps up to 129 below 2^-14, less than the E of the tolerances."""
    from lbm_amd import ops
    D, N = 64, 200
    gen = torch.Generator().manual_seed(22)
    k = torch.zeros(1, N, D)
    k[..., 0] = torch.linspace(-8, 8, N)
    q = torch.zeros(1, N, D)
    q[..., 0] = cap * torch.linspace(-8, 8, N)
    q, k, v, g = q.to(BF), k.to(BF), torch.randn(1, N, D, generator=gen).to(BF), torch.randn(1, N, D, generator=gen).to(BF)
    seen = torch.ones(1, N, N, dtype=torch.bool)
    want = definition(q, k, v, 1, 1, D, seen, torch.arange(N).expand(1, N), D ** -0.5, cap, None, g)
    q, k, v, g = (t.to(cuda) for t in (q, k, v, g))
    o, lse = ops.ranged_attn(q, k, v, 1, 1, D, cap=cap, return_lse=True)
    check("o", o, want["o"])
    dq, dk, dv = ops.ranged_attn_bwd(q, k, v, o, g, lse, 1, 1, D, cap=cap)
    check("dv", dv, want["dv"])
    last = torch.full((1,), N, dtype=I32, device=cuda)
    want = definition(q[:, -1:].cpu(), k.cpu(), v.cpu(), 1, 1, D, seen[:, -1:], torch.zeros(1, 1), D ** -0.5, cap, None)
    check("cache", ops.cached_attn(q[:, -1:].contiguous(), k, v, last, 1, 1, D, cap=cap), want["o"])


def _cpu_operands():
    return dict(q=torch.zeros(2, 5, 128, dtype=BF), k=torch.zeros(2, 7, 64, dtype=BF), v=torch.zeros(2, 7, 64, dtype=BF), heads=2, kv_heads=1, head_dim=64)


# what f32 does not hold, and what is no cap in f32 or overflows scale / cap
@pytest.mark.parametrize("change,text", [(dict(cap=1e-50), "cap"), (dict(cap=1e39), "cap"), (dict(cap=1e-38, scale=100.0), "cap"), (dict(scale=1e-50), "scale"),
                                         (dict(scale=1e39), "scale"), (dict(cap=float("nan")), "cap")])
def test_scales_and_caps_that_f32_does_not_hold(change, text):
    from lbm_amd import ops
    a = {**_cpu_operands(), **change}
    with pytest.raises(ValueError, match=text):
        ops.ranged_attn(**a)
    a["k_cache"], a["v_cache"], a["lens"] = a.pop("k"), a.pop("v"), torch.zeros(2, dtype=I32)
    with pytest.raises(ValueError, match=text):
        ops.cached_attn(**a)


@pytest.mark.parametrize("bad", [dict(cap=math.inf), dict(cap=math.nan), dict(scale=math.inf), dict(scale=math.nan), dict(cap=1e-38, scale=100.0),
                                 dict(scale=1e-42), dict(cap=1e-42)])
def test_entry_points_refuse_scales_and_caps_that_f32_does_not_hold(bad):
    from lbm_amd import _C
    base = dict(q=4096, k=4096, v=4096, o=4096, H=2, Hk=1, B=1, D=64, ldq=128, ldk=64, ldv=64, scale=0.125)
    r, c = _C.RangedAttnDesc(), _C.CachedAttnDesc()
    for d, more in ((r, dict(dout=4096, dq=4096, dk=4096, dv=4096, lse=4096, scratch=4096, Nq=4, Nk=4, ldo=128, ldg=128)),
                    (c, dict(lens=4096, scratch=4096, n=1, cap_rows=4096))):
        for n, x in {**base, **more, **bad}.items():
            setattr(d, n, x)
    assert _C.lib.lbmk_ranged_attn(ctypes.byref(r), None) == 1
    assert _C.lib.lbmk_ranged_attn_bwd(ctypes.byref(r), None) == 1
    assert _C.lib.lbmk_cached_attn(ctypes.byref(c), None) == 1


# ---- values that are not finite where they are seen ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("D", [40, 64, 96, 128, 160])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("at", [10, 70, 140])
def test_a_seen_value_counts_however_small_its_weight(cuda, D, value, at):
    """slopes of 8 take every weight from 14 tokens on below f32's range: 0 times a value that is not finite is NaN, in tiles that have
    masked places and in tiles that have none"""
    from lbm_amd import ops
    B, N, H, Hk = 1, 200, 2, 1
    q, k, v, g, gen = make(23, B, N, N, H, Hk, D)
    ranges, slopes = ranges_of("causal", B, N, N, gen), torch.tensor([8.0, 16.0])
    seen, pos = seen_by(ranges, N), torch.arange(N).expand(B, N)
    want = definition(q, k, v, H, Hk, D, seen, pos, D ** -0.5, 0.0, slopes, g)
    dev = [t.to(cuda) for t in (q, k, v, g, ranges, slopes)]
    good = ops.ranged_attn(*dev[:3], H, Hk, D, dev[4], slopes=dev[5], return_lse=True)
    rows = torch.arange(N)

    def split(name, got, heads, bad):
        """`bad` [N, D]: not finite there in every head, and the definition's values elsewhere"""
        got, ref, tol = (t.detach().double().cpu().view(N, heads, D).transpose(0, 1) for t in (got, *want[name]))
        assert not bool(torch.isfinite(got[:, bad]).any()), name
        assert bool(((got - ref).abs() <= tol)[:, ~bad].all()), name

    # a value: the rows from it on, in its channel
    v2 = v.clone()
    v2[0, at, 3] = value
    bad = torch.zeros(N, D, dtype=torch.bool)
    bad[at:, 3] = True
    split("o", ops.ranged_attn(dev[0], dev[1], v2.to(cuda), H, Hk, D, dev[4], slopes=dev[5]), H, bad)
    # an output gradient: the keys up to its row, in its channel of dv and everywhere in dk (its row's dP is not finite)
    g2 = g.clone().view(B, N, H, D)
    g2[0, at, :, 3] = value
    dq, dk, dv = ops.ranged_attn_bwd(*dev[:3], good[0], g2.view(B, N, -1).to(cuda), good[1], H, Hk, D, dev[4], slopes=dev[5])
    bad = torch.zeros(N, D, dtype=torch.bool)
    bad[:at + 1, 3] = True
    split("dv", dv, Hk, bad)
    bad[:at + 1] = True
    split("dk", dk, Hk, bad)
    bad = (rows == at)[:, None].expand(N, D)
    split("dq", dq, H, bad)
    if value != value:
        return
    # a key whose scores are -inf: no weight, so no change of the output, but 0 times it in the rows' gradients
    q2, k2 = q.clone().view(B, N, H, D), k.clone()
    q2[0, at + 1:, :, 5] = -q2[0, at + 1:, :, 5].abs() if value > 0 else q2[0, at + 1:, :, 5].abs()
    q2[0, at, :, 5] = 0.0                                            # (its own row: 0 * inf)
    q2, k2[0, at, 5] = q2.view(B, N, -1), value
    o, lse = ops.ranged_attn(q2.to(cuda), k2.to(cuda), dev[2], H, Hk, D, dev[4], slopes=dev[5], return_lse=True)
    seen2 = seen.clone()
    seen2[0, :, at] = False
    k0 = k.clone()
    k0[0, at] = 0.0
    want = definition(q2, k0, v, H, Hk, D, seen2, pos, D ** -0.5, 0.0, slopes, g)
    split("o", o, H, (rows == at)[:, None].expand(N, D))
    dq, dk, dv = ops.ranged_attn_bwd(q2.to(cuda), k2.to(cuda), dev[2], o, dev[3], lse, H, Hk, D, dev[4], slopes=dev[5])
    assert not bool(torch.isfinite(dq.cpu().view(N, H, D)[at:, :, 5]).any())
    assert bool(torch.isfinite(dq[0, :at]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [40, 64, 128, 160])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_seen_value_counts_over_a_cache(cuda, D, value):
    from lbm_amd import ops
    B, n, H, Hk, rows = 2, 3, 4, 2, 700
    q, k, v, _, _ = make(24, B, n, rows, H, Hk, D)
    lens, slopes = torch.tensor([650, 90], dtype=I32), torch.full((H,), 16.0)        # weights below f32's range from 7 tokens on
    v[0, 300, 1], v[0, 648, 2], v[0, 640, 3], v[1, 2, 4], v[1, 66, 5], v[1, 89, 6] = [value] * 6
    o = ops.cached_attn(q.to(cuda), k.to(cuda), v.to(cuda), lens.to(cuda), H, Hk, D, slopes=slopes.to(cuda)).cpu().view(B, n, H, D)
    bad = torch.zeros(B, n, D, dtype=torch.bool)
    bad[0, :, 1], bad[0, 1:, 2], bad[0, :, 3], bad[1, :, 4], bad[1, :, 5], bad[1, 2:, 6] = [True] * 6
    assert torch.equal(~torch.isfinite(o), bad[:, :, None].expand(B, n, H, D).logical_and((torch.arange(H) // (H // Hk) == 0)[:, None]))


# ---- gradients that nobody computes ------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["q", "k_cache", "v_cache", "slopes"])
def test_cached_attn_has_no_gradient_and_says_so(name):
    from lbm_amd import ops
    a = _cpu_operands()
    a["k_cache"], a["v_cache"], a["lens"], a["slopes"] = a.pop("k"), a.pop("v"), torch.zeros(2, dtype=I32), torch.zeros(2)
    a[name].requires_grad_(True)
    with pytest.raises(NotImplementedError, match="inference-only"):
        ops.cached_attn(**a)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        ops.cached_attn(**a)


# ---- scratch -----------------------------------------------------------------------------------------------------------
def test_scratch_is_sized_on_the_operands_device(monkeypatch):
    """the size follows the compute units of the current device, so it is asked for with the operands' device current, where the
    launch asks for the same plan; a library and two devices that are not there stand in for the real ones"""
    import contextlib
    from lbm_amd import ops
    current, asked = [0], []

    @contextlib.contextmanager
    def device(n):
        before, current[0] = current[0], n
        yield
        current[0] = before

    class Lib:
        lbmk_ranged_attn_bwd = lbmk_cached_attn = None

        def _floats(self, *sizes):
            asked.append(current[0])
            return 8
        lbmk_ranged_attn_bwd_scratch_floats = lbmk_cached_attn_scratch_floats = _floats
    monkeypatch.setattr(ops, "lib", Lib())
    monkeypatch.setattr(ops, "_one_device", lambda *a: 1)
    monkeypatch.setattr(ops, "_launch", lambda device, *a: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    a = _cpu_operands()
    ops.ranged_attn_bwd(a["q"], a["k"], a["v"], a["q"], a["q"], torch.zeros(2, 2, 5), 2, 1, 64)
    ops.cached_attn(a["q"], a["k"], a["v"], torch.zeros(2, dtype=I32), 2, 1, 64)
    assert asked == [1, 1] and current == [0]


# ---- numbers that 32 bits do not hold ----------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1, 10 ** 30])
def test_a_window_wider_than_32_bits_is_no_window(cuda, window):
    from lbm_amd import ops
    for Nq, Nk in ((40, 40), (3, 200), (9, 4)):
        assert torch.equal(ops.key_ranges(2, Nq, Nk, causal=True, window=window, device=cuda), ops.key_ranges(2, Nq, Nk, causal=True, device=cuda))
    q, k, v, _, _ = make(25, 2, 2, 90, 2, 1, 64)
    args = (q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor([90, 41], dtype=I32, device=cuda), 2, 1, 64)
    assert torch.equal(ops.cached_attn(*args, window=window), ops.cached_attn(*args))


def test_sizes_that_32_bits_do_not_hold():
    from lbm_amd import ops
    for Nq, Nk in ((2 ** 32 + 5, 9), (9, 2 ** 32 + 5), (5, 2 ** 30)):
        with pytest.raises(ValueError, match="key_ranges"):
            ops.key_ranges(0, Nq, Nk)
    wide = lambda *s: torch.empty(*s, dtype=BF, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="tokens"):
        ops.qk_norm_rope(wide(1, 2 ** 32 + 5, 64), wide(1, 2 ** 32 + 5, 64), 64, None, None)
    with pytest.raises(ValueError, match="tokens"):
        ops.ranged_attn(wide(1, 3, 64), wide(1, 2 ** 32 + 5, 64), wide(1, 2 ** 32 + 5, 64), 1, 1, 64)
    pw = ops.PackedWeight(wide(32, 64), None, 32, 64, 64, 64, 1, 1)
    for x, index in ((wide(1, 2 ** 32 + 5, 64), 1), (wide(2 ** 16, 2 ** 15, 64), 2 ** 16)):
        with pytest.raises(ValueError, match="rows"):
            ops.linear_adapters(x, pw, wide(2, 4, 64), wide(2, 32, 4), torch.empty(index, dtype=I32, device="meta"))


# ---- ranked workgroups (over 4096 keys) --------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("D,cap,bias,times", [(64, 0.0, False, 1), (64, 500.0, True, 20), (40, 8.0, False, 1), (128, 0.0, True, 1), (160, 0.0, False, 1), (96, 300.0, False, 10)])
@pytest.mark.parametrize("hole", [None, float("nan"), -float("inf")])
def test_ranked_workgroups_of_two_rows_with_padding_that_holds_anything(cuda, D, cap, bias, times, hole):
    """two rows of a batch with documents of their own, causal inside them, and padding between that holds zeros or values that are not
    finite: the second walk starts with the ranking again.  Many heads: the first ones again, in another order"""
    from lbm_amd import ops
    B, Nq, Nk, H = 2, 500, 4200, 2
    q, k, v, g, gen = make(26, B, Nq, Nk, H, H, D)
    ranges, pad = torch.zeros(B, Nq, 2, dtype=I32), torch.ones(B, Nk, dtype=torch.bool)
    rows = torch.ones(B, Nq, dtype=torch.bool)
    for b, docs in enumerate((((0, 120, 0, 900), (125, 300, 905, 4100), (300, 490, 4100, 4190)), ((3, 260, 10, 4000), (270, 500, 4005, 4200)))):
        for a, e, lo, hi in docs:
            for i in range(a, e):
                ranges[b, i] = torch.tensor([lo, max(lo + 1, hi - (e - 1 - i) * (hi - lo) // (2 * (e - a)))])
            pad[b, lo:hi] = False
            rows[b, a:e] = False
    clean = [t.clone() for t in (q, k, v, g)]
    for t, p in zip((q, k, v, g), (rows, pad, pad, rows)):
        t[p] = 0.0 if hole is None else hole
    for t, p in zip(clean, (rows, pad, pad, rows)):
        t[p] = 0.0
    slopes = torch.tensor([0.5, 0.01]) if bias else None
    want = definition(*clean[:3], H, H, D, seen_by(ranges, Nk), (torch.arange(Nq) + Nk - Nq).expand(B, Nq), D ** -0.5, cap, slopes, clean[3])
    q, k, v, g = (t.to(cuda).repeat(1, 1, times) for t in (q, k, v, g))
    kw = dict(cap=cap, slopes=None if slopes is None else slopes.to(cuda).repeat(times))
    ranges = ranges.to(cuda)
    o, lse, rest = ops.ranged_attn(q, k, v, H * times, H * times, D, ranges, return_lse=True, return_rest=True, **kw)
    got = (o,) + ops.ranged_attn_bwd(q, k, v, o, g, lse, H * times, H * times, D, ranges, rest=rest, **kw)
    for n, x in zip(("o", "dq", "dk", "dv"), got):
        for part in (x[..., :H * D], x[..., -H * D:]):
            check(n, part, want[n])
