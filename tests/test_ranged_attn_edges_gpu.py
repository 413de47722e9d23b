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
