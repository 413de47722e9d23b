"""Head norms with the position rotation (ops.qk_norm_rope, its backward, layers.qk_norm_rope) against the definition in
64 bits.

Tolerances.  One rounding to the output's type is off by at most half a step, eps / 2 of the value (bf16 2^-8, f32 2^-24).
Before it the kernel works in f32: the mean of squares (a tree of at most 256 products: below 20 roundings on any path),
a reciprocal root of 1 ulp, three products and one sum of two products, which cancel: below 40 * 2^-24 of the row's
largest magnitude in all.  The gains' gradients add one f32 sum over tokens and heads: at most (terms on one lane's path
+ 32) * 2^-24 of the sum of the terms' magnitudes."""
import pytest
import torch

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6


def reference(x, w, table, pos, D, rot, inter, eps=EPS, g=None):
    """y (and dx, dw, sum of |terms of dw|) in 64 bits; x [B, N, H*D], pos [B, N, axes] or None"""
    x = x.double().unflatten(-1, (-1, D))
    w = torch.ones(D, dtype=F64) if w is None else w.double()
    rstd = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * rstd
    R = torch.eye(D, dtype=F64).expand(*x.shape[:2], D, D).clone()
    if rot:
        axes = pos.shape[-1]
        F = rot // 2 // axes
        for j in range(rot // 2):
            a, b = (2 * j, 2 * j + 1) if inter else (j, j + rot // 2)
            p = pos[..., j // F].long()
            bad = (p < 0) | (p >= table.shape[0])
            cs = table.double()[p.clamp(0, table.shape[0] - 1), j % F]
            cs = torch.where(bad[..., None], torch.full_like(cs, float("nan")), cs)
            R[..., a, a], R[..., b, b], R[..., a, b], R[..., b, a] = cs[..., 0], cs[..., 0], -cs[..., 1], cs[..., 1]
    turn = lambda m, v: (m[:, :, None] * v[..., None, :]).sum(-1)  # noqa: E731
    y = turn(R, xh * w).flatten(-2)
    if g is None:
        return y
    gy = turn(R.transpose(-1, -2), g.double().unflatten(-1, (-1, D)))
    gx = gy * w
    dx = rstd * (gx - xh * (gx * xh).mean(-1, keepdim=True))
    return y, dx.flatten(-2), (gy * xh).sum((0, 1, 2)), (gy * xh).abs().sum((0, 1, 2))


def near(got, want, D):
    """half a step of the output's type, and 40 f32 roundings of the row's largest magnitude"""
    half = torch.finfo(got.dtype).eps / 2
    got, want = got.double().cpu(), want.double()
    row = want.nan_to_num(0.0).unflatten(-1, (-1, D)).abs().amax(-1, keepdim=True).expand(*want.shape[:-1], want.shape[-1] // D, D).flatten(-2)
    off = (got - want).abs()
    tol = half * want.abs() + 40 * 2.0 ** -24 * row + 1e-37
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert bool(((off <= tol) | torch.isnan(want)).all()), float((off / tol).nan_to_num().max())


def make(seed, dtype, B, N, Hq, Hk, D, axes, F, wdt=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = (r(B, N, Hq * D) * 1.5).to(dtype), (r(B, N, Hk * D) * 0.5).to(dtype)
    wdt = wdt or dtype
    wq, wk = (1 + 0.2 * r(D)).to(wdt), (1 + 0.2 * r(D)).to(wdt)
    gq, gk = r(B, N, Hq * D).to(dtype), r(B, N, Hk * D).to(dtype)
    pos = torch.randint(0, 50, (B, N, axes), generator=g, dtype=torch.int32) if F else None
    ang = torch.rand(50, max(F, 1), generator=g, dtype=F64) * 7
    table = torch.stack((ang.cos(), ang.sin()), -1).to(F32) if F else None
    return q, k, wq, wk, gq, gk, table, pos


CASES = [  # dtype, B, N, Hq, Hk, D, axes, pairs per axis, interleaved
    (BF, 1, 1, 1, 1, 64, 1, 32, False),
    (BF, 2, 37, 20, 5, 64, 1, 32, False),
    (BF, 2, 33, 5, 5, 64, 2, 16, False),
    (BF, 1, 19, 8, 8, 40, 1, 20, False),         # 20 pairs: chunks of four channels
    (BF, 1, 19, 8, 2, 40, 2, 10, False),         # a chunk that crosses two axes
    (BF, 3, 11, 3, 1, 80, 1, 24, False),         # a part of the head, five chunks
    (BF, 1, 9, 8, 8, 160, 1, 80, False),
    (BF, 1, 9, 2, 2, 256, 1, 128, True),
    (BF, 2, 21, 4, 4, 40, 1, 20, True),
    (BF, 2, 21, 4, 4, 72, 1, 32, True),          # nine chunks, the last without a partner
    (BF, 2, 5, 4, 4, 8, 1, 4, False),
    (BF, 2, 45, 7, 3, 128, 0, 0, False),         # the norm alone
    (F32, 2, 37, 20, 5, 64, 2, 16, False),
    (F32, 1, 101, 8, 8, 80, 1, 24, True),
    (F32, 1, 19, 3, 2, 40, 1, 20, False),
    (BF, 2, 1700, 10, 10, 64, 1, 32, False),     # more tokens than one step of the grid, several heads per lane group
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_forward_and_gradients(cuda, case):
    from lbm_amd import ops
    dtype, B, N, Hq, Hk, D, axes, F, inter = case
    q, k, wq, wk, gq, gk, table, pos = make(1, dtype, B, N, Hq, Hk, D, max(axes, 1), F)
    rot = 2 * axes * F
    dev = [None if t is None else t.to(cuda) for t in (q, k, wq, wk, gq, gk, table, pos)]
    yq, yk = ops.qk_norm_rope(dev[0], dev[1], D, dev[2], dev[3], dev[6], dev[7], interleaved=inter)
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(dev[0], dev[1], dev[4], dev[5], D, dev[2], dev[3], dev[6], dev[7], interleaved=inter)
    for x, w, g, y, dx, dw, H in ((q, wq, gq, yq, dq, dwq, Hq), (k, wk, gk, yk, dk, dwk, Hk)):
        ry, rdx, rdw, mag = reference(x, w, table, pos, D, rot, inter, g=g)
        near(y, ry, D)
        # the gradient's row maximum before the cancellation is below rstd * (|g w| + |xh| * mean): bounded by four times its own
        # largest plus the mean's share; 40 roundings of the larger of the two
        big = rdx.unflatten(-1, (-1, D)).abs().amax(-1, keepdim=True).expand(B, N, H, D).flatten(-2)
        half = torch.finfo(dtype).eps / 2
        assert bool(((dx.double().cpu() - rdx).abs() <= half * rdx.abs() + 160 * 2.0 ** -24 * big + 1e-37).all())
        path = B * N * H
        assert bool(((dw.double().cpu() - rdw).abs() <= half * rdw.abs() + (path + 32) * 2.0 ** -24 * mag).all())
    again = ops.qk_norm_rope_bwd(dev[0], dev[1], dev[4], dev[5], D, dev[2], dev[3], dev[6], dev[7], interleaved=inter)
    for a, b in zip((dq, dk, dwq, dwk), again):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_windows_of_a_packed_projection_in_place_and_without_batch(cuda):
    from lbm_amd import ops
    B, N, Hq, Hk, D = 2, 29, 6, 3, 64
    q, k, wq, wk, _, _, table, pos = make(2, BF, B, N, Hq, Hk, D, 1, 32, wdt=F32)
    packed = torch.full((B, N, (Hq + 2 * Hk) * D), 7.0, dtype=BF)
    packed[..., :Hq * D], packed[..., Hq * D:(Hq + Hk) * D] = q, k
    packed = packed.to(cuda)
    a, b = packed[..., :Hq * D], packed[..., Hq * D:(Hq + Hk) * D]
    args = (D, wq.to(cuda), wk.to(cuda), table.to(cuda), pos.to(cuda))
    yq, yk = ops.qk_norm_rope(a, b, *args)
    near(yq, reference(q, wq, table, pos, D, 64, False), D)
    zq, zk = ops.qk_norm_rope(a[1], b[1], args[0], args[1], args[2], args[3], args[4][1, :, 0].contiguous())       # [N, C]
    assert torch.equal(zq, yq[1]) and torch.equal(zk, yk[1])
    ops.qk_norm_rope(a, b, *args, out=(a, b))
    assert torch.equal(a, yq) and torch.equal(b, yk) and bool((packed[..., (Hq + Hk) * D:] == 7.0).all())
    # a gain that does not start on 16 bytes (a slot of a flat parameter buffer)
    flat = torch.zeros(2 * D + 1, dtype=F32, device=cuda)
    flat[1:D + 1], flat[D + 1:] = wq.to(cuda), wk.to(cuda)
    packed[..., :Hq * D], packed[..., Hq * D:(Hq + Hk) * D] = q.to(cuda), k.to(cuda)
    assert torch.equal(ops.qk_norm_rope(a, b, D, flat[1:D + 1], flat[D + 1:], args[3], args[4])[0], yq)


@pytest.mark.gpu
def test_positions_outside_the_table_and_special_values(cuda):
    from lbm_amd import ops
    q, k, wq, wk, gq, gk, table, pos = make(3, BF, 1, 9, 2, 1, 64, 1, 16)         # 32 of 64 channels rotate
    pos[0, 2, 0], pos[0, 5, 0], pos[0, 7, 0] = -1, 50, 2 ** 31 - 1
    q[0, 3], k[0, 4, 5] = 0.0, float("inf")
    d = [t.to(cuda) for t in (q, k, wq, wk, gq, gk, table, pos)]
    yq, yk = ops.qk_norm_rope(d[0], d[1], 64, d[2], d[3], d[6], d[7])
    for t in (2, 5, 7):
        assert bool(torch.isnan(yq[0, t].view(2, 64)[:, :32]).all()) and bool(torch.isfinite(yq[0, t].view(2, 64)[:, 32:]).all())
    assert bool((yq[0, 3] == 0).all())
    near(yq, reference(q, wq, table, pos, 64, 32, False), 64)
    assert bool(torch.isnan(yk[0, 4, 5])) and bool(torch.isfinite(yk[0, 3]).all()) and bool(torch.isfinite(yk[0, 6]).all())
    # zero tokens, and no key heads' gradient wanted
    e = ops.qk_norm_rope(d[0][:, :0], d[1][:, :0], 64, d[2], d[3], d[6], d[7][:, :0])
    assert e[0].shape == (1, 0, 128) and e[1].shape == (1, 0, 64)
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(d[0][:, :0], d[1][:, :0], d[4][:, :0], d[5][:, :0], 64, d[2], None, d[6], d[7][:, :0])
    assert bool((dwq == 0).all()) and dwk is None


@pytest.mark.gpu
def test_autograd_matches_differences_of_the_definition(cuda):
    """directional differences of the 64-bit definition, step h: error h^2 times its third derivative, below 1e-6 of the value
    here; the f32 gradients' own error is bounded by 1e-5 of the summed magnitudes"""
    from lbm_amd.models import layers
    q, k, wq, wk, gq, gk, table, pos = make(4, F32, 2, 13, 4, 2, 64, 2, 16)
    leaves = [t.to(cuda).requires_grad_(True) for t in (q, k, wq, wk)]
    y = layers.qk_norm_rope(leaves[0], leaves[1], 64, leaves[2], leaves[3], table.to(cuda), pos.to(cuda))
    grads = torch.autograd.grad(y, leaves, (gq.to(cuda), gk.to(cuda)))

    def value(q, k, wq, wk):
        return float((reference(q, wq, table, pos, 64, 64, False) * gq.double()).sum() + (reference(k, wk, table, pos, 64, 64, False) * gk.double()).sum())
    base = [t.double() for t in (q, k, wq, wk)]
    gen = torch.Generator().manual_seed(5)
    h = 1e-4
    for i, g in enumerate(grads):
        u = torch.randn(base[i].shape, generator=gen, dtype=F64)
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * u, base[i] - h * u
        diff = (value(*up) - value(*dn)) / (2 * h)
        mine = g.double().cpu() * u
        assert abs(float(mine.sum()) - diff) <= 1e-5 * float(mine.abs().sum()), i
    # an output gradient that autograd expanded from a scalar
    layers.qk_norm_rope(leaves[0], leaves[1], 64, leaves[2], leaves[3], table.to(cuda), pos.to(cuda))[0].sum().backward()
    assert leaves[0].grad is not None and bool(torch.isfinite(leaves[0].grad).all())
    # only one output used, gains without gradients
    yq, _ = layers.qk_norm_rope(leaves[0], leaves[1], 64, None, None, table.to(cuda), pos.to(cuda))
    dq, dk = torch.autograd.grad(yq, leaves[:2], gq.to(cuda), allow_unused=True)
    assert bool((dk == 0).all()) and bool(torch.isfinite(dq).all())


@pytest.mark.gpu
def test_graph_replay_and_side_stream(cuda):
    from lbm_amd import ops
    q, k, wq, wk, gq, gk, table, pos = [t.to(cuda) for t in make(6, BF, 2, 65, 4, 4, 64, 1, 32)]

    def both():
        return ops.qk_norm_rope(q, k, 64, wq, wk, table, pos) + ops.qk_norm_rope_bwd(q, k, gq, gk, 64, wq, wk, table, pos)
    both()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = both()
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(n)).to(BF))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, both()):
            assert torch.equal(a, b), n
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


REFUSED = [
    (lambda a: a.update(q=a["q"].half()), "both bf16"),
    (lambda a: a.update(k=a["k"].float()), "both bf16"),
    (lambda a: a.update(q=a["q"][:, :4]), "qk_norm_rope: q"),
    (lambda a: a.update(q=a["q"][..., :100]), "100 channels"),
    (lambda a: a.update(q=a["q"].transpose(1, 2).contiguous().transpose(1, 2)), "adjacent"),
    (lambda a: a.update(q=torch.zeros(1, 5, 129, dtype=BF)[..., 1:]), "16 bytes"),
    (lambda a: a.update(q_weight=torch.ones(32, dtype=BF)), "vector of 64"),
    (lambda a: a.update(k_weight=torch.ones(64)), "one dtype"),
    (lambda a: a.update(table=None), "go together"),
    (lambda a: a.update(table=a["table"].double()), "table"),
    (lambda a: a.update(positions=a["positions"].long()), "int32"),
    (lambda a: a.update(positions=a["positions"][:, :3].contiguous()), "positions"),
    (lambda a: a.update(table=torch.zeros(9, 33, 2)), "rotate 66"),
    (lambda a: a.update(table=torch.zeros(9, 3, 2)), "multiple of 8"),
    (lambda a: a.update(head_dim=32, q_weight=None, k_weight=None), "rotate 64 of 32"),
    (lambda a: a.update(eps=-1.0), "eps"),
]


@pytest.mark.parametrize("change,text", REFUSED, ids=[t for _, t in REFUSED])
def test_refusals(change, text):
    """every check of the arguments comes before anything touches the GPU: CPU tensors reach them all"""
    from lbm_amd import ops
    a = dict(q=torch.zeros(1, 5, 128, dtype=BF), k=torch.zeros(1, 5, 64, dtype=BF), head_dim=64, q_weight=torch.ones(64, dtype=BF),
             k_weight=torch.ones(64, dtype=BF), table=torch.zeros(9, 32, 2), positions=torch.zeros(1, 5, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.qk_norm_rope(**a)
    change(a)
    with pytest.raises(ValueError, match=text):
        ops.qk_norm_rope(**a)


def test_entry_point_refuses_what_its_kernel_does_not_take():
    """the C ABI returns an argument error, and launches nothing, for sizes and pointers outside its contract"""
    import ctypes
    from lbm_amd import _C

    def desc(**kw):
        d = _C.NormRopeDesc()
        base = dict(q=4096, k=8192, q_out=4096, k_out=8192, dq_out=4096, dk_out=8192, B=1, N=2, Hq=2, Hk=2, D=64, rot=0, ldq=128, ldk=128,
                    ldqo=128, ldko=128, lddq=128, lddk=128, eps=1e-6)
        base.update(kw)
        for n, v in base.items():
            setattr(d, n, v)
        return ctypes.byref(d)
    for bad in (dict(D=12), dict(D=264), dict(rot=72), dict(rot=12), dict(rot=64), dict(q=4104), dict(ldq=64), dict(ldk=132), dict(eps=-1.0),
                dict(rot=64, axes=3, table=4096, pos=4096, positions=4), dict(rot=64, axes=1, table=4096, pos=4096, positions=0),
                dict(q=0), dict(wq=4097), dict(B=70000, N=70000)):
        assert _C.lib.lbmk_norm_rope(desc(**bad), None) == 1, bad
        assert _C.lib.lbmk_norm_rope_bwd(desc(**bad), 4096, None, None, None) == 1, bad
    assert _C.lib.lbmk_norm_rope_bwd(desc(lddq=96), 4096, None, None, None) == 1
    assert _C.lib.lbmk_norm_rope_bwd(desc(), None, None, None, None) == 1
