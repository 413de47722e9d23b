"""Head norms with the position rotation (ops.qk_norm_rope and its backward) where a block takes more than one step over the
tokens: more than 2048 blocks of tokens forward, more than 1024 backward, the last step a part of one.

Tolerances, element by element.  Outputs: half a step of their type, eps / 2 of the value, and 40 f32 roundings (2^-24) of the
head's largest magnitude; dx: 160 of them (both as derived in test_norm_rope_gpu).  The gains' gradients: a lane adds one term per step
and head of its group, a block joins its groups by at most 8 additions, the last kernel adds at most 16 blocks per strip and 64
strips; a term itself carries at most 30 roundings: (steps * heads + 118) * 2^-24 of the sum of the terms' magnitudes.  A step left out
or taken twice changes a gradient by a multiple of that."""
import pytest
import torch

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
EPS = 1e-6


def definition(x, w, table, pos, D, inter, g):
    """y, dx, dw and the sum of |terms of dw| in 64 bits; x [B, N, H D], pos [B, N]"""
    x, w, g = x.double().unflatten(-1, (-1, D)), w.double(), g.double().unflatten(-1, (-1, D))
    F = table.shape[1]
    c, s = (table.double()[pos.long()][..., i].unsqueeze(2) for i in (0, 1))
    first, second = (slice(0, 2 * F, 2), slice(1, 2 * F, 2)) if inter else (slice(0, F), slice(F, 2 * F))

    def turn(v, s):
        out = v.clone()
        a, b = v[..., first], v[..., second]
        out[..., first], out[..., second] = a * c - b * s, b * c + a * s
        return out
    rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh, gy = x * rstd, turn(g, -s)
    gx = gy * w
    dx = rstd * (gx - xh * (gx * xh).mean(-1, keepdim=True))
    terms = gy * xh
    return turn(xh * w, s), dx, terms.sum((0, 1, 2)), terms.abs().sum((0, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,N,Hq,Hk,D,F,inter,steps", [
    (BF, 1, 2 * 16384 + 53, 10, 3, 64, 32, False, 3),        # 16 tokens per block
    (F32, 1, 2 * 16384 + 5, 8, 8, 80, 24, True, 3),          # 16
    (BF, 2, 65536 + 77, 1, 1, 64, 16, False, 3),             # 64
    (BF, 1, 2 * 2048 + 3, 200, 1, 64, 32, False, 5),         # one: 64 groups for 200 heads
], ids=str)
def test_more_tokens_than_a_step_of_the_grid(cuda, dtype, B, N, Hq, Hk, D, F, inter, steps):
    from lbm_amd import ops
    gen = torch.Generator(device=cuda).manual_seed(41)
    r = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    q, k, gq, gk = (r(B, N, H * D).to(dtype) for H in (Hq, Hk, Hq, Hk))
    wq, wk = 1 + 0.2 * r(D), 1 + 0.2 * r(D)
    table = ops.rope_table(300, F, device=cuda)
    pos = torch.randint(0, 300, (B, N), generator=gen, device=cuda, dtype=I32)
    yq, yk = ops.qk_norm_rope(q, k, D, wq, wk, table, pos, eps=EPS, interleaved=inter)
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(q, k, gq, gk, D, wq, wk, table, pos, eps=EPS, interleaved=inter)
    half, one = torch.finfo(dtype).eps / 2, 2.0 ** -24
    for x, w, g, H, y, dx, dw in ((q, wq, gq, Hq, yq, dq, dwq), (k, wk, gk, Hk, yk, dk, dwk)):
        ry, rdx, rdw, mag = definition(x, w, table, pos, D, inter, g)
        for got, want, n in ((y, ry, 40), (dx, rdx, 160)):
            off = (got.double().unflatten(-1, (-1, D)) - want).abs()
            assert bool((off <= half * want.abs() + n * one * want.abs().amax(-1, keepdim=True) + 1e-37).all())
        off = (dw.double() - rdw).abs()
        assert bool((off <= ((steps * min(H, 5) + 118) * one) * mag + one * rdw.abs()).all()), float((off / (one * mag)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("eps", [0.0, 1e-40])
def test_heads_whose_mean_square_is_a_subnormal_number(cuda, dtype, eps):
    """values around 2^-65: squares around 2^-130, which f32 holds in 19 bits and fewer.  A square is off by half a step of 2^-149, so
    the mean square by 2^-149 (of at least 2^-132: 2^-17 of it, and half of that in the root), and the outputs by 2^-17 of their
    head's largest magnitude beside the usual roundings; the gradient's two terms likewise."""
    from lbm_amd import ops
    B, N, H, D, F = 1, 37, 3, 64, 32
    gen = torch.Generator(device=cuda).manual_seed(42)
    r = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    q, k = ((r(B, N, H * D) * 2.0 ** -64.5).to(dtype) for _ in range(2))
    # (gradients as small as the heads: dx holds their quotient)
    gq, gk = ((r(B, N, H * D) * 2.0 ** -60).to(dtype) for _ in range(2))
    w = 1 + 0.2 * r(D)
    table = ops.rope_table(300, F, device=cuda)
    pos = torch.randint(0, 300, (B, N), generator=gen, device=cuda, dtype=I32)
    y = ops.qk_norm_rope(q, k, D, w, w, table, pos, eps=eps)
    d = ops.qk_norm_rope_bwd(q, k, gq, gk, D, w, w, table, pos, eps=eps)
    half = torch.finfo(dtype).eps / 2
    for x, g, got, dx in ((q, gq, y[0], d[0]), (k, gk, y[1], d[1])):
        xd, wd, gd = x.double().unflatten(-1, (-1, D)).requires_grad_(True), w.double(), g.double().unflatten(-1, (-1, D))
        c, s = (table.double()[pos.long()][..., i].unsqueeze(2) for i in (0, 1))
        v = xd * (xd.square().mean(-1, keepdim=True) + eps).rsqrt() * wd
        want = torch.cat((v[..., :F] * c - v[..., F:] * s, v[..., F:] * c + v[..., :F] * s), -1)
        wdx = torch.autograd.grad(want, xd, gd)[0]
        big = want.detach().abs().amax(-1, keepdim=True)
        off = (got.double().unflatten(-1, (-1, D)) - want.detach()).abs()
        assert bool((off <= half * want.detach().abs() + 2.0 ** -17 * big).all())
        off = (dx.double().unflatten(-1, (-1, D)) - wdx).abs()
        assert bool((off <= half * wdx.abs() + 2.0 ** -14 * wdx.abs().amax(-1, keepdim=True)).all())


def test_destinations_whose_rows_overlap_are_refused():
    """two groups would write one address; batches between the rows of a wider buffer do not"""
    from lbm_amd import ops
    B, N, C = 2, 4, 64
    q, k = torch.zeros(B, N, C, dtype=BF), torch.zeros(B, N, C, dtype=BF)
    good = torch.zeros(B, N, C, dtype=BF)
    buf = torch.zeros(4096, dtype=BF)
    for strides in ((0, C, 1), (C, C, 1), (3 * C, C, 1), (C // 2, 2 * C, 1), (4 * C, 2 * C, 1), (2 * C + 8, 2 * C, 1)):
        bad = buf.as_strided((B, N, C), strides)
        for out in ((bad, good), (good, bad)):
            with pytest.raises(ValueError, match="out"):
                ops.qk_norm_rope(q, k, 64, None, None, out=out)
    for strides in ((N * C, C, 1), (N * C + 8, C, 1), (C, B * C, 1), (C, 3 * C, 1), (3 * C, 2 * C, 1)):
        with pytest.raises(RuntimeError, match="GPU only"):
            ops.qk_norm_rope(q, k, 64, None, None, out=(buf.as_strided((B, N, C), strides), good))


def test_overlap_of_rows_against_every_address():
    import itertools
    from lbm_amd.ops import _rows_overlap
    for B, N, c in itertools.product((0, 1, 2, 4), (0, 1, 2, 3), (1, 3)):
        for ld, sb in itertools.product(range(c, 12), range(0, 26)):
            rows = [set(range(b * sb + n * ld, b * sb + n * ld + c)) for b in range(B) for n in range(N)]
            assert _rows_overlap(B, N, c, ld, sb) == (len(set().union(*rows)) < B * N * c), (B, N, c, ld, sb)
