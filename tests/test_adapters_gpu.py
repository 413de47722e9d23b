"""A linear layer with the low-rank adapters of many requests (ops.linear_adapters) against the definition in 64 bits.

Tolerance, element by element: y's own rounding, half a step (2^-8 of it); t's, half a step of each of its `rank` values
(2^-8 sum |t| |up|); and the f32 sums, (K + rank + 16) * 2^-24 of the sums of the products' magnitudes."""
import pytest
import torch

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
H8 = 2.0 ** -8


def make(seed, R, rows, K, N, count, rank, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k).to(BF)  # noqa: E731
    x, w, b = r(R, rows, K), r(N, K, k=K ** -0.5), torch.randn(N, generator=g) if bias else None
    down, up = r(count, rank, K, k=K ** -0.5), r(count, N, rank, k=rank ** -0.5)
    return x, w, b, down, up, torch.rand(count, generator=g) + 0.5, torch.randint(-1, count, (R,), generator=g, dtype=I32)


def definition(x, w, b, down, up, scaling, index):
    K, rank = x.shape[-1], up.shape[-1]
    x, w = x.double(), w.double()
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        y, mag = y + b.double(), mag + b.double().abs()
    tol = torch.zeros_like(y)
    for r, a in enumerate(index.tolist()):
        if 0 <= a < down.shape[0]:
            s = 1.0 if scaling is None else float(scaling[a])
            t = s * (x[r] @ down[a].double().t())
            y[r] += t @ up[a].double().t()
            tol[r] += H8 * (t.abs() @ up[a].double().abs().t())
            mag[r] += s * (x[r].abs() @ down[a].double().abs().t()) @ up[a].double().abs().t()
    return y, tol + H8 * y.abs() + (K + rank + 16) * 2.0 ** -24 * mag


def check(got, want):
    off = (got.double().cpu() - want[0]).abs()
    assert bool((off <= want[1]).all()), float((off / want[1]).max())


def on(cuda, *ts):
    return [None if t is None else t.to(cuda) for t in ts]


CASES = [  # requests, rows, K, N, adapters, rank, bias
    (1, 1, 64, 64, 1, 16, True),
    (1, 1, 8, 8, 1, 1, False),
    (16, 1, 1280, 1280, 7, 16, True),
    (5, 1, 640, 328, 3, 4, True),
    (17, 1, 320, 200, 4, 8, False),
    (33, 1, 72, 40, 5, 64, True),
    (3, 20, 200, 136, 2, 3, True),
    (64, 1, 2560, 640, 8, 32, True),
    (4, 16, 1280, 72, 2, 256, True),
    (65, 1, 320, 328, 5, 16, True),
    (100, 1, 328, 72, 5, 5, True),
    (5, 77, 640, 1000, 3, 8, True),
    (3, 130, 72, 200, 2, 40, False),
    (2, 300, 1280, 640, 2, 16, True),
    (7, 33, 128, 96, 3, 100, True),
    (2, 1024, 640, 640, 2, 32, True),
    (129, 1, 320, 72, 5, 16, True),            # several workgroups' rows in the few-rows kernel, a last row alone
    (250, 2, 328, 136, 3, 6, False),
    (513, 1, 128, 200, 4, 8, True),            # one row per request in the tiled product
    (43, 3, 128, 200, 4, 8, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_against_the_definition(cuda, case):
    from lbm_amd import ops
    *sizes, bias = case
    x, w, b, down, up, scaling, index = make(1, *sizes, bias)
    want = definition(x, w, b, down, up, scaling, index)
    xd, wd, bd, dd, ud, sd, idx = on(cuda, x, w, b, down, up, scaling, index)
    pw = ops.pack_linear_weight(wd, bd)
    y = ops.linear_adapters(xd, pw, dd, ud, idx, sd)
    check(y, want)
    assert torch.equal(y, ops.linear_adapters(xd, pw, dd, ud, idx, sd))
    if sizes[1] == 1:
        assert torch.equal(y[:, 0], ops.linear_adapters(xd[:, 0], pw, dd, ud, idx, sd))
    check(ops.linear_adapters(xd, pw, dd, ud, idx), definition(x, w, b, down, up, None, index))
    # rows of a wider buffer
    wide = torch.full((sizes[0], sizes[1], sizes[2] + 24), float("nan"), dtype=BF, device=cuda)
    wide[..., 8:8 + sizes[2]] = xd
    assert torch.equal(y, ops.linear_adapters(wide[..., 8:8 + sizes[2]], pw, dd, ud, idx, sd))


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [12, 13, 14, 17, 18])
@pytest.mark.parametrize("rows,rank", [(1, 16), (33, 7), (300, 64)])
def test_every_tile(cuda, tile, rows, rank):
    from lbm_amd import ops
    R = 600 // rows
    x, w, b, down, up, scaling, index = make(2, R, rows, 192, 328, 4, rank)
    args = on(cuda, x, w, b, down, up, scaling, index)
    pw = ops.pack_linear_weight(args[1], args[2])
    y = ops.linear_adapters(args[0], pw, args[3], args[4], args[6], args[5], tile=tile)
    check(y, definition(x, w, b, down, up, scaling, index))
    assert torch.equal(y, ops.linear_adapters(args[0], pw, args[3], args[4], args[6], args[5], tile=13))


@pytest.mark.gpu
@pytest.mark.parametrize("R,rows", [(12, 1), (40, 5), (6, 130)])
def test_a_request_sees_its_own_adapter_only(cuda, R, rows):
    """an adapter that holds NaN and infinities, and rows of NaN, stay with their own request; without an adapter the result is
    the shared layer's"""
    from lbm_amd import ops
    x, w, b, down, up, scaling, _ = make(3, R, rows, 320, 264, 3, 16)
    index = torch.tensor([i % 4 - 1 for i in range(R)], dtype=I32)          # -1, 0, 1, 2, ...
    index[index == -1] = torch.tensor([-1, 3, 2 ** 31 - 1, -2 ** 31, 3, -5, 7, 100, 3, 3], dtype=I32)[:int((index == -1).sum())]
    want = definition(x, w, b, down, up, scaling, index)
    down[1, 3], up[1, 200:] = float("nan"), float("inf")
    bad = index == 1
    x[1, 0] = x[1, 0] if rows == 1 else float("nan")
    args = on(cuda, x, w, b, down, up, scaling, index)
    y = ops.linear_adapters(args[0], ops.pack_linear_weight(args[1], args[2]), args[3], args[4], args[6], args[5]).cpu()
    keep = ~bad[:, None].expand(R, rows).clone()
    if rows > 1:
        keep[1, 0] = False
        assert bool(torch.isnan(y[1, 0]).all())
    off = (y.double() - want[0]).abs()
    assert bool((off <= want[1])[keep].all())
    assert not bool(torch.isfinite(y[bad]).any())


@pytest.mark.gpu
def test_graph_replay_follows_the_index_and_zero_rows(cuda):
    from lbm_amd import ops
    for R, rows in ((12, 1), (4, 100)):
        x, w, b, down, up, scaling, index = on(cuda, *make(4, R, rows, 320, 640, 4, 16))
        pw = ops.pack_linear_weight(w, b)
        run = lambda: ops.linear_adapters(x, pw, down, up, index, scaling)  # noqa: E731
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        for n in range(3):
            index.copy_(torch.randint(-1, 4, (R,), generator=torch.Generator().manual_seed(n), dtype=I32))
            x.mul_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, run())
    assert ops.linear_adapters(x[:0], pw, down, up, index[:0], scaling).shape == (0, 100, 640)
    assert ops.linear_adapters(x[:, :0], pw, down, up, index, scaling).shape == (4, 0, 640)


@pytest.mark.gpu
def test_layer_form(cuda):
    from lbm_amd.models.layers import HipLinear
    layer = HipLinear(320, 640).to(cuda).to(BF)
    x, _, _, down, up, scaling, index = make(5, 6, 10, 320, 640, 2, 8)
    want = definition(x, layer.weight.detach().cpu(), layer.bias.detach().cpu(), down, up, scaling, index)
    args = on(cuda, x, down, up, index, scaling)
    with torch.no_grad():
        check(layer.forward_adapters(*args), want)
    with pytest.raises(NotImplementedError, match="inference-only"):
        layer.forward_adapters(*args)


def _args():
    from lbm_amd import ops
    return dict(x=torch.zeros(3, 5, 64, dtype=BF), pw=ops.PackedWeight(torch.zeros(32, 64, dtype=BF), None, 32, 64, 64, 64, 1, 1),
                down=torch.zeros(2, 4, 64, dtype=BF), up=torch.zeros(2, 32, 4, dtype=BF), index=torch.zeros(3, dtype=I32), scaling=torch.ones(2))


REFUSED = [
    (dict(x=torch.zeros(64, dtype=BF)), "expected"), (dict(x=torch.zeros(3, 5, 64)), "bf16"), (dict(x=torch.zeros(3, 5, 72, dtype=BF)), "72 channels"),
    (dict(down=torch.zeros(2, 4, 64)), "bf16"), (dict(down=torch.zeros(3, 4, 64, dtype=BF)), "down"), (dict(down=torch.zeros(2, 5, 64, dtype=BF)), "down"),
    (dict(up=torch.zeros(2, 4, 32, dtype=BF)), "up"), (dict(up=torch.zeros(2, 4, 32, dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(down=torch.zeros(2, 257, 64, dtype=BF), up=torch.zeros(2, 32, 257, dtype=BF)), "rank"),
    (dict(down=torch.zeros(0, 4, 64, dtype=BF), up=torch.zeros(0, 32, 4, dtype=BF)), "count"),
    (dict(index=torch.zeros(3, dtype=torch.long)), "index"), (dict(index=torch.zeros(15, dtype=I32)), "index"),
    (dict(scaling=torch.ones(3)), "scaling"), (dict(scaling=torch.ones(2, dtype=BF)), "scaling"),
    (dict(x=torch.zeros(5, 3, 64, dtype=BF).transpose(0, 1)), "strides"), (dict(x=torch.zeros(3, 5, 65, dtype=BF)[..., 1:]), "strides"),
    (dict(x=torch.zeros(3, 64, 5, dtype=BF).transpose(1, 2)), "strides"),
]


@pytest.mark.parametrize("change,text", REFUSED, ids=range(len(REFUSED)))
def test_refusals(change, text):
    from lbm_amd import ops
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.linear_adapters(**_args())
    with pytest.raises(ValueError, match=text):
        ops.linear_adapters(**{**_args(), **change})
    with pytest.raises(NotImplementedError, match="inference-only"):
        ops.linear_adapters(**{**_args(), "x": torch.zeros(3, 5, 64, dtype=BF, requires_grad=True)})


def test_entry_points_refuse_what_their_kernels_do_not_take():
    import ctypes
    from lbm_amd import _C
    P = 4096

    def down(x=P, dn=P, index=P, scaling=P, t=P, requests=2, rows=3, K=64, ldx=64, rank=4, tk=32, count=2):
        return _C.lib.lbmk_adapter_down(x, dn, index, scaling, t, requests, rows, K, ldx, rank, tk, count, None)
    for bad in (dict(x=0), dict(x=P + 8), dict(dn=0), dict(index=0), dict(t=0), dict(t=P + 8), dict(K=60), dict(K=0), dict(ldx=56), dict(ldx=68), dict(rank=0),
                dict(rank=33), dict(tk=64), dict(tk=40), dict(count=0), dict(requests=-1), dict(rows=1 << 21), dict(requests=1 << 20, rows=1 << 12), dict(scaling=P + 2)):
        assert down(**bad) == 1, bad

    def few(x=P, w=P, bias=P, t=P, up=P, index=P, y=P, requests=2, rows=3, N=32, K=64, ldx=64, ldw=64, ldy=32, rank=8, tk=32, count=2):
        return _C.lib.lbmk_adapter_linear_few(x, w, bias, t, up, index, y, requests, rows, N, K, ldx, ldw, ldy, rank, tk, count, None)
    for bad in (dict(requests=1 << 20, rows=1 << 3), dict(rows=-1), dict(N=30), dict(K=60), dict(ldw=56), dict(ldy=28), dict(up=P + 8), dict(y=P + 4), dict(w=0), dict(tk=16),
                dict(rank=33), dict(count=0), dict(bias=P + 2)):
        assert few(**bad) == 1, bad

    def gemm(**kw):
        d = _C.IgemmDesc()
        base = dict(a=P, w=P, out=P, M=130, N=64, K=64, Kp=64, Cin=64, a_cs=64, IH=1, IW=1, OH=1, OW=1, KH=1, KW=1, stride=1, ldo=64, alpha=1.0, batch=1,
                    tile=-1, lr_t=P, lr_up=P, lr_index=P, lr_rank=8, lr_k=32, lr_rows=65, lr_count=2)
        base.update(kw)
        for n, v in base.items():
            setattr(d, n, v)
        return _C.lib.lbmk_igemm(ctypes.byref(d), None)
    for bad in (dict(lr_t=0), dict(lr_index=0), dict(lr_rows=0), dict(lr_rows=60), dict(lr_count=0), dict(lr_rank=0), dict(lr_rank=40), dict(lr_k=24), dict(alpha=2.0),
                dict(batch=2), dict(in_f32=1, out_f32=1), dict(smx_mode=1), dict(tile=0), dict(tile=3), dict(lr_up=P + 8), dict(act=2), dict(rowvec=P, rowvec_ld=64)):
        assert gemm(**bad) == 1, bad
