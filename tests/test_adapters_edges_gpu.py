"""A linear layer with the adapters of many requests (ops.linear_adapters) at the edges of what its arguments allow, against the
definition in 64 bits (that of test_adapters_gpu, with its tolerances)."""
import ctypes

import pytest
import torch

from test_adapters_gpu import BF, I32, check, definition, make, on

ERR_ARG = 1


# ---- row strides -------------------------------------------------------------------------------------------------------
# A tile of the tiled product addresses its rows by 32-bit offsets from the first one, below 2^31: 256 rows of 2^22 elements
def test_row_strides_beyond_a_tiles_offsets_are_refused():
    from lbm_amd import _C, ops
    pw = ops.PackedWeight(torch.zeros(32, 64, dtype=BF), None, 32, 64, 64, 64, 1, 1)
    wide = torch.empty(600, 1 << 23, dtype=BF, device="meta")[:, :64]
    meta = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    pw.w = meta(32, 64)
    with pytest.raises(ValueError, match="row stride"):
        ops.linear_adapters(wide, pw, meta(2, 4, 64), meta(2, 32, 4), meta(600, dtype=I32))
    with pytest.raises(RuntimeError, match="GPU only"):                  # few rows are addressed one by one
        ops.linear_adapters(wide[:100], pw, meta(2, 4, 64), meta(2, 32, 4), meta(100, dtype=I32))
    for M, a_cs, status in ((256, 1 << 23, ERR_ARG), (600, 1 << 23, ERR_ARG), (130, (1 << 23) + (1 << 18), ERR_ARG)):
        d = _C.IgemmDesc()
        for n, v in dict(a=4096, w=4096, out=4096, M=M, N=64, K=64, Kp=64, Cin=64, a_cs=a_cs, IH=1, IW=1, OH=1, OW=1, KH=1, KW=1, stride=1, ldo=64, alpha=1.0,
                         batch=1, tile=-1, lr_t=4096, lr_up=4096, lr_index=4096, lr_rank=8, lr_k=32, lr_rows=1, lr_count=2).items():
            setattr(d, n, v)
        assert _C.lib.lbmk_igemm(ctypes.byref(d), None) == status, (M, a_cs)


@pytest.mark.gpu
@pytest.mark.parametrize("R,rows", [(513, 1), (3, 50), (1, 300)])
def test_wide_row_strides(cuda, R, rows):
    """rows four million elements apart: 4 GB between the first and the last of 513"""
    from lbm_amd import ops
    x, w, b, down, up, scaling, index = make(31, R, rows, 128, 72, 3, 8)
    buf = torch.empty(R * rows, 1 << 22, dtype=BF, device=cuda)
    view = buf[:, 8:136].unflatten(0, (R, rows))
    view.copy_(x)
    args = on(cuda, w, b, down, up, index, scaling)
    y = ops.linear_adapters(view, ops.pack_linear_weight(args[0], args[1]), *args[2:])
    check(y, definition(x, w, b, down, up, scaling, index))


# ---- many rows: two groups of 16 rows share one reading of the factor (from 512 groups of 16 rows on) --------------------
@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    (18, 451, 128, 72, 3, 40, True),           # 29 groups of a request in 15 pairs, the last rows 3 of 32; two blocks of ranks
    (33, 250, 320, 40, 5, 7, False),
    (512, 17, 72, 200, 4, 16, True),           # the second group of a pair holds one row
    (1, 8200, 64, 64, 1, 64, True),
], ids=lambda c: "-".join(map(str, c)))
def test_many_rows(cuda, case):
    from lbm_amd import ops
    *sizes, bias = case
    x, w, b, down, up, scaling, index = make(32, *sizes, bias)
    index[0] = 0
    want = definition(x, w, b, down, up, scaling, index)
    xd, wd, bd, dd, ud, sd, idx = on(cuda, x, w, b, down, up, scaling, index)
    pw = ops.pack_linear_weight(wd, bd)
    y = ops.linear_adapters(xd, pw, dd, ud, idx, sd)
    check(y, want)
    assert torch.equal(y, ops.linear_adapters(xd, pw, dd, ud, idx, sd))


# ---- more requests than a launch's grid takes ------------------------------------------------------------------------
@pytest.mark.gpu
def test_more_requests_than_a_grid(cuda):
    """70001 requests of one row: the factors' product in two launches, the second from request 65535 on"""
    from lbm_amd import ops
    R, K, N, rank = 70001, 64, 64, 8
    x, w, b, down, up, scaling, index = make(33, R, 1, K, N, 3, rank)
    has, a, x0 = (index >= 0).double()[:, None], index.clamp(min=0).long(), x[:, 0].double()
    s = scaling.double()[a][:, None] * has
    t = s * torch.stack([x0 @ d.double().t() for d in down])[a, torch.arange(R)]
    each = torch.stack([t @ u.double().t() for u in up])[a, torch.arange(R)]
    y = x0 @ w.double().t() + b.double() + each
    mag = x0.abs() @ w.double().abs().t() + b.double().abs()
    mag += torch.stack([(s * (x0.abs() @ d.double().abs().t())) @ u.double().abs().t() for d, u in zip(down, up)])[a, torch.arange(R)]
    tol = 2.0 ** -8 * (y.abs() + torch.stack([t.abs() @ u.double().abs().t() for u in up])[a, torch.arange(R)]) + (K + rank + 16) * 2.0 ** -24 * mag
    args = on(cuda, x[:, 0].contiguous(), w, b, down, up, index, scaling)
    check(ops.linear_adapters(args[0], ops.pack_linear_weight(args[1], args[2]), *args[3:]), (y, tol))
