"""The token operators one after the other, as a layer uses them: projection (with each request's adapter), head norms with
rotation, attention (a prompt, single tokens over a cache, packed documents in training), output projection; against the whole
chain in 64 bits.

Tolerance.  A rounding to bf16 is off by at most 2^-8 of the value (E).  The chain rounds the projection (q, k, v), the normed
heads, the attention weights, the attention's output, the result, and an adapter's factor: v, weights, output and result
enter y once each, 4 E in all, the adapter's factor its own share, below 1 E.  A score is a sum over the head's channels of
products with four roundings, each of them of random sign: its error is below sqrt(4) E times the score, which is about 1 here
(normed heads, scale 1 / sqrt(D)), and moves the output by p (v - o) times that, below 2 E of it with the same number of keys
averaged.  7 E; 10 E is allowed, in the norm of a whole tensor.  A gradient passes the forward's roundings and its own
(projection, attention's ds, p and outputs, norm), each at most as often again: 20 E."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
E = 2.0 ** -8


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def norm_rope(x, w, D, table, pos, eps=1e-6):
    """[B, N, H D] in 64 bits; pos [B, N]"""
    x = x.unflatten(-1, (-1, D))
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
    F = table.shape[1]
    c, s = (table[pos][..., i].unsqueeze(2) for i in (0, 1))
    a, b = y[..., :F], y[..., F:2 * F]
    return torch.cat((a * c - b * s, a * s + b * c, y[..., 2 * F:]), -1).flatten(-2)


def attention(q, k, v, H, Hk, D, seen, cap=0.0):
    heads = lambda t, g: t.unflatten(-1, (-1, D)).transpose(1, 2).repeat_interleave(g, 1)  # noqa: E731
    q, k, v = heads(q, 1), heads(k, H // Hk), heads(v, H // Hk)
    x = q @ k.transpose(-1, -2) * D ** -0.5
    if cap:
        x = cap * torch.tanh(x / cap)
    return (torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v).transpose(1, 2).flatten(-2)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,D,window", [(4, 2, 64, 0), (5, 5, 40, 9), (3, 1, 128, 0)])
def test_serving_prompt_then_single_tokens(cuda, H, Hk, D, window):
    from lbm_amd import ops
    from lbm_amd.models import layers
    gen = torch.Generator().manual_seed(31)
    R, L, steps, rank, rows = 3, 37, 6, 8, 64
    C, W = H * D, (H + 2 * Hk) * D
    T = L + steps
    rand = lambda *s, by=1.0: (torch.randn(*s, generator=gen) * by).to(BF)  # noqa: E731
    x = rand(R, T, C)
    proj, out = layers.HipLinear(C, W), layers.HipLinear(C, C, bias=False)
    with torch.no_grad():
        for m in (proj, out):
            m.weight.copy_(rand(*m.weight.shape, by=C ** -0.5))
        proj.bias.copy_(rand(W, by=0.1))
    proj, out = proj.to(cuda, BF), out.to(cuda, BF)
    down, up = rand(2, rank, C, by=C ** -0.5), rand(2, W, rank, by=rank ** -0.5)
    odown, oup = rand(2, rank, C, by=C ** -0.5), rand(2, C, rank, by=rank ** -0.5)
    scaling, index = torch.tensor([0.5, 0.25]), torch.tensor([1, -1, 0], dtype=I32)
    wq, wk = (1 + 0.2 * torch.randn(D, generator=gen)).to(BF), (1 + 0.2 * torch.randn(D, generator=gen)).to(BF)
    table = ops.rope_table(rows, D // 2)

    # the chain in 64 bits over all tokens
    def linear(m, x, down, up):
        y = x @ m.weight.detach().double().cpu().t() + (0 if m.bias is None else m.bias.detach().double().cpu())
        for r, a in enumerate(index.tolist()):
            if a >= 0:
                y[r] += float(scaling[a]) * (x[r] @ down[a].double().t()) @ up[a].double().t()
        return y
    qkv = linear(proj, x.double(), down, up)
    at = torch.arange(T).expand(R, T)
    q, k, v = qkv.split([C, Hk * D, Hk * D], -1)
    q, k = norm_rope(q, wq.double(), D, table.double().cpu(), at), norm_rope(k, wk.double(), D, table.double().cpu(), at)
    i = torch.arange(T)
    seen = i[None] <= i[:, None]
    if window:
        seen = seen & (i[None] > i[:, None] - window)
    want = linear(out, attention(q, k, v, H, Hk, D, seen), odown, oup)

    x, down, up, odown, oup, scaling, index, wq, wk, table = (t.to(cuda) for t in (x, down, up, odown, oup, scaling, index, wq, wk, table))
    kc, vc = (torch.full((R, rows, Hk * D), float("nan"), dtype=BF, device=cuda) for _ in range(2))
    with torch.no_grad():
        def heads(x):
            qkv = proj.forward_adapters(x, down, up, index, scaling)
            return qkv[..., :C], qkv[..., C:C + Hk * D], qkv[..., C + Hk * D:]
        # the prompt: normed keys go straight into the cache
        q, k, v = heads(x[:, :L].contiguous())
        pos = torch.arange(L, dtype=I32, device=cuda).expand(R, L).contiguous()
        ops.qk_norm_rope(q, k, D, wq, wk, table, pos, out=(q, kc[:, :L]))
        vc[:, :L].copy_(v)
        o = ops.ranged_attn(q, kc[:, :L], vc[:, :L], H, Hk, D, ops.key_ranges(R, L, causal=True, window=window, device=cuda))
        y = out.forward_adapters(o, odown, oup, index, scaling)
        assert off(y, want[:, :L]) <= 10 * E
        # the same through the cache's kernel, as a chunk of new tokens
        lens = torch.full((R,), L, dtype=I32, device=cuda)
        assert off(out.forward_adapters(ops.cached_attn(q, kc, vc, lens, H, Hk, D, window=window), odown, oup, index, scaling), want[:, :L]) <= 10 * E

        # single tokens: one captured step, replayed
        token, at, pos = x[:, L:L + 1].clone(), torch.full((1,), L, device=cuda), torch.full((R, 1), L, dtype=I32, device=cuda)
        lens.fill_(L + 1)

        def step():
            q, k, v = heads(token)
            q, k = ops.qk_norm_rope(q, k, D, wq, wk, table, pos)
            kc.index_copy_(1, at, k)
            vc.index_copy_(1, at, v)
            return out.forward_adapters(ops.cached_attn(q, kc, vc, lens, H, Hk, D, window=window), odown, oup, index, scaling)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for n in range(steps):
            token.copy_(x[:, L + n:L + n + 1])
            graph.replay()
            torch.cuda.synchronize()
            assert off(held, want[:, L + n:L + n + 1]) <= 10 * E, n
            assert torch.equal(held, step())
            for t in (at, pos, lens):
                t.add_(1)
    assert bool(torch.isnan(kc[:, T:].float()).all()) and bool(torch.isnan(vc[:, T:].float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,D,N", [(4, 2, 64, 150), (2, 2, 80, 65), (3, 1, 128, 77)])
def test_training_over_packed_documents(cuda, H, Hk, D, N):
    from lbm_amd import ops
    from lbm_amd.models import layers
    gen = torch.Generator().manual_seed(32)
    B, C, W = 2, H * D, (H + 2 * Hk) * D
    rand = lambda *s, by=1.0: (torch.randn(*s, generator=gen) * by).to(BF)  # noqa: E731
    docs = torch.tensor([0, 1, N // 3, N - 5], dtype=I32)                 # the last five rows belong to no document
    lo = torch.tensor([0] + [1] * (N // 3 - 1) + [N // 3] * (N - 5 - N // 3) + [0] * 5)
    i = torch.arange(N)
    seen = (i[None] <= i[:, None]) & (i[None] >= lo[:, None]) & (i[:, None] < N - 5)
    pos = torch.where(i < N - 5, i - lo, 0).to(I32).expand(B, N).contiguous()
    table = ops.rope_table(N, D // 4)
    leaves = {"x": rand(B, N, C), "proj": rand(W, C, by=C ** -0.5), "out": rand(C, C, by=C ** -0.5),
              "wq": (1 + 0.2 * torch.randn(D, generator=gen)).to(BF), "wk": (1 + 0.2 * torch.randn(D, generator=gen)).to(BF)}
    g = rand(B, N, C)

    ref = {n: t.double().requires_grad_(True) for n, t in leaves.items()}
    q, k, v = (ref["x"] @ ref["proj"].t()).split([C, Hk * D, Hk * D], -1)
    q, k = (norm_rope(t, ref[w], D, table.double().cpu(), pos.long()) for t, w in ((q, "wq"), (k, "wk")))
    o = torch.cat((attention(q[:, :N - 5], k, v, H, Hk, D, seen[:N - 5], cap=5.0), torch.zeros(B, 5, C, dtype=F64)), 1)
    y = o @ ref["out"].t()
    want = dict(zip(ref, torch.autograd.grad((y * g.double()).sum(), list(ref.values()))), y=y.detach())

    proj, out = (layers.HipLinear(C, n, bias=False).to(cuda, BF) for n in (W, C))
    with torch.no_grad():
        proj.weight.copy_(leaves["proj"])
        out.weight.copy_(leaves["out"])
    x, wq, wk = (leaves[n].to(cuda).requires_grad_(True) for n in ("x", "wq", "wk"))
    table, pos, docs, g = (t.to(cuda) for t in (table, pos, docs, g))
    ranges = ops.key_ranges(B, N, causal=True, documents=docs)
    qkv = proj(x)
    q, k = layers.qk_norm_rope(qkv[..., :C], qkv[..., C:C + Hk * D], D, wq, wk, table, pos)
    o = layers.ranged_attention(q, k, qkv[..., C + Hk * D:], H, Hk, D, ranges, cap=5.0)
    y = out(o)
    y.backward(g)
    got = {"x": x.grad, "proj": proj.weight.grad, "out": out.weight.grad, "wq": wq.grad, "wk": wk.grad}
    assert off(y.detach(), want["y"]) <= 10 * E
    assert bool((y[:, N - 5:] == 0).all())
    for n in got:
        assert off(got[n], want[n]) <= 20 * E, n


@pytest.mark.gpu
def test_training_pair_captured_and_replayed(cuda):
    """forward and backward of the two differentiable operators in one graph, replayed between eager passes"""
    import gc
    from lbm_amd import ops
    from lbm_amd.models import layers
    gen = torch.Generator().manual_seed(33)
    B, N, H, Hk, D = 2, 130, 4, 2, 64
    q, k, v, g = (torch.randn(B, N, h * D, generator=gen).to(cuda, BF) for h in (H, Hk, Hk, H))
    wq, wk = (torch.ones(D, device=cuda) for _ in range(2))
    table, pos = ops.rope_table(N, D // 2).to(cuda), torch.arange(N, dtype=I32, device=cuda).expand(B, N).contiguous()
    ranges = ops.key_ranges(B, N, causal=True, device=cuda)

    def grads():
        # leaves of the pass's own: a captured backward must not meet the accumulation nodes of an eager one
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, wq.to(BF), wk.to(BF))]
        a, b = layers.qk_norm_rope(leaves[0], leaves[1], D, leaves[3], leaves[4], table, pos)
        o = layers.ranged_attention(a, b, leaves[2], H, Hk, D, ranges)
        return (o.detach(),) + torch.autograd.grad(o, leaves, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = grads()
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(BF))
        g.copy_(torch.randn(g.shape, generator=gen).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, grads()):
            assert torch.equal(a, b), n


def test_descriptors_have_the_headers_layout(tmp_path):
    from lbm_amd import _C
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    descs = {"lbmk_norm_rope_desc": _C.NormRopeDesc, "lbmk_ranged_attn_desc": _C.RangedAttnDesc, "lbmk_cached_attn_desc": _C.CachedAttnDesc}
    lines = [f'printf("{c}.{n} %zu\\n", offsetof({c}, {n}));' for c, d in descs.items() for n in (f[0] for f in d._fields_)]
    lines += [f'printf("{c} %zu\\n", sizeof({c}));' for c in descs]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "lbmk.h"\nint main(void){' + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for c, d in descs.items():
        assert int(out[c]) == ctypes.sizeof(d), c
        for n, _ in d._fields_:
            assert int(out[f"{c}.{n}"]) == getattr(d, n).offset, (c, n)
