"""The differentiable token operators (models.layers.qk_norm_rope, ranged_attention) where a gradient is not theirs to give."""
import pytest
import torch

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "attention"])
def test_a_gradient_of_the_gradients_is_refused(cuda, op):
    """create_graph builds the first gradients as ever; a term of a loss that goes through them (a gradient penalty) raises, where it was
    left out"""
    from lbm_amd.models import layers
    q, k, v = (torch.randn(1, 9, 128, device=cuda).to(BF).requires_grad_(True) for _ in range(3))
    w = torch.ones(64, device=cuda, dtype=BF, requires_grad=True)
    run = (lambda: layers.qk_norm_rope(q, k, 64, w, w)[0]) if op == "norm" else (lambda: layers.ranged_attention(q, k, v, 2, 2, 64))
    y = run()
    plain, = torch.autograd.grad(y.float().square().sum(), q, retain_graph=True)
    first, = torch.autograd.grad(y.float().square().sum(), q, create_graph=True)
    assert torch.equal(plain, first)
    for leaf in (q, k):
        with pytest.raises(NotImplementedError, match="gradient of their gradients"):
            torch.autograd.grad(run().float().sum() + first.float().square().sum(), leaf, retain_graph=True)
    with pytest.raises(NotImplementedError, match="gradient of their gradients"):
        (run().float().sum() + first.float().square().sum()).backward()
    # other parts of the loss keep theirs: the first gradients as constants
    a, = torch.autograd.grad(run().float().sum() + first.detach().float().square().sum(), q)
    assert torch.equal(a, torch.autograd.grad(run().float().sum(), q)[0])
