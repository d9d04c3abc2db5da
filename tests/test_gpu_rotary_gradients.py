"""Which gradients rotary positions hand on where only one of q and k takes part."""
import pytest
import torch

from diffusion_model_amd.embedding import grid_positions, rotary

pytestmark = pytest.mark.gpu


def _x(heads, seed):
    return torch.randn(2, 9, heads, 8, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("first", [False, True])
def test_the_gradient_of_one_is_that_of_a_call_alone(first):
    pos = grid_positions(3, 3)
    x, g = _x(2, 1).requires_grad_(True), _x(2, 2)
    other, h = _x(3, 3), _x(3, 4)
    want, = torch.autograd.grad(rotary(x, None, pos, (4, 4)), x, g)
    both = rotary(x, other, pos, (4, 4)) if first else rotary(other, x, pos, (4, 4))
    mine, others = both if first else both[::-1]
    assert mine.requires_grad and torch.equal(mine.detach(), rotary(x.detach(), None, pos, (4, 4)))
    assert torch.equal(others.detach(), rotary(other, None, pos, (4, 4)))
    got, = torch.autograd.grad((mine * g).sum() + (others * h).sum(), x)
    assert torch.equal(got, want) and other.grad is None


def test_an_output_that_the_loss_leaves_out():
    pos = grid_positions(3, 3)
    q, k, g = _x(2, 1).requires_grad_(True), _x(3, 2).requires_grad_(True), _x(3, 3)
    alone = k.detach().requires_grad_(True)
    want, = torch.autograd.grad(rotary(alone, None, pos, (4, 4)), alone, g)
    _, turned = rotary(q, k, pos, (4, 4))
    (turned * g).sum().backward()
    assert torch.equal(k.grad, want) and q.grad is None
