"""`optim.Adam` in calls that a training loop may make beside the ordinary one. All comparisons are bit for bit: the same updates are
made in another way."""
import copy
import pickle
import warnings

import pytest
import torch

from diffusion_model_amd import optim

pytestmark = pytest.mark.gpu
SIZES = [1, 5, 2047, 2048, 2049, 5000]


def _params(seed):
    g = torch.Generator().manual_seed(seed)
    out = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in SIZES]
    for p in out:
        p.grad = torch.randn(p.shape, generator=g).cuda()
    return out


def _adam(params, **how):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")                         # torch warns of parameters listed twice
        return optim.Adam(params, lr=1e-2, **how)


def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("max_grad_norm", [None, 0.3])
def test_a_parameter_listed_twice_takes_two_steps(max_grad_norm):
    """As two steps of an optimizer that lists it once, with the same gradients."""
    a, b = _params(1), _params(1)
    twice, once = _adam(a + a[2:], max_grad_norm=max_grad_norm), _adam(b, max_grad_norm=max_grad_norm)
    twice.step()
    once.step()
    if max_grad_norm is not None:
        assert torch.equal(twice.grad_norm, once.grad_norm)
    first = [p.detach().clone() for p in b[:2]]
    once.step()
    assert _equal(a[:2], first) and _equal(a[2:], b[2:])
    for p, q in zip(a[2:], b[2:]):
        assert float(twice.state[p]["step"]) == 2.0
        assert all(torch.equal(twice.state[p][k], once.state[q][k]) for k in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("max_grad_norm", [None, 0.3])
@pytest.mark.parametrize("through", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
def test_a_copied_optimizer_goes_on_as_the_first(max_grad_norm, through):
    a = _params(2)
    grads = [p.grad for p in a]
    first = _adam(a, max_grad_norm=max_grad_norm)
    first.step()
    second = through(first)
    b = second.param_groups[0]["params"]
    for p, q, g in zip(a, b, grads):
        p.grad, q.grad = g, g.clone()
    first.step()
    second.step()
    assert _equal(a, b) and (max_grad_norm is None or torch.equal(first.grad_norm, second.grad_norm))


def test_a_gradient_that_parameters_share():
    """The norm counts it for each of them, and so does the clipped step, which reads gradients alone; scaling it twice is refused."""
    a, b = _params(3), _params(3)
    a[4].grad = a[5].grad[:2049]                                # the same memory, of two sizes
    b[4].grad = a[4].grad.clone()
    a.append(torch.nn.Parameter(a[5].detach().clone()))
    a[-1].grad = a[5].grad
    b.append(torch.nn.Parameter(a[5].detach().clone()))
    b[-1].grad = a[5].grad.clone()
    want = optim.grad_norm(b)
    assert torch.equal(optim.grad_norm(a), want)
    assert float(want) == pytest.approx(float(torch.cat([p.grad.double() for p in a]).norm()), rel=2.0 ** -23)
    with pytest.raises(ValueError, match="twice"):
        optim.clip_grad_norm_(a, 0.3)
    for params in (a, b):
        opt = _adam(params, max_grad_norm=0.3)
        opt.step()
        assert torch.equal(opt.grad_norm, want)
    assert _equal(a, b)


def test_clipping_takes_the_arguments_of_torch():
    tol = sum(SIZES) * 2.0 ** -24                               # what adding up that many squares in fp32 is off by at most
    for foreach in (None, False, True):
        a, b = _params(4), _params(4)
        got = optim.clip_grad_norm_(a, 0.5, 2.0, False, foreach)
        want = torch.nn.utils.clip_grad_norm_(b, 0.5, 2.0, False, foreach)
        assert float(got) == pytest.approx(float(want), rel=tol)
        assert all(torch.allclose(p.grad, q.grad, rtol=tol, atol=0) for p, q in zip(a, b))
