"""Host side of `optim.Adam`: which launches a step makes and what travels with a copied optimizer, on a machine without a GPU.
The launch itself is replaced by a record of its arguments."""
import contextlib
import copy
import pickle
import warnings

import pytest
import torch

from diffusion_model_amd import optim


class OnGpu(torch.nn.Parameter):
    """A parameter that says it is on GPU 0."""
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


@pytest.fixture
def launches(monkeypatch):
    """[(step, data pointers of the parameters)] of every launch, in order."""
    made = []
    monkeypatch.setattr(optim, "on_gpu", lambda gpu: contextlib.nullcontext())
    monkeypatch.setattr(optim, "_update", lambda lists, pointers, sizes, step, *rest: made.append((step, pointers[0])))
    return made


def _param(n=4):
    p = OnGpu(torch.zeros(n))
    p.grad = torch.ones(n)
    return p


def _adam(params, **how):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")                         # torch warns of parameters listed twice
        return optim.Adam(params, **how)


def test_a_parameter_listed_twice_takes_two_steps(launches):
    """Each in a launch of its own: two entries of one launch would read and write the same memory at once."""
    p, q = _param(), _param()
    opt = _adam([p, q, p])
    opt.step()
    assert launches == [(1, [p.data_ptr(), q.data_ptr()]), (2, [p.data_ptr()])]
    assert float(opt.state[p]["step"]) == 2.0 and float(opt.state[q]["step"]) == 1.0


def test_the_steps_of_a_parameter_listed_twice_stay_in_order(launches):
    p, q = _param(), _param()
    opt = _adam([q, p, p])
    p.grad = None
    opt.step()
    p.grad = torch.ones(4)
    del launches[:]
    opt.step()                                                  # q's second step, p's first and second
    assert launches == [(1, [p.data_ptr()]), (2, [q.data_ptr(), p.data_ptr()])]
    assert float(opt.state[p]["step"]) == 2.0 and float(opt.state[q]["step"]) == 2.0


def test_the_norm_counts_a_parameter_listed_twice_once(launches, monkeypatch):
    seen = []

    class Norm:
        state = torch.zeros(2)

        def __init__(self, what, grads, *rest):
            seen.extend(g.data_ptr() for g in grads)

        def factor(self):
            return None

    monkeypatch.setattr(optim, "_Norm", Norm)
    p, q = _param(), _param()
    _adam([p, q, p], max_grad_norm=1.0).step()
    assert seen == [p.grad.data_ptr(), q.grad.data_ptr()]
    assert [step for step, _ in launches] == [1, 2]


@pytest.mark.parametrize("max_grad_norm", [None, 0.5])
@pytest.mark.parametrize("through", [copy.deepcopy, lambda opt: pickle.loads(pickle.dumps(opt))])
def test_a_copied_optimizer_keeps_its_clipping_and_steps(launches, monkeypatch, max_grad_norm, through):
    clipped = []

    class Norm:
        state = torch.zeros(2)

        def __init__(self, what, grads, max_norm, *rest):
            clipped.append(max_norm)

        def factor(self):
            return None

    monkeypatch.setattr(optim, "_Norm", Norm)
    p = torch.nn.Parameter(torch.zeros(4))
    first = _adam([p], lr=0.25, max_grad_norm=max_grad_norm)
    first.grad_norm = torch.tensor(3.0)
    opt = through(first)
    assert opt.max_grad_norm == max_grad_norm and float(opt.grad_norm) == 3.0 and opt.param_groups[0]["lr"] == 0.25
    opt.param_groups[0]["params"] = [_param()]
    opt.step()
    assert [step for step, _ in launches] == [1] and clipped == ([] if max_grad_norm is None else [max_grad_norm])


def test_an_optimizer_pickled_without_a_bound_has_none(launches):
    opt = _adam([_param()], max_grad_norm=2.0)
    old = {k: v for k, v in opt.__getstate__().items() if k in ("defaults", "state", "param_groups")}
    new = optim.Adam.__new__(optim.Adam)
    new.__setstate__(old)
    assert new.max_grad_norm is None and new.grad_norm is None
    new.step()
    assert [step for step, _ in launches] == [1]


def test_loading_a_state_dict_keeps_the_bound():
    p = torch.nn.Parameter(torch.zeros(4))
    opt, other = optim.Adam([p], max_grad_norm=2.0), torch.optim.Adam([p], lr=0.5)
    opt.load_state_dict(other.state_dict())
    assert opt.max_grad_norm == 2.0 and opt.param_groups[0]["lr"] == 0.5
    opt.load_state_dict(optim.Adam([p], max_grad_norm=7.0).state_dict())
    assert opt.max_grad_norm == 2.0
