"""A step that AdamW refuses leaves weights, moments and step counts as they were (CPU)."""
import pytest
import torch

from abacus_b200.optim.adamw import AdamW


def _after_one_step(state_bits, **kwargs):
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(4, 3), torch.nn.Linear(3, 2))
    opt = AdamW(model, state_bits=state_bits, **({k: f(model) for k, f in kwargs.items()}))
    for p in model.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    return model, opt


def _record(model, opt):
    out = [p.detach().clone() for p in model.parameters()]
    for p in model.parameters():
        for key, value in opt.state[id(p)].items():
            out.append(torch.tensor(value) if key == "step" else value.float().clone().reshape(-1))
    return out


def _refused(model, opt, error, match):
    before = _record(model, opt)
    with pytest.raises(error, match=match):
        opt.step()
    for a, b in zip(_record(model, opt), before):
        assert torch.equal(a, b)


@pytest.mark.parametrize("state_bits", [8, 32])
def test_sparse_gradient(state_bits):
    model, opt = _after_one_step(state_bits)
    model[1].bias.grad = torch.ones(2).to_sparse()
    _refused(model, opt, RuntimeError, "sparse")


@pytest.mark.parametrize("state_bits", [8, 32])
def test_missing_gradient_of_an_owned_range(state_bits):
    model, opt = _after_one_step(state_bits, owned=lambda m: {id(p): (0, p.numel()) for p in m.parameters()})
    model[1].bias.grad = None
    _refused(model, opt, RuntimeError, "missing a gradient")


def test_new_parameter_of_another_type_in_8_bits():
    model, opt = _after_one_step(8)
    other = torch.nn.Parameter(torch.zeros(3, dtype=torch.bfloat16))
    other.grad = torch.zeros_like(other)
    opt.params.append(other)
    _refused(model, opt, ValueError, "fp32 weights")
    opt.params.pop()
    opt.step()
    assert all(opt.state[id(p)]["step"] == 2 for p in model.parameters())


@pytest.mark.parametrize("state_bits,error", [(8, ValueError), (32, RuntimeError)])
def test_moments_of_another_size(state_bits, error):
    model, opt = _after_one_step(state_bits)
    donor, donor_opt = _after_one_step(state_bits)
    opt.state[id(model[1].bias)] = donor_opt.state[id(donor[0].weight)]
    _refused(model, opt, error, "moments of a parameter|shape")
