"""Muon's step around the orthogonalisation, against the documented formula in
64 bits: displacements, decays and updates far below a bf16 step, state that is
saved and continued, parameters that others change.  On the CPU with the plain
products in place of the kernel; on a GPU with the kernel."""
import copy

import pytest
import torch

from bitsparse_b200 import optim
from bitsparse_b200.optim import COEFFICIENTS, Muon

BF16, F32 = torch.bfloat16, torch.float32
SHAPES = [(64, 32), (32, 64), (64, 32), (8, 4, 3, 3)]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def formula(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    x = g.double()
    x = x / (x.pow(2).sum((-2, -1), keepdim=True).sqrt() + eps)
    a, b, c = coefficients
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + b * (s @ x) + c * (s @ (s @ x))
    return x


@pytest.fixture(params=DEVICES)
def device(request, monkeypatch):
    if request.param == "cpu":
        monkeypatch.setattr(optim, "orthogonalize",
                            lambda u, steps=5, coefficients=COEFFICIENTS, eps=1e-7:
                            formula(u, steps, coefficients, eps).to(BF16))
    return request.param


def rand(*shape, device, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(device=device, dtype=dtype)


def parameters(device, dtype):
    return [torch.nn.Parameter(rand(*s, device=device, dtype=dtype, seed=i))
            for i, s in enumerate(SHAPES)]


def give_gradients(params, step):
    for i, p in enumerate(params):
        p.grad = rand(*p.shape, device=p.device, dtype=p.dtype, seed=1000 * step + i + 100)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_displacement(device, dtype, nesterov):
    """Three steps of lr 0.1 with a decay of 0.05 each.  An update is right to
    2^-7 of itself in 2-norm (its bf16 result, 2^-9, and the kernel's operands),
    and the decays make the displacement longer than the three updates
    together, so 2^-7 of it holds their errors; a bf16 parameter is rounded
    once, by 2^-8 of itself at most."""
    params = parameters(device, dtype)
    start = [p.detach().double() for p in params]
    want, bufs = [s.clone() for s in start], [torch.zeros_like(s) for s in start]
    opt = Muon(params, lr=0.1, momentum=0.9, weight_decay=0.5, nesterov=nesterov)
    for step in range(3):
        give_gradients(params, step)
        opt.step()
        for i, p in enumerate(params):
            g = p.grad.double()
            bufs[i] = 0.9 * bufs[i] + g
            u = (g + 0.9 * bufs[i] if nesterov else bufs[i]).reshape(p.shape[0], -1)
            scale = max(1.0, u.shape[0] / u.shape[1]) ** 0.5
            want[i] = want[i] - 0.1 * (scale * formula(u).view(p.shape) + 0.5 * want[i])
    for p, s, w in zip(params, start, want):
        error = (p.detach().double() - w).norm()
        rounding = 2.0 ** -8 * w.norm() if dtype is BF16 else 0.0
        assert error <= 2.0 ** -7 * (w - s).norm() + rounding


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_small_decays_add_up(device, dtype):
    """lr * weight_decay = 2e-4 is below half a step of a bf16 value; 500 such
    decays take a tenth.  A fp32 rounding a step, 500 * 2^-24 = 3e-5 in all,
    and one of bf16 at the end, 2^-8 at most."""
    params = parameters(device, dtype)
    start = [p.detach().double() for p in params]
    opt = Muon(params, lr=0.02, weight_decay=0.01)
    for p in params:
        p.grad = torch.zeros_like(p)
    for _ in range(500):
        opt.step()
    bound = 3e-5 + (2.0 ** -8 if dtype is BF16 else 0.0)
    for p, s in zip(params, start):
        want = s * (1 - 0.02 * 0.01) ** 500
        assert ((p.detach().double() - want).abs() <= bound * want.abs()).all()


def test_small_updates_add_up_in_bf16(device):
    """A constant gradient at a learning rate whose step is a small part of a
    bf16 step: 200 of them move a parameter as far as their sum."""
    start = (5 + rand(64, 64, device=device, seed=3).clamp(-0.9, 0.9)).to(BF16)
    p = torch.nn.Parameter(start.clone())
    opt = Muon([p], lr=1e-3, momentum=0.0, nesterov=False)
    p.grad = rand(64, 64, device=device, dtype=BF16, seed=4)
    for _ in range(200):
        opt.step()
    moved, want = p.detach().double() - start.double(), -0.2 * formula(p.grad)
    # values of [4, 8) have steps of 2^-5: half of one is lost at most, and the
    # updates are right to 2^-7
    assert (moved - want).norm() <= 2.0 ** -7 * want.norm() + 64 * 2.0 ** -6
    # along the updates' own direction the roundings, 2^-5 / sqrt(12) each in the
    # mean, make one of that size (four of them: once in 10^4)
    along = (moved * want).sum() / want.pow(2).sum()
    assert abs(along - 1) <= 2.0 ** -7 + 4 * 2.0 ** -5 / 12 ** 0.5 / want.norm()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_state_is_saved_and_continued(device, dtype):
    params = parameters(device, dtype)
    opt = Muon(params, lr=0.05, momentum=0.9, weight_decay=0.1)
    for step in range(2):
        give_gradients(params, step)
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    twin = Muon(twins)
    twin.load_state_dict(saved)
    before = copy.deepcopy(saved)
    for p, q in zip(params, twins):
        for k, v in opt.state[p].items():
            assert twin.state[q][k].dtype == F32 and torch.equal(twin.state[q][k], v)
    for step in range(2, 5):
        give_gradients(params, step)
        give_gradients(twins, step)
        opt.step()
        twin.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
    for k, v in before["state"].items():  # what was loaded is the caller's
        for name, t in v.items():
            assert torch.equal(t, saved["state"][k][name])


def test_state_is_fp32(device):
    for dtype in (F32, BF16):
        params = parameters(device, dtype)
        opt = Muon(params)
        give_gradients(params, 0)
        opt.step()
        for p in params:
            assert all(v.dtype == F32 for v in opt.state[p].values())


def test_older_bf16_state_is_widened(device):
    params = parameters(device, BF16)
    opt = Muon(params)
    give_gradients(params, 0)
    opt.step()
    saved = opt.state_dict()
    saved = {"param_groups": saved["param_groups"], "state": {
        k: {"momentum_buffer": v["momentum_buffer"].to(BF16)} for k, v in saved["state"].items()}}
    opt = Muon(params)
    opt.load_state_dict(saved)
    give_gradients(params, 1)
    opt.step()
    for p in params:
        assert all(v.dtype == F32 for v in opt.state[p].values())
        assert torch.isfinite(p).all()


def test_parameters_changed_between_steps(device):
    """What a parameter's rounding left belongs to the value that was rounded,
    not to one that others put in its place."""
    params = parameters(device, BF16)
    opt = Muon(params, lr=0.05, weight_decay=0.3, momentum=0.0, nesterov=False)
    give_gradients(params, 0)
    opt.step()
    with torch.no_grad():
        for p in params:
            p.zero_()
    for p in params:
        p.grad = torch.zeros_like(p)
    opt.step()
    for p in params:
        assert p.abs().sum() == 0


def test_types_without_a_step_are_refused_before_anything_changes(device):
    for dtype in (torch.float16, torch.float64):
        params = [torch.nn.Parameter(rand(4, 8, device=device, dtype=dtype))]
        opt = Muon(params)
        give_gradients(params, 0)
        start = params[0].detach().clone()
        with pytest.raises(TypeError):
            opt.step()
        assert not opt.state[params[0]] and torch.equal(params[0], start)


def test_added_groups_are_checked_too():
    opt = Muon([torch.nn.Parameter(torch.zeros(3, 4))])
    for bad in (torch.zeros(4), torch.zeros(())):
        with pytest.raises(ValueError):
            opt.add_param_group({"params": [torch.nn.Parameter(bad)]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, 2))], "lr": 0.5})
    assert len(opt.param_groups) == 2
