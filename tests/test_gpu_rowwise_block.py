"""Layer norm, dropout and the residual join in a block's radial MLP, as they are used together."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from oracle import rowwise_oracle as orc
from tests.helpers import random_case, rel_l2

pytestmark = pytest.mark.gpu

CFG = dict(lmax=2, mmax=1, sphere_channels=16, hidden_channels=16, edge_channels=32, num_distance_basis=16,
           cutoff=5.0)


def block_with(layers, seed=0):
    from zippel_b200.blocks.eso2 import BlockConfig, ESO2Block
    torch.manual_seed(seed)
    block = ESO2Block(BlockConfig(**CFG))
    w_in, w_out = block.rad_func[0].in_features, block.rad_func[-1].out_features
    block.rad_func = layers(w_in, CFG["edge_channels"], w_out)
    return block.cuda()


def residual_stack(w_in, c, w_out):
    from zippel_b200.blocks.rowwise import ResidualNorm
    return nn.Sequential(nn.Linear(w_in, c), nn.LayerNorm(c), nn.Dropout(0.1),
                         ResidualNorm([nn.Linear(c, 2 * c), nn.LayerNorm(2 * c), nn.SiLU(), nn.Linear(2 * c, c)], c, p=0.2),
                         ResidualNorm([nn.Linear(c, c), nn.LayerNorm(c, bias=False), nn.Dropout(0.3)], c),
                         nn.Linear(c, w_out))


def stack64(mods, h, states):
    """The same stack in FP64, dropping with ``states`` in the order in which they are drawn."""
    from zippel_b200.blocks.rowwise import ResidualNorm
    drop = lambda v, p: v * orc.factors(v.shape, p, next(states).tolist())          # noqa: E731
    for m in mods:
        if isinstance(m, ResidualNorm):
            inner = stack64(m.layers, h, states)
            h = orc.layer_norm(h + (drop(inner, m.p) if m.training and m.p else inner), m.weight, m.bias, m.eps)[0]
        elif isinstance(m, nn.Dropout):
            h = drop(h, m.p) if m.training else h
        else:
            h = m(h)
    return h


@pytest.mark.parametrize("training", [True, False])
def test_radial_mlp_with_residual_layers(training):
    """Values and gradients of the whole stack within 1e-5, the bound that this package's tests hold its
    fp32 path to."""
    from zippel_b200.blocks.rowwise import dropout_state
    import copy
    block = block_with(residual_stack).train(training)
    x = torch.randn(200, block.rad_func[0].in_features, device="cuda")
    up = torch.randn(200, block.rad_func[-1].out_features, device="cuda")
    torch.manual_seed(3)
    states = [dropout_state("cuda").cpu() for _ in range(3)]
    torch.manual_seed(3)
    leaf = x.clone().requires_grad_()
    y = block.radial_mlp(block.plan(x.device), leaf)
    params = list(block.rad_func.parameters())
    got = torch.autograd.grad(y, [leaf, *params], up)
    ref = copy.deepcopy(block.rad_func).cpu().double()
    x64 = x.cpu().double().requires_grad_()
    y64 = stack64(ref, x64, iter(states))
    want = torch.autograd.grad(y64, [x64, *ref.parameters()], up.cpu().double())
    assert rel_l2(y, y64) < 1e-5
    for g, r in zip(got, want):
        assert rel_l2(g, r) < 1e-5


def call(block, case, pos, x):
    d = lambda k, t=torch.float32: case[k].to("cuda", t)                             # noqa: E731
    return block.node_output(pos, case["atomic_numbers"].cuda(), x, case["edge_index"].cuda(), d("shifts"),
                             d("cos_gamma_k"), d("sin_gamma_k"))


@pytest.mark.parametrize("limit", [None, 100])
def test_block_with_dropout_in_training(limit, monkeypatch):
    """One seed, one result, and gradients of exactly the masks that the forward drew: against central
    differences along one direction of all parameters, the graph whole and in chunks that the backward
    recomputes.  h = 2^-8: truncation of order h^2, rounding of order 1e-6 / h = 2.6e-4 of the value."""
    from zippel_b200.blocks import eso2
    monkeypatch.setattr(eso2, "MAX_EDGES_PER_CALL", limit)
    block = block_with(residual_stack).train()
    case = random_case(dict(CFG, mmax=1), 20, 240, seed=1)
    pos, x, up = (case[k].float().cuda() for k in ("pos", "x_node", "upstream"))
    params = list(block.parameters())[:-4]

    def value():
        torch.manual_seed(11)
        return (call(block, case, pos, x).double() * up.double()).sum()

    pos.requires_grad_(True)
    grads = torch.autograd.grad(value(), [*params, pos])
    again = torch.autograd.grad(value(), [*params, pos])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    g = torch.Generator("cuda").manual_seed(0)
    with torch.no_grad():
        d = [torch.randn(p.shape, generator=g, device="cuda") * p.abs().mean() for p in params]
        h, f = 2.0 ** -8, []
        for k in (1, -2):
            for p, v in zip(params, d):
                p.add_(k * h * v)
            f.append(value().item())
        for p, v in zip(params, d):
            p.add_(h * v)
    slope = (f[0] - f[1]) / (2 * h)
    want = sum((a.double() * b.double()).sum().item() for a, b in zip(grads, d))
    size = sum((a.double() * b.double()).pow(2).sum().item() for a, b in zip(grads, d)) ** 0.5
    assert abs(slope - want) < 0.02 * max(abs(want), size)
    block.eval()
    assert torch.equal(value(), value())
    torch.manual_seed(12)
    plain = call(block, case, pos, x)
    assert torch.isfinite(plain).all()


def test_captured_training_step_draws_new_masks():
    from zippel_b200.captured import CapturedStep
    block = block_with(residual_stack).train()
    case = random_case(CFG, 20, 240, seed=1)
    example = {k: v.float() if v.is_floating_point() else v for k, v in case.items()}
    step = CapturedStep(block, example, "cuda")
    seen = []
    for _ in range(2):
        step.run()
        seen.append(step.loss_host.item())
    assert seen[0] != seen[1]
    block.eval()
    step = CapturedStep(block, example, "cuda")
    seen = []
    for _ in range(2):
        step.run()
        seen.append(step.loss_host.item())
    assert seen[0] == seen[1]


def test_layers_without_a_kernel_are_still_refused():
    from zippel_b200._lib import ZpError
    block = block_with(lambda a, c, b: nn.Sequential(nn.Linear(a, c), nn.GELU(), nn.Linear(c, b)))
    with pytest.raises(ZpError):
        block.radial_mlp(block.plan("cuda:0"), torch.randn(5, block.rad_func[0].in_features, device="cuda"))
