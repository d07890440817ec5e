"""Layers of a radial MLP that do not fit what comes in: refused before anything is launched (their parameters would be
read past their ends, or a norm taken over other channels than it names).  No device is needed for it."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn


def run(layers, width=32):
    from zippel_b200.blocks import eso2
    return eso2.radial_mlp(None, torch.randn(5, width), layers)


def residual(layers, width):
    from zippel_b200.blocks.rowwise import ResidualNorm
    return ResidualNorm(layers, width)


@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("width", [16, 64])
@pytest.mark.parametrize("inside", [False, True])
def test_a_norm_of_another_width(width, affine, inside):
    for behind in ([], [nn.SiLU()]):
        layers = [nn.LayerNorm(width, elementwise_affine=affine), *behind]
        with pytest.raises(ValueError, match="32"):
            run([residual(layers, 32)] if inside else layers)


@pytest.mark.parametrize("n_in", [8, 16, 31, 33, 64])
def test_a_linear_layer_of_another_width(n_in):
    for layers in ([nn.Linear(n_in, 24)], [nn.Linear(n_in, 24, bias=False)], [residual([nn.Linear(n_in, 32)], 32)],
                   [("linear", torch.zeros(24, n_in), torch.zeros(24))]):
        with pytest.raises(ValueError, match="32"):
            run(layers)
    with pytest.raises(ValueError, match="bias"):
        run([("linear", torch.zeros(24, 32), torch.zeros(8))])


@pytest.mark.parametrize("shape", [(16,), (64,), (1,), (32, 1)])
def test_a_norm_with_parameters_of_another_width(shape):
    """For a functional caller, which names no width."""
    fit, other = torch.zeros(32), torch.zeros(shape)
    for gamma, beta in ((other, other), (fit, other), (other, fit)):
        with pytest.raises(ValueError, match="32"):
            run([("ln_silu", gamma, beta, 1e-5)])


def test_a_norm_without_parameters_in_front_of_a_silu_is_not_refused_for_them():
    """(The refusal that is left is that there is no CPU path.)"""
    for norm in (nn.LayerNorm(32, elementwise_affine=False), nn.LayerNorm(32, bias=False)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            run([norm, nn.SiLU()])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["no parameters", "no bias"])
def test_a_norm_without_parameters_in_front_of_a_silu(kind):
    """Values and gradients within 1e-5 of the same layers in FP64, the bound that this package's tests hold its fp32
    path to."""
    import copy

    from tests.helpers import rel_l2
    from zippel_b200.blocks.eso2 import Plan, radial_mlp
    torch.manual_seed(0)
    norm = nn.LayerNorm(32, elementwise_affine=False) if kind == "no parameters" else nn.LayerNorm(32, bias=False)
    layers = nn.Sequential(nn.Linear(16, 32), norm, nn.SiLU(), nn.Linear(32, 24)).cuda()
    if kind == "no bias":
        nn.init.normal_(norm.weight)
    x, up = torch.randn(100, 16, device="cuda", requires_grad=True), torch.randn(100, 24, device="cuda")
    y = radial_mlp(Plan.get(2, 1, 16, 16, x.device), x, list(layers))
    got = torch.autograd.grad(y, [x, *layers.parameters()], up)
    ref = copy.deepcopy(layers).cpu().double()
    x64 = x.detach().cpu().double().requires_grad_()
    y64 = ref(x64)
    want = torch.autograd.grad(y64, [x64, *ref.parameters()], up.cpu().double())
    assert rel_l2(y, y64) < 1e-5
    for g, r in zip(got, want, strict=True):
        assert rel_l2(g, r) < 1e-5


STACKS = {"dropout for silu": lambda c, w: [nn.Linear(w, c), nn.LayerNorm(c), nn.Dropout(0.1), nn.Linear(c, c),
                                             nn.LayerNorm(c), nn.SiLU()],
          "residual layers": lambda c, w: [nn.Linear(w, c), nn.LayerNorm(c), nn.SiLU(), residual([nn.Linear(c, c)], c),
                                            nn.LayerNorm(c), nn.SiLU()],
          "one layer more": lambda c, w: [nn.Linear(w, c), nn.LayerNorm(c), nn.SiLU(), nn.Linear(c, c), nn.LayerNorm(c),
                                           nn.SiLU(), nn.Linear(c, c), nn.Dropout(0.1)],
          "another eps": lambda c, w: [nn.Linear(w, c), nn.LayerNorm(c, eps=1e-3), nn.SiLU(), nn.Linear(c, c),
                                        nn.LayerNorm(c), nn.SiLU()]}


@pytest.mark.parametrize("name", STACKS)
def test_a_program_is_not_bound_to_other_layers(name):
    """The programs have the reference's radial MLP written out, eps 1e-5 included."""
    from tests.helpers import random_case
    from zippel_b200.blocks.eso2 import BlockConfig, ESO2Block, load_jd
    from zippel_b200.blocks.ir_bind import bind
    cfg = dict(lmax=2, mmax=1, sphere_channels=8, hidden_channels=8, edge_channels=16, num_distance_basis=8, cutoff=5.0)
    block, case = ESO2Block(BlockConfig(**cfg)), random_case(cfg, 6, 20, seed=1)
    bind(block, case, load_jd(2))
    last = block.rad_func[-1]
    block.rad_func = nn.Sequential(*STACKS[name](16, block.rad_func[0].in_features), last)
    with pytest.raises(ValueError, match="radial"):
        bind(block, case, load_jd(2))
