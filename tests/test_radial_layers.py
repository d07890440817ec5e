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
