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
