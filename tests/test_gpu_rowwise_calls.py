"""A block with norms, dropout and residual layers in its radial MLP, through the calls that a block has: whole and in
chunks, value and gradients in one sweep, energies, frozen parameters, FP64 parameters, no edges."""

from __future__ import annotations

import pytest
import torch

from tests.helpers import random_case, rel_l2
from tests.test_gpu_rowwise_block import CFG, block_with, residual_stack

pytestmark = pytest.mark.gpu
KEYS = ("pos", "atomic_numbers", "x_node", "edge_index", "shifts", "cos_gamma_k", "sin_gamma_k")


def args_of(edges=240, dtype=torch.float32):
    case = random_case(CFG, 20, edges, seed=1)
    on = lambda t: t.to("cuda", dtype) if t.is_floating_point() else t.cuda()        # noqa: E731
    return [on(case[k]) for k in KEYS], on(case["upstream"])


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("limit", [None, 100])
def test_value_and_gradients_in_one_sweep(limit, training, monkeypatch):
    """node_output_vjp draws and drops what node_output does from the same seed, chunk by chunk; sums over chunks are
    taken in another order: 1e-5."""
    from zippel_b200.blocks import eso2
    monkeypatch.setattr(eso2, "MAX_EDGES_PER_CALL", limit)
    block = block_with(residual_stack).train(training)
    args, up = args_of()
    torch.manual_seed(5)
    out, gx, gpos, gparams = block.node_output_vjp(*args, up)
    pos, x = args[0].clone().requires_grad_(), args[2].clone().requires_grad_()
    torch.manual_seed(5)
    ref = block.node_output(pos, args[1], x, *args[3:])
    want = torch.autograd.grad(ref, [x, pos, *block.parameters()], up, allow_unused=True)
    assert torch.equal(out, ref)
    for got, w in zip((gx, gpos, *gparams), want, strict=True):
        assert (got is None) == (w is None)
        assert got is None or rel_l2(got, w) < 1e-5


def test_energy_force_and_frozen_parameters():
    block = block_with(residual_stack).eval()
    args, _ = args_of()
    pos = args[0].clone().requires_grad_()
    energy = block(pos, *args[1:])
    force, = torch.autograd.grad(energy, pos)
    assert torch.equal(energy, block.energy(block.node_output(pos, *args[1:])))
    block.requires_grad_(False)
    again = block(pos, *args[1:])
    frozen, = torch.autograd.grad(again, pos)
    assert torch.equal(again, energy) and torch.equal(frozen, force)
    with torch.no_grad():
        assert torch.equal(block(*args), energy)


def test_parameters_in_fp64():
    """The kernels' fp32 path with parameters and inputs held in FP64, as the blocks' own layers take them."""
    block = block_with(residual_stack).eval()
    args, up = args_of()
    want = torch.autograd.grad(block.node_output(*args), list(block.parameters())[:-4], up)
    block.double()
    args, up = args_of(dtype=torch.float64)
    got = torch.autograd.grad(block.node_output(*args), list(block.parameters())[:-4], up)
    for g, w in zip(got, want, strict=True):
        assert g.dtype == torch.float64 and rel_l2(g, w) < 1e-5


@pytest.mark.parametrize("training", [True, False])
def test_no_edges(training):
    block = block_with(residual_stack).train(training)
    args, up = args_of(0)
    pos, x = args[0].clone().requires_grad_(), args[2].clone().requires_grad_()
    out = block.node_output(pos, args[1], x, *args[3:])
    grads = torch.autograd.grad((out * up).sum(), [pos, x, *block.parameters()], allow_unused=True)
    assert not out.any() and not any(g.any() for g in grads if g is not None)
