"""The example stack: steps after prompts agree with the whole sequences at once.

Both ways run the same layers on the same tokens; what differs is how each layer's
recurrence is computed (chunks with bf16 operands, or token by token), and every
layer's output is rounded to bf16, 2^-8 at most.  Through four layers, each of whose
norms passes a relative error on at its size and whose recurrence adds a few roundings
of its own, 5e-2 in the 2-norm is many times what roundings give and far below what a
wrong state, slot or order would (order one)."""

import importlib.util
import os

import pytest
import torch

from conftest import ROOT
from gdn_kernel_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[700, 1, 129, 40], [5], [64, 64, 3]])
def test_steps_follow_prompts(lengths):
    spec = importlib.util.spec_from_file_location(
        "hybrid_stack", os.path.join(ROOT, "examples", "hybrid_stack.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got, want = example.prompts_then_steps(lengths, steps=4)
    assert got.shape == want.shape == (len(lengths), 4, example.HIDDEN)
    err = (got.float() - want.float()).flatten(1).norm(dim=1) / want.float().flatten(1).norm(dim=1)
    assert torch.isfinite(got).all() and err.max().item() <= 5e-2, err
    assert _lib.device_status(torch.cuda.current_device()) == 0
