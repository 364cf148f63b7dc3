"""Verification steps over drafted trees on the CPU: the types of mixed batches, and refused steps."""

from __future__ import annotations

import pytest
import torch

from llmserve.speculative import tree_attention
from spec_steps import typed_step


@pytest.mark.parametrize("dtype,kind", [(torch.float32, "int8"), (torch.float32, "own"), (torch.bfloat16, "own"),
                                        (torch.float16, "own")])
@pytest.mark.parametrize("long", [False, True])
def test_a_batch_with_trees_has_the_type_it_has_without(dtype, kind, long):
    """Trees with a decode token, and with a prompt that is no tree: the result's type is that of the same call
    without parents, a tree's values those of float32, rounded once."""
    step = typed_step(dtype, kind, long, torch.device("cpu"))
    got, caches, meta = step(trees=True)
    plain, *_ = step(trees=False)
    assert got.dtype == plain.dtype == dtype and got.shape == plain.shape
    want = tree_attention(step.q[:5].float(), *caches, meta.draft, 0.2)
    assert torch.equal(got[:5], want.to(dtype)) and torch.equal(got[5:], plain[5:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["int8", "fp32"])
def test_trees_in_16_bits_over_other_caches(dtype, kind):
    step = typed_step(dtype, kind, False, torch.device("cpu"))
    got, caches, meta = step(trees=True)
    assert got.dtype == dtype
    assert torch.equal(got, tree_attention(step.q.float(), *caches, meta.draft, 0.2).to(dtype))
