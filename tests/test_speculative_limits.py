"""Verification steps over drafted trees on the CPU: the types of mixed batches, and refused steps."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from llmserve._native import capi
from llmserve.model_runner import ModelRunner
from llmserve.sampling import SampleRow, SamplingParams
from llmserve.speculative import draft_batch, tree_attention, verify_draft
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


def test_a_refused_step_leaves_the_cache_as_it_was():
    """Requests, probabilities, tables, ids and trees that are refused: before a block is copied or the model runs."""
    copied = []

    class Model:
        cfg = SimpleNamespace(vocab_size=50, num_attention_heads=4, num_key_value_heads=2)

        def __call__(self, *args):
            raise LookupError("the model runs")

    runner = ModelRunner.__new__(ModelRunner)
    runner.cache, runner.block_size, runner.model = SimpleNamespace(layers=[], num_blocks=4), 16, Model()
    runner.device, runner.attention_backend = torch.device("cpu"), "torch"
    runner.copy_blocks = copied.append

    def sched(drafts=(8, 9, 3), up=(-1, -1, 0), table=(0,), known=(5, 6, 7)):
        seq = SimpleNamespace(token_ids=lambda: list(known), num_computed_tokens=2, spec_tokens=list(drafts),
                              spec_parents=None if up is None else list(up), block_table=list(table))
        item = SimpleNamespace(seq=seq, num_new_tokens=len(known) - 2 + len(drafts))
        return SimpleNamespace(scheduled=[item], block_copies=[(1, 2)])

    def row(**kw):
        return SampleRow(SamplingParams(**{k: v for k, v in kw.items() if k != "banned"}), [], [], None,
                         **({"banned_token_ids": kw["banned"]} if "banned" in kw else {}))

    ok = row()
    for rows, kw in (([row(presence_penalty=1.0)], {}), ([row(repetition_penalty=1.1)], {}), ([row(banned=[3])], {}), ([], {}),
                     ([ok], dict(draft_probs=torch.ones(4, 49))), ([ok], dict(draft_probs=torch.ones(4, 50).double()))):
        with pytest.raises(ValueError):
            runner.verify_step(sched(), rows, **kw)
    chain = [1] * 64
    for bad, error in ((sched(table=(9,)), IndexError), (sched(drafts=(8, 9, 50)), IndexError), (sched(up=(-1, 1, 0)), ValueError),
                       (sched(up=(-1, -1)), ValueError), (sched(known=(5, 6)), ValueError),
                       (sched(chain, None, (0, 1, 2, 3, 0)), ValueError), (sched(table=()), ValueError)):
        with pytest.raises(error):
            runner.verify_step(bad, [ok])
        if bad.scheduled[0].seq.spec_parents is not None and len(bad.scheduled[0].seq.token_ids()) > 2:
            with pytest.raises(error):
                runner.execute(bad, [0])
    assert copied == []
    for run in (lambda: runner.verify_step(sched(), [ok]), lambda: runner.execute(sched(), [0])):
        with pytest.raises(LookupError):
            run()
    assert copied == [[(1, 2)], [(1, 2)]]
    assert runner.verify_step(SimpleNamespace(scheduled=[], block_copies=[(0, 3)]), []) == [] and copied[2] == [(0, 3)]


def test_rows_without_sequences():
    empty = torch.empty(0, dtype=torch.long)
    d = draft_batch(empty, torch.zeros(1, dtype=torch.long), torch.tensor([-1] * 7), torch.empty(0, 3, dtype=torch.long), 16, 2, 1)
    assert d.positions.tolist() == d.ancestors.tolist() == [0] * 7 and d.slots.tolist() == [-1] * 7
    f = capi().llmserve_draft_metadata
    assert f(*[None] * 4, 0, 7, 3, 16, 1, 1, *[None] * 4, 0, None) == 1
    assert "null pointer" in capi().llmserve_last_error().decode()


def test_trees_larger_than_max_nodes_are_taken():
    """``max_nodes`` gives the depth limit only: a larger tree is whole, its path ends at the limit."""
    one = torch.zeros(1, dtype=torch.long)
    d = draft_batch(one, torch.tensor([0, 4]), torch.tensor([-1, 0, 1, 2]), one[None], 16, 2, 1, max_nodes=2)
    assert d.max_depth == 1 and d.ancestors.tolist() == [1, 3, 7, 15] and d.slots.tolist() == [0, 1, 2, 3]
    x = torch.zeros(4, 5)
    x[:, 3] = 9
    got = verify_draft(x, d, torch.tensor([0, 3, 3, 3]), torch.zeros(1), torch.zeros(4), torch.ones(1, 5))
    assert got.path.tolist() == [[0, 1]] and got.tokens.tolist() == [[3, 3]]
