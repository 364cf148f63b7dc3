"""Verification steps over drafted trees on the GPU, where arithmetic is at its limits: drafts that cover all
of a row, logits far from 0, channels of very different size beside each other, batches of large and small trees.

Tolerances are those of ``test_gpu_speculative.py`` unless a test derives its own.
"""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from llmserve import speculative as sp
from spec_steps import typed_step
from spec_util import Batch, check_walks, random_tree

pytestmark = pytest.mark.gpu
F32 = np.float32
NEAR = 2e-5
UNDER_ONE = F32(1 - 2.0 ** -24)  # the largest uniform number


# ---- drafts that cover a row ------------------------------------------------------------------


@pytest.mark.parametrize("seqs,v,max_depth", [(40, 4099, 63), (1600, 4099, 3), (90, 262147, 3), (90, 262147, 63)])
def test_siblings_that_cover_a_row(gpu, seqs, v, max_depth):
    """Two or three tokens have all of a row's mass and all are drafted, or all but one: a first token may have
    all but 2^-20 of it. With uniform numbers just below 1 every child but the last is rejected; the last
    one's r is 1, so it is kept; where one token is not drafted, that is the next token. The walks in the race's
    launch, in one of their own, after launches for a path's nodes, and by workgroups that read rows."""
    rng = np.random.default_rng(seqs)
    trees = [[-1] + [0] * (2 if i % 3 else 3) for i in range(seqs)]
    b = Batch(41, [2] * seqs, trees, 16, gpu, max_nodes=max_depth + 1)
    if v > 200000:
        assert b.T * v > 75 << 20  # rows too many to be read ahead of the walks
    x = torch.full((b.T, v), -float("inf"), device=gpu)
    tokens, want, set_at = np.zeros(b.T, np.int64), [], []
    for i, tree in enumerate(trees):
        a, kids = int(b.start[i]), len(tree) - 1
        support = rng.choice(v, 3 if i % 3 != 1 else 2, replace=False)
        # below e^-13.31 of the first: the rest of 1 is under 1.7e-6, rounded as 1 is; else shares of a few per cent and more
        first = 13.31 if i % 2 else rng.random() * 2
        low = [0.0] + [first + rng.random() for _ in support[1:]]
        set_at += [(a, int(t), -y) for t, y in zip(support, low)]
        end = int(rng.integers(v))
        set_at += [(a + j, end, 1.0) for j in range(1, kids + 1)]
        tokens[a + 1: a + 1 + kids] = support[:kids]
        covered = kids == len(support)
        want.append(([0, kids], [int(support[kids - 1]), end]) if covered else ([0], [int(support[-1])]))
    rows, at, values = (np.array(z) for z in zip(*set_at))
    x[torch.from_numpy(rows).to(gpu), torch.from_numpy(at).to(gpu)] = torch.from_numpy(values.astype(F32)).to(gpu)
    noise = torch.empty(seqs, v, device=gpu).exponential_(generator=torch.Generator(gpu).manual_seed(2))
    got = sp.verify_draft(x, b.draft, b.put(tokens), torch.ones(seqs, device=gpu), b.put([UNDER_ONE] * b.T, F32), noise)
    for s, (path, out) in enumerate(want):
        assert got.accepted[s] == len(path) - 1 and got.path[s, : len(path)].tolist() == path, (s, got.path[s, :4])
        assert got.tokens[s, : len(out)].tolist() == out, s


def test_walks_of_rows_just_too_many_to_read_ahead(gpu):
    """Between the limits of given and of drawn drafts: a launch for each of a path's nodes."""
    v, rng = 98511, np.random.default_rng(12)
    trees = [random_tree(rng, 58) for _ in range(16)]
    b = Batch(42, [2] * len(trees), trees, 16, gpu, max_depth=8)
    assert 75 << 20 < b.T * v < 150 << 20
    x, tokens, u, noise, _ = b.logits(v, lift=0.6)
    temps = [0.0 if i % 5 == 0 else 0.9 for i in range(len(trees))]
    got = b.verify(x, tokens, temps, u, noise)
    assert check_walks(got, b.walks(x, tokens, temps, u, noise, max_depth=8), NEAR) >= len(trees) - 2


# ---- the race far from 0 ------------------------------------------------------------------------


@pytest.mark.parametrize("seqs,drawn", [(40, False), (1600, False), (40, True)])
@pytest.mark.parametrize("offset,temp", [(0.0, 0.01), (1000.0, 0.01), (1e4, 0.01), (-1e4, 1.0), (3e5, 1.0)])
def test_the_race_does_not_see_a_shift(gpu, seqs, drawn, offset, temp):
    """Logits around an offset, most of them equal to the largest: the noise decides among those, and a softmax does
    not change with the offset. The rows hold multiples of 2^-5, so that they are the same numbers in 32 bits
    with every offset here. The race in the walks' launch and in one of its own, a last slice that is short or empty of
    likely tokens, rejected drafts."""
    v, rng = 8192 + 1003, np.random.default_rng(int(abs(offset)) + seqs)
    trees = [[-1] if i % 2 else [-1, 0, 0] for i in range(seqs)]
    b = Batch(43, [2] * seqs, trees, 16, gpu, max_nodes=3)
    x = (offset - np.where(rng.random((b.T, v)) < 0.7, 0, rng.integers(1, 64, (b.T, v))) / 32).astype(F32)
    x[::5, 8000:] = -np.inf
    assert (np.diff(np.unique(x[0, :8000])) >= 1 / 32).all()
    noise = rng.exponential(size=(seqs, v)).astype(F32)
    tokens, u = rng.integers(0, v, b.T), np.full(b.T, 0.9, F32)
    probs = np.full((b.T, v), 1 / v, F32) if drawn else None
    temps = [temp] * seqs
    got = b.verify(x, tokens, temps, u, noise, probs)
    assert check_walks(got, b.walks(x, tokens, np.full(seqs, temp, F32), u, noise, probs), NEAR) >= seqs - 4


# ---- channels and trees of very different size --------------------------------------------------


@pytest.mark.parametrize("hq", [2, 16])
@pytest.mark.parametrize("v_size,k_size", [(1.0, 1.0), (1e4, 1.0), (1e6, 1.0), (1e8, 1.0), (1.0, 1e3), (1.0, 1e4), (1e6, 1e4)])
def test_channels_of_very_different_size(gpu, hq, v_size, k_size):
    """A float32 cache with one channel of V v_size times the others, one of K k_size times the others (its q as much
    smaller) and one of q k_size times the others (its K as much smaller): every channel of the result by
    itself is as near as with channels of one size, on the fp32 matrix instructions (few rows) and in fp16 pieces: a
    float32 product's rounding is relative to each term, so that the bound on a result's 2-norm holds for a channel's."""
    b = Batch(44, [333], [random_tree(np.random.default_rng(6), 24)], 16, gpu, heads=(hq, 2))
    d = 128
    (kc, vc), (k, v) = b.caches(d, "fp32")
    q = b.rng.standard_normal((b.T, hq, d)).astype(F32)
    v[..., 5] *= F32(v_size)
    k[..., 9] *= F32(k_size)
    q[..., 9] /= F32(k_size)
    k[..., 77] /= F32(k_size)
    q[..., 77] *= F32(k_size)
    kc.copy_(torch.from_numpy(k))
    vc.copy_(torch.from_numpy(v))
    out = sp.tree_attention(b.put(q, F32), kc, vc, b.draft, d ** -0.5).cpu().numpy().astype(np.float64)
    want = b.attend64(q, k, v, (None, None), d ** -0.5)
    error = np.linalg.norm(out - want, axis=(0, 1)) / np.linalg.norm(want, axis=(0, 1))
    assert (error <= 2e-6).all(), (error.argmax(), error.max())


@pytest.mark.parametrize("kind", ["int8", "fp32"])
@pytest.mark.parametrize("nodes", [[64] + [1] * 30, [1, 2, 60, 64, 1, 3, 64, 50]])
def test_large_trees_beside_small_ones(gpu, kind, nodes):
    """Few rows on average with one large tree among them, and many with small ones among them: every tree by itself."""
    rng = np.random.default_rng(len(nodes))
    b = Batch(45, rng.integers(0, 700, len(nodes)).tolist(), [random_tree(rng, n) for n in nodes], 16, gpu, heads=(16, 2))
    caches, (k, v) = b.caches(128, kind)
    q = rng.standard_normal((b.T, 16, 128)).astype(F32)
    out = sp.tree_attention(b.put(q, F32), *caches, b.draft, 0.09).cpu().numpy().astype(np.float64)
    want = b.attend64(q, k, v, caches, 0.09)
    for s in range(len(nodes)):
        r = b.rows(s)
        assert np.linalg.norm(out[r] - want[r]) <= 2e-6 * np.linalg.norm(want[r]), s


# ---- types --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["int8", "fp32"])
@pytest.mark.parametrize("long", [False, True])
def test_a_batch_with_trees_has_the_type_it_has_without(gpu, dtype, kind, long):
    """The kernels give float32 for every type of q, with trees and without."""
    step = typed_step(dtype, kind, long, gpu, 64)
    got, caches, meta = step(trees=True)
    plain, *_ = step(trees=False)
    assert got.dtype == plain.dtype == torch.float32 and got.shape == plain.shape
    assert torch.equal(got[:5], sp.tree_attention(step.q[:5].contiguous(), *caches, meta.draft, 0.2))
    assert long == (len(got) > 5)
    assert (got[5:] - plain[5:]).norm() <= 2e-6 * plain[5:].norm()


# ---- a batch without sequences --------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 7, 1000])
def test_rows_without_sequences(gpu, rows):
    put = lambda x: torch.tensor(x, dtype=torch.long, device=gpu)  # noqa: E731
    tables = torch.empty(0, 3, dtype=torch.long, device=gpu)
    d = sp.draft_batch(put([]), put([0]), put([-1] * rows), tables, 16, 2, 1)
    assert d.native and len(d.positions) == len(d.slots) == len(d.ancestors) == rows
    assert bool((d.positions == 0).all()) and bool((d.slots == -1).all()) and bool((d.ancestors == 0).all())


def test_a_step_without_sequences(gpu):
    """Attention leaves every row alone, verification and commit have nothing to do."""
    put = lambda x: torch.tensor(x, dtype=torch.long, device=gpu)  # noqa: E731
    d = sp.draft_batch(put([]), put([0]), put([-1] * 5), torch.empty(0, 3, dtype=torch.long, device=gpu), 16, 4, 2)
    kc, vc = (torch.randn(48, 2, 128, device=gpu) for _ in range(2))
    before = kc.clone()
    q = torch.randn(5, 4, 128, device=gpu)
    out = sp.tree_attention(q, kc, vc, d, 0.1, out=torch.full_like(q, -7.5))
    assert bool((out == -7.5).all())
    got = sp.verify_draft(torch.randn(5, 11, device=gpu), d, put([0] * 5), torch.empty(0, device=gpu), torch.rand(5, device=gpu),
                          torch.empty(0, 11, device=gpu))
    assert got.accepted.shape == (0,) and got.path.shape == got.tokens.shape == (0, 64)
    sp.commit_draft(SimpleNamespace(layers=[(kc, vc)]), d, got)
    assert torch.equal(kc, before)


def test_sums_over_a_row_in_a_graph(gpu):
    """Rows whose rest is summed, captured and replayed with other rows between eager calls: every replay the eager result."""
    v, seqs = 4099, 12
    b = Batch(46, [2] * seqs, [[-1, 0, 0]] * seqs, 16, gpu)
    rng = np.random.default_rng(46)
    sets = []
    for i in range(3):
        x = np.full((b.T, v), -np.inf, F32)
        tokens = np.zeros(b.T, np.int64)
        for s in range(seqs):
            pair = rng.choice(v, 2, replace=False)
            x[3 * s, pair] = [0.0, -13.31 - rng.random()]
            x[3 * s + 1: 3 * s + 3, rng.integers(v)] = 1.0
            tokens[3 * s + 1: 3 * s + 3] = pair
        sets.append((b.put(x, F32), b.put(tokens)))
    x, tokens = (t.clone() for t in sets[0])
    numbers = [torch.ones(seqs, device=gpu), b.put([UNDER_ONE] * b.T, F32), b.put(rng.exponential(size=(seqs, v)), F32)]
    eager = [sp.verify_draft(y, b.draft, t, *numbers) for y, t in sets]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sp.verify_draft(x, b.draft, tokens, *numbers)
    for i in (1, 0, 2, 1):
        x.copy_(sets[i][0])
        tokens.copy_(sets[i][1])
        graph.replay()
        assert bool((got.accepted == 1).all())
        for a, w in ((got.accepted, eager[i].accepted), (got.path, eager[i].path), (got.tokens, eager[i].tokens)):
            assert torch.equal(a, w)
        sp.verify_draft(x, b.draft, tokens, *numbers)


@pytest.mark.parametrize("hq,d,nodes", [(2, 128, [24]), (4, 64, [24, 3]), (16, 128, [24, 40]), (32, 64, [64, 1, 7])])
@pytest.mark.parametrize("size", [30.0, 1e3, 1e5])
@pytest.mark.parametrize("rows", ["all", "some"])
@pytest.mark.parametrize("share", [0.0, 0.4])
def test_queries_of_uneven_channels_over_int8(gpu, hq, d, nodes, size, rows, share):
    """A channel of q, or a share of them, `size` times the others where K's codes are as much smaller, so that every score is a sum of products of
    one size; in all nodes or in one of each tree. A float32 product's rounding is relative to each term: every node is
    as near as with even channels."""
    b = Batch(47, [333, 90, 2][: len(nodes)], [random_tree(np.random.default_rng(6 + n), n) for n in nodes], 16, gpu, heads=(hq, 2))
    shape = (b.blocks * b.bs, 2, d)
    k = b.rng.standard_normal(shape).astype(F32)
    at = [7] if not share else np.flatnonzero(b.rng.random(d) < share)
    k[..., at] /= F32(size)
    (kc, vc), (_, v) = b.caches(d, "int8")
    idx = torch.arange(len(k), device=gpu)
    kc.write(idx, torch.from_numpy(k).to(gpu))
    kc.set_smoothing(torch.ones(2, d), hq)
    k = kc.rows(idx).cpu().numpy()
    q = b.rng.standard_normal((b.T, hq, d)).astype(F32)
    big = np.arange(b.T) if rows == "all" else b.start[:-1] + np.array(nodes) // 2
    q[np.ix_(big, range(hq), at)] *= F32(size)
    out = sp.tree_attention(b.put(q, F32), kc, vc, b.draft, d ** -0.5).cpu().numpy().astype(np.float64)
    want = b.attend64(q, k, v, (kc, vc), d ** -0.5)
    error = np.linalg.norm(out - want, axis=(1, 2)) / np.linalg.norm(want, axis=(1, 2))
    assert (error <= 2e-6).all(), (error.argmax(), error.max())


def test_uneven_queries_of_very_many_short_sequences(gpu):
    """Tens of sequences to a workgroup, a few of them with uneven queries."""
    n, d, rng = 20000, 64, np.random.default_rng(48)
    b = Batch(48, rng.integers(0, 4, n).tolist(), [[-1]] * n, 4, gpu, heads=(4, 2), max_nodes=1)
    (kc, vc), (k, v) = b.caches(d, "int8")
    kc.data[..., 7] = 0
    k[..., 7] = 0
    q = rng.standard_normal((n, 4, d)).astype(F32)
    q[5::97, :, 7] *= 1e4
    out = sp.tree_attention(b.put(q, F32), kc, vc, b.draft, 0.125).cpu().numpy().astype(np.float64)
    want = b.attend64(q, k, v, (kc, vc), 0.125)
    error = np.linalg.norm(out - want, axis=(1, 2)) / np.linalg.norm(want, axis=(1, 2))
    assert (error <= 2e-6).all(), (error.argmax(), error.max())


@pytest.mark.parametrize("kind", ["int8", "fp32"])
@pytest.mark.parametrize("hq,d", [(2, 128), (16, 128), (4, 64)])
def test_queries_that_are_not_finite_stay_in_their_rows(gpu, kind, hq, d):
    """A NaN or an infinity in a node's query makes that row of that head NaN, and no other."""
    b = Batch(49, [150], [random_tree(np.random.default_rng(3), 24)], 16, gpu, heads=(hq, 2))
    caches, (k, v) = b.caches(d, kind)
    q = b.rng.standard_normal((b.T, hq, d)).astype(F32)
    want = b.attend64(q, k, v, caches, d ** -0.5)
    odd = np.zeros((b.T, hq), bool)
    for node, head, value in ((0, 0, np.nan), (5, hq - 1, np.inf), (23, 0, -np.inf)):
        q[node, head, 9], odd[node, head] = value, True
    out = sp.tree_attention(b.put(q, F32), *caches, b.draft, d ** -0.5).cpu().numpy().astype(np.float64)
    assert np.isnan(out[odd]).all() and np.isfinite(out[~odd]).all()
    assert np.linalg.norm(out[~odd] - want[~odd]) <= 2e-6 * np.linalg.norm(want[~odd])
