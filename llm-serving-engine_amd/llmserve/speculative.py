"""Verification steps of speculative decoding: trees of drafted tokens over the paged cache.

The reference verifies chains of drafted tokens as prompt rows (``ModelRunner.execute`` with
``spec_tokens`` and ``num_logits``, model_runner.py:40-87). Here a sequence's drafts may form a tree
of up to 64 nodes: node 0 is the sequence's last token (not in the cache yet), every other node a
drafted token with an earlier node as its parent. The nodes of a batch lie end to end in a flat
``[T]`` stream; node ``i`` of a sequence with ``c`` cached tokens is written at position ``c + i`` of
its block table and rotated for position ``c + depth``. One step:

* ``draft_batch``: positions, cache slots and ancestor masks of the nodes, from lengths, parents and
  block tables on the device (no host round trip: the lengths may be a step's own results);
* ``tree_attention``: a node sees the cached tokens, its ancestors and itself;
* ``verify_draft``: the drafts that the target's probabilities keep, and the token after them, from
  given random numbers (``verify`` draws these for ``SampleRow`` requests);
* ``commit_draft``: the cache rows of the kept path moved to consecutive positions. The sequence then
  has ``c + accepted + 1`` cached tokens and its new last token is the last one of ``tokens``.

On a ROCm device these are HIP kernels (``llmserve_draft_metadata``, ``llmserve_paged_attention_tree``,
``llmserve_verify_draft``, ``llmserve_commit_draft``) on the current stream without synchronization,
so a step of these four can be captured into a graph; elsewhere, or without the native library, torch ops.
``verify`` draws its numbers request by request and copies parameters from the host: it is not for a graph.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .attention import QuantizedKV
from .kernels import load_speculative
from .sampling import GREEDY_TEMPERATURE, SampleRow, _exponential, _penalized, _top_k_top_p_min_p

MAX_NODES = 64  # nodes of a tree: an ancestor mask is one 64-bit word


@dataclass
class DraftBatch:
    """The trees of one step and what its layers share (``draft_batch`` makes it)."""

    parents: torch.Tensor  # [T] the parent of each node, an index into its tree (-1: a root)
    block_tables: torch.Tensor  # [S, max_blocks]
    block_size: int
    q_heads: int
    kv_heads: int
    max_depth: int  # most drafts of a path
    positions: torch.Tensor  # [T] rotary position of each node
    slots: torch.Tensor  # [T] cache slot of each node (-1: none)
    ancestors: torch.Tensor  # [T] bit j: node j of the tree is an ancestor of the node, or the node itself
    plan: torch.Tensor  # native: the step's plan; torch: int64 [S, 3] first node, nodes, cached tokens

    @property
    def sequences(self) -> int:
        return self.block_tables.shape[0]

    @property
    def native(self) -> bool:
        return self.plan.dtype == torch.uint8


@dataclass
class Verified:
    """The result of a verification; ``path`` and ``tokens`` hold -1 past their last entry."""

    accepted: torch.Tensor  # [S] accepted drafts
    path: torch.Tensor  # [S, max_depth + 1] node 0, then the accepted nodes
    tokens: torch.Tensor  # [S, max_depth + 1] the accepted drafts' tokens, then the next token


def _ops(t: torch.Tensor):
    """The native kernels for tensors on a ROCm device (None: torch ops)."""
    return load_speculative() if t.is_cuda else None


def _int64(name: str, t: torch.Tensor, dim: int, device) -> torch.Tensor:
    if t.dtype != torch.long or t.dim() != dim or t.device != device:
        raise ValueError(f"{name} must be an int64 tensor of {dim} dimension(s) on {device}")
    return t if t.is_contiguous() else t.contiguous()


def draft_batch(context_lens: torch.Tensor, draft_start: torch.Tensor, parents: torch.Tensor,
                block_tables: torch.Tensor, block_size: int, q_heads: int, kv_heads: int,
                max_nodes: int = MAX_NODES, max_depth: int | None = None, native: bool = True) -> DraftBatch:
    """The trees of one step. ``context_lens`` [S]: cached tokens of each sequence, without its tree;
    ``draft_start`` [S + 1]: where each tree begins in the flat stream, and the end of the last;
    ``parents`` [T]; ``block_tables`` [S, max_blocks]: blocks of the cached tokens and the nodes; all
    int64 on one device. ``max_depth`` is the most drafts of a path: a walk ends there. ``max_nodes`` (at most 64)
    is the largest tree that the caller has, and gives ``max_depth`` when that is not given (``max_nodes - 1``);
    trees are taken as they come, up to 64 nodes, whatever it says. The values are read on the device: a parent that is no
    earlier node makes a root, and rows of no tree (past a tree's 64th node, outside
    ``draft_start``) get slot -1 and are left alone by the step's kernels. ``native=False``: torch ops
    for the whole step, also on a ROCm device."""
    dev = context_lens.device
    if not 1 <= max_nodes <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got max_nodes={max_nodes}")
    depth = max_nodes - 1 if max_depth is None else max_depth
    if not 0 <= depth < max_nodes:
        raise ValueError(f"max_depth must lie in [0, max_nodes), got {depth}")
    if block_size < 1 or q_heads < 1 or kv_heads < 1 or q_heads % kv_heads:
        raise ValueError("block_size must be positive and q_heads a multiple of kv_heads")
    context_lens = _int64("context_lens", context_lens, 1, dev)
    draft_start = _int64("draft_start", draft_start, 1, dev)
    parents = _int64("parents", parents, 1, dev)
    block_tables = _int64("block_tables", block_tables, 2, dev)
    s = block_tables.shape[0]
    if context_lens.numel() != s or draft_start.numel() != s + 1:
        raise ValueError("context_lens, draft_start and block_tables must describe the same sequences")
    ops = _ops(context_lens) if native else None
    make = _metadata_torch if ops is None else ops.draft_metadata
    positions, slots, ancestors, plan = make(context_lens, draft_start, parents, block_tables, block_size,
                                             q_heads, kv_heads)
    return DraftBatch(parents, block_tables, block_size, q_heads, kv_heads, depth, positions, slots,
                      ancestors, plan)


def tree_attention(q: torch.Tensor, k_cache, v_cache, draft: DraftBatch, scale: float,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the nodes (q [T, Hq, D]) over a layer's caches, which hold the nodes' K/V already
    (``draft.slots``): ``QuantizedKV`` pairs (key smoothing as ``paged_attention`` applies it) or float32
    tensors [slots, Hk, D]; float32 for every type of q. Rows of no tree keep what ``out`` holds (they are undefined when it is not given);
    ``out`` must not share memory with ``q``."""
    quantized = isinstance(k_cache, QuantizedKV)
    if quantized != isinstance(v_cache, QuantizedKV):
        raise ValueError("K and V caches of one kind")
    data = (k_cache.data, v_cache.data, k_cache.scale, v_cache.scale) if quantized else (
        k_cache, v_cache, None, None)
    if q.dim() != 3 or (q.shape[0], q.shape[1]) != (draft.parents.numel(), draft.q_heads) or (
            data[0].shape[1] != draft.kv_heads):
        raise ValueError("q and the caches must have the draft batch's nodes and heads")
    if out is not None and (out.shape != q.shape or out.dtype != torch.float32 or out.device != q.device
                            or not out.is_contiguous()):
        raise ValueError("out must be a contiguous float32 tensor shaped like q, on its device")
    mult = k_cache._q_mult if quantized and k_cache.smooth is not None else None
    q = q.float().contiguous()
    if out is not None and abs(out.data_ptr() - q.data_ptr()) < 4 * q.numel():
        raise ValueError("out must not share q's memory")
    ops = _ops(q) if draft.native else None
    if ops is None or (not quantized and k_cache.dtype != torch.float32):
        return _attend_torch(q, data, mult, draft, scale, torch.zeros_like(q) if out is None else out)
    if out is None:
        out = torch.empty_like(q)
    ops.paged_attention_tree_(out, q, *data, draft.block_tables, draft.ancestors, draft.plan, draft.block_size,
                              scale, mult)
    return out


def verify_draft(logits: torch.Tensor, draft: DraftBatch, draft_tokens: torch.Tensor, temperature: torch.Tensor,
                 uniforms: torch.Tensor, noise: torch.Tensor,
                 draft_probs: torch.Tensor | None = None) -> Verified:
    """Which drafts the target keeps. ``logits`` [T, V] float32: the target's at every node;
    ``draft_tokens`` [T] int64; ``temperature`` [S] (below 1e-5: greedy); ``uniforms`` [T] in [0, 1), one
    for each node's test; ``noise`` [S, V] Exp(1), for the token after the kept path; ``draft_probs``
    [T, V]: row n the distribution that node n's children were drawn from (None: the drafts are given
    tokens). Children are tested in order, child x accepted when u q(x) < r(x), r the target's
    distribution at the node less what its rejected children took (``max(r - q, 0)``, normalised): the
    emitted tokens are distributed as the target's."""
    t, s = draft.parents.numel(), draft.sequences
    if logits.dim() != 2 or logits.shape[0] != t or logits.dtype != torch.float32:
        raise ValueError("logits must be a float32 [T, V] tensor, a row for every node")
    v = logits.shape[1]
    f32 = (("temperature", temperature, (s,)), ("uniforms", uniforms, (t,)), ("noise", noise, (s, v)))
    if draft_probs is not None:
        f32 += (("draft_probs", draft_probs, (t, v)),)
    for name, x, shape in f32:
        if x.dtype != torch.float32 or x.shape != shape or x.device != logits.device:
            raise ValueError(f"{name} must be a float32 {list(shape)} tensor on {logits.device}")
    draft_tokens = _int64("draft_tokens", draft_tokens, 1, logits.device)
    if draft_tokens.numel() != t:
        raise ValueError("draft_tokens must have an entry for every node")
    args = (logits.contiguous(), draft_tokens, draft.parents, draft.plan, temperature.contiguous(),
            uniforms.contiguous(), noise.contiguous(),
            None if draft_probs is None else draft_probs.contiguous(), draft.max_depth)
    ops = _ops(logits) if draft.native else None
    return Verified(*(_verify_torch(*args) if ops is None else ops.verify_draft(*args)))


def commit_draft(cache, draft: DraftBatch, verified: Verified) -> None:
    """Moves the accepted paths' rows of every layer of ``cache`` (a ``KVCache``) to the positions behind
    their sequences' cached tokens (as they were when ``draft`` was made), in place."""
    tensors = [c for layer in cache.layers for c in layer]
    if not tensors:
        return
    quantized = isinstance(tensors[0], QuantizedKV)
    data, scales = ([c.data for c in tensors], [c.scale for c in tensors]) if quantized else (tensors, [])
    path, accepted = verified.path, verified.accepted
    ops = _ops(data[0]) if draft.native else None
    if ops is None or data[0].element_size() * data[0].shape[1] * data[0].shape[2] % 4:
        _commit_torch(data + scales, draft, path, accepted)
    else:
        ops.commit_draft_(data, scales, draft.plan, path, accepted, draft.block_tables, draft.block_size)


def check_requests(rows: list[SampleRow]) -> None:
    """Refuses requests that ``verify`` cannot serve."""
    for r in rows:
        if _penalized(r.params) or r.allowed_token_ids is not None or r.banned_token_ids:
            raise ValueError("penalties and allowed / banned tokens are not supported with drafted tokens")


def verify(logits: torch.Tensor, draft: DraftBatch, draft_tokens: torch.Tensor, rows: list[SampleRow],
           nodes: list[int], draft_probs: torch.Tensor | None = None) -> Verified:
    """``verify_draft`` for requests: ``rows[s]`` the sampling parameters and generator of sequence ``s``,
    ``nodes[s]`` the nodes of its tree. The uniform numbers and then the noise of a sampled row come
    from its generator, as ``sampling.sample`` draws the noise. Top-k / top-p / min-p cut the target's
    distribution at every node. Penalties and token masks, which depend on the tokens a path has
    emitted, are refused."""
    if len(rows) != draft.sequences or len(nodes) != len(rows) or sum(nodes) != logits.shape[0]:
        raise ValueError("one row and one node count per sequence")
    check_requests(rows)
    dev, v = logits.device, logits.shape[1]
    uniforms, noise, temps, at = [], [], [], 0
    cut = logits
    for r, n in zip(rows, nodes):
        p = r.params
        temp = p.temperature
        if p.greedy:
            uniforms.append(torch.zeros(n, device=dev))
            noise.append(torch.ones(v, device=dev))
        else:
            g = r.generator
            uniforms.append((torch.rand(n, generator=g) if g is None or g.device.type == "cpu" else
                             torch.rand(n, generator=g, device=g.device)).to(dev))
            noise.append(_exponential((v,), g).to(dev))
            if n and (p.top_k > 0 or p.top_p < 1 or p.min_p > 0):
                if cut is logits:
                    cut = logits.clone()
                each = [torch.full((n,), x) for x in (p.top_k, p.top_p, p.min_p)]
                cut[at: at + n] = _top_k_top_p_min_p(logits[at: at + n] / temp, *each)
                temp = 1.0
        temps.append(0.0 if p.greedy else temp)
        at += n
    empty = torch.empty(0, device=dev)
    return verify_draft(cut, draft, draft_tokens, torch.tensor(temps, dtype=torch.float32).to(dev),
                        torch.cat([empty, *uniforms]),
                        torch.stack(noise) if noise else torch.empty(0, v, device=dev), draft_probs)


# ---- torch ops: CPU tensors, or no native library -------------------------------------------------


def _metadata_torch(context_lens, draft_start, parents, block_tables, block_size, q_heads, kv_heads):
    dev, t = parents.device, parents.numel()
    cap = block_tables.shape[1] * block_size
    first = draft_start[:-1].clamp(0, t)
    nodes = (torch.minimum(draft_start[1:].clamp(0, t) - first, torch.tensor(MAX_NODES, device=dev))).clamp_min(0)
    ctx = context_lens.clamp(0, cap)
    plan = torch.stack([first, nodes, ctx], 1)
    positions = torch.zeros(t, dtype=torch.long, device=dev)
    slots = torch.full((t,), -1, dtype=torch.long, device=dev)
    ancestors = torch.zeros(t, dtype=torch.long, device=dev)
    for s, (a, n, c) in enumerate(plan.tolist()):
        i = torch.arange(n, device=dev)
        p = parents[a: a + n]
        up = torch.where((p >= 0) & (p < i), p, i)
        mask, depth = torch.ones_like(i) << i, (up != i).long()
        for _ in range(6):  # paths of up to 64 nodes by doubling
            mask, depth, up = mask | mask[up], depth + depth[up], up[up]
        pos = c + i
        block = pos // block_size
        inside = block < block_tables.shape[1]
        ids = block_tables[s, torch.where(inside, block, 0)]
        positions[a: a + n] = c + depth
        slots[a: a + n] = torch.where(inside & (ids >= 0), ids * block_size + pos % block_size, -1)
        ancestors[a: a + n] = mask
    return positions, slots, ancestors, plan


def _trees(draft: DraftBatch) -> list[list[int]]:
    """(first node, nodes, cached tokens) of every sequence, on the host."""
    if draft.native:
        from ._native import plan_trees

        return plan_trees(draft.plan, draft.sequences)
    return draft.plan.tolist()


def _attend_torch(q, data, mult, draft: DraftBatch, scale: float, out: torch.Tensor) -> torch.Tensor:
    k_cache, v_cache, k_scale, v_scale = data
    if mult is not None:
        q = q * mult
    hk = k_cache.shape[1]
    bs, width, blocks = draft.block_size, draft.block_tables.shape[1], k_cache.shape[0] // draft.block_size
    for s, (a, n, c) in enumerate(_trees(draft)):
        if n == 0:
            continue
        pos = torch.arange(min(c + n, width * bs), device=q.device)
        ids = draft.block_tables[s, pos // bs]
        there = (ids >= 0) & (ids < blocks)
        slots = torch.where(there, ids, 0) * bs + pos % bs
        k, v = k_cache[slots].float(), v_cache[slots].float()
        if k_scale is not None:
            k, v = k * k_scale[slots][..., None], v * v_scale[slots][..., None]
        k, v = (torch.where(there[:, None, None], x, 0.0) for x in (k, v))
        node = (pos - c).clamp_min(0)
        see = there & ((pos < c) | ((draft.ancestors[a: a + n, None] >> node & 1) == 1))
        rows = q[a: a + n].unflatten(1, (hk, -1))
        w = torch.einsum("nhgd,thd->hgnt", rows, k) * scale
        w = torch.softmax(w.masked_fill(~see, float("-inf")), -1)
        # a row that a node does not see reaches nothing, also where it is not finite
        bad = ~torch.isfinite(v)
        o = torch.einsum("hgnt,thd->nhgd", w, torch.where(bad, 0.0, v))
        if bool(bad.any()):
            wv = torch.where(see[:, None, None, :, None], w.permute(2, 0, 1, 3)[..., None] * v.permute(1, 0, 2)[:, None],
                             0.0)
            o = wv.sum(3)
        out[a: a + n] = o.flatten(1, 2)
    return out


def _verify_torch(logits, draft_tokens, parents, plan, temperature, uniforms, noise, draft_probs, max_depth):
    """The walks on the host's control flow, in float64."""
    dev, v = logits.device, logits.shape[1]
    s_count = temperature.numel()
    path = torch.full((s_count, max_depth + 1), -1, dtype=torch.long)
    tokens, accepted = path.clone(), torch.zeros(s_count, dtype=torch.long)
    up, drafts, u = parents.tolist(), draft_tokens.tolist(), uniforms.double().tolist()
    for s, (a, n, _) in enumerate(plan.tolist()):
        if n == 0:
            continue
        temp, node, kept = float(temperature[s]), 0, [0]
        while True:
            x = logits[a + node].double()
            greedy = temp < GREEDY_TEMPERATURE
            if greedy:
                left = torch.zeros_like(x)
                left[int(x.argmax())] = 1.0
            else:
                left = torch.softmax(x / temp, -1)
            taken = 0
            for i in range(node + 1, n):
                if len(kept) > max_depth or up[a + i] != node:
                    continue
                t = drafts[a + i]
                inside = 0 <= t < v
                q = torch.zeros_like(left) if draft_probs is None or greedy else draft_probs[a + node].double()
                if inside and (draft_probs is None or greedy):
                    q[t] = 1.0
                if inside and u[a + i] * float(q[t]) < float(left[t]):
                    taken = i
                    break
                rest = (left - q).clamp_min(0)
                total = float(rest.sum())
                left = rest / total if total > 0 else left
            if not taken:
                break
            node = taken
            kept.append(node)
        m = len(kept) - 1
        path[s, : m + 1] = torch.tensor(kept)
        accepted[s] = m
        tokens[s, :m] = torch.tensor([drafts[a + i] for i in kept[1:]], dtype=torch.long)
        race = left if greedy else torch.where(left > 0, left / noise[s].double(), left)
        tokens[s, m] = int(race.argmax())
    return accepted.to(dev), path.to(dev), tokens.to(dev)


def _commit_torch(tensors, draft: DraftBatch, path: torch.Tensor, accepted: torch.Tensor) -> None:
    bs, width = draft.block_size, draft.block_tables.shape[1]
    tables, blocks = draft.block_tables.tolist(), tensors[0].shape[0] // bs
    paths, counts = path.tolist(), accepted.tolist()

    def slot(s: int, pos: int) -> int:
        if pos // bs >= width or not 0 <= tables[s][pos // bs] < blocks:
            return -1
        return tables[s][pos // bs] * bs + pos % bs

    for s, (_, n, c) in enumerate(_trees(draft)):
        for j in range(1, min(counts[s], len(paths[s]) - 1) + 1):
            if not 0 <= paths[s][j] < n or paths[s][j] == j:
                continue
            src, dst = slot(s, c + paths[s][j]), slot(s, c + j)
            if src >= 0 and dst >= 0:
                for t in tensors:
                    t[dst] = t[src]


__all__ = ["MAX_NODES", "DraftBatch", "Verified", "check_requests", "commit_draft", "draft_batch", "tree_attention", "verify",
           "verify_draft"]
