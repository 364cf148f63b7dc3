"""Steps of ``paged_attention`` for the tests of batches with trees."""

from __future__ import annotations

import torch

from llmserve.attention import AttentionMetadata, QuantizedKV, paged_attention


def typed_step(dtype, kind: str, long: bool, device, d: int = 32):
    """A step over a tree, a decode token and, with ``long``, a prompt of more tokens than a tree has, q / k / v of
    ``dtype`` over a cache of ``kind`` (int8, fp32, or the tensors' own type). ``step(trees)`` runs it with or without
    parents and returns (result, caches, metadata); ``step.q`` is its q."""
    bs, hq, hk = 16, 4, 2
    backend = "hip" if device.type == "cuda" else "torch"
    q_lens, ctx, tables = [4, 1], [40, 33], [[0, 1, 2], [3, 4, 5]]
    parents = [[-1, 0, 0, 2], None]
    if long:
        q_lens, ctx, tables, parents = [*q_lens, 70], [*ctx, 90], [*tables, list(range(6, 12))], [*parents, None]
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(sum(q_lens), h, d, generator=g).to(device, dtype) for h in (hq, hk, hk))
    fills = [torch.randn(12 * bs, hk, d, generator=g).to(device) for _ in range(2)]

    def step(trees: bool):
        caches = []
        for fill in fills:
            if kind == "int8":
                caches.append(QuantizedKV(12 * bs, hk, d, device))
                caches[-1].write(torch.arange(12 * bs, device=device), fill)
            else:
                caches.append(fill.to(dtype if kind == "own" else torch.float32))
        meta = AttentionMetadata.build(q_lens, ctx, tables, bs, device, backend, parents if trees else None, (hq, hk))
        assert (meta.draft is not None) == trees and (meta.rest is not None) == (long and trees)
        return paged_attention(q, k, v, *caches, meta, 0.2), caches, meta

    step.q = q
    return step
