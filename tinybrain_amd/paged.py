"""PagedKVCache: one key/value cache that many requests share.

The reference's KVCache is paged as well (16 tokens a page,
Sources/TinyBrainRuntime/KVCache.swift:61-120) but holds one sequence; here
requests of any lengths draw blocks from one pool.  All state lives on the GPU
(block table, lengths, stack of free blocks) and every call only enqueues work,
so a step can be captured in a graph and replayed with other lengths.
"""
from __future__ import annotations

from typing import Any, NamedTuple

from .quantized import PreconditionFailure


class PagedPlan(NamedTuple):
    """What tbh_paged_plan_device computes for one step (int32 device tensors)."""
    queryStart: Any     # [requests + 1]: first row of each request among the step's tokens
    granted: Any        # [requests]: tokens that got slots (its new tokens, or 0)
    slots: Any          # [maxTokens]: where a row is stored; -1: nowhere
    positions: Any      # [maxTokens]: a row's position in its request; -1 likewise
    contextLens: Any    # [requests]: lengths after the step
    freeCount: Any      # [1]: free blocks after the step


class PagedKVCache:
    """The cache arrays of every layer and the state that the calls share.

        cache = PagedKVCache(backend, layers, blocks, blockSize, kvHeads, headDim, requests, blocksPerRequest)
        plan = cache.plan(newLens, maxTokens)            # int32 cuda [requests]; -1 releases a request
        for layer in range(layers):
            q = cache.append(layer, plan, k, v, q, ropeBase=10000.0)
            y = cache.attention(layer, plan, q, numHeads)

    A plan advances the lengths, so it is made once a step, before the layers.
    """

    def __init__(self, backend, numLayers: int, numBlocks: int, blockSize: int, numKVHeads: int, headDim: int,
                 maxRequests: int, blocksPerRequest: int, dtype=None):
        import torch

        dtype = torch.float32 if dtype is None else dtype
        if dtype not in (torch.float32, torch.bfloat16):
            raise PreconditionFailure("the cache is float32 or bfloat16")
        if min(numLayers, numBlocks, blockSize, numKVHeads, headDim, maxRequests, blocksPerRequest) <= 0:
            raise PreconditionFailure("sizes must be positive")
        if blockSize > 1024 or blockSize & (blockSize - 1):
            raise PreconditionFailure("blockSize must be a power of two, at most 1024")
        dev = torch.device("cuda", backend.device)
        shape = (numBlocks, numKVHeads, blockSize, headDim)
        self.backend, self.blockSize = backend, blockSize
        self.keys = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(numLayers)]
        self.values = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(numLayers)]
        self.blockTable = torch.full((maxRequests, blocksPerRequest), -1, dtype=torch.int32, device=dev)
        self.contextLens = torch.zeros(maxRequests, dtype=torch.int32, device=dev)
        # block 0 is handed out first
        self.freeBlocks = torch.arange(numBlocks - 1, -1, -1, dtype=torch.int32, device=dev)
        self.freeCount = torch.full((1,), numBlocks, dtype=torch.int32, device=dev)

    def plan(self, newLens, maxTokens: int, stream=None) -> PagedPlan:
        """Blocks, slots and positions of the next newLens[b] tokens of each
        request (0: idle, negative: released); advances the cache's state.  A
        request waits (granted 0) if there are no blocks for it or the step's
        tokens up to its own are more than maxTokens."""
        return self.backend.paged_plan_device(newLens, self.contextLens, self.blockTable, self.freeBlocks,
                                              self.freeCount, self.blockSize, maxTokens,
                                              contextOut=self.contextLens, freeCountOut=self.freeCount,
                                              stream=stream)

    def append(self, layer: int, plan: PagedPlan, k, v, q=None, ropeBase: float = 0.0, qOut=None, stream=None):
        """Stores a layer's new keys and values; returns the (rotated) queries."""
        return self.backend.paged_append_device(self.keys[layer], self.values[layer], plan.slots, k, v, q=q,
                                                positions=plan.positions, ropeBase=ropeBase, qOut=qOut,
                                                stream=stream)

    def attention(self, layer: int, plan: PagedPlan, q, numHeads: int, scale: float = 0.0, maxQueryLen: int = 0,
                  maxContextLen: int = 0, out=None, stream=None):
        """Attention of the step's tokens over the layer's cache."""
        return self.backend.paged_attention_device(q, self.keys[layer], self.values[layer], self.blockTable,
                                                   plan.queryStart, plan.contextLens, numHeads, scale=scale,
                                                   maxQueryLen=maxQueryLen, maxContextLen=maxContextLen, out=out,
                                                   stream=stream)

    def reorder(self, parents, beams: int, sharedLens=None, reordered=None, stream=None) -> None:
        """Lets row i of every group of `beams` requests go on where row parents[i]
        stood (a beam search's selection), in place: the block table, and in every
        layer the contents of rows that several follow.  sharedLens [groups]: lengths
        of the prompts that a group's rows share.  The rows of a group hold
        equally many tokens; else, or with a parent outside its group, it is left
        as it is (reordered [groups], if given: 0)."""
        self.backend.paged_reorder_device(self.keys, self.values, self.blockTable, self.contextLens, parents, beams,
                                          sharedLens=sharedLens, tableOut=self.blockTable, reordered=reordered,
                                          stream=stream)
