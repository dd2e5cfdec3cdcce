"""Drafts for the rollout engine's speculative decode step: prompt lookup, as token trees.

A sequence's draft is what followed the latest earlier occurrences of its last tokens - rollouts repeat their prompt, their tools'
output and themselves.  Up to two different continuations are merged into one tree; the engine scores all of its nodes in one pass
(``ops.fused.tree_attn``), keeps what the target's own distribution confirms (``ops.fused.verify_tree``) and writes the keys and
values of what was kept (``ops.fused.kv_commit_``).  Whatever is drafted, the emitted tokens are distributed as without drafts.
"""

from __future__ import annotations

import numpy as np

from .sampler import _M0, _M1, _W0, _W1


class PromptLookup:
    """Where the n-grams of one growing token list were seen last: the positions of the tokens behind them, the two latest."""

    def __init__(self, ngram: int = 3):
        self.ngram = ngram
        self.seen = 0   # tokens whose predecessors are in the index
        self.behind: dict[tuple, tuple] = {}

    def update(self, tokens: list) -> None:
        n = self.ngram
        for p in range(max(self.seen, n), len(tokens)):
            key = tuple(tokens[p - n:p])
            old = self.behind.get(key)
            self.behind[key] = (p, old[0]) if old else (p,)
        self.seen = len(tokens)

    def continuations(self, tokens: list, length: int) -> list:
        """What followed the last n-gram before, latest first: lists of at most ``length`` tokens."""
        self.update(tokens)
        at = self.behind.get(tuple(tokens[-self.ngram:])) if len(tokens) >= self.ngram and length > 0 else None
        return [tokens[p:p + length] for p in at] if at else []


def draft_tree(last_token: int, continuations: list, most: int):
    """(tokens, parents, depths) of a tree whose node 0 is the sequence's newest token, with at most ``most`` drafted nodes.  With two
    different continuations the latest gets two thirds of them."""
    tokens, parents, depths = [last_token], [-1], [0]
    share = most if len(continuations) < 2 else -(-2 * most // 3)
    for k, chain in enumerate(continuations[:2]):
        at = 0
        for depth, token in enumerate(chain, 1):
            known = next((j for j in range(at + 1, len(tokens)) if parents[j] == at and tokens[j] == token), None)
            if known is None:
                if len(tokens) - 1 >= (share if k == 0 else most):
                    break
                known = len(tokens)
                tokens.append(int(token))
                parents.append(at)
                depths.append(depth)
            at = known
    return tokens, parents, depths


def uniforms(seeds: np.ndarray, counters: np.ndarray, index: np.ndarray) -> np.ndarray:
    """Philox4x32-10 numbers in [0, 1) keyed like the sampler's (seed, step counter, index), one for each entry of the arrays; the
    engine's indices start at 2^31, above every token id, so no number is used twice."""
    mask = np.uint64(0xFFFFFFFF)
    seeds = seeds.astype(np.int64).astype(np.uint64)
    c0, c1 = index.astype(np.uint64) & mask, counters.astype(np.int64).astype(np.uint64) & mask
    c2, c3 = np.zeros_like(c0), np.zeros_like(c0)
    k0, k1 = seeds & mask, seeds >> np.uint64(32)
    for _ in range(10):
        p0, p1 = np.uint64(_M0) * c0, np.uint64(_M1) * c2
        c0, c1, c2, c3 = ((p1 >> np.uint64(32)) ^ c1 ^ k0) & mask, p1 & mask, ((p0 >> np.uint64(32)) ^ c3 ^ k1) & mask, p0 & mask
        k0, k1 = (k0 + np.uint64(_W0)) & mask, (k1 + np.uint64(_W1)) & mask
    return (c0 >> np.uint64(8)).astype(np.float32) * np.float32(2.0 ** -24)
