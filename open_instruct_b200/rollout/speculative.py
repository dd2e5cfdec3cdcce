"""Drafts for the rollout engine's speculative decode step: prompt lookup, as token trees.

A sequence's draft is what followed the latest earlier occurrences of its last tokens - rollouts repeat their prompt, their tools'
output and themselves.  Up to two different continuations are merged into one tree; the engine scores all of its nodes in one pass
(``ops.fused.tree_attn``), keeps what the target's own distribution confirms (``ops.fused.verify_tree``) and writes the keys and
values of what was kept (``ops.fused.kv_commit_``).  Whatever is drafted, the emitted tokens are distributed as without drafts.

A verified step costs more than an ordinary one, so it is taken only where it is expected to emit more tokens a millisecond
(``plan_drafts``): the sequences' drafts are judged by how often they were right lately (``Acceptance``), the steps by a model of
their time (``step_ms``).  Both are functions of the batch alone, so the same requests take the same steps again.
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
        """What followed the last n-gram before, latest first: lists of at most ``length`` tokens, none the beginning of another."""
        self.update(tokens)
        at = self.behind.get(tuple(tokens[-self.ngram:])) if len(tokens) >= self.ngram and length > 0 else None
        found = [tokens[p:p + length] for p in at] if at else []
        if len(found) == 2:
            short, long = sorted(found, key=len)
            if long[:len(short)] == short:
                return [long]
        return found


class Acceptance:
    """How often the next token of one sequence was among those drafted for it: over its last ten steps or so, starting at one half."""

    def __init__(self):
        self.hits = self.trials = 0.0

    def record(self, hits: int, trials: int) -> None:
        self.hits = 0.9 * self.hits + hits
        self.trials = 0.9 * self.trials + trials

    def rate(self) -> float:
        return (self.hits + 1.0) / (self.trials + 2.0)


def expected_tokens(rate, depth):
    """What drafts of ``depth`` tokens in a row are expected to add, each token being right with probability ``rate`` < 1."""
    return rate * (1.0 - rate ** depth) / (1.0 - rate)


DECODE_ROWS = 256  # rows up to which the projections run on the decode GEMMs


def step_ms(rows: int, layers: int, weights: int, eager: bool) -> float:
    """Milliseconds of a decode step over ``rows`` tokens of a model with ``weights`` bf16 numbers on one B200: reading the weights,
    the products (the rate falls where the decode GEMMs end), 0.03 a layer for its small kernels, or the launches from the host where
    no graph is replayed, and what a step takes whatever the model.  Against steps of Llama 8B and Qwen3 1.7B at contexts of 250,
    the ratio of a verified to an ordinary step is within 25 % from 32 sequences on (8B, 64 sequences of 5 nodes: 2.0 measured, 1.7 here;
    256 of 5: 3.2 and 3.0; 1.7B, 32 of 5: 2.9 and 2.8).  With fewer, 8B's ordinary steps take longer than this says (6.7 ms at 16,
    10 at 4), so that drafts are judged more strictly than they had to be."""
    device = 0.03 * layers + weights * 2 / 5.2e9 + rows * 2 * weights / (1.6e12 if rows <= DECODE_ROWS else 1.2e12)
    return 0.6 + max(device, 0.2 * layers if eager else 0.0)


def plan_drafts(ahead: list, chances: list, most: int, rows: int, plain: float, verified) -> int:
    """How many nodes each sequence may draft in this step, 0 where an ordinary step emits more tokens a millisecond.  Looked at are
    as many as ``most`` and ``rows`` tokens in all allow, the halves of that, and as many as the decode GEMMs' rows allow.  ``ahead``:
    the sequences' continuations; ``chances``: their ``Acceptance``; ``plain``: the time of an ordinary step; ``verified(rows)``: of a
    verified one."""
    batch = len(ahead)
    # drafts without end add rate / (1 - rate): most steps that do not pay are told by that alone
    if batch + sum((c.hits + 1.0) / (c.trials - c.hits + 1.0) for c, chains in zip(chances, ahead) if chains) <= batch / plain * verified(batch + 1):
        return 0
    nodes = np.array([sum(map(len, chains)) for chains in ahead])
    first = np.array([len(chains[0]) if chains else 0 for chains in ahead])
    several = np.array([len(chains) > 1 for chains in ahead])
    rate = np.array([chance.rate() for chance in chances])

    def total(share):
        return batch + int(np.minimum(nodes, share).sum())

    def largest(limit):  # share whose total fits
        low, high = 0, most
        while low < high:
            mid = (low + high + 1) // 2
            low, high = (mid, high) if total(mid) <= limit else (low, mid - 1)
        return low

    shares = {largest(min(rows, DECODE_ROWS))}
    share = largest(rows)
    while share:
        shares.add(share)
        share //= 2
    best, speed = 0, batch / plain
    for share in sorted(shares - {0}):
        depth = np.minimum(first, np.where(several, _first_share(share, 2), share))
        got = (batch + float(expected_tokens(rate, depth).sum())) / verified(total(share))
        if got > speed:
            best, speed = share, got
    return best


def _first_share(most: int, continuations: int) -> int:
    """Nodes for the latest continuation: all of them, or two thirds beside a second one."""
    return most if continuations < 2 else -(-2 * most // 3)


def draft_tree(last_token: int, continuations: list, most: int):
    """(tokens, parents, depths) of a tree whose node 0 is the sequence's newest token, with at most ``most`` drafted nodes.  With two
    different continuations the latest gets two thirds of them."""
    tokens, parents, depths = [last_token], [-1], [0]
    share = _first_share(most, len(continuations))
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
