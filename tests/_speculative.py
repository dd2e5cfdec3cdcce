"""Inputs and 64-bit oracles of the speculative-decoding operators, shared by the CPU and the GPU tests."""

import math

import torch

PAGE, DIM = 64, 128
BF16_STEP = 2.0 ** -8   # a rounding to bf16 is off by at most this much of the value


def make_parents(counts, shape, gen):
    """Parents of all nodes: ``chain``, ``tree`` (random earlier parent), ``star`` (all children of node 0)."""
    out = []
    for n in counts:
        for j in range(n):
            if j == 0:
                out.append(-1)
            elif shape == "chain":
                out.append(j - 1)
            elif shape == "star":
                out.append(0)
            else:
                out.append(int(torch.randint(0, j, (1,), generator=gen)))
    return out


def make_attn(heads, kv_heads, ctx, counts, shape="tree", seed=0, device="cpu", dtype=torch.bfloat16, row_extra=0, extra_rows=0, table_extra=0,
              blocks=None, garbage=True):
    """Inputs of ``tree_attn``: pages scattered over the cache; everything that must not matter (rows past a context, unused pages,
    unused table entries, columns between rows) is NaN, infinity or an impossible page."""
    g = torch.Generator().manual_seed(seed)
    B, N, width = len(ctx), sum(counts) + extra_rows, (heads + 2 * kv_heads) * DIM
    need = [-(-c // PAGE) for c in ctx]
    total = blocks or sum(need) + 2
    order = torch.randperm(total, generator=g)[: sum(need)]
    wide = max(need + [0]) + table_extra
    table = torch.full((B, wide), -7, dtype=torch.int32)
    shape_c = (total, kv_heads, PAGE, DIM)
    fill = float("nan") if garbage else 0.0
    k = torch.full(shape_c, fill, dtype=dtype, device=device)
    v = torch.full(shape_c, fill, dtype=dtype, device=device)
    if garbage:
        v[..., ::2] = float("inf")
    at = 0
    for b, c in enumerate(ctx):
        for i in range(need[b]):
            blk = int(order[at])
            table[b, i] = blk
            m = min(PAGE, c - i * PAGE)
            k[blk, :, :m] = torch.randn(kv_heads, m, DIM, generator=g).to(device, dtype)
            v[blk, :, :m] = torch.randn(kv_heads, m, DIM, generator=g).to(device, dtype)
            at += 1
    room = torch.full((N, width + row_extra), float("nan"), dtype=dtype)
    room[: sum(counts), :width] = torch.randn(sum(counts), width, generator=g).to(dtype)
    room[:, : heads * DIM] *= 1.5
    cu = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    parents = torch.tensor(make_parents(counts, shape, g) + [-2] * extra_rows, dtype=torch.int32)
    wide_table = torch.full((B, wide + 5), 1 << 30, dtype=torch.int32)
    wide_table[:, :wide] = table
    return dict(qkv=room.to(device)[:, :width], k_cache=k, v_cache=v, block_table=wide_table.to(device)[:, :wide],
                ctx=torch.tensor(ctx, dtype=torch.int32, device=device), cu_nodes=cu.to(device), parents=parents.to(device), n_q=heads,
                n_kv=kv_heads, head_dim=DIM, scale=DIM ** -0.5, max_nodes=max(1, max(counts + [1])))


def attn_oracle(a):
    """(output, sum_j p_j |v_j|) in 64 bits; rows that no sequence owns are zero in both."""
    hq, hk, dev = a["n_q"], a["n_kv"], a["qkv"].device
    N = a["qkv"].shape[0]
    out = torch.zeros(N, hq * DIM, dtype=torch.float64, device=dev)
    mag = torch.zeros_like(out)
    cu, par, blocks = a["cu_nodes"].tolist(), a["parents"].tolist(), a["k_cache"].shape[0]
    for b in range(len(cu) - 1):
        lo, n, c = cu[b], cu[b + 1] - cu[b], int(a["ctx"][b])
        if n == 0:
            continue
        x = a["qkv"][lo:lo + n].double().view(n, hq + 2 * hk, DIM)
        ks, vs = [], []
        for i in range(-(-c // PAGE)):
            blk, m = int(a["block_table"][b, i]), min(PAGE, c - i * PAGE)
            if 0 <= blk < blocks:
                ks.append(a["k_cache"][blk, :, :m].double())
                vs.append(a["v_cache"][blk, :, :m].double())
            else:
                ks.append(torch.zeros(hk, m, DIM, dtype=torch.float64, device=dev))
                vs.append(ks[-1])
        k = torch.cat(ks + [x[:, hq:hq + hk].transpose(0, 1)], 1)
        v = torch.cat(vs + [x[:, hq + hk:].transpose(0, 1)], 1)
        for t in range(n):
            if par[lo + t] < -1:
                continue
            keep, at = list(range(c)), t
            own = []
            while at >= 0:
                own.append(c + at)
                at = par[lo + at]
            keep = torch.tensor(keep + sorted(own), device=dev)
            for h in range(hq):
                kk, vv = k[h // (hq // hk)][keep], v[h // (hq // hk)][keep]
                p = torch.softmax(kk @ x[t, h] * a["scale"], 0)
                out[lo + t, h * DIM:(h + 1) * DIM] = p @ vv
                mag[lo + t, h * DIM:(h + 1) * DIM] = p @ vv.abs()
    return out, mag


def attn_bound(ref, mag):
    """The result is rounded to bf16 once (2^-8 of it), every weight may be rounded to bf16 before it meets its value (2^-8 of
    sum p |v|); scores and sums are fp32: 128 products of magnitude about 1 are off by 2^-17 at most, the exponentials by 2^-21,
    the rescaling of partial sums by a few 2^-23 - together below 2^-13 of sum p |v|."""
    return BF16_STEP * ref.abs() + (BF16_STEP + 2.0 ** -13) * mag + 1e-30


def make_verify(counts, vocab, shape="tree", drafted=False, temps=(1.0,), seed=0, device="cpu", row_extra=0, likely=0.0, extra_rows=0):
    """Inputs of ``verify_tree``; ``likely`` shifts how often a draft is accepted."""
    g = torch.Generator().manual_seed(seed)
    N, B = sum(counts) + extra_rows, len(counts)
    room = torch.full((N, vocab + row_extra), float("nan"), dtype=torch.bfloat16)
    room[:, :vocab] = (2.0 * torch.randn(N, vocab, generator=g)).bfloat16()
    tokens = torch.randint(0, vocab, (N,), generator=g)
    parents = make_parents(counts, shape, g) + [-2] * extra_rows
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    for b, n in enumerate(counts):
        for j in range(1, n):
            row = cu[b] + parents[cu[b] + j]
            room[row, tokens[cu[b] + j]] = math.log(vocab) + 2.0 + likely + 3.0 * float(torch.rand(1, generator=g) - 0.5)
    draft = None
    if drafted:
        draft = torch.softmax(room[:, :vocab].float() + 0.7 * torch.randn(N, vocab, generator=g), -1)
        for b, n in enumerate(counts):
            for j in range(1, n):
                tokens[cu[b] + j] = torch.multinomial(draft[cu[b] + parents[cu[b] + j]], 1, generator=g)[0]
        draft = draft.to(device)
    temperature = torch.tensor([temps[b % len(temps)] for b in range(B)], dtype=torch.float32)
    return dict(logits=room.to(device)[:, :vocab], tokens=tokens.to(device), parents=torch.tensor(parents, dtype=torch.int32, device=device),
                cu_nodes=torch.tensor(cu, dtype=torch.int32, device=device), temperature=temperature.to(device),
                u_accept=torch.rand(N, generator=g).to(device), u_sample=torch.rand(B, generator=g).to(device), max_nodes=max(1, max(counts + [1])),
                draft_probs=draft)


def verify_oracle(a):
    """(count, tokens, path, logprobs) from the definition, 64 bits, on the CPU."""
    logits, tok, par, cu = a["logits"].float().cpu(), a["tokens"].tolist(), a["parents"].tolist(), a["cu_nodes"].tolist()
    ua, us, temp = a["u_accept"].tolist(), a["u_sample"].tolist(), a["temperature"].tolist()
    draft = None if a["draft_probs"] is None else a["draft_probs"].double().cpu()
    V, B, T = logits.shape[1], len(cu) - 1, a["max_nodes"]
    count, emitted, path, lps = torch.zeros(B, dtype=torch.int32), torch.full((B, T), -1), torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, T).double()
    for b in range(B):
        nodes = list(range(cu[b], cu[b + 1]))
        if not nodes:
            continue

        def target(row):
            z = logits[row].double() / (temp[b] if temp[b] > 0 else 1.0)
            lp = z - z.max() - math.log(float(torch.exp(z - z.max()).sum()))
            if temp[b] > 0:
                return lp, torch.exp(lp)
            one = torch.zeros(V, dtype=torch.float64)
            one[int((z == z.max()).nonzero()[0])] = 1.0
            return lp, one

        out, walk = [], [nodes[0]]
        lp, r = target(nodes[0])
        again = True
        while again:
            again = False
            for j in [n for n in nodes if n > walk[-1] and par[n] == walk[-1] - cu[b]]:
                x, q = tok[j], None if draft is None else draft[walk[-1]]
                inside = 0 <= x < V
                if inside and ua[j] * (1.0 if q is None else float(q[x])) < float(r[x]):
                    out.append((x, float(lp[x])))
                    walk.append(j)
                    lp, r = target(j)
                    again = True
                    break
                left = r.clone() if q is None else torch.clamp(r - q, min=0)
                if q is None and inside:
                    left[x] = 0
                if float(left.sum()) > 0:
                    r = left / left.sum()
        edge = torch.cumsum(r, 0)
        over = (edge > us[b] * float(edge[-1])).nonzero()
        x = int(over[0]) if len(over) else int(r.nonzero()[-1])
        out.append((x, float(lp[x])))
        count[b] = len(out)
        for k, (x, l) in enumerate(out):
            emitted[b, k], lps[b, k], path[b, k] = x, l, walk[k]
    return count, emitted, path, lps


def logprob_bound(vocab):
    """A log-probability is z - max - log(sum): one fp32 rounding of the argument (|z| <= 64: 2^-18), a sum of fp32 weights (each
    off by 2^-22 of itself, so the sum is), one logarithm and one rounding of the result (below 2^-18 for results up to 32)."""
    return 2.0 ** -16


ALMOST_ONE = 1.0 - 2.0 ** -24


def make_covered(vocab=64, device="cpu"):
    """Certain drafts whose siblings take up all, or nearly all, that a row allows: (inputs, expected first tokens, expected counts).
    A case is the finite logits of a row, the children, their coins and what has to come out."""
    lone = 1.0 / (1.0 + math.exp(-1.0))          # share of the heavier of two tokens that lie 1 apart
    cases = [
        ([(5, 0.0), (9, -12.0)], [5, 9], [ALMOST_ONE, 0.995], 9, 2),     # the first is rejected, so the second is certain
        ([(5, 0.0), (9, -12.0)], [5, 9], [ALMOST_ONE, ALMOST_ONE], 9, 2),
        ([(1, 0.3), (2, -0.7), (3, 0.9)], [1, 2, 3], [ALMOST_ONE] * 3, 3, 2),
        ([(1, 2.5), (2, -3.0), (3, -9.0)], [3, 1, 2], [ALMOST_ONE] * 3, 2, 2),
        ([(7, 0.0), (8, 0.0), (9, 0.0)], [8, 9, 7], [ALMOST_ONE] * 3, 7, 2),
        ([(7, 1.0), (8, 0.0)], [7, 7, 8], [ALMOST_ONE] * 3, 8, 2),       # the same token twice: rejected once and for all
        ([(4, -2.0)], [6, 4], [0.0, ALMOST_ONE], 4, 2),                  # the only token that is left
    ]
    for low in (-8.0, -10.0, -12.0, -13.0):      # a heavy token rejected, then one of two light ones with a coin beside its share
        for off in (-1e-3, -2e-4, 2e-4, 1e-3):
            cases.append(([(5, 0.0), (9, low), (30, low - 1.0)], [5, 9], [ALMOST_ONE, lone + off], 9 if off < 0 else 30, 2 if off < 0 else 1))
    counts = [1 + len(c[1]) for c in cases]
    a = make_verify(counts, vocab, "star", seed=4, device=device)
    at = 0
    for finite, kids, coins, _, _ in cases:
        a["logits"][at] = float("-inf")
        for x, z in finite:
            a["logits"][at, x] = z
        a["tokens"][at + 1:at + 1 + len(kids)] = torch.tensor(kids, device=device)
        a["u_accept"][at + 1:at + 1 + len(kids)] = torch.tensor(coins, device=device)
        at += 1 + len(kids)
    return a, [c[3] for c in cases], [c[4] for c in cases]


def make_cold(vocab=2000, drafted=False, device="cpu", seed=21):
    """Logits around 20 at temperatures down to 0.05, so that logits / temperature reach several hundreds."""
    a = make_verify([3, 1, 7, 5, 12, 2, 4, 6], vocab, "tree", drafted, temps=(0.05, 0.1, 0.3, 0.07), seed=seed, device=device)
    a["logits"] = (0.5 * a["logits"].float() + 20.0).bfloat16()
    return a


def make_borders(ctx, nodes, heads=4, device="cpu", seed=0):
    """A long context in which every key at a page's border, the last one too, shows in the output: those keys answer the queries
    with a score of 6 and have a value of 1 in one dimension each (the i-th in dimension i mod 128, the other keys' values are 0),
    so an element of the output is the weight of at most ceil(keys / 128) border keys of the same weight, and losing one of them
    changes it by that share or more.  Returns the inputs and the borders' positions."""
    a = make_attn(heads, 1, [ctx], [nodes], "chain", seed=seed, device=device, garbage=False)
    g = torch.Generator().manual_seed(seed + 1)
    base = torch.randn(DIM, generator=g)
    q = base + 0.05 * torch.randn(nodes, heads, DIM, generator=g)
    a["qkv"][:, : heads * DIM] = q.view(nodes, -1).to(device, torch.bfloat16)
    a["qkv"][:, (heads + 1) * DIM:] = 0.0
    a["v_cache"].zero_()
    borders = sorted({p for p in range(ctx) if p % PAGE in (0, PAGE - 1)} | {ctx - 1})
    key = (base * (6.0 / a["scale"]) / float(base @ base)).to(device, torch.bfloat16)
    for i, p in enumerate(borders):
        blk = int(a["block_table"][0, p // PAGE])
        a["k_cache"][blk, 0, p % PAGE] = key
        a["v_cache"][blk, 0, p % PAGE, i % DIM] = 1.0
    return a, borders
