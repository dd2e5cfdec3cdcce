"""Speculative-decoding operators of the rollout engine as measurable cases: attention of a tree of drafted tokens over the
paged KV cache, verification of the tree against the target's probabilities, and the commit of the accepted path's keys and
values into the cache.

Every case runs in two forms on the same inputs: the plain form (elementary torch operations, also on a tree without the
kernels) and, with ``own = True``, the calls of ``open_instruct_b200.ops.fused`` that a user's program makes.

Conventions, the same for all three operators: sequence ``b`` of a batch owns the nodes ``cu_nodes[b] .. cu_nodes[b + 1]``;
``parents[n]`` is the position of a node's parent inside its own sequence, smaller than the node's own position, ``-1`` for a
root and ``-2`` for padding; node 0 of a sequence is its newest token, whose keys and values are not in the cache yet.  A node
attends to the sequence's ``ctx[b]`` cached tokens, to its ancestors and to itself.
"""

import math

import torch

own = False

PAGE = 64      # tokens of one cache page
DIM = 128      # head dimension of the kernel path
_GOLDEN = 0.6180339887498949


def listed():
    return [
        # one new token for each of a few sequences: a decode step without drafts, latency counts
        dict(name="attn single token", op="attn", batch=8, nodes=1, ragged=False, shape="chain", ctx=512, ctx_low=64, heads=32, kv_heads=8),
        # prompt-lookup drafts in the middle of a rollout batch: short chains, ragged contexts
        dict(name="attn chains", op="attn", batch=64, nodes=5, ragged=True, shape="chain", ctx=2048, ctx_low=100, heads=32, kv_heads=8),
        # draft trees on a model with seven query heads per KV head, odd context lengths
        dict(name="attn trees, group of 7", op="attn", batch=32, nodes=27, ragged=True, shape="tree", ctx=8189, ctx_low=1, heads=28, kv_heads=4),
        # as many KV heads as query heads: the cache is four times as large per token
        dict(name="attn one head a group", op="attn", batch=128, nodes=8, ragged=False, shape="tree", ctx=1024, ctx_low=256, heads=32, kv_heads=32),
        # full 64-node trees over long reasoning traces of a large model
        dict(name="attn long contexts", op="attn", batch=16, nodes=64, ragged=False, shape="tree", ctx=32768, ctx_low=8192, heads=64, kv_heads=8),
        # a handful of sequences at the tail of a batch: latency counts
        dict(name="verify few chains", op="verify", batch=4, nodes=5, ragged=False, shape="chain", vocab=128256, drafted=False, temps="one"),
        # a draft model's chains with its probabilities
        dict(name="verify drafted chains", op="verify", batch=64, nodes=6, ragged=True, shape="chain", vocab=128256, drafted=True, temps="mixed"),
        # a full rollout batch with trees, the largest vocabulary
        dict(name="verify trees", op="verify", batch=256, nodes=16, ragged=False, shape="tree", vocab=152064, drafted=False, temps="one"),
        # a vocabulary of odd size (logit rows are not 16-byte aligned), a draft model's trees
        dict(name="verify odd vocabulary", op="verify", batch=31, nodes=9, ragged=True, shape="tree", vocab=50281, drafted=True, temps="mixed"),
        # the accepted tokens of four sequences, all layers
        dict(name="commit few", op="commit", batch=4, nodes=5, layers=32, ctx=512, ctx_low=60, heads=32, kv_heads=8),
        # the accepted tokens of a full batch, all layers
        dict(name="commit batch", op="commit", batch=128, nodes=8, layers=32, ctx=256, ctx_low=1, heads=32, kv_heads=8),
    ]


_HEADS = [(32, 8), (28, 4), (40, 8), (64, 8), (32, 32), (16, 16), (16, 8), (40, 40), (48, 4), (4, 2)]
_VOCABS = [32768, 50304, 50281, 100278, 100352, 128256, 151936, 152064]


def _log_between(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "verify", "verify", "commit"])
    shape, ragged = rng.choice(["chain", "tree"]), rng.random() < 0.6
    while True:
        batch, nodes = _log_between(rng, 1, 256), _log_between(rng, 1, 64)
        heads, kv_heads = rng.choice(_HEADS)
        if op == "attn":
            ctx = _log_between(rng, 1, 32768)
            if batch * ctx * kv_heads > 16 * 32768 * 8 or batch * ctx * heads * nodes > 16 * 32768 * 64 * 64:
                continue
            return dict(op=op, batch=batch, nodes=nodes, ragged=ragged, shape=shape, ctx=ctx, ctx_low=rng.randint(0, ctx), heads=heads, kv_heads=kv_heads)
        if op == "verify":
            vocab = rng.choice(_VOCABS + [rng.randint(1000, 60000)])
            drafted = rng.random() < 0.5
            if batch * nodes * vocab > 256 * 16 * 152064 // (3 if drafted else 1) or (drafted and nodes > 24):
                continue
            return dict(op=op, batch=batch, nodes=nodes, ragged=ragged, shape=shape, vocab=vocab, drafted=drafted, temps=rng.choice(["one", "mixed"]))
        layers, ctx = rng.randint(1, 48), _log_between(rng, 1, 4096)
        nodes = min(nodes, 16)
        if batch * nodes * layers * (heads + 2 * kv_heads) > 128 * 8 * 32 * 48 or batch * (ctx // PAGE + 2) * layers * kv_heads > 128 * 6 * 32 * 8:
            continue
        return dict(op=op, batch=batch, nodes=nodes, layers=layers, ctx=ctx, ctx_low=rng.randint(0, ctx), heads=heads, kv_heads=kv_heads)


# ------------------------------------------------------------------------------------------------ sizes and inputs
def _spread(count, low, high):
    """``count`` whole numbers over [low, high], the largest among them: the same ones for every seed."""
    return [high if i == 0 else low + int((high - low + 1) * ((i * _GOLDEN) % 1.0)) for i in range(count)]


def _sizes(case):
    """(nodes of each sequence, context of each sequence) before the seed shuffles the sequences."""
    n = _spread(case["batch"], 1, case["nodes"]) if case.get("ragged") else [case["nodes"]] * case["batch"]
    return n, _spread(case["batch"], case["ctx_low"], case["ctx"]) if "ctx" in case else None


def _parents(counts, shape, gen):
    """Parents of every node; the trees branch more near their roots, as trees of a drafter's best guesses do."""
    out = []
    draws = torch.rand(sum(counts), generator=gen).tolist()
    for n in counts:
        for j in range(n):
            r = draws[len(out)]
            out.append(j - 1 if shape == "chain" or j == 0 else int(j * r ** 0.7) if r < 0.6 else j - 1)
    return out


def _pages(ctx, extra, gen):
    """A block table whose pages are scattered over the cache, and how many pages the cache has."""
    need = [-(-(c + e) // PAGE) for c, e in zip(ctx, extra)]
    width, total = max(1, max(need)), sum(need) + 3
    order = torch.randperm(total, generator=gen)
    table, at = torch.zeros(len(ctx), width, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    return table, total


def prepare(case, seed):
    host, dev = torch.Generator().manual_seed(seed), torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    counts, ctx = _sizes(case)
    order = torch.randperm(case["batch"], generator=host).tolist()
    counts = [counts[i] for i in order]
    cu = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    N = int(cu[-1])
    s = dict(op=case["op"], cu=cu.to(dev), max_nodes=case["nodes"])

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.bfloat16).mul_(std)

    if case["op"] in ("attn", "commit"):
        heads, kv_heads = case["heads"], case["kv_heads"]
        ctx = [ctx[i] for i in order]
        width = (heads + 2 * kv_heads) * DIM
        s.update(heads=heads, kv_heads=kv_heads, ctx=torch.tensor(ctx, dtype=torch.int32, device=dev))
    if case["op"] == "attn":
        table, total = _pages(ctx, [0] * len(ctx), host)
        qkv = normal(N, width)
        qkv[:, : heads * DIM] *= 2.0   # peaked scores, as trained models have them
        s.update(qkv=qkv, k_cache=normal(total, kv_heads, PAGE, DIM), v_cache=normal(total, kv_heads, PAGE, DIM), table=table.to(dev),
                 parents=torch.tensor(_parents(counts, case["shape"], host), dtype=torch.int32, device=dev), scale=DIM ** -0.5)
    elif case["op"] == "commit":
        accepted = _spread(case["batch"], 1, case["nodes"])
        accepted = [accepted[i] for i in torch.randperm(case["batch"], generator=host).tolist()]
        table, total = _pages(ctx, [case["nodes"]] * len(ctx), host)
        path = torch.full((case["batch"], case["nodes"]), -1, dtype=torch.int32)
        for b, a in enumerate(accepted):  # the root, then ever later nodes
            later = torch.randperm(case["nodes"] - 1, generator=host)[: a - 1].sort().values + 1
            path[b, 0] = cu[b]
            path[b, 1:a] = cu[b] + later.int()
        s.update(layers=[normal(N, width) for _ in range(case["layers"])], table=table.to(dev), path=path.to(dev),
                 k_cache=normal(case["layers"], total, kv_heads, PAGE, DIM), v_cache=normal(case["layers"], total, kv_heads, PAGE, DIM))
    else:
        V, B = case["vocab"], case["batch"]
        parents = _parents(counts, case["shape"], host)
        start = cu[:-1].tolist()
        owner = [b for b, n in enumerate(counts) for _ in range(n)]
        choice = [0.0, 0.7, 1.0, 1.3] if case["temps"] == "mixed" else [1.0]
        temp = torch.tensor([choice[i % len(choice)] for i in order], dtype=torch.float32, device=dev)
        logits = normal(N, V, std=2.0)
        tokens = torch.randint(0, V, (N,), generator=gen, device=dev)
        child = [j for j in range(N) if parents[j] >= 0]
        above = torch.tensor([start[owner[j]] + parents[j] for j in child], dtype=torch.long, device=dev)
        below = torch.tensor(child, dtype=torch.long, device=dev)
        # a draft that the target finds likely: about as heavy as everything else in its row, more or less
        level = math.log(V) + 2.0 + 5.0 * torch.rand(len(child), generator=gen, device=dev) - 2.5
        logits[above, tokens[below]] = level.to(torch.bfloat16)
        s.update(logits=logits, tokens=tokens, parents=torch.tensor(parents, dtype=torch.int32, device=dev), temperature=temp,
                 u_accept=torch.rand(N, generator=gen, device=dev), u_sample=torch.rand(B, generator=gen, device=dev), draft_probs=None)
        if case["drafted"]:  # the drafter: the target with noise on its logits; children are drawn from its row
            draft = torch.softmax(logits.float() + 0.7 * torch.randn(N, V, generator=gen, device=dev), -1)
            if child:
                tokens[below] = torch.multinomial(draft[above], 1, generator=gen).squeeze(1)
            s["draft_probs"] = draft
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _attn_plain(s):
    hq, hk, T, cu = s["heads"], s["kv_heads"], s["max_nodes"], s["cu"].long()
    B, g, dev = cu.numel() - 1, s["heads"] // s["kv_heads"], s["qkv"].device
    n = cu[1:] - cu[:-1]
    here = torch.arange(T, device=dev) < n[:, None]
    rows = torch.where(here, cu[:-1, None] + torch.arange(T, device=dev), 0)
    x = s["qkv"][rows].float().view(B, T, hq + 2 * hk, DIM).masked_fill(~here[:, :, None, None], 0.0)
    par = torch.where(here, s["parents"].long()[rows], -2)
    q = x[:, :, :hq].view(B, T, hk, g, DIM).permute(0, 2, 3, 1, 4).reshape(B, hk, g * T, DIM)
    pages, span = s["table"].long(), s["table"].shape[1] * PAGE
    old = torch.arange(span, device=dev) < s["ctx"][:, None]

    def keys(cache, new):
        c = cache[pages].permute(0, 2, 1, 3, 4).reshape(B, hk, span, DIM).float()
        return torch.cat([c.masked_fill_(~old[:, None, :, None], 0.0), new.permute(0, 2, 1, 3)], 2)

    k = keys(s["k_cache"], x[:, :, hq:hq + hk])
    up = torch.eye(T, device=dev) + (par[:, :, None] == torch.arange(T, device=dev)).float()
    sees = (torch.linalg.matrix_power(up, T) > 0) & (par > -2)[:, :, None]        # ancestors and the node itself
    live = torch.cat([old[:, None, :] & (par > -2)[:, :, None], sees], 2)          # [B, T, span + T]
    e = (q @ k.transpose(-1, -2)).mul_(s["scale"]).view(B, hk, g, T, span + T)
    del k
    e.masked_fill_(~live[:, None, None], -math.inf)
    top = e.amax(-1, keepdim=True).clamp_(min=-1e30)
    e.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = e.view(B, hk, g * T, span + T) @ keys(s["v_cache"], x[:, :, hq + hk:])
    o = o.view(B, hk, g, T, DIM) / total.clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, hq * DIM)[here].to(torch.bfloat16)


def _verify_plain(s):
    logits, tokens, par, cu, draft = s["logits"], s["tokens"], s["parents"].long(), s["cu"].long(), s["draft_probs"]
    N, V = logits.shape
    B, T, dev = cu.numel() - 1, s["max_nodes"], logits.device
    n = cu[1:] - cu[:-1]
    owner = torch.repeat_interleave(torch.arange(B, device=dev), n, output_size=N)
    temp = s["temperature"]
    z = logits.float() / torch.where(temp > 0, temp, 1.0)[owner][:, None]
    top = z.amax(-1)
    w = z.sub_(top[:, None]).exp()            # z is relative to the row's largest from here on
    total = w.sum(-1, dtype=torch.float64)
    best = logits.float().argmax(-1)
    greedy = temp <= 0
    seq, cols = torch.arange(B, device=dev), torch.arange(V, device=dev)

    def weights(row):  # [B, V], 64 bits: the target's probabilities at one node of each sequence
        p = w[row].double() / total[row][:, None]
        return torch.where(greedy[:, None], (cols == best[row][:, None]).double(), p)

    out_tokens = torch.full((B, T), -1, dtype=torch.int64, device=dev)
    path = torch.full((B, T), -1, dtype=torch.int32, device=dev)
    logprobs = torch.zeros(B, T, dtype=torch.float32, device=dev)
    some = n > 0
    cur, count = torch.where(some, cu[:-1], 0), torch.zeros(B, dtype=torch.int64, device=dev)
    r = weights(cur)
    path[:, 0] = torch.where(some, cur, -1).int()

    def emit(token, where):
        lp = (z[cur, token].double() - torch.log(total[cur])).float()
        out_tokens[seq, count] = torch.where(where, token, out_tokens[seq, count])
        logprobs[seq, count] = torch.where(where, lp, logprobs[seq, count])

    for j in range(1, T):  # siblings and descendants come in the order of their positions
        node = (cu[:-1] + j).clamp(max=N - 1)
        child = (j < n) & (par[node] == cur - cu[:-1]) & (par[node] >= 0)
        x = tokens[node]
        q = draft[cur].double() if draft is not None else (cols == x[:, None]).double()
        yes = child & (s["u_accept"][node].double() * q[seq, x] < r[seq, x])
        no = child & ~yes
        emit(x, yes)
        left = (r - q).clamp_(min=0.0) if draft is not None else r * (1.0 - q)
        mass = left.sum(-1, keepdim=True)
        r = torch.where((no[:, None]) & (mass > 0), left / mass, r)
        cur = torch.where(yes, node, cur)
        count = count + yes
        path[seq, count] = torch.where(yes, node.int(), path[seq, count])
        r = torch.where(yes[:, None], weights(cur), r)
    c = r.cumsum(-1)
    token = (c <= s["u_sample"].double()[:, None] * c[:, -1:]).sum(-1)
    last = torch.where(r > 0, cols, 0).amax(-1)
    emit(torch.minimum(token, last), some)
    return (count + 1).mul(some).int(), out_tokens, path, logprobs


def _commit_plain(s):
    hq, hk = s["heads"], s["kv_heads"]
    b, j = torch.nonzero(s["path"] >= 0, as_tuple=True)
    rows = s["path"][b, j].long()
    at = s["ctx"][b].long() + j
    page, off = s["table"][b, at // PAGE].long(), at % PAGE
    new = torch.stack([x[rows, hq * DIM:] for x in s["layers"]], 1).view(rows.numel(), len(s["layers"]), 2, hk, DIM)
    s["k_cache"][:, page, :, off] = new[:, :, 0]
    s["v_cache"][:, page, :, off] = new[:, :, 1]
    return s["k_cache"], s["v_cache"]


def run(state):
    s = state
    if not own:
        return {"attn": _attn_plain, "verify": _verify_plain, "commit": _commit_plain}[s["op"]](s)
    from open_instruct_b200.ops import fused

    if s["op"] == "attn":
        return fused.tree_attn(s["qkv"], s["k_cache"], s["v_cache"], s["table"], s["ctx"], s["cu"], s["parents"], s["heads"], s["kv_heads"],
                               DIM, s["scale"], s["max_nodes"])
    if s["op"] == "verify":
        return fused.verify_tree(s["logits"], s["tokens"], s["parents"], s["cu"], s["temperature"], s["u_accept"], s["u_sample"],
                                 s["max_nodes"], draft_probs=s["draft_probs"])
    fused.kv_commit_(s["layers"], s["k_cache"], s["v_cache"], s["table"], s["ctx"], s["path"], s["heads"], s["kv_heads"], DIM)
    return s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------ work and 64-bit values
def work(case):
    counts, ctx = _sizes(case)
    if case["op"] == "attn":
        hq, hk = case["heads"], case["kv_heads"]
        pairs = sum(n * (c + (n + 1) / 2) for n, c in zip(counts, ctx))
        nbytes = 2 * DIM * (2 * hk * sum(ctx) + (hq + 2 * hk + hq) * sum(counts))
        return {"bytes": nbytes, "flops": 4 * DIM * hq * pairs}
    if case["op"] == "verify":
        # every node's logits; a drafter's probabilities at the node where the path ends
        nbytes = 2 * case["vocab"] * sum(counts) + (4 * case["vocab"] * case["batch"] if case["drafted"] else 0)
        return {"bytes": nbytes, "flops": 4 * case["vocab"] * sum(counts)}
    rows = sum(_spread(case["batch"], 1, case["nodes"]))
    return {"bytes": 2 * rows * case["layers"] * 2 * case["kv_heads"] * DIM * 2, "flops": 0}


def _chain_of(parents, node):
    seen = []
    while node >= 0:
        seen.append(node)
        node = parents[node]
    return seen


def _attn_exact(s):
    hq, hk, cu, par = s["heads"], s["kv_heads"], s["cu"].tolist(), s["parents"].tolist()
    outs = []
    for b in range(len(cu) - 1):
        lo, hi, c = cu[b], cu[b + 1], int(s["ctx"][b])
        pos = torch.arange(c, device=s["qkv"].device)
        page = s["table"][b].long()[pos // PAGE]
        new = s["qkv"][lo:hi].double().view(hi - lo, hq + 2 * hk, DIM)
        sees = torch.zeros(hi - lo, hi - lo, dtype=torch.bool)
        for t in range(hi - lo):
            sees[t, _chain_of(par[lo:hi], t)] = True
        bias = torch.zeros(hi - lo, c + hi - lo, dtype=torch.float64)
        bias[:, c:][~sees] = -math.inf
        bias = bias.to(s["qkv"].device)
        heads = []
        for h in range(hk):
            k = torch.cat([s["k_cache"][page, h, pos % PAGE].double(), new[:, hq + h]])
            v = torch.cat([s["v_cache"][page, h, pos % PAGE].double(), new[:, hq + hk + h]])
            for i in range(h * (hq // hk), (h + 1) * (hq // hk)):
                heads.append(torch.softmax(new[:, i] @ k.t() * s["scale"] + bias, -1) @ v)
        outs.append(torch.stack(heads, 1).reshape(hi - lo, hq * DIM))
    return torch.cat(outs)


def _verify_exact(s):
    cu, par, tok = s["cu"].tolist(), s["parents"].tolist(), s["tokens"].tolist()
    ua, us, temp = s["u_accept"].tolist(), s["u_sample"].tolist(), s["temperature"].tolist()
    B, T = len(cu) - 1, s["max_nodes"]
    counts, tokens = torch.zeros(B, dtype=torch.int32), torch.full((B, T), -1, dtype=torch.int64)
    path, logprobs = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, T, dtype=torch.float64)

    def at(row, t):
        lp = torch.log_softmax(s["logits"][row].double() / (t if t > 0 else 1.0), -1)
        if t > 0:
            return lp, lp.exp()
        p = torch.zeros_like(lp)
        p[int((s["logits"][row] == s["logits"][row].max()).nonzero()[0])] = 1.0
        return lp, p

    for b in range(B):
        cur, k = cu[b], 0
        lp, r = at(cur, temp[b])
        path[b, 0] = cur
        kids = [j for j in range(cu[b] + 1, cu[b + 1]) if par[j] == 0]
        while kids:
            j = kids.pop(0)
            x = tok[j]
            q = 1.0 if s["draft_probs"] is None else float(s["draft_probs"][cur, x].double())
            if ua[j] * q < float(r[x]):
                tokens[b, k], logprobs[b, k] = x, float(lp[x])
                k += 1
                path[b, k] = cur = j
                lp, r = at(cur, temp[b])
                kids = [i for i in range(j + 1, cu[b + 1]) if par[i] == j - cu[b]]
            else:
                if s["draft_probs"] is None:
                    left = r.clone()
                    left[x] = 0.0
                else:
                    left = torch.relu(r - s["draft_probs"][cur].double())
                if float(left.sum()) > 0:
                    r = left / left.sum()
        edge = torch.cumsum(r, 0)
        over = (edge > us[b] * edge[-1]).nonzero()
        x = int(over[0]) if over.numel() else int(r.nonzero()[-1])
        tokens[b, k], logprobs[b, k], counts[b] = x, float(lp[x]), k + 1
    return counts, tokens, path, logprobs


def _commit_exact(s):
    path, ctx, table = s["path"].tolist(), s["ctx"].tolist(), s["table"].tolist()
    hq, hk = s["heads"], s["kv_heads"]
    for b, nodes in enumerate(path):
        for j, node in enumerate(nodes):
            if node < 0:
                continue
            page, off = table[b][(ctx[b] + j) // PAGE], (ctx[b] + j) % PAGE
            row = torch.stack([x[node] for x in s["layers"]]).view(len(s["layers"]), hq + 2 * hk, DIM)
            s["k_cache"][:, page, :, off] = row[:, hq:hq + hk]
            s["v_cache"][:, page, :, off] = row[:, hq + hk:]
    return s["k_cache"], s["v_cache"]


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _attn_exact, "verify": _verify_exact, "commit": _commit_exact}[s["op"]](s)
