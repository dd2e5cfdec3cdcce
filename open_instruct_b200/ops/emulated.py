"""The kernel wrappers of ``ops.fused`` restated in PyTorch, call for call.

``LlamaModel(ops="emulated")`` runs the SAME hand-driven forward / backward as ``ops="fused"`` (layer stash, activation
recomputation, chunked output head, in-place gradient rewrites) with these functions in place of the sm_100a kernels, on any
device and dtype.  That is how the driver's bookkeeping - which tensor is saved, which gradient is added where - is tested on a
CPU against autograd over the plain PyTorch path; the kernels themselves are tested one by one on the GPU against the same
PyTorch operations.  Nothing here is a training path: every function allocates and none is fast.

Each function keeps the contract of its namesake: argument order, in-place behaviour, what is returned and in which dtype
(statistics and log-probabilities fp32; activations in the dtype of the input).
"""

from __future__ import annotations

import torch

from . import ref

OUT_BF16, OUT_F32, OUT_F32_ACC, OUT_F32_RED = 0, 1, 2, 3


def gemm(a, b, out=None, *, a_mn: bool = False, b_mn: bool = False, out_mode: int = OUT_BF16, max_ctas: int = 0, impl=None):
    """``C[M, N] (op)= A_op[M, K] @ B_op[N, K]^T``; ``a_mn`` / ``b_mn`` say that the operand is stored transposed.  Mode 0
    stores in the operands' dtype (bf16 on the GPU), mode 1 stores fp32, modes 2 / 3 add into the fp32 ``out``."""
    A = (a.t() if a_mn else a).float()
    B = (b if b_mn else b.t()).float()
    c = A @ B
    if out_mode == OUT_BF16:
        c = c.to(a.dtype)
        if out is None:
            return c
        out.copy_(c)
        return out
    if out is None:
        if out_mode != OUT_F32:
            raise ValueError("accumulate mode needs an output tensor")
        return c
    if out.dtype != torch.float32:
        raise TypeError("fp32 output modes need an fp32 out")
    if out_mode == OUT_F32:
        out.copy_(c)
    else:
        out.add_(c)
    return out


def rmsnorm_fwd(x, w, eps: float, res=None):
    """(y, h, rstd): ``h = x (+ res)`` in the input dtype, ``rstd`` fp32 [T], ``y = w * (h * rstd)``."""
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.pow(2).mean(-1) + eps)
    y = w * (hf * rstd[:, None]).to(x.dtype)
    return y.to(x.dtype), h, rstd


def rmsnorm_bwd(h, w, rstd, dy, dres, dw_out):
    """``dx = dRMSNorm/dh (+ dres)``; the weight gradient is ADDED into ``dw_out`` (fp32 [D]) when given."""
    hf, dyf, wf = h.float(), dy.float(), w.float()
    xhat = hf * rstd[:, None]
    if dw_out is not None:
        dw_out.add_((dyf * xhat).sum(0))
    dxhat = dyf * wf
    dx = rstd[:, None] * (dxhat - xhat * (dxhat * xhat).mean(-1, keepdim=True))
    if dres is not None:
        dx = dx + dres.float()
    return dx.to(h.dtype)


def rope_table(pos, inv_freq, head_dim: int):
    ang = pos.float()[:, None] * inv_freq[None, :].to(pos.device)
    return torch.stack([ang.cos(), ang.sin()], dim=-1)  # [T, head_dim / 2, 2]


def rope_(qkv, pos, inv_freq, n_q: int, n_kv: int, head_dim: int, backward: bool = False, table=None):
    """In-place rotation of the q and k heads (half-split convention); ``backward`` rotates by the negative angle, which
    is the transpose of the rotation and so its gradient."""
    T = qkv.shape[0]
    tab = table if table is not None else rope_table(pos, inv_freq, head_dim)
    cos, sin = tab[..., 0][:, None, :], tab[..., 1][:, None, :]
    if backward:
        sin = -sin
    x = qkv.view(T, n_q + 2 * n_kv, head_dim)
    rot = x[:, : n_q + n_kv].float()
    half = head_dim // 2
    x1, x2 = rot[..., :half], rot[..., half:]
    x[:, : n_q + n_kv].copy_(torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(qkv.dtype))
    return qkv


def swiglu_fwd(gate_up):
    return ref.swiglu(gate_up.float()).to(gate_up.dtype)


def swiglu_bwd_(gate_up, dact):
    """Overwrites ``gate_up`` with d(gate | up)."""
    F = gate_up.shape[1] // 2
    g, u, d = gate_up[:, :F].float(), gate_up[:, F:].float(), dact.float()
    sig = torch.sigmoid(g)
    dg = d * u * sig * (1 + g * (1 - sig))
    du = d * g * sig
    gate_up.copy_(torch.cat([dg, du], dim=1).to(gate_up.dtype))
    return gate_up


def embedding_fwd(table, ids):
    return table[ids.reshape(-1)].clone()


def embedding_bwd(grad_table, ids, dout) -> None:
    grad_table.index_add_(0, ids.reshape(-1), dout.to(grad_table.dtype))


def logprob_fwd(logits, labels, temperature: float = 1.0, want_entropy: bool = False):
    """(logp, lse, entropy | None), fp32; ``lse`` is the log-sum-exp of ``logits / temperature``."""
    lp, ent = ref.token_logprobs(logits, labels, temperature, with_entropy=want_entropy)
    return lp, torch.logsumexp(logits.float() / temperature, dim=-1), ent


def logprob_bwd_(logits, labels, lse, g, temperature: float = 1.0):
    """Rewrites ``logits`` in place with dL/dlogits given ``g = dL/dlogp``; rows with a negative label give zeros."""
    return logprob_bwd_vp_(logits, labels, lse, g, 0, temperature)


def logprob_fwd_vp(logits, labels, label_offset: int, temperature: float = 1.0):
    """Partials of this rank's logit columns ``[label_offset, label_offset + V_local)``: (the label's logit / temperature if
    the label is one of mine else 0, log-sum-exp over my columns, mean of my scaled logits under MY columns' softmax); zeros
    for rows without a label."""
    z = logits.float() / temperature
    V = z.shape[1]
    loc = labels - label_offset
    mine = (labels >= 0) & (loc >= 0) & (loc < V)
    zl = torch.where(mine, z.gather(1, loc.clamp(0, V - 1)[:, None]).squeeze(1), torch.zeros_like(z[:, 0]))
    valid = labels >= 0
    lse = torch.where(valid, torch.logsumexp(z, dim=-1), torch.zeros_like(zl))
    ez = torch.where(valid, (torch.softmax(z, dim=-1) * z).sum(-1), torch.zeros_like(zl))
    return zl, lse, ez


def logprob_bwd_vp_(logits, labels, lse_global, g, label_offset: int, temperature: float = 1.0):
    z = logits.float() / temperature
    V = z.shape[1]
    p = torch.exp(z - lse_global[:, None])
    loc = labels - label_offset
    mine = (labels >= 0) & (loc >= 0) & (loc < V)
    onehot = torch.zeros_like(p)
    onehot[mine, loc[mine]] = 1.0
    d = (onehot - p) * (g.float() / temperature)[:, None]
    d = torch.where((labels >= 0)[:, None], d, torch.zeros_like(d))
    logits.copy_(d.to(logits.dtype))
    return logits


def attn_max_tiles(total_tokens: int, num_docs: int) -> int:
    return (total_tokens + 127) // 128 + num_docs


def attn_fwd(qkv, cu_seqlens, n_q: int, n_kv: int, head_dim: int, scale: float):
    """(out [T, n_q * head_dim], lse [n_q, T] fp32).  The emulated backward recomputes the scores, so ``lse`` only has the
    kernel's shape."""
    out = ref.attention_varlen(qkv.float(), cu_seqlens, n_q, n_kv, head_dim, scale).to(qkv.dtype)
    return out, torch.zeros(n_q, qkv.shape[0], dtype=torch.float32, device=qkv.device)


def attn_bwd(qkv, out, d_out, lse, cu_seqlens, n_q: int, n_kv: int, head_dim: int, scale: float):
    """Gradient with respect to the post-RoPE fused qkv, by autograd over the explicit-softmax attention."""
    with torch.enable_grad():
        x = qkv.detach().float().requires_grad_(True)
        y = ref.attention_varlen(x, cu_seqlens, n_q, n_kv, head_dim, scale)
        (dx,) = torch.autograd.grad(y, x, d_out.float())
    return dx.to(qkv.dtype)


def attn_fwd_window(qkv, cu_seqlens, n_q: int, n_kv: int, head_dim: int, scale: float, window: int, max_len: int):
    return ref.attention_varlen(qkv.float(), cu_seqlens, n_q, n_kv, head_dim, scale, window=window).to(qkv.dtype)


def attn_bwd_window(qkv, d_out, cu_seqlens, n_q: int, n_kv: int, head_dim: int, scale: float, window: int, max_len: int):
    with torch.enable_grad():
        x = qkv.detach().float().requires_grad_(True)
        y = ref.attention_varlen(x, cu_seqlens, n_q, n_kv, head_dim, scale, window=window)
        (dx,) = torch.autograd.grad(y, x, d_out.float())
    return dx.to(qkv.dtype)


# ---------------------------------------------------------------------------------- speculative decoding
def _ancestors(parents: list, t: int) -> list:
    """The node at position ``t`` and its ancestors; nothing for padding."""
    if parents[t] < -1:
        return []
    seen = [t]
    while 0 <= parents[t] < t and parents[parents[t]] >= -1:   # padding has no descendants: its children are roots
        t = parents[t]
        seen.append(t)
    return sorted(seen)


def _spans(cu_nodes, total: int, max_nodes: int) -> list:
    """(first row, nodes) of every sequence, held inside the batch."""
    cu = cu_nodes.tolist()
    first = [min(max(c, 0), total) for c in cu[:-1]]
    return [(lo, min(max(hi - lo, 0), max_nodes, total - lo)) for lo, hi in zip(first, cu[1:])]


def tree_attn(qkv, k_cache, v_cache, block_table, ctx, cu_nodes, parents, n_q: int, n_kv: int, head_dim: int, scale: float, max_nodes: int, out=None):
    """Attention of drafted token trees over the paged cache, sequence by sequence."""
    from . import fused

    fused._check_tree_attn(qkv, k_cache, v_cache, block_table, ctx, cu_nodes, parents, n_q, n_kv, head_dim, scale, max_nodes, out, qkv.dtype)
    N, group, page = qkv.shape[0], n_q // n_kv, fused.KV_PAGE
    if out is None:
        out = torch.empty(N, n_q * head_dim, dtype=qkv.dtype, device=qkv.device)
    par = parents.tolist()
    for b, (lo, n) in enumerate(_spans(cu_nodes, N, max_nodes)):
        if n == 0:
            continue
        x = qkv[lo:lo + n].float().view(n, n_q + 2 * n_kv, head_dim)
        c = min(max(int(ctx[b]), 0), block_table.shape[1] * page)
        at = torch.arange(c, device=qkv.device)
        blk = block_table[b].long()[at // page]
        there = ((blk >= 0) & (blk < k_cache.shape[0])).view(-1, 1, 1)
        blk = torch.where(there.view(-1), blk, 0)
        old_k = k_cache[blk, :, at % page].float().masked_fill(~there, 0.0) if c else x[:0, :n_kv]
        old_v = v_cache[blk, :, at % page].float().masked_fill(~there, 0.0) if c else x[:0, :n_kv]
        pad = torch.tensor([p < -1 for p in par[lo:lo + n]], device=qkv.device)
        k = torch.cat([old_k, x[:, n_q:n_q + n_kv]]).repeat_interleave(group, 1)
        v = torch.cat([old_v, x[:, n_q + n_kv:].masked_fill(pad[:, None, None], 0.0)]).repeat_interleave(group, 1)  # 0 * NaN
        live = torch.ones(n, c + n, dtype=torch.bool)
        live[:, c:] = False
        for t in range(n):
            live[t, [c + a for a in _ancestors(par[lo:lo + n], t)]] = True
        s = torch.einsum("nhd,jhd->hnj", x[:, :n_q], k) * scale
        s = s.masked_fill(~live.to(s.device), float("-inf"))
        o = torch.einsum("hnj,jhd->nhd", torch.softmax(s, -1), v).reshape(n, -1)
        out[lo:lo + n] = o.masked_fill(pad[:, None], 0.0).to(qkv.dtype)
    return out


def verify_tree(logits, tokens, parents, cu_nodes, temperature, u_accept, u_sample, max_nodes: int, draft_probs=None):
    """Verification of drafted trees, node by node in 64 bits; returns (count, tokens, path, logprobs)."""
    from . import fused

    fused._check_verify_tree(logits, tokens, parents, cu_nodes, temperature, u_accept, u_sample, max_nodes, draft_probs, logits.dtype)
    (N, V), B, dev = logits.shape, temperature.shape[0], logits.device
    count = torch.zeros(B, dtype=torch.int32)
    emitted = torch.full((B, max_nodes), -1, dtype=torch.int64)
    path = torch.full((B, max_nodes), -1, dtype=torch.int32)
    logprobs = torch.zeros(B, max_nodes, dtype=torch.float32)
    par, tok, coin = parents.tolist(), tokens.tolist(), u_accept.double().tolist()
    for b, (lo, n) in enumerate(_spans(cu_nodes, N, max_nodes)):
        if n == 0:
            continue
        t = float(temperature[b])

        def arrive(node):
            lp = torch.log_softmax(logits[node].double() / (t if t > 0 else 1.0), -1)
            if t > 0:
                return lp, lp.exp()
            p = torch.zeros_like(lp)
            p[int(torch.argmax((logits[node] == logits[node].max()).int()))] = 1.0
            return lp, p

        cur, k = lo, 0
        lp, r = arrive(cur)
        path[b, 0] = cur
        for j in range(1, n):
            if par[lo + j] != cur - lo:
                continue
            x = tok[lo + j]
            known = 0 <= x < V
            q = draft_probs[cur].double() if draft_probs is not None else None
            qx = 1.0 if q is None else float(q[x]) if known else 0.0
            if known and coin[lo + j] * qx < float(r[x]):
                emitted[b, k], logprobs[b, k] = x, float(lp[x])
                k, cur = k + 1, lo + j
                path[b, k] = cur
                lp, r = arrive(cur)
                continue
            left = r.clone()
            if q is not None:
                left = (r - q).clamp(min=0.0)
            elif known:
                left[x] = 0.0
            if float(left.sum()) > 0:
                r = left / left.sum()
        c = r.cumsum(0)
        over = torch.nonzero(c > float(u_sample[b].double()) * c[-1])
        live = torch.nonzero(r > 0)
        x = int(over[0]) if len(over) else int(live[-1]) if len(live) else 0
        emitted[b, k], logprobs[b, k], count[b] = x, float(lp[x]), k + 1
    return count.to(dev), emitted.to(dev), path.to(dev), logprobs.to(dev)


def kv_commit_(qkv_layers, k_cache, v_cache, block_table, ctx, path, n_q: int, n_kv: int, head_dim: int) -> None:
    """Keys and values of the accepted nodes into the paged cache of every layer."""
    from . import fused

    fused._check_kv_commit(qkv_layers, k_cache, v_cache, block_table, ctx, path, n_q, n_kv, head_dim, k_cache.dtype)
    page, (N, L) = fused.KV_PAGE, (qkv_layers[0].shape[0], len(qkv_layers))
    for b, nodes in enumerate(path.tolist()):
        for j, node in enumerate(nodes):
            at = int(ctx[b]) + j
            if not 0 <= node < N or at < 0 or at // page >= block_table.shape[1]:
                continue
            blk = int(block_table[b, at // page])
            if not 0 <= blk < k_cache.shape[1]:
                continue
            for i in range(L):
                x = qkv_layers[i][node].view(n_q + 2 * n_kv, head_dim)
                k_cache[i, blk, :, at % page] = x[n_q:n_q + n_kv]
                v_cache[i, blk, :, at % page] = x[n_q + n_kv:]
