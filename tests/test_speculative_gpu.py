"""Speculative-decoding kernels on a B200 against 64-bit oracles."""

import pytest
import torch

from _speculative import DIM, PAGE, attn_bound, attn_oracle, logprob_bound, make_attn, make_borders, make_cold, make_covered, make_verify, verify_oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    from open_instruct_b200.ops import lib

    yield
    lib.check_status()


def _check_attn(a, out=None):
    from open_instruct_b200.ops import fused

    got = fused.tree_attn(**a, out=out)
    ref, mag = attn_oracle(a)
    n = int(a["cu_nodes"][-1])
    off = (got[:n].double() - ref[:n]).abs()
    assert torch.isfinite(got[:n].float()).all()
    assert (off <= attn_bound(ref[:n], mag[:n])).all(), float((off / attn_bound(ref[:n], mag[:n])).max())
    return got


HEADS = [(8, 2), (7, 1), (3, 3), (10, 2), (12, 1), (2, 1), (32, 8), (128, 1), (65, 1), (43, 1)]


@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_tree_attention_short(heads, kv_heads):
    _check_attn(make_attn(heads, kv_heads, [0, 1, 63, 64, 65, 127, 128, 129, 200], [1, 3, 0, 5, 9, 2, 4, 1, 17], device="cuda", table_extra=2))


@pytest.mark.parametrize("shape", ["chain", "tree", "star"])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (7, 1), (8, 1), (1, 1)])
def test_tree_attention_full_trees(heads, kv_heads, shape):
    """64 nodes: several row tiles for every KV head."""
    _check_attn(make_attn(heads, kv_heads, [0, 257, 64, 1000], [64, 63, 0, 64], shape, device="cuda", row_extra=8))


@pytest.mark.parametrize("nodes", [1, 2, 5])
@pytest.mark.parametrize("ctx", [1, 64, 383, 4097, 20011])
def test_tree_attention_one_sequence(ctx, nodes):
    """One sequence: its keys are shared out over the whole GPU and joined again."""
    _check_attn(make_attn(4, 1, [ctx], [nodes], device="cuda"))


@pytest.mark.parametrize("seed", range(4))
def test_tree_attention_ragged(seed):
    g = torch.Generator().manual_seed(seed)
    B = int(torch.randint(2, 40, (1,), generator=g))
    ctx = [int(600 * float(r) ** 2) for r in torch.rand(B, generator=g)]
    counts = torch.randint(0, 12, (B,), generator=g).tolist()
    heads, kv_heads = [(8, 2), (14, 2), (5, 1), (3, 3)][seed]
    _check_attn(make_attn(heads, kv_heads, ctx, counts, device="cuda", seed=seed, extra_rows=seed))


@pytest.mark.parametrize("heads,kv_heads", [(7, 1), (8, 2), (16, 1), (64, 1), (3, 3)])
@pytest.mark.parametrize("seed", range(3))
def test_tree_attention_uneven_trees(heads, kv_heads, seed):
    """Trees of one to many row tiles next to each other: shares of the work that end inside a unit of two row tiles."""
    g = torch.Generator().manual_seed(100 + seed)
    counts = torch.randint(0, 65, (9,), generator=g).tolist()
    ctx = [int(1500 * float(r) ** 2) for r in torch.rand(9, generator=g)]
    _check_attn(make_attn(heads, kv_heads, ctx, counts, device="cuda", seed=seed, extra_rows=seed))


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 1)])
def test_tree_attention_many_sequences(heads, kv_heads):
    """More sequences than a CTA has threads, the first 500 of them empty."""
    counts = [0] * 500 + [i % 6 for i in range(500)]
    _check_attn(make_attn(heads, kv_heads, [(37 * i) % 150 for i in range(1000)], counts, device="cuda"))


@pytest.mark.parametrize("most", [1, 40])
def test_tree_attention_scores_below_the_range(most):
    """A whole tile of keys whose scores are -inf in fp32 (narrow and wide kernel): no weight, and nothing else is disturbed."""
    a = make_attn(1, 1, [200, 5], [1, most], device="cuda")
    far = -3.0e38 * torch.sign(a["qkv"][0, :DIM].float())
    a["k_cache"][a["block_table"][0, :2].long(), 0] = far.bfloat16()
    _check_attn(a)


def test_tree_attention_between_decode_gemms():
    """As in the engine's layers: the decode GEMMs around it allocate tensor memory for CTA pairs and are launched early."""
    from open_instruct_b200.ops import fused

    a = make_attn(32, 8, [300], [5], device="cuda", garbage=False)
    g = torch.Generator(device="cuda").manual_seed(3)
    w = [(torch.randn(n, k, device="cuda", generator=g) / k ** 0.5).bfloat16() for n, k in ((4096, 4096), (28672, 4096), (4096, 14336), (6144, 4096))]
    norm = torch.ones(4096, device="cuda", dtype=torch.bfloat16)
    x = a.pop("qkv")

    def layer(x, sync):
        o = fused.tree_attn(x, **a)
        if sync:
            torch.cuda.synchronize()
        y = fused.rmsnorm_fwd(fused.gemm_decode(o, w[0]), norm, 1e-6)[0]
        y = fused.gemm_decode(fused.swiglu_fwd(fused.gemm_decode(y, w[1])), w[2])
        y = fused.gemm_decode(fused.rmsnorm_fwd(y, norm, 1e-6)[0], w[3])
        if sync:
            torch.cuda.synchronize()
        return y

    want = x
    for _ in range(8):
        want = layer(want, True)
    for _ in range(60):
        got = x
        for _ in range(8):
            got = layer(got, False)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_tree_attention_shared_pages():
    """Two sequences on the same pages and one table row for both."""
    a = make_attn(8, 2, [150, 150], [5, 9], device="cuda", garbage=False)
    a["block_table"] = a["block_table"][:1].expand(2, -1)
    _check_attn(a)


def test_tree_attention_peaked_and_large_scores():
    """Scores of a few tens and more: the running maximum moves far.  A query has a standard deviation of 18, the 128 products of
    a score add up to less than 2^12 in magnitude, so fp32 sums leave it off by at most 128 * 2^-24 * 2^12 = 2^-5, times the scale
    of 2^-3.5 that is 2^-8.5 in the exponent: numerator and denominator together get less than 2^-7 of sum p |v| on top."""
    a = make_attn(4, 1, [700, 129], [6, 9], device="cuda")
    a["qkv"][:, : 4 * DIM] *= 12.0
    from open_instruct_b200.ops import fused

    got = fused.tree_attn(**a)
    ref, mag = attn_oracle(a)
    assert ((got.double() - ref).abs() <= attn_bound(ref, mag) + 2.0 ** -7 * mag).all()


def test_tree_attention_padding_bad_pages_and_untouched_rows():
    a = make_attn(4, 2, [70, 130, 65], [6, 5, 3], device="cuda", extra_rows=3)
    a["parents"][[4, 5, 10]] = -2
    a["parents"][9] = 0
    a["block_table"][0, 1] = -3
    a["block_table"][1, 0] = a["k_cache"].shape[0]
    a["block_table"][2, 0] = 1 << 30
    out = torch.full((17, 4 * DIM), 7.0, device="cuda", dtype=torch.bfloat16)
    got = _check_attn(a, out)
    assert got is out and (out[[4, 5, 10]] == 0).all() and (out[14:] == 7.0).all()


def test_tree_attention_contexts_past_the_table_are_cut():
    a = make_attn(4, 2, [128, 64], [3, 2], device="cuda")
    want = attn_oracle(a)
    a["ctx"][0] = 100000
    a["block_table"][1, 1] = a["block_table"][1, 0]
    from open_instruct_b200.ops import fused

    got = fused.tree_attn(**a)
    assert ((got.double() - want[0]).abs() <= attn_bound(*want)).all()


def test_tree_attention_of_nothing():
    from open_instruct_b200.ops import fused

    a = make_attn(4, 2, [5, 9], [0, 0], device="cuda")
    assert fused.tree_attn(**a).shape == (0, 4 * DIM)
    a = make_attn(4, 2, [], [], device="cuda")
    assert fused.tree_attn(**a).shape == (0, 4 * DIM)


def test_tree_attention_far_pages():
    """Pages behind 2^32 bytes and 2^32 elements of the cache."""
    a = make_attn(4, 2, [200, 77], [5, 3], device="cuda", garbage=False)
    big = 280000   # blocks of 2 * 64 * 128 elements: 4.6e9 elements, 9.2 GB
    old = a["block_table"].clone()
    new = torch.where(old >= 0, big - 1 - 7 * old.clamp(min=0), old)
    for name in ("k_cache", "v_cache"):
        cache = torch.empty(big, 2, PAGE, DIM, device="cuda", dtype=torch.bfloat16)
        cache[new[old >= 0].long()] = a[name][old[old >= 0].long()]
        a[name] = cache
    a["block_table"] = new
    _check_attn(a)


def test_tree_attention_other_stream_and_graph():
    from open_instruct_b200.ops import fused

    a = make_attn(8, 2, [300, 1000, 64], [5, 9, 1], device="cuda")
    b = make_attn(8, 2, [10, 500, 900], [9, 1, 5], device="cuda", seed=9)
    for x in (a, b):
        x["max_nodes"] = 9
    width = max(a["block_table"].shape[1], b["block_table"].shape[1])
    blocks = max(a["k_cache"].shape[0], b["k_cache"].shape[0])

    def grown(x):
        t = torch.zeros(3, width, dtype=torch.int32, device="cuda")
        t[:, : x["block_table"].shape[1]] = x["block_table"]
        x["block_table"] = t
        for n in ("k_cache", "v_cache"):
            c = torch.zeros(blocks, 2, PAGE, DIM, device="cuda", dtype=torch.bfloat16)
            c[: x[n].shape[0]] = x[n]
            x[n] = c
        x["qkv"] = x["qkv"].contiguous()
        return x

    a, b = grown(a), grown(b)
    want_a, want_b = attn_oracle(a), attn_oracle(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # two calls at once, on two streams
        ys = [fused.tree_attn(**b) for _ in range(5)]
    xs = [fused.tree_attn(**a) for _ in range(5)]
    torch.cuda.synchronize()
    for x in xs:
        assert ((x.double() - want_a[0]).abs() <= attn_bound(*want_a)).all() and torch.equal(x, xs[0])
    for y in ys:
        assert ((y.double() - want_b[0]).abs() <= attn_bound(*want_b)).all() and torch.equal(y, ys[0])
    live = {k: v.clone() if torch.is_tensor(v) else v for k, v in a.items()}
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one = fused.tree_attn(**live)
    with torch.cuda.graph(second, pool=graph.pool()):
        two = fused.tree_attn(**live)
    graph.replay()
    second.replay()
    torch.cuda.synchronize()
    assert torch.equal(one, xs[0]) and torch.equal(two, xs[0])
    for k, v in b.items():   # other contents in the same buffers
        if torch.is_tensor(v):
            live[k].copy_(v)
    second.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(one, ys[0]) and torch.equal(two, ys[0])


def _check_verify(a):
    from open_instruct_b200.ops import fused

    got, want = fused.verify_tree(**a), verify_oracle(a)
    for name, x, y in zip(("count", "tokens", "path"), got, want):
        assert torch.equal(x.cpu(), y.to(x.dtype)), name
    assert (got[3].cpu().double() - want[3]).abs().max() <= logprob_bound(a["logits"].shape[1])
    return got


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("shape", ["chain", "tree", "star"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 97, 1000, 16384, 16391, 50257])
def test_verification(vocab, shape, drafted):
    counts = [3, 1, 0, 7, 5, 12, 2, 4]
    _check_verify(make_verify(counts, vocab, shape, drafted, temps=(1.0, 0.0, 0.6, 1.7, 1.0), seed=vocab, device="cuda", row_extra=3, extra_rows=2))


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("likely", [-3.0, 0.0, 3.0])
def test_verification_large_vocabulary(likely, drafted):
    """Rows of 16-byte aligned logits, few and many accepted drafts."""
    _check_verify(make_verify([6, 2, 9, 64, 5, 1], 128256, "tree", drafted, temps=(1.0, 0.8), seed=4, device="cuda", likely=likely))


def test_verification_many_sequences():
    _check_verify(make_verify([1 + i % 5 for i in range(300)], 512, "tree", False, temps=(1.0, 0.0, 0.7), seed=6, device="cuda"))


def test_verification_of_nothing():
    from open_instruct_b200.ops import fused

    for counts in ([], [0, 0, 0]):
        for drafted in (False, True):
            a = make_verify(counts, 50, "chain", drafted, device="cuda")
            count, tokens, path, logprobs = fused.verify_tree(**a)
            assert count.tolist() == counts and (tokens == -1).all() and (path == -1).all() and (logprobs == 0).all()


def test_verification_broadcast_rows():
    """One row of logits and one drafter's row for all nodes (stride 0)."""
    a = make_verify([4, 1, 6], 1003, "tree", True, temps=(1.0, 0.7), seed=3, device="cuda")
    a["logits"], a["draft_probs"] = a["logits"][:1].expand(11, -1), a["draft_probs"][2:3].expand(11, -1)
    _check_verify(a)


@pytest.mark.parametrize("drafted", [False, True])
def test_verification_edges(drafted):
    """Masked vocabularies, ties at temperature 0, the same token twice among siblings, tokens outside the vocabulary, coins of 0
    and just below 1, drafts of probability 0 and 1."""
    a = make_verify([5, 5, 5, 5, 5, 5], 300, "star", drafted, temps=(1.0, 0.0, 1.0, 1.0, 0.0, 1.0), seed=2, device="cuda")
    a["logits"][0:5, 7:] = float("-inf")                 # few tokens are left
    a["logits"][5:10] = 1.25                              # all tie: token 0
    a["tokens"][6] = 0
    a["logits"][10:15, 1:] = float("-inf")               # one token is left
    a["tokens"][11:15] = 5
    a["tokens"][16:20] = torch.tensor([9, 9, 9, 200], device="cuda")
    a["tokens"][[2, 22, 27]] = torch.tensor([-1, 300, 1 << 40], device="cuda")
    a["u_accept"][[16, 17, 18]] = 1.0 - 2.0 ** -24
    a["u_accept"][26] = 0.0
    a["u_sample"][:] = torch.tensor([0.0, 0.5, 1.0 - 2.0 ** -24, 0.0, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -24], device="cuda")
    if drafted:
        a["draft_probs"][25] = 0.0
        a["draft_probs"][0, :] = 0.0
        a["draft_probs"][0, 3] = 1.0
    want = verify_oracle(a)
    from open_instruct_b200.ops import fused

    got = fused.verify_tree(**a)
    for x, y in zip(got[:3], want[:3]):
        assert torch.equal(x.cpu(), y.to(x.dtype))
    assert (got[3].cpu().double() - want[3]).abs().max() <= logprob_bound(300)


@pytest.mark.parametrize("vocab", [300, 20011])
def test_verification_where_a_rejection_leaves_nothing(vocab):
    """A drafter's row that is nowhere below the target's: the residual is empty and stays what it was, before the next sibling and
    before the last draw."""
    a = make_verify([2, 4, 4, 3], vocab, "star", True, temps=(1.0, 0.9), seed=12, device="cuda")
    a["draft_probs"][:] = 1.0
    a["u_accept"][:] = 1.0 - 2.0 ** -24
    a["u_accept"][3] = 0.0
    a["draft_probs"][6] = 0.5 * torch.softmax(a["logits"][6].float(), -1)   # something is left here
    _check_verify(a)


def test_verification_rows_without_a_finite_logit_stay_in_range():
    from open_instruct_b200.ops import fused

    a = make_verify([3, 3, 3], 500, "chain", False, device="cuda")
    a["logits"][0] = float("-inf")
    a["logits"][3] = float("nan")
    a["logits"][6] = float("inf")
    count, tokens, path, _ = fused.verify_tree(**a)
    assert ((tokens >= -1) & (tokens < 500)).all() and ((path >= -1) & (path < 9)).all() and ((count >= 1) & (count <= 3)).all()


def test_verification_stream_and_graph():
    from open_instruct_b200.ops import fused

    a, b = (make_verify([6, 2, 5, 1], 32003, "tree", True, temps=(1.0, 0.0), seed=s, device="cuda", row_extra=5) for s in (1, 2))
    wa, wb = fused.verify_tree(**a), fused.verify_tree(**b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [fused.verify_tree(**b) for _ in range(4)]
    xs = [fused.verify_tree(**a) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for x in xs for p, q in zip(x, wa)) and all(torch.equal(p, q) for y in ys for p, q in zip(y, wb))
    live = {k: v.clone() if torch.is_tensor(v) else v for k, v in a.items()}
    live["logits"] = a["logits"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused.verify_tree(**live)
    for src, want in ((a, wa), (b, wb), (a, wa)):
        for k, v in src.items():
            if torch.is_tensor(v):
                live[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out[:3], want[:3]))
        # the clone's rows start at other 16-byte offsets, so a row's sum is grouped differently: each result is within
        # logprob_bound of the exact value, the two within twice that of each other
        assert (out[3] - want[3]).abs().max() <= 2 * logprob_bound(32003)


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("layers,heads,kv_heads", [(1, 4, 2), (3, 7, 1), (130, 2, 2)])
def test_commit(layers, heads, kv_heads, bad):
    from open_instruct_b200.ops import fused
    from test_speculative_cpu import _commit_inputs, _commit_oracle

    a = _commit_inputs(layers, kv_heads, heads, torch.bfloat16, "cuda")
    if bad:
        a["block_table"][1, 0], a["block_table"][0, 0], a["path"][3, 1], a["ctx"][4] = -1, a["k_cache"].shape[1], 19, 64 * a["block_table"].shape[1]
        a["path"][4, 0] = 17
    want = _commit_oracle(a)
    fused.kv_commit_(**a)
    assert torch.equal(a["k_cache"], want[0]) and torch.equal(a["v_cache"], want[1])


def test_commit_far_pages():
    from open_instruct_b200.ops import fused
    from test_speculative_cpu import _commit_inputs

    a = _commit_inputs(2, 8, 8, torch.bfloat16, "cuda")
    blocks = 33000   # 2 layers of 33000 * 8 * 64 * 128 elements: 4.3e9 elements
    a["k_cache"], a["v_cache"] = (torch.zeros(2, blocks, 8, PAGE, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    a["block_table"] += blocks - 100
    fused.kv_commit_(**a)
    for b, nodes in enumerate(a["path"].tolist()):
        for j, node in enumerate(nodes):
            if node < 0:
                continue
            pos = int(a["ctx"][b]) + j
            blk = int(a["block_table"][b, pos // PAGE])
            for i, x in enumerate(a["qkv_layers"]):
                row = x[node].view(24, DIM)
                assert torch.equal(a["k_cache"][i, blk, :, pos % PAGE], row[8:16]) and torch.equal(a["v_cache"][i, blk, :, pos % PAGE], row[16:])


def test_one_speculative_step():
    """The three operators as a decode step uses them: attention of a tree, verification, commit of the path - and the next step's
    single-node attention over the grown cache equals attention over the text that was kept."""
    from open_instruct_b200.ops import fused

    heads, kv_heads = 8, 2
    ctx, counts = [130, 5, 63], [6, 4, 5]
    a = make_attn(heads, kv_heads, [c + n for c, n in zip(ctx, counts)], counts, device="cuda", garbage=False)   # pages with room for the path
    a["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    _check_attn(a)
    v = make_verify(counts, 1000, "tree", False, seed=3, device="cuda", likely=2.0)
    v["parents"] = a["parents"]
    count, _, path, _ = _check_verify(v)
    assert int(count.max()) > 1
    k, w = a["k_cache"][None].clone(), a["v_cache"][None].clone()
    fused.kv_commit_([a["qkv"]], k, w, a["block_table"], a["ctx"], path, heads, kv_heads, DIM)
    step = make_attn(heads, kv_heads, [1, 1, 1], [1, 1, 1], device="cuda", seed=8)
    step.update(k_cache=k[0], v_cache=w[0], block_table=a["block_table"], ctx=a["ctx"] + count)
    _check_attn(step)
    for b in range(3):   # what the cache holds now is the path's own rows
        for j in range(int(count[b])):
            pos = ctx[b] + j
            row = a["qkv"][int(path[b, j])].view(heads + 2 * kv_heads, DIM)
            assert torch.equal(k[0, int(a["block_table"][b, pos // PAGE]), :, pos % PAGE], row[heads:heads + kv_heads])


@pytest.mark.parametrize("temperature", [0.0, 0.05, 0.8])
def test_engine_with_drafts(temperature):
    """The fused engine with drafted tokens: every emitted token's log-probability is the model's own (fp32 PyTorch statement on the
    same weights; the two-layer model's bf16 activations leave its logits off by less than 0.08, the bound of the engine tests
    without drafts), greedy tokens are within that of the largest logit, and drafts are accepted."""
    from open_instruct_b200.data_types import SamplingConfig
    from open_instruct_b200.models import LlamaModel, get_spec
    from open_instruct_b200.rollout.engine import RolloutEngine

    spec = get_spec("tiny128")
    eng = RolloutEngine(spec, device="cuda", ops="fused", num_blocks=128, max_model_len=1024, seed=3, eos_token_ids=[], speculative_tokens=7)
    g = torch.Generator().manual_seed(1)
    base = torch.randint(4, spec.vocab_size, (50,), generator=g).tolist()
    prompts = [base * 4, base + base[:30], torch.randint(4, spec.vocab_size, (9,), generator=g).tolist(), base[:20] * 12]
    res = eng.generate(prompts, SamplingConfig(temperature=temperature, max_tokens=60, min_tokens=60, n=2, seed=5))
    # at 0.8 a random model's text hardly repeats three tokens, so there is nothing to look up and nothing is drafted
    assert eng.stats.get("accepted_tokens", 0) > 0 or temperature == 0.8
    assert eng.host.free_blocks() == 128
    oracle = LlamaModel(spec, device="cuda", dtype=torch.float32, ops="ref", flat=eng.model.flat.detach().float().clone())
    t = temperature or 1.0
    for prompt, r in zip(prompts, res):
        for text, lps in zip(r.responses, r.logprobs):
            assert len(text) == 60
            ids = torch.tensor(prompt + text, device="cuda")
            with torch.no_grad():
                logits = oracle.logits(ids, torch.arange(len(ids), device="cuda"), torch.tensor([0, len(ids)], dtype=torch.int32, device="cuda")).float() / t
            rows = torch.log_softmax(logits, -1)[len(prompt) - 1:-1]
            want = rows.gather(1, ids[len(prompt):, None]).squeeze(1)
            # a log-probability is a difference of two numbers that are logits / t: what the logits are off by counts 1 / t times
            assert (want.cpu() - torch.tensor(lps)).abs().max() < 0.08 / min(t, 1.0)
            if not temperature:
                assert (rows.amax(-1) - want).max() < 0.08


@pytest.mark.parametrize("vocab", [64, 20011])
def test_drafts_that_cover_all_that_a_row_allows(vocab):
    """Certain drafts: a last sibling that is all that is left is accepted, whatever its coin, and what is left beside rejected heavy
    tokens is shared out by its own weights, not by what a subtraction from 1 leaves of them."""
    a, first, counts = make_covered(vocab, "cuda")
    got = _check_verify(a)
    assert got[1][:, 0].tolist() == first and got[0].tolist() == counts


@pytest.mark.parametrize("vocab", [64, 9001])
def test_coins_of_one_leave_the_last_rejected_draft(vocab):
    """Coins outside of [0, 1) reject what is certain.  Then nothing is left, the last rejected token stays and is drawn."""
    from open_instruct_b200.ops import fused

    a, first, _ = make_covered(vocab, "cuda")
    a["u_accept"].fill_(1.0)
    want = verify_oracle(a)
    got = fused.verify_tree(**a)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1]) and torch.isfinite(got[3]).all()


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("vocab", [2000, 40013])
def test_verification_at_low_temperatures(vocab, drafted):
    _check_verify(make_cold(vocab, drafted, "cuda"))


@pytest.mark.parametrize("heads,kv_heads,ctx,counts", [
    (4, 2, [20, 0, 63], [6, 5, 3]),        # narrow kernel, every unit in one piece
    (4, 2, [70, 64, 129], [6, 5, 3]),      # the tree beside a page and alone
    (4, 2, [9000, 0, 30], [6, 5, 3]),      # narrow kernel, joined from parts
    (16, 1, [20, 0, 100], [6, 5, 3]),      # wide kernel, one row tile
    (8, 1, [9000, 64, 20], [40, 5, 64]),   # wide kernel, several row tiles
])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf")])
def test_tree_attention_padding_nodes_may_hold_anything(heads, kv_heads, ctx, counts, garbage):
    """A padding node's row of qkv is never used: its result is zero and no other node's result is touched."""
    from open_instruct_b200.ops import fused

    a = make_attn(heads, kv_heads, ctx, counts, device="cuda")
    first = counts[0]
    pads = [4, 5, first + 1, first + 4, first + counts[1] + 1]
    at = torch.tensor(pads, device="cuda")
    par = a["parents"]
    lost = torch.isin(par, torch.tensor([1, 4, 5], device="cuda", dtype=par.dtype))   # children of padding hang on node 0 instead
    par[lost] = 0
    par[at] = -2
    ref, mag = attn_oracle(a)
    a["qkv"][at] = garbage
    got = fused.tree_attn(**a)
    assert (got[at] == 0).all() and ((got.double() - ref).abs() <= attn_bound(ref, mag)).all()


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (16, 1)])
def test_tree_attention_children_of_padding_are_roots(heads, kv_heads):
    """In both kernels; the second sequence is padding alone."""
    from open_instruct_b200.ops import fused

    a = make_attn(heads, kv_heads, [70, 300, 5], [6, 3, 9], "chain", device="cuda")
    a["parents"][[2, 6, 7, 8]] = -2
    roots = {**a, "parents": a["parents"].clone()}
    roots["parents"][3] = -1
    got = fused.tree_attn(**a)
    ref, mag = attn_oracle(roots)
    assert ((got.double() - ref).abs() <= attn_bound(ref, mag)).all() and (got[6:9] == 0).all()


@pytest.mark.parametrize("nodes", [1, 5, 40])
@pytest.mark.parametrize("ctx", [383, 4097, 20011])
def test_tree_attention_loses_no_key_of_a_long_context(ctx, nodes):
    """Every key at a page's border shows in the output (the CPU test of these inputs removes them one by one)."""
    _check_attn(make_borders(ctx, nodes, device="cuda")[0])


def test_a_verified_step_takes_no_more_memory_than_is_set_aside():
    from open_instruct_b200.data_types import SamplingConfig
    from open_instruct_b200.models import get_spec
    from open_instruct_b200.rollout.engine import RolloutEngine

    spec = get_spec("llama3.2-1b").replace(head_dim=128, num_heads=16, num_kv_heads=4, num_layers=6, eos_token_id=None)
    eng = RolloutEngine(spec, device="cuda", ops="fused", num_blocks=400, max_running=32, max_model_len=1024, seed=3, eos_token_ids=[], speculative_tokens=31)
    assert eng.draft_rows == 1024
    eng._step_ms = lambda rows, drafts: 1.0 if drafts else 100.0
    peaks, drafts = [], eng._decode_drafts

    def watched(seqs, trees):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        drafts(seqs, trees)
        rows = sum(len(t) for t, _, _ in trees)
        peaks.append((rows, torch.cuda.max_memory_allocated() - before))

    eng._decode_drafts = watched
    ahead = eng._ahead
    eng._ahead = lambda q: (ahead(q), [[(q.tokens[-1] + i) % spec.vocab_size for i in range(1, 32)]] if len(q.tokens) < 60 else [])[1]
    eng.generate([[5 + i, 6, 7] for i in range(32)], SamplingConfig(temperature=0.0, max_tokens=70, min_tokens=70, n=1))
    assert max(peaks)[0] == 1024
    for rows, peak in peaks:
        assert peak <= eng.draft_bytes(spec, rows), (rows, peak, eng.draft_bytes(spec, rows))
