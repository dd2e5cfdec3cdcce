"""Speculative-decoding operators on the CPU: the PyTorch restatements against 64-bit oracles, and the refusals, which the kernel
wrappers share with them."""

import pytest
import torch

from open_instruct_b200.ops import emulated, fused
from _speculative import DIM, PAGE, attn_bound, attn_oracle, logprob_bound, make_attn, make_borders, make_cold, make_covered, make_verify, verify_oracle


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (7, 1), (2, 2)])
@pytest.mark.parametrize("shape", ["chain", "tree", "star"])
def test_tree_attention(heads, kv_heads, shape):
    a = make_attn(heads, kv_heads, [0, 1, 63, 64, 65, 200, 10], [1, 3, 0, 5, 9, 2, 4], shape, dtype=torch.float32, row_extra=8, table_extra=1)
    out = emulated.tree_attn(**a)
    ref, mag = attn_oracle(a)
    assert ((out.double() - ref).abs() <= 2.0 ** -13 * mag + 1e-30).all()   # fp32 throughout: the bound's fp32 share


def test_tree_attention_padding_and_bad_pages():
    a = make_attn(4, 2, [70, 130], [6, 5], dtype=torch.float32, extra_rows=3)
    a["parents"][[4, 5, 10]] = -2
    a["parents"][9] = 0
    a["block_table"][0, 1] = -3
    a["block_table"][1, 0] = a["k_cache"].shape[0]
    out = torch.full((14, 4 * DIM), 7.0)
    assert emulated.tree_attn(**a, out=out) is out
    ref, mag = attn_oracle(a)
    assert ((out[:11].double() - ref[:11]).abs() <= 2.0 ** -13 * mag[:11] + 1e-30).all()
    assert (out[[4, 5, 10]] == 0).all() and (out[11:] == 7.0).all()


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("shape", ["chain", "tree", "star"])
@pytest.mark.parametrize("vocab", [1, 2, 97, 1000])
def test_verification(vocab, shape, drafted):
    a = make_verify([3, 1, 0, 7, 5, 12, 2, 4] * 3, vocab, shape, drafted, temps=(1.0, 0.0, 0.6, 1.7, 1.0), seed=vocab, row_extra=3, extra_rows=2)
    got, want = emulated.verify_tree(**a), verify_oracle(a)
    for x, y in zip(got[:3], want[:3]):
        assert torch.equal(x, y.to(x.dtype))
    assert (got[3].double() - want[3]).abs().max() <= logprob_bound(vocab)


@pytest.mark.parametrize("drafted", [False, True])
def test_emitted_tokens_follow_the_target(drafted):
    """The first emitted token over many independent draws has the target's distribution, whatever is drafted: each bin's count is
    within six standard deviations."""
    g = torch.Generator().manual_seed(5)
    V, trials, kids = 6, 4000, 3
    z = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5, -3.0]).bfloat16()
    q = torch.softmax(torch.tensor([0.0, 1.0, 0.5, 0.0, 2.0, -1.0]), -1)
    counts = [kids + 1] * trials
    a = make_verify(counts, V, "star", seed=1)
    a["logits"] = z.expand(len(a["tokens"]), V).contiguous()
    a["tokens"] = torch.multinomial(q, len(a["tokens"]), replacement=True, generator=g)
    a["draft_probs"] = q.expand(len(a["tokens"]), V).contiguous() if drafted else None
    _, tokens, _, _ = emulated.verify_tree(**a)
    p = torch.softmax(z.double(), -1)
    seen = torch.bincount(tokens[:, 0], minlength=V).double()
    assert ((seen - trials * p).abs() <= 6 * (trials * p * (1 - p)).sqrt()).all(), (seen / trials, p)


def _commit_inputs(layers, kv_heads=2, heads=4, dtype=torch.float32, device="cpu"):
    a = make_attn(heads, kv_heads, [0, 60, 64, 127, 200], [3, 8, 1, 5, 2], dtype=dtype, garbage=False, table_extra=1, device=device, row_extra=16)
    g = torch.Generator().manual_seed(3)
    total = a["k_cache"].shape[0] + 8
    table = torch.randperm(total, generator=g)[: 5 * a["block_table"].shape[1]]
    total = max(total, 5 * a["block_table"].shape[1])
    table = torch.randperm(total, generator=g)[: 5 * a["block_table"].shape[1]].view(5, -1).int().to(device)
    width = (heads + 2 * kv_heads) * DIM
    qkv = [torch.randn(19, width + 16, generator=g).to(device, dtype)[:, :width] for _ in range(layers)]
    path = torch.full((5, 4), -1, dtype=torch.int32)
    path[0, :3] = torch.tensor([0, 1, 2])
    path[1] = torch.tensor([3, 5, 6, 10])
    path[2, 0] = 11
    path[3, :2] = torch.tensor([12, 16])
    shape = (layers, total, kv_heads, PAGE, DIM)
    k, v = (torch.randn(shape, generator=g).to(device, dtype) for _ in range(2))
    return dict(qkv_layers=qkv, k_cache=k, v_cache=v, block_table=table, ctx=a["ctx"], path=path.to(device), n_q=heads, n_kv=kv_heads, head_dim=DIM)


def _commit_oracle(a):
    k, v = a["k_cache"].clone(), a["v_cache"].clone()
    hq, hk = a["n_q"], a["n_kv"]
    for b, nodes in enumerate(a["path"].tolist()):
        for j, node in enumerate(nodes):
            pos = int(a["ctx"][b]) + j
            if not 0 <= node < a["qkv_layers"][0].shape[0] or pos // PAGE >= a["block_table"].shape[1]:
                continue
            blk = int(a["block_table"][b, pos // PAGE])
            if not 0 <= blk < k.shape[1]:
                continue
            for i, x in enumerate(a["qkv_layers"]):
                row = x[node].view(hq + 2 * hk, DIM)
                k[i, blk, :, pos % PAGE], v[i, blk, :, pos % PAGE] = row[hq:hq + hk], row[hq + hk:]
    return k, v


@pytest.mark.parametrize("bad", [False, True])
def test_commit(bad):
    a = _commit_inputs(3)
    if bad:   # a page outside the cache on either side, a node outside the batch, a context past the table
        a["block_table"][1, 0], a["block_table"][0, 0], a["path"][3, 1], a["ctx"][4] = -1, a["k_cache"].shape[1], 19, 64 * a["block_table"].shape[1]
        a["path"][4, 0] = 17
    want = _commit_oracle(a)
    emulated.kv_commit_(**a)
    assert torch.equal(a["k_cache"], want[0]) and torch.equal(a["v_cache"], want[1])


def _change(a, **kw):
    return {**a, **kw}


def test_refusals_of_tree_attention():
    a = make_attn(4, 2, [70, 3], [3, 2], dtype=torch.float32)
    with pytest.raises(TypeError, match="CUDA"):
        fused.tree_attn(**a)
    odd = torch.zeros(5, 8 * DIM + 4)[:, : 8 * DIM]
    bad = [
        dict(head_dim=64), dict(n_kv=3), dict(n_kv=0), dict(n_q=2 * 129), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
        dict(scale=float("nan")), dict(max_nodes=0), dict(max_nodes=65), dict(qkv=a["qkv"][:, :-DIM]), dict(qkv=odd), dict(qkv=a["qkv"][:, None]),
        dict(k_cache=a["k_cache"].double()), dict(v_cache=a["v_cache"][:-1]), dict(k_cache=a["k_cache"].transpose(1, 2)),
        dict(block_table=a["block_table"].long()), dict(block_table=a["block_table"][:1]), dict(block_table=a["block_table"].t()),
        dict(ctx=a["ctx"].long()), dict(ctx=a["ctx"][:1]), dict(cu_nodes=a["cu_nodes"][:-1]), dict(cu_nodes=a["cu_nodes"].long()),
        dict(parents=a["parents"][:-1]), dict(parents=a["parents"].long()), dict(out=torch.zeros(5, 4 * DIM, dtype=torch.float64)),
        dict(out=torch.zeros(4, 4 * DIM)), dict(out=torch.zeros(5, 8 * DIM)[:, ::2]),
    ]
    for kw in bad:
        with pytest.raises((TypeError, ValueError)):
            emulated.tree_attn(**_change(a, **kw))


def test_refusals_of_verification():
    a = make_verify([3, 2], 10, drafted=True)
    with pytest.raises(TypeError, match="CUDA"):
        fused.verify_tree(**a)
    with pytest.raises(TypeError):
        fused._check_verify_tree(**_change(a, logits=a["logits"].float()), dtype=torch.bfloat16)
    bad = [
        dict(max_nodes=0), dict(max_nodes=65), dict(logits=a["logits"][0]), dict(logits=a["logits"][:, :0]), dict(logits=torch.zeros(5, 20)[:, ::2]),
        dict(tokens=a["tokens"].int()), dict(tokens=a["tokens"][1:]), dict(parents=a["parents"].long()), dict(cu_nodes=a["cu_nodes"][1:]),
        dict(temperature=a["temperature"].double()), dict(temperature=a["temperature"][:, None]), dict(u_accept=a["u_accept"][:4]),
        dict(u_accept=a["u_accept"].double()), dict(u_sample=a["u_sample"][:1]), dict(draft_probs=a["draft_probs"].bfloat16()),
        dict(draft_probs=a["draft_probs"][:, :9]), dict(draft_probs=a["draft_probs"].t().contiguous().t()),
    ]
    for kw in bad:
        with pytest.raises((TypeError, ValueError)):
            emulated.verify_tree(**_change(a, **kw))


def test_refusals_of_commit():
    a = _commit_inputs(2)
    with pytest.raises(TypeError, match="CUDA"):
        fused.kv_commit_(**a)
    x = a["qkv_layers"]
    bad = [
        dict(qkv_layers=[]), dict(qkv_layers=x[:1]), dict(qkv_layers=[x[0], x[1][:-1]]), dict(qkv_layers=[x[0], x[1].contiguous()]),
        dict(qkv_layers=[x[0], x[1].double()]), dict(head_dim=64), dict(n_kv=0), dict(n_q=5), dict(k_cache=a["k_cache"][:, :-1]),
        dict(v_cache=a["v_cache"].double()), dict(path=a["path"].long()), dict(path=a["path"][:-1]), dict(path=a["path"][0]),
        dict(ctx=a["ctx"].long()), dict(block_table=a["block_table"][:2]),
    ]
    for kw in bad:
        with pytest.raises((TypeError, ValueError)):
            emulated.kv_commit_(**_change(a, **kw))


# ------------------------------------------------------------------------------------------------ the rollout engine
def _engine(speculative_tokens, **kw):
    from open_instruct_b200.models import get_spec
    from open_instruct_b200.rollout.engine import RolloutEngine

    spec = get_spec("tiny128").replace(eos_token_id=3)
    return RolloutEngine(spec, device="cpu", ops="ref", seed=1, speculative_tokens=speculative_tokens, **kw)


def _prompts():
    g = torch.Generator().manual_seed(0)
    base = torch.randint(4, 512, (40,), generator=g).tolist()
    return [base * 3, base + base[:20], torch.randint(4, 512, (7,), generator=g).tolist()]


def test_draft_trees():
    from open_instruct_b200.rollout.speculative import PromptLookup, draft_tree

    look = PromptLookup(2)
    toks = [1, 2, 3, 4, 1, 2, 5, 6, 1, 2]
    assert look.continuations(toks, 3) == [[5, 6, 1], [3, 4, 1]]
    assert look.continuations(toks + [3], 2) == [[4, 1]] and look.continuations([9], 4) == [] and look.continuations(toks, 0) == []
    tokens, parents, depths = draft_tree(2, [[5, 6, 1], [5, 7, 8]], 5)
    assert tokens == [2, 5, 6, 1, 7, 8] and parents == [-1, 0, 1, 2, 1, 4] and depths == [0, 1, 2, 3, 2, 3]
    tokens, parents, _ = draft_tree(2, [[5, 6, 1, 1, 1], [3, 4]], 3)
    assert len(tokens) == 4 and tokens[:3] == [2, 5, 6] and tokens[3] == 3 and parents[3] == 0
    assert draft_tree(4, [], 3) == ([4], [-1], [0])


def test_drafting_coins_are_the_samplers_numbers():
    """The vectorised generator is the sampler's Philox: its numbers lie half a step above these."""
    import numpy as np

    from open_instruct_b200.rollout.sampler import philox_uniform
    from open_instruct_b200.rollout.speculative import uniforms

    seeds, ctr, idx = np.array([5, 1 << 40, 12345678901]), np.array([0, 7, 100]), np.array([0x80000000, 0x80000003, 0xFFFFFFFF])
    got = uniforms(seeds, ctr, idx)
    want = [philox_uniform(int(s), int(c), np.array([i], dtype=np.uint32))[0] for s, c, i in zip(seeds, ctr, idx)]
    assert np.abs(got - (np.array(want) - 0.5 / 16777216.0)).max() == 0.0 and got.dtype == np.float32


@pytest.mark.parametrize("drafts", [1, 4, 63])
def test_engine_with_drafts_emits_the_same_greedy_text(drafts):
    from open_instruct_b200.data_types import SamplingConfig

    cfg = SamplingConfig(temperature=0.0, max_tokens=70, n=2)
    plain, spec = _engine(0, num_blocks=64), _engine(drafts, num_blocks=64)
    a, b = plain.generate(_prompts(), cfg), spec.generate(_prompts(), cfg)
    assert [r.responses for r in a] == [r.responses for r in b] and [r.finish_reasons for r in a] == [r.finish_reasons for r in b]
    for x, y in zip(a, b):   # fp32 on both sides, other summation orders
        for p, q in zip(x.logprobs, y.logprobs):
            assert len(p) == len(q) and max(abs(u - v) for u, v in zip(p, q)) < 1e-3
    assert spec.stats["accepted_tokens"] > 0 and spec.stats["steps"] < plain.stats["steps"]
    assert spec.host.free_blocks() == 64


def test_engine_with_drafts_samples_reproducibly_and_reports_the_targets_logprobs():
    from open_instruct_b200.data_types import SamplingConfig

    cfg = SamplingConfig(temperature=0.7, max_tokens=20, n=3, seed=11)
    eng = _engine(6, num_blocks=64)
    a, b = eng.generate(_prompts(), cfg), eng.generate(_prompts(), cfg)
    assert [r.responses for r in a] == [r.responses for r in b]
    for prompt, r in zip(_prompts(), a):
        for text, lps in zip(r.responses, r.logprobs):
            ids = torch.tensor(prompt + text)
            logits = eng.model.logits(ids, torch.arange(len(ids)), torch.tensor([0, len(ids)], dtype=torch.int32)).float() / 0.7
            want = torch.log_softmax(logits, -1)[len(prompt) - 1:-1].gather(1, ids[len(prompt):, None]).squeeze(1)
            assert (want - torch.tensor(lps)).abs().max() < 1e-3


def test_engine_with_drafts_under_preemption_and_with_a_nucleus():
    from open_instruct_b200.data_types import SamplingConfig

    prompts = [list(range(5, 5 + n)) * 2 for n in (50, 55, 60)]
    cfg = SamplingConfig(temperature=0.0, max_tokens=40, n=1)
    big, small = _engine(5, num_blocks=64), _engine(5, num_blocks=7)
    assert [r.responses for r in big.generate(prompts, cfg)] == [r.responses for r in small.generate(prompts, cfg)]
    assert small.host.preemptions() > 0 and small.host.free_blocks() == 7
    nucleus = SamplingConfig(temperature=1.0, top_p=0.9, max_tokens=8, n=1, seed=3)
    eng = _engine(5, num_blocks=64)
    assert [r.responses for r in eng.generate(prompts, nucleus)] == [r.responses for r in _engine(0, num_blocks=64).generate(prompts, nucleus)]
    assert "drafted_tokens" not in eng.stats


def test_engine_with_drafts_and_prefix_caching():
    """Pages filled by verified steps are found again by a follow-up turn."""
    from open_instruct_b200.data_types import SamplingConfig

    cfg = SamplingConfig(temperature=0.0, max_tokens=90, n=1)
    plain, spec = _engine(0, num_blocks=64), _engine(4, num_blocks=64, enable_prefix_caching=True)
    prompts = _prompts()
    for _ in range(2):
        a, b = plain.generate(prompts, cfg), spec.generate(prompts, cfg)
        assert [r.responses for r in a] == [r.responses for r in b]
        prompts = [p + r.responses[0] + [7, 8, 9] for p, r in zip(prompts, a)]
    assert spec.stats["prefix_cached_tokens"] > 0 and spec.stats["accepted_tokens"] > 0


def test_engine_refuses_drafts_it_cannot_verify():
    from open_instruct_b200.models import get_spec
    from open_instruct_b200.rollout.engine import RolloutEngine

    with pytest.raises(ValueError):
        _engine(64)
    with pytest.raises(ValueError):
        _engine(-1)
    with pytest.raises(NotImplementedError):
        RolloutEngine(get_spec("tiny"), device="cpu", ops="ref", num_blocks=16, speculative_tokens=4)


def test_rows_that_overlap_are_refused():
    a = make_attn(2, 1, [5], [3])
    for qkv in (a["qkv"][:1].expand(3, -1), torch.empty(4096, dtype=torch.bfloat16).as_strided((3, 512), (256, 1))):
        with pytest.raises(ValueError, match="overlap"):
            fused._check_tree_attn(**{**a, "qkv": qkv}, out=None, dtype=torch.bfloat16)
    a["qkv"] = a["qkv"][:1].expand(1, -1)   # one row alone has no stride
    a["parents"] = a["parents"][:1]
    fused._check_tree_attn(**a, out=None, dtype=torch.bfloat16)


def test_drafts_that_cover_all_that_a_row_allows():
    a, first, counts = make_covered()
    got, want = emulated.verify_tree(**a), verify_oracle(a)
    for x, y in zip(got[:3], want[:3]):
        assert torch.equal(x, y.to(x.dtype))
    assert got[1][:, 0].tolist() == first and got[0].tolist() == counts
    assert torch.isfinite(got[3]).all()


@pytest.mark.parametrize("drafted", [False, True])
def test_verification_at_low_temperatures(drafted):
    a = make_cold(drafted=drafted)
    got, want = emulated.verify_tree(**a), verify_oracle(a)
    for x, y in zip(got[:3], want[:3]):
        assert torch.equal(x, y.to(x.dtype))
    assert (got[3].double() - want[3]).abs().max() <= logprob_bound(2000)


def test_padding_nodes_may_hold_anything():
    """A padding node's row of qkv is never used: its result is zero and no other node's result is touched."""
    a = make_attn(4, 2, [70, 0, 30], [6, 5, 3], dtype=torch.float32)
    pads = [4, 5, 10, 12]
    a["parents"][pads] = -2
    a["parents"][[9, 13]] = 0
    ref, mag = attn_oracle(a)
    a["qkv"][pads] = float("nan")
    out = emulated.tree_attn(**a)
    assert (out[pads] == 0).all() and ((out.double() - ref).abs() <= 2.0 ** -13 * mag + 1e-30).all()


def test_children_of_padding_are_roots():
    a = make_attn(4, 2, [70, 0], [6, 3], "chain", dtype=torch.float32)
    a["parents"][[2, 6, 7, 8]] = -2
    roots = {**a, "parents": a["parents"].clone()}
    roots["parents"][3] = -1
    assert a["parents"][3] == 2
    assert torch.equal(emulated.tree_attn(**a), emulated.tree_attn(**roots))
    ref, mag = attn_oracle(roots)
    assert ((emulated.tree_attn(**a).double() - ref).abs() <= 2.0 ** -13 * mag + 1e-30).all()


@pytest.mark.parametrize("ctx", [383, 4097, 20011])
def test_long_context_inputs_show_every_border_key(ctx):
    """What the GPU test of long contexts relies on: leaving out any one key at a page's border moves the result by more than its
    tolerance (every border key of the shorter contexts, every 37th and the last of the longest)."""
    a, borders = make_borders(ctx, 1)
    ref, mag = attn_oracle(a)
    bound = attn_bound(ref, mag)
    full = [a["block_table"][0].long(), torch.arange(ctx)]
    k = a["k_cache"][full[0][full[1] // PAGE], 0, full[1] % PAGE].double()
    v = a["v_cache"][full[0][full[1] // PAGE], 0, full[1] % PAGE].double()
    x = a["qkv"][0].double().view(6, DIM)
    s = torch.cat([x[:4] @ k.t(), x[:4] @ x[4:5].t()], 1) * a["scale"]
    v = torch.cat([v, x[5:6]])
    w = torch.exp(s - s.max())
    top, total = w @ v, w.sum(1, keepdim=True)
    assert torch.allclose((top / total).reshape(-1), ref[0], rtol=1e-9, atol=1e-15)
    for p in borders if ctx < 10000 else borders[::37] + [ctx - 1]:
        less = (top - w[:, p:p + 1] * v[p]) / (total - w[:, p:p + 1])
        assert ((less.reshape(-1) - ref[0]).abs() > bound[0]).any(), p


def test_a_verified_step_has_to_pay():
    """Which steps draft: the expected tokens against the steps' modelled times."""
    from open_instruct_b200.rollout.speculative import DECODE_ROWS, Acceptance, expected_tokens, plan_drafts, step_ms

    def chance(hits, trials):
        c = Acceptance()
        for _ in range(30):
            c.record(hits, trials)
        return c

    assert Acceptance().rate() == 0.5 and [expected_tokens(0.5, d) for d in (0, 1, 3)] == [0.0, 0.5, 0.875]
    good, poor = chance(4, 4), chance(0, 1)
    assert 0.95 < good.rate() < 1.0 and poor.rate() < 0.1

    def plan(ahead, chances, most=4, rows=1 << 20, graphs=True):
        model = lambda rows, eager: step_ms(rows, 32, 8_030_000_000, eager)
        return plan_drafts(ahead, chances, most, rows, model(len(ahead), not graphs), lambda n: model(n, True))

    draft, none = [[1, 2, 3, 4]], []
    for batch, nodes in ((16, 4), (64, 3), (256, 4)):                                  # 64 of 1 + 3 nodes are the decode GEMMs' 256 rows
        assert plan([draft] * batch, [good] * batch) == nodes                          # nearly all is accepted
        assert plan([draft] * batch, [poor] * batch) == 0                              # nearly nothing is
        assert plan([draft] + [none] * (batch - 1), [good] * batch) == 0               # one sequence of many
    assert plan([draft], [poor], graphs=False) == 4                                    # a lone sequence has little to lose
    # two tokens each would leave the decode GEMMs, one stays
    fair = chance(3, 5)
    assert plan([[[1, 2]]] * 120, [fair] * 120, most=2) in (0, 1)
    assert plan([[[1, 2]]] * 120, [good] * 120, most=2, rows=240) == 1 and DECODE_ROWS == 256
    assert plan([draft] * 8, [good] * 8, rows=8) == 0                                  # no room for a single node
    assert plan([draft] * 8, [good] * 8, rows=16) == 1
    # as many as the drafter offers are too many, fewer pay
    assert 0 < plan([[list(range(32))]] * 256, [good] * 256, most=32) < 32


def test_one_drafting_sequence_does_not_move_a_batch_off_its_ordinary_steps():
    from open_instruct_b200.data_types import SamplingConfig

    prompts = [list(range(5 + 9 * i, 25 + 9 * i)) for i in range(8)]
    cfg = SamplingConfig(temperature=0.0, max_tokens=12, min_tokens=12, n=1)
    want = [r.responses for r in _engine(0, num_blocks=64).generate(prompts, cfg)]
    right = {tuple(p): r[0] for p, r in zip(prompts, want)}

    def run(drafting):
        eng = _engine(3, num_blocks=64)
        eng._step_ms = lambda rows, drafts: 1.5 if drafts else 1.0
        ahead = eng._ahead

        def foresee(q):   # the right tokens for the drafting sequences
            ahead(q)
            prompt, n = tuple(q.tokens[: q.prompt_len]), len(q.tokens) - q.prompt_len
            chain = right[prompt][n:n + 3][: q.request.sampling.max_tokens - n - 1]
            return [chain] if chain and prompts.index(list(prompt)) < drafting else []

        eng._ahead = foresee
        assert [r.responses for r in eng.generate(prompts, cfg)] == want
        return eng.stats

    assert "drafted_tokens" not in run(1) and run(8)["accepted_tokens"] > 20


def test_continuations_that_agree_are_one_draft():
    from open_instruct_b200.rollout.speculative import PromptLookup

    toks = [1, 2, 3, 4, 5, 9, 1, 2, 3, 4, 5, 8, 1, 2]
    assert PromptLookup(2).continuations(toks, 3) == [[3, 4, 5]]
    assert PromptLookup(2).continuations(toks, 4) == [[3, 4, 5, 8], [3, 4, 5, 9]]
    assert PromptLookup(1).continuations([7, 7, 7], 4) == [[7, 7]]   # the latest one is cut by the end of the text


def test_a_verified_step_is_bounded_and_its_memory_is_set_aside(monkeypatch):
    """No step has more nodes than ``draft_rows``, whatever the sequences offer, and an engine that sizes its own cache leaves room
    for such a step."""
    from open_instruct_b200.data_types import SamplingConfig
    from open_instruct_b200.models import get_spec
    from open_instruct_b200.rollout.engine import DRAFT_ROWS, RolloutEngine

    eng = _engine(63, num_blocks=64, max_running=8)
    assert eng.draft_rows == 8 * 64 and _engine(0, num_blocks=16).draft_rows == 0
    eng.draft_rows, seen = 20, []
    drafts = eng._decode_drafts
    eng._decode_drafts = lambda seqs, trees: (seen.append(sum(len(t) for t, _, _ in trees)), drafts(seqs, trees))
    cfg = SamplingConfig(temperature=0.0, max_tokens=70, n=2)
    a, b = eng.generate(_prompts(), cfg), _engine(0, num_blocks=64).generate(_prompts(), cfg)
    assert [r.responses for r in a] == [r.responses for r in b] and 6 < max(seen) <= 20
    spec = get_spec("llama3.1-8b")
    rows = min(256 * 64, DRAFT_ROWS)
    assert RolloutEngine.draft_bytes(spec, 0) == 0
    assert RolloutEngine.draft_bytes(spec, rows) > rows * 2 * (32 * 48 * 128 + spec.vocab_size)


def test_nothing_is_launched_early_behind_the_join_of_the_tree_attention():
    """The decode GEMMs' pairs of CTAs must not start on SMs that the attention is leaving (their allocation of tensor memory has no
    limit on its wait): the join waits for the attention and lets nothing start before its own end."""
    from pathlib import Path

    import open_instruct_b200.ops as ops

    src = (Path(ops.__file__).parent / "csrc" / "tree_attn.cu").read_text()
    at = src.index("tree_join_kernel(const __grid_constant__ TreeArgs a) {")
    body = src[at:src.index("\n}\n", at)]
    assert "griddep_wait();" in body and "griddep_launch_dependents" not in body
    launch = src[src.index('extern "C" int b200_tree_attn('):]
    assert launch.index("ta_launch<true>") < launch.index("tree_join_kernel")   # and it is the last kernel of the call
    assert "launch" not in launch[launch.index("tree_join_kernel"):].split("\n", 1)[1]
