"""Drafted trees, the 8-bit KV cache and log-probabilities on the CPU oracle."""
import math

import pytest
import torch

from cascadia_b200.engine.base import InvalidConfig
from cascadia_b200.engine.llm import LLMBuilder, LLMEngine
from cascadia_b200.models.config import get_config
from cascadia_b200.models.llama import LlamaModel
from cascadia_b200.ops import reference as ref
from cascadia_b200.runtime.generator import BatchGenerator
from cascadia_b200.runtime.kv_cache import KVCache
from cascadia_b200.runtime.spec import (DraftTree, NGramDraft, TreeSpecDecoder, verify_trees)
from cascadia_b200.types import GenerationTask, ShardSpec


def _model(kv_dtype="bf16", seed=5, name="tiny-llama"):
    m = LlamaModel(get_config(name), "cpu").init_random(seed=seed, gen_device="cpu")
    m.allocate_kv(256, kv_dtype=kv_dtype)
    return m


def _prompts():
    g = torch.Generator().manual_seed(3)
    rep = torch.randint(3, 500, (6,), generator=g).tolist()
    return [rep * 4, torch.randint(3, 500, (11,), generator=g).tolist(), [7]]


# ------------------------------------------------------------ the oracle
def test_quantised_rows_round_trip():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 3, 64, generator=g) * torch.exp(3 * torch.randn(40, 3, 1, generator=g))
    x[0] = 0
    codes, s = ref.quantise_rows(x)
    y = ref.dequantise_rows(codes, s)
    # half a step of a 4-bit significand, and of the smallest step 2^-9 s
    tol = torch.maximum(x.abs() / 16, s.unsqueeze(-1) * 2.0 ** -10) * (1 + 1e-5)
    assert bool(((y - x).abs() <= tol).all()) and bool((y[0] == 0).all())
    x[1, 2, 5] = float("inf")
    x[2, 0, 1] = float("nan")
    codes, s = ref.quantise_rows(x)
    assert bool(s[1, 2].isnan()) and bool(s[2, 0].isnan()) and bool(s[1, :2].isfinite().all())
    assert bool((codes[1, 2].float() == 0).all())


@pytest.mark.parametrize("n,ctx", [(1, 0), (1, 9), (5, 0), (7, 6)])
def test_tree_attention_is_the_formula(n, ctx):
    """Row by row: an ordinary softmax over the keys it sees, in 64 bits."""
    g = torch.Generator().manual_seed(n + ctx)
    q = torch.randn(n, 4, 8, generator=g, dtype=torch.float64)
    k, v = torch.randn(2, ctx + n, 2, 8, generator=g, dtype=torch.float64)
    tree = DraftTree()
    for i in range(1, n):
        tree.add((i - 1) // 2, i)
    masks = tree.masks()
    out = ref.tree_attention(q, k, v, 0.3, masks)
    chain = ref.tree_attention(q, k, v, 0.3)
    for i in range(n):
        for mask, got in ((masks[i], out), ((1 << (i + 1)) - 1, chain)):
            keys = list(range(ctx)) + [ctx + j for j in range(n) if mask >> j & 1]
            for h in range(4):
                p = torch.softmax(k[keys, h // 2] @ q[i, h] * 0.3, 0)
                assert torch.allclose(got[i, h], p @ v[keys, h // 2], atol=1e-12)


def test_tree_attention_row_that_sees_nothing():
    x = torch.randn(2, 1, 8)
    out = ref.tree_attention(x, x, x, 1.0, [0, 2])
    assert bool((out[0] == 0).all()) and torch.allclose(out[1], x[1])


def test_token_logprobs_reference():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5, 40, generator=g, dtype=torch.float64) * 4
    x[1] = -math.inf
    x[2, 3] = math.nan
    x[3, :] = 1.0
    lp, ent, ids, top = ref.token_logprobs(x, torch.tensor([0, 1, 2, 3, 40]), 4)
    want = torch.log_softmax(x[0], 0)
    assert abs(float(lp[0] - want[0])) < 1e-12
    assert abs(float(ent[0]) + float((want.exp() * want).sum())) < 1e-12
    assert float(lp[1]) == -math.inf and float(ent[1]) == 0.0 and ids[1].tolist() == [0, 1, 2, 3]
    assert math.isnan(float(lp[2])) and int(ids[2, 0]) == 3
    assert ids[3].tolist() == [0, 1, 2, 3] and abs(float(ent[3]) - math.log(40)) < 1e-12
    assert math.isnan(float(lp[4]))  # no such token


# ------------------------------------------------------------ trees
def test_tree_from_chains_and_masks():
    t = DraftTree.from_chains([[5, 6, 7], [5, 8], [9]], 10)
    assert (t.tokens, t.parents) == ([5, 6, 7, 8, 9], [0, 1, 2, 1, 0])
    assert t.depths() == [0, 1, 2, 3, 2, 1]
    assert t.masks() == [1, 3, 7, 15, 0b10011, 0b100001]
    assert t.cut(1).tokens == [5, 9] and t.cut(0).tokens == []
    assert DraftTree.from_chains([[5, 6, 7], [5, 8]], 2).tokens == [5, 6]
    assert t.accepted_chain([5, 6, 7]) == 3 and t.accepted_chain([5, 8]) == 1
    assert t.accepted_chain([9]) == 0
    deep = DraftTree()
    for i in range(63):
        deep.add(i, i)
    assert deep.masks()[63] == -1  # all 64 bits, as a signed number


def test_ngram_tree_branches_where_the_text_did():
    d = NGramDraft(4)
    d.extend([1, 2, 3, 4, 9, 2, 3, 4, 8, 7, 3, 4, 6, 1, 2, 3, 4])
    t = d.propose_tree(3, 16)
    roots = [tok for tok, p in zip(t.tokens, t.parents) if p == 0]
    assert roots == [9, 8, 6]  # after 1 2 3 4, after 2 3 4, after 3 4


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("draft", ["ngram", "self", "other"])
def test_tree_decoding_equals_greedy(kv_dtype, draft):
    m = _model(kv_dtype)
    want = BatchGenerator(m, use_graph=False).generate(_prompts(), 20)
    dm = None if draft == "ngram" else _model(seed=5 if draft == "self" else 6)
    dec = TreeSpecDecoder(m, draft=dm, k=3, branch=3, max_nodes=12, use_graph=False)
    lps = []
    got = dec.generate(_prompts(), 20, logprobs=lps)
    assert got == want
    assert [len(x) for x in lps] == [19] * 3
    assert all(-1e-6 < -x < 20 for row in lps for x in row)
    assert m.kv.allocator.num_free == m.kv.num_blocks
    if draft == "self" and kv_dtype == "bf16":
        assert dec.stats.accepted >= dec.stats.rounds  # the chain is the target's own


def test_accepted_path_closes_ranks():
    """After a verification the cache holds the accepted path's rows, as
    plain decoding would have left them."""
    a, b = _model(), _model()
    prompt = _prompts()[0]
    plain = BatchGenerator(a, use_graph=False)
    toks = [int(plain.prefill(["s"], [prompt])[0])]
    for _ in range(3):
        toks.append(int(plain.decode(["s"], [toks[-1]], 16)[0]))
    BatchGenerator(b, use_graph=False).prefill(["s"], [prompt])
    # Wrong siblings before the right ones: the path's slots are not in order.
    tree = DraftTree()
    at = 0
    for t in toks[1:3]:
        tree.add(at, (t + 1) % 500)
        at = tree.add(at, t)
    r = verify_trees(b, ["s"], [toks[0]], [tree], [len(prompt)], top_k=3)[0]
    assert r.tokens == toks[1:4]
    assert b.kv.seqs["s"].length == len(prompt) + 3
    for layer in range(2):
        for x, y in zip(a.kv.gather(layer, "s"), b.kv.gather(layer, "s")):
            n = len(prompt) + 3
            assert torch.allclose(x[:n].float(), y[:n].float(), atol=2e-2)
    assert [len(t) for t in r.top_ids] == [3, 3, 3] and r.top_ids[0][0] == toks[1]


def test_moved_rows_are_read_before_any_is_written():
    kv = KVCache(2, 4, 1, 64, "cpu", kv_dtype="fp8")
    kv.add_sequence("s")
    kv.reserve("s", 40)
    x = torch.randn(40, 1, 64)
    slots = torch.tensor(kv.seqs["s"].slots(0, 40))
    for layer in range(2):
        kv.write_rows(layer, slots, x * (layer + 1), -x)
    want = [kv.gather(layer, "s") for layer in range(2)]
    kv.move_rows("s", [20, 21, 35], [19, 20, 21])
    for layer in range(2):
        for got, old in zip(kv.gather(layer, "s"), want[layer]):
            assert torch.equal(got[[19, 20, 21]], old[[20, 21, 35]])
            assert torch.equal(got[22:35], old[22:35])


def test_fp8_cache_is_close_and_smaller():
    a, b = _model(), _model("fp8")
    assert b.kv_bytes_per_block("fp8") < 0.54 * a.kv_bytes_per_block()
    prompt = _prompts()[0]
    outs = []
    for m in (a, b):
        g = BatchGenerator(m, use_graph=False)
        g.prefill(["s"], [prompt])
        outs.append(g.last_logits.float())
    assert float((outs[0] - outs[1]).norm() / outs[0].norm()) < 0.1


# ------------------------------------------------------------ engine
def _drain(e, ids, steps=200):
    out = {t: [] for t in ids}
    for _ in range(steps):
        for tid, c in e.step():
            out[tid].append(c)
        if all(out[t] and out[t][-1].is_final for t in ids):
            break
    return out


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_engine_trees_match_plain_and_carry_logprobs(kv_dtype):
    results = {}
    for spec in (None, "tree"):
        e = LLMEngine(_model(kv_dtype), max_model_len=512, spec=spec, use_graph=False)
        for i, p in enumerate(_prompts()):
            t = GenerationTask(f"t{i}", "", max_tokens=15, prompt_ids=p)
            t.logprobs = 0 if i == 2 else 1 + i
            e.submit(t)
        out = _drain(e, ["t0", "t1", "t2"])
        results[spec] = {k: [(c.token_id, c.logprobs) for c in v if not c.is_final]
                         for k, v in out.items()}
    for tid, rows in results[None].items():
        got = results["tree"][tid]
        assert [t for t, _ in got] == [t for t, _ in rows]
        for (_, a), (_, b) in zip(rows, got):
            assert (a is None) == (b is None)
            if a is not None:
                assert a.token_id == b.token_id and abs(a.logprob - b.logprob) < 0.05
                assert len(a.top_logprobs) == len(b.top_logprobs)
                assert a.top_logprobs[0].token_id == b.top_logprobs[0].token_id


def test_refusals():
    with pytest.raises(ValueError):
        KVCache(1, 4, 1, 64, "cpu", kv_dtype="int3")
    m = _model()
    with pytest.raises(ValueError):
        TreeSpecDecoder(m, max_nodes=64)
    big = DraftTree()
    for i in range(64):
        big.add(0, i)
    BatchGenerator(m, use_graph=False).prefill(["s"], [[3, 4]])
    with pytest.raises(ValueError):
        verify_trees(m, ["s"], [5], [big], [2])
    for name in ("tiny-mla", "tiny-gemma4", "tiny-qwen36"):
        b = LLMBuilder(name, device="cpu", kv_blocks=32, kv_dtype="fp8")
        with pytest.raises(InvalidConfig):
            n = get_config(name).num_layers
            list(b.load(ShardSpec(name, 0, n, n, "cpu", True, True)))


def test_builder_and_moe_family_take_the_8_bit_cache():
    cfg = get_config("tiny-moe")
    b = LLMBuilder("tiny-moe", device="cpu", kv_blocks=64, kv_dtype="fp8", spec="tree",
                   use_graph=False)
    list(b.load(ShardSpec("tiny-moe", 0, cfg.num_layers, cfg.num_layers, "cpu", True, True)))
    e = b.build()
    assert e.model.kv.fp8
    e.submit(GenerationTask("a", "", max_tokens=8, prompt_ids=[5, 6, 7, 5, 6, 7, 5, 6]))
    out = _drain(e, ["a"])["a"]
    assert len([c for c in out if not c.is_final]) in range(1, 9)


# ------------------------------------------------------------ a tight pool
def _tight(blocks, kv_dtype="bf16", seed=5):
    m = LlamaModel(get_config("tiny-llama"), "cpu").init_random(seed=seed, gen_device="cpu")
    m.allocate_kv(blocks, kv_dtype=kv_dtype)
    return m


@pytest.mark.parametrize("draft", ["ngram", "self"])
def test_trees_in_a_pool_that_plain_decoding_just_fits(draft):
    new = 20
    blocks = sum(-(-(len(p) + new - 1) // 16) for p in _prompts())
    want = BatchGenerator(_tight(blocks), use_graph=False).generate(_prompts(), new)
    with pytest.raises(MemoryError):
        BatchGenerator(_tight(blocks - 1), use_graph=False).generate(_prompts(), new)
    m = _tight(blocks)
    dm = None if draft == "ngram" else _model(seed=5)
    dec = TreeSpecDecoder(m, draft=dm, k=4, branch=4, max_nodes=40, use_graph=False)
    assert dec.generate(_prompts(), new) == want
    assert m.kv.allocator.num_free == blocks
    if draft == "self":  # there is still room for some drafts
        assert dec.stats.accepted > 0


def test_engine_trees_in_a_pool_that_plain_decoding_just_fits():
    new = 20
    got = {}
    blocks = sum(-(-(len(p) + new) // 16) for p in _prompts())
    for spec in (None, "tree"):
        e = LLMEngine(_tight(blocks), max_model_len=48, spec=spec, spec_k=6, use_graph=False)
        for i, p in enumerate(_prompts()):
            e.submit(GenerationTask(f"t{i}", "", max_tokens=new, prompt_ids=p))
        if spec:
            # Drafts of many branches for every sequence, wrong ones.
            from cascadia_b200.runtime import spec as spec_mod

            old = spec_mod.NGramDraft.propose_tree
            spec_mod.NGramDraft.propose_tree = lambda self, k, most: DraftTree.from_chains(
                [[3 + i, 4 + i, 5 + i] for i in range(9)], most)
        try:
            out = _drain(e, ["t0", "t1", "t2"])
        finally:
            if spec:
                spec_mod.NGramDraft.propose_tree = old
        got[spec] = [[c.token_id for c in out[f"t{i}"] if not c.is_final] for i in range(3)]
        assert e.model.kv.allocator.num_free == blocks
    assert got["tree"] == got[None] and all(len(x) >= 1 for x in got[None])


def test_a_failed_reservation_gives_back_what_it_took():
    m = _tight(6)
    g = BatchGenerator(m, use_graph=False)
    prompts = [list(range(3, 18)), list(range(3, 34)), [5]]
    g.prefill(["a", "b", "c"], prompts)
    lens = [len(p) for p in prompts]
    before = {s: list(m.kv.seqs[s].blocks) for s in "abc"}
    wide = DraftTree()
    for i in range(40):
        wide.add(0, i)
    with pytest.raises(MemoryError):
        verify_trees(m, ["a", "b", "c"], [4, 4, 4], [DraftTree(), wide, DraftTree()], lens)
    assert {s: m.kv.seqs[s].blocks for s in "abc"} == before
    assert [m.kv.seqs[s].length for s in "abc"] == lens
    # What fits is drafted, in the order of the nodes.
    from cascadia_b200.runtime.spec import fit_trees

    cut = fit_trees(m.kv, ["a", "b", "c"], lens, [wide, wide, wide])
    assert [len(t.tokens) for t in cut] == [32, 0, 14]
    assert cut[0].tokens == wide.tokens[:32]
    verify_trees(m, ["a", "b", "c"], [4, 4, 4], cut, lens)
