"""The 8-bit KV cache, drafted trees and log-probabilities through the model
and the engine on the GPU kernels."""
import pytest
import torch

from cascadia_b200 import ops
from cascadia_b200.engine.llm import LLMEngine
from cascadia_b200.models.config import get_config
from cascadia_b200.models.llama import LlamaModel
from cascadia_b200.models.moe import MoEModel
from cascadia_b200.ops import reference as ref
from cascadia_b200.runtime.generator import BatchGenerator
from cascadia_b200.runtime.spec import DraftTree, SpecDecoder, TreeSpecDecoder, build_tree_batch
from cascadia_b200.types import GenerationTask

pytestmark = pytest.mark.gpu


def _model(kv_dtype="bf16", seed=5, name="tiny-llama-128", device="cuda"):
    cfg = get_config(name)
    m = (MoEModel if cfg.is_moe else LlamaModel)(cfg, device).init_random(seed=seed,
                                                                         gen_device="cpu")
    m.allocate_kv(256, kv_dtype=kv_dtype)
    return m


def _prompts(vocab=500):
    g = torch.Generator().manual_seed(3)
    rep = torch.randint(3, vocab, (6,), generator=g).tolist()
    return [rep * 4, torch.randint(3, vocab, (11,), generator=g).tolist(),
            torch.randint(3, vocab, (40,), generator=g).tolist()]


def _agree(a, b):
    n = 0
    for x, y in zip(a, b):
        if x != y:
            break
        n += 1
    return n


@pytest.mark.parametrize("name", ["tiny-llama-128", "tiny-llama", "tiny-moe"])
@pytest.mark.parametrize("graph", [False, True])
def test_fp8_model_matches_its_cpu_oracle(name, graph):
    """Prefill (read-back) and decode (single-token attention, captured or
    not) logits against the CPU path on the same 8-bit cache."""
    gpu, cpu = _model("fp8", name=name), _model("fp8", name=name, device="cpu")
    gg, gc = BatchGenerator(gpu, use_graph=graph), BatchGenerator(cpu, use_graph=False)
    ids = ["a", "b", "c"]
    last = None
    for step in range(5):
        if step == 0:
            gg.prefill(ids, _prompts())
            last = gc.prefill(ids, _prompts()).tolist()
        else:
            gg.decode(ids, last, 16)
            last = gc.decode(ids, last, 16).tolist()
        torch.cuda.synchronize()
        x, y = gg.last_logits[:3].float().cpu(), gc.last_logits.float()
        assert float((x - y).norm() / y.norm()) < 0.05, step
    assert ops.read_status(torch.device("cuda")) == 0


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_chunked_prefill_reads_what_the_whole_one_computed(kv_dtype):
    m = _model(kv_dtype)
    prompt = (_prompts()[2] * 5)[:170]
    g = BatchGenerator(m, use_graph=False)
    g.prefill(["a"], [prompt])
    whole = g.last_logits.float()
    g.prefill(["b"], [prompt[:100]])
    g.prefill(["b"], [prompt[100:]], [100])
    assert float((g.last_logits.float() - whole).norm() / whole.norm()) < 0.05


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("nodes", [4, 60])
def test_tree_rows_equal_their_chains(kv_dtype, nodes):
    """Every node's logits are those of a chain that ends at it."""
    m = _model(kv_dtype)
    prompt = _prompts()[1]
    g = BatchGenerator(m, use_graph=False)
    g.prefill(["t"], [prompt])
    gen = torch.Generator().manual_seed(nodes)
    tree = DraftTree()
    for i in range(nodes):
        tree.add(int(torch.randint(max(0, i - 6), i + 1, (1,), generator=gen)),
                 int(torch.randint(3, 500, (1,), generator=gen)))
    batch = build_tree_batch(m, ["t"], [tree], [len(prompt)])
    hidden = m.embed_tokens(torch.tensor([9] + tree.tokens, dtype=torch.int32).cuda())
    m.forward(batch, hidden)
    logits = m.head(hidden).float()
    for node in (0, 1, nodes // 2, nodes):
        path, at = [], node
        while at:
            path.append(tree.tokens[at - 1])
            at = tree.parents[at - 1]
        sid = f"c{node}"
        g.prefill([sid], [prompt + [9] + path[::-1]])
        want = g.last_logits.float()[0]
        assert float((logits[node] - want).norm() / want.norm()) < 0.05, node
    assert ops.read_status(torch.device("cuda")) == 0


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("draft", ["ngram", "self", "other"])
def test_tree_decoding_matches_greedy(kv_dtype, draft):
    m = _model(kv_dtype)
    want = BatchGenerator(m).generate(_prompts(), 24)
    dm = None if draft == "ngram" else _model(seed=5 if draft == "self" else 6)
    dec = TreeSpecDecoder(m, draft=dm, k=4, branch=3, max_nodes=20)
    lps = []
    got = dec.generate(_prompts(), 24, logprobs=lps)
    torch.cuda.synchronize()
    assert ops.read_status(torch.device("cuda")) == 0
    # Different kernels and batch sizes: near-tied picks may differ.
    assert sum(_agree(a, b) for a, b in zip(got, want)) >= 0.8 * 72, (got, want)
    assert [len(x) for x in lps] == [23] * 3
    assert m.kv.allocator.num_free == m.kv.num_blocks
    if draft == "self":
        assert dec.stats.accepted / dec.stats.rounds > 2


def test_chain_speculation_on_the_8_bit_cache():
    """The chain verify paths (captured graph, ragged prefill) on fp8."""
    m = _model("fp8")
    want = BatchGenerator(m).generate(_prompts(), 24)
    got = SpecDecoder(m, draft=_model(seed=5), k=4).generate(_prompts(), 24)
    assert sum(_agree(a, b) for a, b in zip(got, want)) >= 0.7 * 72


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("spec", [None, "tree"])
def test_engine_logprobs(kv_dtype, spec):
    """Each token's logprob and alternatives as the engine reports them."""
    e = LLMEngine(_model(kv_dtype, name="tiny-llama"), max_model_len=512, spec=spec)
    t = GenerationTask("a", "", max_tokens=12, prompt_ids=_prompts()[0])
    t.logprobs = 5
    e.submit(t)
    got = []
    for _ in range(60):
        out = e.step()
        got += [c for _, c in out if not c.is_final]
        if any(c.is_final for _, c in out):
            break
    # The same positions by one forward over prompt + output on the CPU.
    cpu = _model(kv_dtype, name="tiny-llama", device="cpu")
    g = BatchGenerator(cpu, use_graph=False)
    toks = [c.token_id for c in got]
    assert len(toks) >= 1
    for i, c in enumerate(got):
        g.prefill([f"s{i}"], [_prompts()[0] + toks[:i]])
        lp, _, ids, top = ref.token_logprobs(g.last_logits, torch.tensor([toks[i]]), 5)
        assert abs(c.logprobs.logprob - float(lp[0])) < 0.1
        assert len(c.logprobs.top_logprobs) == 5
        assert c.logprobs.top_logprobs[0].logprob >= c.logprobs.top_logprobs[4].logprob
        assert abs(c.logprobs.top_logprobs[0].logprob - float(top[0, 0])) < 0.1


def test_more_sequences_than_one_attention_call_takes():
    """Decoding and chain verification of thousands of rows on the 8-bit cache."""
    g = torch.Generator().manual_seed(8)
    few = torch.randint(3, 500, (60, 5), generator=g).tolist()
    prompts = [few[i % 60] for i in range(2100)]
    m = LlamaModel(get_config("tiny-llama"), "cuda").init_random(seed=5, gen_device="cpu")
    m.allocate_kv(2100, kv_dtype="fp8")
    want = BatchGenerator(m).generate(few, 6)
    got = BatchGenerator(m).generate(prompts, 6)
    same = sum(_agree(a, want[i % 60]) for i, a in enumerate(got))
    assert same >= 0.8 * 6 * 2100
    # 600 sequences of 5 rows each in a captured verification.
    draft = LlamaModel(get_config("tiny-llama"), "cuda").init_random(seed=5, gen_device="cpu")
    draft.allocate_kv(1200)
    got = SpecDecoder(m, draft=draft, k=4).generate(few * 10, 6)
    assert sum(_agree(a, want[i % 60]) for i, a in enumerate(got)) >= 0.7 * 6 * 600
    assert ops.read_status(torch.device("cuda")) == 0
