"""Speculative decoding with drafted trees on the bf16 or the 8-bit KV cache.

    python bench/bench_tree_spec.py [--model llama-3.1-8b] [--batch 8] [--prompt-len 2048]
                                    [--new 128] [--kv-dtype fp8] [--draft ngram|exit|none]
                                    [--follow-text 0]

Every prompt repeats a short passage.  Weights are random (INT4, seeded), but for the
embedding's size and the LM head's rows of the passages' tokens, which are set so that the
model goes on with the passage: n-gram drafts are right then, and so are those of ``exit``
(the target's own first layers), as the best case of speculation.  ``--follow-text 0``
leaves the weights as they are: nothing predicts what the model emits, n-gram drafts find
nothing to propose and the others are not accepted, the cost of speculation where it does
not help.  Prints one JSON line: tokens per second of plain decoding and of tree decoding,
nodes drafted and tokens emitted per round, and the mean log-probability of the emitted
tokens.
"""
import argparse
import json
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from cascadia_b200 import ops  # noqa: E402
from cascadia_b200.models.config import get_config  # noqa: E402
from cascadia_b200.models.llama import Int4Weight, LlamaModel, QLinear  # noqa: E402
from cascadia_b200.runtime.generator import BatchGenerator  # noqa: E402
from cascadia_b200.runtime.spec import TreeSpecDecoder  # noqa: E402


def follow_text(m, passages):
    """Make the token after each of a passage's the model's own choice: the residual is
    mostly the embedding, and the head's row of the next token points along it."""
    head = torch.randn(m.cfg.vocab_size, m.cfg.hidden_size, device=m.device,
                       generator=torch.Generator(m.device).manual_seed(2)) * 0.02
    for text in passages:
        at = torch.tensor(text, device=m.device)
        head[at.roll(-1)] = m.embed[at].float() / m.embed.float().std() * 0.1
    m.embed.mul_(100.0 / m.embed.float().std())
    m.lm_head = QLinear(Int4Weight.quantize(head, m.cfg.group_size), m.device)


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--model", default="llama-3.1-8b")
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--prompt-len", type=int, default=2048)
    p.add_argument("--new", type=int, default=128)
    p.add_argument("--kv-dtype", default="fp8", choices=["bf16", "fp8"])
    p.add_argument("--draft", default="ngram", choices=["ngram", "exit", "none"])
    p.add_argument("--exit-layers", type=int, default=4)
    p.add_argument("--k", type=int, default=6, help="depth of a tree")
    p.add_argument("--branch", type=int, default=3)
    p.add_argument("--nodes", type=int, default=31)
    p.add_argument("--follow-text", type=int, default=1)
    a = p.parse_args()
    dev = torch.device("cuda")
    m = LlamaModel(get_config(a.model), dev).init_random(seed=0)
    width = -(-(a.prompt_len + a.new + 80) // 16)
    m.allocate_kv(a.batch * width + 64, kv_dtype=a.kv_dtype)
    g = torch.Generator().manual_seed(1)
    passages = [torch.randint(3, m.cfg.vocab_size, (61,), generator=g).tolist()
                for _ in range(a.batch)]
    prompts = [(text * (a.prompt_len // 61 + 1))[:a.prompt_len] for text in passages]
    if a.follow_text:
        follow_text(m, passages)
    out = {"model": a.model, "batch": a.batch, "prompt_len": a.prompt_len, "new": a.new,
           "follow_text": a.follow_text, "kv_dtype": a.kv_dtype, "kv_bytes_per_token": m.kv_bytes_per_block(a.kv_dtype) // 16}

    def timed(fn):
        fn(8)  # captures, caches
        torch.cuda.synchronize()
        t = [time.perf_counter()]
        fn(1)  # prefill alone
        torch.cuda.synchronize()
        t.append(time.perf_counter())
        fn(a.new)
        torch.cuda.synchronize()
        t.append(time.perf_counter())
        return a.batch * (a.new - 1) / (t[2] - t[1] - (t[1] - t[0]))

    plain = BatchGenerator(m)
    out["plain_tok_s"] = round(timed(lambda n: plain.generate(prompts, n, width)), 1)
    if a.draft != "none":
        draft = None
        if a.draft == "exit":
            draft = m.early_exit(a.exit_layers)
            draft.allocate_kv(a.batch * width + 64)
        lps = []

        def run(n):
            lps.clear()
            run.dec = TreeSpecDecoder(m, draft=draft, k=a.k, branch=a.branch, max_nodes=a.nodes)
            run.dec.generate(prompts, n, logprobs=lps)

        out["tree_tok_s"] = round(timed(run), 1)
        st = run.dec.stats
        out["rounds"] = st.rounds
        out["drafted_per_round"] = round(st.drafted / max(1, st.rounds) / a.batch, 2)
        out["emitted_per_round"] = round(st.emitted / max(1, st.rounds) / a.batch, 2)
        out["verify_ms"] = round(1e3 * st.verify_s / max(1, st.rounds), 3)
        flat = [x for row in lps for x in row]
        out["mean_logprob"] = round(sum(flat) / max(1, len(flat)), 3)
    assert ops.read_status(dev) == 0
    print(json.dumps(out))


if __name__ == "__main__":
    main()
