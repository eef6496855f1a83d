"""Cases that time the 8-bit KV cache, tree attention and log-probability operators.

Four operators that one speculative decoding step uses together:

* ``write``: RoPE of a fused q/k/v row, K and V quantised to e4m3 into the paged cache;
* ``read``: blocks of the 8-bit cache back to bf16 (what the prefill attention reads);
* ``attn``: attention of the newest tokens of every sequence (one token, a chain or a
  tree of drafted tokens) over the paged bf16 or 8-bit cache;
* ``logp``: log-probability of a given token, entropy and top alternatives of logit rows.

``run`` computes them in plain torch operations when ``own`` is false and through
``cascadia_b200.ops`` when it is true.
"""
import math

import torch

own = False

BLOCK = 16
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -100


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One decode step of one sequence: a single row per layer; latency counts.
        _write("write_decode_1", 1, 32, 8, 128, 128, False, 0),
        # A decode bucket of 64 rows, a few of them padding, partial interleaved rotation.
        _write("write_decode_61_of_64", 64, 32, 8, 64, 32, True, 3),
        # A full prefill budget of packed prompts.
        _write("write_prefill_8192", 8192, 32, 8, 128, 128, False, 0),
        # The cached prefix of one short prompt (79 tokens: the last block is ragged).
        _read("read_prefix_5_blocks", 5, 8, 128),
        # Chunked prefill of long prompts: 64k context tokens read back for one layer.
        _read("read_context_4096_blocks", 4096, 8, 128),
        # Plain decoding of one sequence in mid generation, one token.
        _attn("attn_decode_1", "fp8", 1, 32, 8, 128, 1151, 1151, 1, 1, False),
        # Plain decoding of a batch whose contexts differ widely.
        _attn("attn_decode_64_ragged", "fp8", 64, 32, 8, 128, 517, 8191, 1, 1, False),
        # Draft trees of different sizes on the bf16 cache, head dim 64.
        _attn("attn_tree_bf16_8x24", "bf16", 8, 32, 8, 64, 1001, 4003, 7, 24, True),
        # The widest trees on the 8-bit cache.
        _attn("attn_tree_fp8_8x64", "fp8", 8, 32, 8, 128, 8129, 8192, 64, 64, True),
        # The sampled token of one sequence, five alternatives.
        _logp("logp_1_top5", 1, 128256, "bf16", 5, 0),
        # A decode batch, most alternatives a client may ask for; a grammar masks part of it.
        _logp("logp_64_top20_masked", 64, 151936, "bf16", 20, 1),
        # Scoring the tokens of a prompt.
        _logp("logp_prompt_2047", 2047, 128256, "bf16", 1, 0),
    ]


def _write(name, tokens, hq, hkv, d, rot, interleaved, padded):
    return dict(name=name, op="write", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot,
                interleaved=interleaved, padded=padded)


def _read(name, blocks, hkv, d):
    return dict(name=name, op="read", blocks=blocks, hkv=hkv, d=d)


def _attn(name, cache, batch, hq, hkv, d, len_lo, len_hi, nodes_lo, nodes_hi, tree):
    return dict(name=name, op="attn", cache=cache, batch=batch, hq=hq, hkv=hkv, d=d,
                len_lo=len_lo, len_hi=len_hi, nodes_lo=nodes_lo, nodes_hi=nodes_hi, tree=tree)


def _logp(name, rows, vocab, dtype, top_k, masked):
    return dict(name=name, op="logp", rows=rows, vocab=vocab, dtype=dtype, top_k=top_k,
                masked=masked)


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, kv heads, head dim): whole models and their tensor-parallel shards.
HEADS = [(32, 8, 128), (32, 8, 64), (32, 4, 128), (16, 4, 128), (8, 2, 128), (4, 1, 128),
         (16, 4, 64)]


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    op = rng.choice(["write", "read", "attn", "attn", "attn", "logp", "logp"])
    hq, hkv, d = rng.choice(HEADS)
    if op == "write":
        tokens = _log_int(rng, 1, 8192)
        rot = rng.choice([d, d, 32, 16])
        case = _write("", tokens, hq, hkv, d, rot, rng.random() < 0.4,
                      rng.randrange(0, 1 + tokens // 8))
    elif op == "read":
        case = _read("", _log_int(rng, 1, 4096), hkv, d)
    elif op == "attn":
        cache = rng.choice(["fp8", "fp8", "bf16"])
        kind = rng.choice(["decode", "chain", "tree", "tree"])
        batch = _log_int(rng, 1, 64)
        nodes_hi = 1 if kind == "decode" else _log_int(rng, 2, 64)
        nodes_lo = max(1, nodes_hi - rng.randrange(0, 1 + nodes_hi // 2))
        # Within the largest listed case: keys x bytes, and keys x query rows.
        row = 2 * hkv * (2 * d if cache == "bf16" else d + 4)
        most = min(131072, 400_000_000 // (row * batch),
                   60_000_000_000 // (4 * d * hq * nodes_hi * batch),
                   130_000_000 // (hq * nodes_hi * batch))
        len_hi = _log_int(rng, nodes_hi, max(nodes_hi, most))
        len_lo = rng.randrange(min(len_hi, max(nodes_hi, len_hi // 8)), len_hi + 1)
        case = _attn("", cache, batch, hq, hkv, d, len_lo, len_hi, nodes_lo, nodes_hi,
                     kind == "tree")
    else:
        vocab = rng.choice([128256, 151936, 32000, 50257, 128255])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        rows = _log_int(rng, 1, min(2047, 250_000_000 // (vocab * (1 if dtype == "bf16" else 2))))
        case = _logp("", rows, vocab, dtype, rng.choice([0, 1, 2, 5, 8, 20]),
                     rng.choice([0, 0, 1]))
    del case["name"]
    return case


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo, evenly."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def work(case):
    """Bytes and operations that one pass cannot do without."""
    op = case["op"]
    if op == "write":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        return {"bytes": t * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + case["rot"] * 4 + 8)
                + (t - case["padded"]) * 2 * hkv * (d + 4),
                "flops": t * ((hq + hkv) * case["rot"] * 3 + 2 * hkv * d * 3)}
    if op == "read":
        n = case["blocks"] * case["hkv"] * BLOCK
        return {"bytes": 2 * n * (case["d"] + 4) + 2 * n * case["d"] * 2 + case["blocks"] * 4,
                "flops": 2 * n * case["d"]}
    if op == "attn":
        b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
        lens = _spread(case["len_lo"], case["len_hi"], b)
        nodes = _spread(case["nodes_lo"], case["nodes_hi"], b)
        row = hkv * 2 * (d + 4 if case["cache"] == "fp8" else 2 * d)
        return {"bytes": sum(lens) * row + sum(nodes) * hq * d * 4
                + sum(-(-n // BLOCK) for n in lens) * 4,
                "flops": 4 * d * hq * sum(n * (l - n + (n + 1) // 2) for n, l in zip(nodes, lens))}
    r, v, k = case["rows"], case["vocab"], case["top_k"]
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": r * v * size + r * 4 + r * (8 + 8 * k), "flops": r * v * 6}


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _quantised(x):
    """Codes and scales of random rows, a cache as earlier steps left it."""
    scale = (x.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
    codes = (x / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes, scale


def _cache(g, blocks, hkv, d, fp8):
    """K and V pools [1, blocks, hkv, 16, d]; token rows of different magnitude."""
    made = []
    for _ in range(2):
        x = _randn(g, 1, blocks, hkv, BLOCK, d)
        x *= torch.exp(0.3 * _randn(g, 1, blocks, hkv, BLOCK, 1))
        made.append(_quantised(x) if fp8 else (x.to(torch.bfloat16), None))
    return made[0][0], made[1][0], made[0][1], made[1][1]


def _tree_mask(parents):
    masks = []
    for i, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | (1 << i))
    return [m - (1 << 64) if m >= 1 << 63 else m for m in masks]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case)
    if op == "write":
        t, hq, hkv, d, rot = (case[k] for k in ("tokens", "hq", "hkv", "d", "rot"))
        s["qkv"] = (_randn(g, t, (hq + 2 * hkv) * d) * 1.5).to(torch.bfloat16)
        max_pos = 16384
        inv = 500000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / rot)
        ang = torch.outer(torch.arange(max_pos, device="cuda", dtype=torch.float32), inv)
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=1).contiguous()
        s["positions"] = torch.randint(0, max_pos, (t,), generator=g, device="cuda",
                                       dtype=torch.int32)
        blocks = -(-t // BLOCK) + 1
        slots = torch.randperm(blocks * BLOCK, generator=g, device="cuda")[:t].to(torch.int32)
        if case["padded"]:
            slots[t - case["padded"]:] = -1
        s["slots"] = slots
        kv = torch.zeros(2, 2, blocks, hkv, BLOCK, d, dtype=torch.uint8, device="cuda")
        s["k"], s["v"] = kv.view(torch.float8_e4m3fn).unbind(0)
        s["ks"], s["vs"] = torch.ones(2, 2, blocks, hkv, BLOCK, device="cuda").unbind(0)
        s["q_out"] = torch.empty(t, hq * d, dtype=torch.bfloat16, device="cuda")
        s["layer"] = 1
    elif op == "read":
        n, hkv, d = case["blocks"], case["hkv"], case["d"]
        pool = n + 3
        s["k"], s["v"], s["ks"], s["vs"] = _cache(g, pool, hkv, d, True)
        s["table"] = torch.randperm(pool, generator=g, device="cuda")[:n].to(torch.int32)
        s["k_out"] = torch.empty(n, hkv, BLOCK, d, dtype=torch.bfloat16, device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
        s["layer"] = 0
    elif op == "attn":
        b, hq, hkv, d = (case[k] for k in ("batch", "hq", "hkv", "d"))
        order = torch.randperm(b, generator=g, device="cuda").tolist()
        lens = _spread(case["len_lo"], case["len_hi"], b)
        nodes = _spread(case["nodes_lo"], case["nodes_hi"], b)
        lens, nodes = [lens[i] for i in order], [nodes[i] for i in order]
        need = [-(-n // BLOCK) for n in lens]
        s["k"], s["v"], s["ks"], s["vs"] = _cache(g, sum(need) + 1, hkv, d,
                                                  case["cache"] == "fp8")
        perm = (torch.randperm(sum(need), generator=g, device="cuda") + 1).to(torch.int32)
        s["table"] = torch.zeros(b, max(need), dtype=torch.int32, device="cuda")
        for i, part in enumerate(perm.split(need)):
            s["table"][i, :need[i]] = part
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        starts = [0]
        for n in nodes:
            starts.append(starts[-1] + n)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["masks"] = None
        if case["tree"]:
            pick = torch.randint(1, 7, (starts[-1],), generator=g, device="cuda").tolist()
            masks = []
            for a, n in zip(starts, nodes):
                masks += _tree_mask([max(-1 if i == 0 else 0, i - pick[a + i])
                                     for i in range(n)])
            s["masks"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
        s["q"] = (_randn(g, starts[-1], hq * d) * 2.0).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(d)
        s["layer"] = 0
    else:
        r, v = case["rows"], case["vocab"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        x = _randn(g, r, v) * (1.0 + 2.0 * torch.rand(r, 1, generator=g, device="cuda"))
        if case["masked"]:
            x.masked_fill_(torch.rand(r, v, generator=g, device="cuda") < 0.4, -math.inf)
        s["logits"] = x.to(dtype)
        # The token a sampler took: among the likely ones, as often as not the best.
        likely = x.topk(4, dim=-1).indices
        s["tokens"] = likely.gather(1, torch.randint(0, 4, (r, 1), generator=g, device="cuda"))[
            :, 0].to(torch.int32)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn,
            "logp": _plain_logp}[s["op"]](s)


def _run_own(s):
    from cascadia_b200 import ops

    op = s["op"]
    if op == "write":
        ops.rope_kv_write_fp8(s["qkv"], s["positions"], s["cos_sin"], s["slots"], s["k"], s["v"],
                              s["ks"], s["vs"], s["layer"], s["hq"], s["hkv"], s["d"], s["rot"],
                              interleaved=s["interleaved"], q_out=s["q_out"])
        return _written(s)
    if op == "read":
        k, v = ops.kv_read_fp8(s["k"], s["v"], s["ks"], s["vs"], s["table"], s["layer"],
                               k_out=s["k_out"], v_out=s["v_out"])
        return {"k": k, "v": v}
    if op == "attn":
        return ops.attn_tree(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"], s["out"],
                             s["layer"], s["scale"], masks=s["masks"], k_scale=s["ks"],
                             v_scale=s["vs"], max_nodes=s["nodes_hi"])
    logprob, entropy, ids, top = ops.token_logprobs(s["logits"], s["tokens"], s["top_k"])
    return {"logprob": logprob, "entropy": entropy, "ids": ids, "top": top}


def _written(s):
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


def _rotate(x, cos, sin, rot, interleaved):
    """x [T, H, D] fp32."""
    if interleaved:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    turned = torch.stack([y0, y1], dim=-1).flatten(-2) if interleaved else torch.cat([y0, y1], -1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _plain_write(s):
    t, hq, hkv, d, rot = (s[k] for k in ("tokens", "hq", "hkv", "d", "rot"))
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    cs = s["cos_sin"][s["positions"].long()]
    cos, sin = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    s["q_out"].copy_(_rotate(x[:, :hq], cos, sin, rot, s["interleaved"]).reshape(t, hq * d))
    y = torch.cat([_rotate(x[:, hq:hq + hkv], cos, sin, rot, s["interleaved"]),
                   x[:, hq + hkv:]], dim=1)
    peak = y.abs().amax(-1)
    fine = torch.isfinite(peak)
    scale = torch.where(fine, (peak * (1.0 / E4M3_MAX)).clamp_min(SCALE_MIN), math.nan)
    code = (y * (1.0 / scale)[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    code = torch.where(fine[..., None], code, 0.0).to(torch.float8_e4m3fn).view(torch.uint8)
    kept = t - s["padded"]  # the padded rows come last
    slot = s["slots"][:kept].long()
    at = (s["layer"], slot // BLOCK, slice(None), slot % BLOCK)
    s["k"].view(torch.uint8)[at] = code[:kept, :hkv]
    s["v"].view(torch.uint8)[at] = code[:kept, hkv:]
    s["ks"][at] = scale[:kept, :hkv]
    s["vs"][at] = scale[:kept, hkv:]
    return _written(s)


def _plain_read(s):
    at = s["table"].long()
    for name in ("k", "v"):
        code = s[name][s["layer"]].view(torch.uint8)[at].view(torch.float8_e4m3fn)
        s[name + "_out"].copy_(code.float() * s[name + "s"][s["layer"]][at][..., None])
    return {"k": s["k_out"], "v": s["v_out"]}


def _keys(s, name):
    """[B, hkv, W * 16, d] fp32 values of every table entry."""
    pool = s[name][s["layer"]]
    at = s["table"].long()
    if s["cache"] == "fp8":
        x = pool.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        x = x * s[name + "s"][s["layer"]][at][..., None]
    else:
        x = pool[at].float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attn(s):
    b, hq, hkv, d, n = (s[k] for k in ("batch", "hq", "hkv", "d", "nodes_hi"))
    lens, starts = s["lens"].long(), s["starts"].long()
    node = torch.arange(n, device="cuda")
    count = starts[1:] - starts[:-1]
    real = node < count[:, None]                                  # [B, n]
    row = torch.where(real, starts[:-1, None] + node, 0)
    q = s["q"].float().view(-1, hkv, hq // hkv, d)[row]           # [B, n, hkv, G, d]
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)                    # [B, hkv, G * n, d]
    k, v = _keys(s, "k"), _keys(s, "v")
    key = torch.arange(k.shape[2], device="cuda")
    j = key - (lens - count)[:, None]                             # node number of each key
    if s["masks"] is None:
        sees = j[:, None, :] <= node[:, None]
    else:
        bits = s["masks"][row][:, :, None] >> j.clamp(0, 63)[:, None, :]
        sees = (bits & 1).bool() | (j < 0)[:, None, :]
    sees = sees & (key < lens[:, None])[:, None, :]               # [B, n, keys]
    score = (q @ k.transpose(2, 3)).view(b, hkv, hq // hkv, n, -1) * s["scale"]
    score = score.masked_fill(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, 1.0)).flatten(2, 3)
    o = (p @ v).view(b, hkv, hq // hkv, n, d).permute(0, 3, 1, 2, 4)
    s["out"].copy_(o[real].reshape(-1, hq * d))
    return s["out"]


def _plain_logp(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    shift = x - top
    p = torch.exp(shift)
    total = p.sum(-1, keepdim=True)
    logp = shift - total.log()
    entropy = -(torch.where(p > 0, p * logp, 0.0) / total).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["top_k"]]
    return {"logprob": logp.gather(1, s["tokens"].long()[:, None])[:, 0], "entropy": entropy,
            "ids": order.to(torch.int32), "top": logp.gather(1, order)}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attn": _exact_attn,
            "logp": _exact_logp}[case["op"]](s)


def _exact_write(s):
    t, hq, hkv, d, rot = (s[k] for k in ("tokens", "hq", "hkv", "d", "rot"))
    x = s["qkv"].double().view(t, hq + 2 * hkv, d)
    cs = s["cos_sin"].double()[s["positions"].long()]
    turn = torch.complex(cs[:, :rot // 2], cs[:, rot // 2:])[:, None]
    y = x.clone()
    a = x[:, :hq + hkv, :rot]
    pairs = a.unflatten(-1, (rot // 2, 2)) if s["interleaved"] else \
        a.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y[:, :hq + hkv, :rot] = (z if s["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    scale = (y.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
    u = y / scale[..., None]
    # e4m3: three bits after the leading one, exponents from -6, ties to even.
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
    code = (torch.round(u / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
    keep = s["slots"] >= 0
    slot = s["slots"][keep].long()
    out = {"q": y[:, :hq].reshape(t, hq * d)}
    for name, lo in (("k", hq), ("v", hq + hkv)):
        pool = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
        scales = torch.ones(s[name + "s"].shape, dtype=torch.float64, device="cuda")
        pool[s["layer"]][slot // BLOCK, :, slot % BLOCK] = code[keep, lo:lo + hkv]
        scales[s["layer"]][slot // BLOCK, :, slot % BLOCK] = scale[keep, lo:lo + hkv]
        out[name], out[name + "s"] = pool, scales
    return out


def _exact_read(s):
    out = {}
    for name in ("k", "v"):
        value = s[name][s["layer"]].float().double() * s[name + "s"][s["layer"]].double()[..., None]
        out[name] = value[s["table"].long()]
    return out


def _exact_attn(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    out = torch.zeros(starts[-1], hq, d, dtype=torch.float64, device="cuda")
    pools = []
    for name in ("k", "v"):
        scales = s[name + "s"]
        pools.append((s[name][s["layer"]], None if scales is None else scales[s["layer"]]))
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        at = s["table"][b, :-(-length // BLOCK)].long()
        kv = []
        for pool, scales in pools:
            x = (pool.view(torch.uint8)[at].view(pool.dtype).float().double() if scales is not None
                 else pool[at].double())
            if scales is not None:
                x = x * scales[at].double()[..., None]
            kv.append(x.permute(0, 2, 1, 3).reshape(-1, hkv, d)[:length])
        seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
        for i in range(n):
            m = (1 << (i + 1)) - 1 if s["masks"] is None else int(s["masks"][starts[b] + i])
            seen[i, length - n:] = torch.tensor([bool(m >> j & 1) for j in range(n)])
        q = s["q"][starts[b]:starts[b + 1]].double().view(n, hkv, hq // hkv, d)
        score = torch.einsum("nhgd,khd->hgnk", q, kv[0]) * s["scale"]
        score.masked_fill_(~seen, -math.inf)
        p = torch.exp(score - torch.logsumexp(score, -1, keepdim=True))
        out[starts[b]:starts[b + 1]] = torch.einsum("hgnk,khd->nhgd", p, kv[1]).reshape(n, hq, d)
    return out.view(starts[-1], hq * d)


def _exact_logp(s):
    got = {"logprob": [], "entropy": [], "ids": None, "top": []}
    for x, token in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double()
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        got["logprob"].append(logp.gather(1, token.long()[:, None])[:, 0])
        got["entropy"].append(torch.special.entr(logp.exp()).sum(-1))
        got["top"].append(logp.topk(s["top_k"], dim=-1).values)
    return {k: None if v is None else torch.cat(v) for k, v in got.items()}
