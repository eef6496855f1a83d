"""Plain-PyTorch fp32 restatement of every device op.

These are the CPU oracle for the kernel tests and the compute path of the CPU
engine (the BASELINE CPU config: Llama-3.2-1B shape, 2-stage loopback
pipeline).  They follow the reference's math:

* INT4 dequant ``(q - 8) * scale``: crates/cascadia-int4-gemm/src/kernel.rs:46-70
* RMSNorm: crates/cascadia-int4-gemm/src/shell.rs:371-394
* RoPE / llama3 scaling: crates/cascadia-engine-openvino/src/rotary.rs:111-185
* sampling: crates/cascadia-engine-sparse-moe/src/sampling.rs:52-187
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence

import torch

from ..quant import Int4Weight


def dequant(w: Int4Weight) -> torch.Tensor:
    """bf16-rounded dequantised weight [N, K] (what the GPU kernel feeds the MMA)."""
    return w.dequant_bf16()


def linear(x: torch.Tensor, w: Int4Weight) -> torch.Tensor:
    """x[M, K] @ dequant(W)^T in fp32; returns fp32."""
    return x.float() @ w.dequant_bf16().float().t()


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    inv = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return xf * inv * w.float()


def silu_mul(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    g = g.float()
    return g / (1.0 + torch.exp(-g)) * u.float()


def apply_rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, rot: int,
               interleaved: bool = False) -> torch.Tensor:
    """x: [T, H, D] float; rotate the first `rot` dims of each head."""
    half = rot // 2
    cs = cos_sin[positions.long()]  # [T, rot]
    cos = cs[:, :half].unsqueeze(1)
    sin = cs[:, half:].unsqueeze(1)
    out = x.clone()
    if interleaved:
        x0 = x[..., 0:rot:2]
        x1 = x[..., 1:rot:2]
        out[..., 0:rot:2] = x0 * cos - x1 * sin
        out[..., 1:rot:2] = x1 * cos + x0 * sin
    else:
        x0 = x[..., :half]
        x1 = x[..., half:rot]
        out[..., :half] = x0 * cos - x1 * sin
        out[..., half:rot] = x1 * cos + x0 * sin
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_pos: torch.Tensor,
              scale: float, window: int = 0, sinks: int = 0) -> torch.Tensor:
    """Causal GQA attention for one sequence.

    q: [Tq, Hq, D], k/v: [Tk, Hkv, D] (positions 0..Tk-1), q_pos: [Tq].
    window > 0: a query at q sees keys q - window < k <= q and k < sinks.
    """
    tq, hq, d = q.shape
    tk, hkv, _ = k.shape
    g = hq // hkv
    kf = k.float().repeat_interleave(g, dim=1)  # [Tk, Hq, D]
    vf = v.float().repeat_interleave(g, dim=1)
    s = torch.einsum("qhd,khd->hqk", q.float(), kf) * scale
    kpos = torch.arange(tk)
    mask = kpos[None, :] > q_pos.long()[:, None]  # [Tq, Tk]
    if window > 0:
        far = kpos[None, :] <= q_pos.long()[:, None] - window
        mask = mask | (far & (kpos[None, :] >= sinks))
    s = s.masked_fill(mask[None], float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("hqk,khd->qhd", p, vf)


# ----------------------------------------------------------------- 8-bit cache

E4M3_MAX = 448.0
KV_SCALE_MIN = 2.0 ** -100


def quantise_rows(y: torch.Tensor):
    """e4m3 codes and fp32 scales of rows [..., D]: s = max(max |y| / 448,
    2^-100), code = e4m3(y / s) (nearest even, saturating).  A row with a NaN
    or an infinity gets s = NaN and zero codes."""
    y = y.float()
    peak = y.abs().amax(-1)
    fine = torch.isfinite(peak)
    s = torch.where(fine, (peak * (1.0 / E4M3_MAX)).clamp_min(KV_SCALE_MIN),
                    torch.full_like(peak, float("nan")))
    c = (y * (1.0 / s).unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX)
    c = torch.where(fine.unsqueeze(-1), c, torch.zeros_like(c))
    return c.to(torch.float8_e4m3fn), s


def dequantise_rows(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return codes.float() * scales.unsqueeze(-1)


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                   masks: Optional[Sequence[int]] = None) -> torch.Tensor:
    """Attention of one sequence's newest tokens: q [n, Hq, D], k / v
    [len, Hkv, D] whose last n rows are the nodes' own.  Row i sees every key
    before them and node j iff bit j of masks[i] (no masks: j <= i); a row
    that sees nothing gives zeros."""
    n, hq, d = q.shape
    tk, hkv, _ = k.shape
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    ctx = tk - n
    j = torch.arange(tk, device=q.device) - ctx  # node number of each key
    if masks is None:
        sees = j[None, :] <= torch.arange(n, device=q.device)[:, None]
    else:
        m = torch.as_tensor(masks, dtype=torch.int64, device=q.device)
        sees = (j < 0)[None, :] | ((j < 64)[None, :] &
                                   (m[:, None] >> j.clamp(0, 63)[None, :] & 1).bool())
    g = hq // hkv
    kf, vf = (x.to(dt).repeat_interleave(g, dim=1) for x in (k, v))
    s = torch.einsum("qhd,khd->hqk", q.to(dt), kf) * scale
    s = s.masked_fill(~sees[None], float("-inf"))
    top = s.amax(-1, keepdim=True) if tk else s.new_zeros(hq, n, 1)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    # A hidden key's value must not meet its weight of zero: it may be a NaN.
    o = torch.zeros(n, hq, d, dtype=dt, device=q.device)
    for i in range(n):
        o[i] = torch.einsum("hk,khd->hd", p[:, i, sees[i]], vf[sees[i]])
    total = p.sum(-1).t().unsqueeze(-1)
    return torch.where(total == 0, torch.zeros_like(o), o / total)


def top_ids(x: torch.Tensor, k: int) -> torch.Tensor:
    """Indices [R, k] of the largest values of rows, larger first, then lower
    index; a NaN comes before every number."""
    k = min(k, x.shape[1])
    if k == 0:
        return torch.zeros(x.shape[0], 0, dtype=torch.long, device=x.device)
    least = x.topk(k, dim=-1).values[:, -1:]
    out = torch.empty(x.shape[0], k, dtype=torch.long, device=x.device)
    for row, reach, ids in zip(x, x >= least, out):
        # (a NaN reaches nothing, and nothing reaches a NaN: such rows are sorted whole)
        at = reach.nonzero()[:, 0]
        if len(at) < k or bool(row.amax().isnan()):
            at = torch.arange(len(row), device=x.device)
        ids.copy_(at[torch.sort(row[at], descending=True, stable=True).indices[:k]])
    return out


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0):
    """(logprob, entropy, ids, top) of logit rows; see ops.token_logprobs."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    m = x.amax(-1, keepdim=True)
    bad = ~(m < float("inf"))
    empty = m == float("-inf")
    sh = x - torch.where(empty, torch.zeros_like(m), m)
    e = torch.exp(sh)
    S = e.sum(-1, keepdim=True)
    log_s = S.log()

    def lp_of(at):
        lp = sh.gather(1, at) - log_s
        lp = torch.where(empty, torch.full_like(lp, float("-inf")), lp)
        return torch.where(bad, torch.full_like(lp, float("nan")), lp)

    # (0 log 0 = 0: a value of -inf takes no part in the sum of e sh)
    spread = (e * sh.clamp_min(torch.finfo(x.dtype).min)).sum(-1) / S[:, 0]
    ent = log_s[:, 0] - spread
    ent = torch.where(bad[:, 0], torch.full_like(ent, float("nan")),
                      torch.where(empty[:, 0], torch.zeros_like(ent), ent))
    ids = top_ids(x, top_k)
    t = tokens.long()
    known = (t >= 0) & (t < x.shape[1])
    got = lp_of(t.clamp(0, x.shape[1] - 1).unsqueeze(1))[:, 0]
    got = torch.where(known, got, torch.full_like(got, float("nan")))
    return got, ent, ids.to(torch.int32), lp_of(ids)


def argmax(logits: torch.Tensor) -> torch.Tensor:
    """Row argmax, lowest index on ties (the reference's strict `>` scan)."""
    return torch.argmax(logits.float(), dim=-1).to(torch.int32)


# ----------------------------------------------------------------- sampling

_MASK64 = (1 << 64) - 1


def xorshift64_next(state: List[int]) -> int:
    """xorshift64* step (crates/cascadia-engine-sparse-moe/src/sampling.rs:191)."""
    x = state[0]
    x ^= (x << 13) & _MASK64
    x ^= x >> 7
    x ^= (x << 17) & _MASK64
    state[0] = x
    return (x * 0x2545F4914F6CDD1D) & _MASK64


def next_uniform(state: List[int]) -> float:
    r = xorshift64_next(state)
    return float(r >> 40) / float(1 << 24)


def init_rng(seed: Optional[int]) -> List[int]:
    if seed is not None:
        return [max(int(seed) & _MASK64, 1)]
    import time

    t = time.time_ns()
    return [max(((t % 10**9) | ((t // 10**9) << 32)) & _MASK64, 1)]


def apply_penalties(work: torch.Tensor, history: Sequence[int], rep_pen: float, rep_window: int,
                    freq_pen: float, pres_pen: float) -> torch.Tensor:
    work = work.clone()
    if abs(rep_pen - 1.0) > 1.1920929e-07:
        start = 0 if rep_window == 0 else max(0, len(history) - rep_window)
        for tok in history[start:]:
            if 0 <= tok < work.numel():
                l = float(work[tok])
                work[tok] = l / rep_pen if l > 0 else l * rep_pen
    if freq_pen != 0.0 or pres_pen != 0.0:
        seen = set()
        for tok in history:
            if 0 <= tok < work.numel():
                work[tok] -= freq_pen
                if tok not in seen:
                    seen.add(tok)
                    work[tok] -= pres_pen
    return work


def sample(logits: torch.Tensor, history: Sequence[int], temperature: float, top_p: float,
           top_k: int, freq_pen: float, pres_pen: float, rep_pen: float, rep_window: int,
           rng_state: List[int]) -> int:
    """Sample one token with the reference's exact semantics and PRNG."""
    work = apply_penalties(logits.float().flatten(), history, rep_pen, rep_window, freq_pen,
                           pres_pen)
    if temperature <= 0.0:
        return int(torch.argmax(work))
    work = work / temperature
    work = torch.softmax(work, dim=0)
    n = work.numel()
    if 0 < top_k < n:
        idx = torch.argsort(work, descending=True, stable=True)
        keep = torch.zeros(n, dtype=torch.bool)
        keep[idx[:top_k]] = True
        work = torch.where(keep, work, torch.zeros_like(work))
        s = work.sum()
        if s > 0:
            work = work / s
    if 0.0 < top_p < 1.0:
        idx = torch.argsort(work, descending=True, stable=True)
        cum = torch.cumsum(work[idx], 0)
        cut = int(torch.searchsorted(cum, torch.tensor(top_p, dtype=cum.dtype)).item())
        keep = torch.zeros(n, dtype=torch.bool)
        keep[idx[: min(n, cut + 1)]] = True
        work = torch.where(keep, work, torch.zeros_like(work))
        s = work.sum()
        if s > 0:
            work = work / s
    u = next_uniform(rng_state)
    cum = torch.cumsum(work, 0)
    hit = torch.nonzero(cum >= u)
    return int(hit[0]) if hit.numel() else n - 1


def spec_verify(target: Sequence[int], draft: Sequence[int]):
    """Greedy acceptance: longest matching prefix plus the correction token."""
    acc = 0
    while acc < len(draft) and draft[acc] == target[acc]:
        acc += 1
    return list(draft[:acc]) + [int(target[acc])]
