"""The CPU oracle of token log-probabilities: order of the alternatives, and its cost."""
import math
import time

import pytest
import torch

from cascadia_b200.ops import reference as ref


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("k", [0, 1, 5, 40])
def test_alternatives_are_those_of_a_stable_sort(dtype, k):
    g = torch.Generator().manual_seed(k)
    x = torch.randint(-3, 4, (9, 40), generator=g).to(dtype)  # ties everywhere
    x[1] = -math.inf
    x[2] = 1.0
    x[3, [4, 30]] = math.nan
    x[4, ::3] = -math.inf
    x[4, 1::3] = math.nan
    x[5, 7] = math.inf
    x[6, ::2], x[6, 1::2] = -0.0, 0.0
    x[7, 5:] = -math.inf
    t = torch.randint(0, 40, (9,), generator=g)
    lp, ent, ids, top = ref.token_logprobs(x, t, k)
    wide = x.double()
    order = torch.sort(wide, dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids.long(), order)
    # The rest by the formulas, row by row (fp32 sums of 40 terms: 2^-18).
    for r in range(9):
        row = wide[r]
        if bool(row.isnan().any()) or bool((row == math.inf).any()):
            assert math.isnan(float(lp[r])) and math.isnan(float(ent[r]))
            assert bool(top[r].isnan().all())
            continue
        want = row - torch.logsumexp(row, 0)
        if bool((row == -math.inf).all()):
            want = torch.full_like(row, -math.inf)
        p = want.exp()
        for got, w in [(lp[r], want[t[r]])] + list(zip(top[r], want[order[r]])):
            assert float(got) == float(w) or abs(float(got) - float(w)) < 2.0 ** -18 * (
                1 + abs(float(w)))
        h = -float(torch.where(p > 0, p * want, 0.0).sum())
        assert float(ent[r]) >= 0 and abs(float(ent[r]) - h) < 2.0 ** -18 * (1 + h)


def test_cost_is_that_of_a_pass_not_of_a_sort():
    """Within a few times a log-softmax with its largest values (a stable sort of
    every row takes twenty and more; on a busy machine this one takes seven)."""
    x = torch.randn(4, 128256, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int32)

    def least(f):
        best = math.inf
        for _ in range(9):
            t0 = time.perf_counter()
            f()
            best = min(best, time.perf_counter() - t0)
        return best

    plain = least(lambda: torch.log_softmax(x.float(), -1).topk(5, -1))
    assert least(lambda: ref.token_logprobs(x, t, 5)) < 14 * plain
