"""Token log-probabilities, entropy and top alternatives against 64 bits."""
import pytest
import torch

from cascadia_b200 import ops
from cascadia_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")


def _check(logits, tokens, k, **kw):
    """Whole values equal; log-probabilities within the rounding of fp32:
    2^-23 (|x - m| + |ln S|) for the subtractions, and for S the error of its
    terms (2^-22 each) and of a sum of n terms by 512 threads, (n / 512 + 32)
    2^-24; the entropy has W / S besides: the same relative errors of
    sum p |x - m|."""
    lp, ent, ids, top = (t.cpu() for t in ops.token_logprobs(logits, tokens, k, **kw))
    x = logits.cpu()
    w_lp, w_ent, w_ids, w_top = ref.token_logprobs(x.double(), tokens.cpu(), k)
    assert torch.equal(ids, w_ids)
    n = x.shape[1]
    rel_s = (n / 512 + 32) * 2.0 ** -24 + 2.0 ** -21
    m = x.double().amax(-1)
    ln_s = torch.logsumexp(x.double() - m[:, None], -1).abs()

    def close(got, want, extra):
        fine = want.isfinite()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~fine & ~want.isnan()].double(), want[~fine & ~want.isnan()])
        tol = rel_s + 2.0 ** -22 * extra
        assert bool(((got.double() - want).abs()[fine] <= tol[fine]).all()), float(
            ((got.double() - want).abs() / tol)[fine].max())

    close(lp, w_lp, w_lp.abs() + ln_s)
    close(top, w_top, w_top.abs() + ln_s[:, None])
    p = torch.softmax(x.double(), -1)
    spread = torch.where(p > 0, p * (x.double() - m[:, None]).abs(), 0.0).sum(-1)
    fine = w_ent.isfinite()
    assert torch.equal(ent.isnan(), w_ent.isnan())
    # (a row of -inf has neither spread nor sum: its entropy is 0)
    tol = 2 * rel_s * (1 + spread.nan_to_num(0.0) + ln_s.nan_to_num(0.0))
    assert bool(((ent.double() - w_ent).abs()[fine] <= tol[fine]).all())
    return lp, ent, ids, top


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 7), (3, 8), (5, 33), (1, 4095), (4, 4097),
                                        (2, 50257), (1, 128256), (70, 9001), (601, 1500)])
@pytest.mark.parametrize("k", [0, 1, 5, 20, 32])
def test_random_rows(dtype, rows, vocab, k):
    if k > vocab:
        pytest.skip("more alternatives than tokens")
    g = torch.Generator().manual_seed(rows * 7 + vocab + k)
    x = (torch.randn(rows, vocab, generator=g) * 4).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32)
    _check(x.to(DEV), t.to(DEV), k)


@pytest.mark.parametrize("offset,pitch", [(0, 1003), (1, 1003), (3, 1005), (8, 1024), (5, 1008)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(offset, pitch, dtype):
    g = torch.Generator().manual_seed(offset + pitch)
    whole = torch.full((9, pitch + 8), 1e4).to(dtype)
    x = (torch.randn(9, 990, generator=g) * 3).to(dtype)
    whole[:, offset:offset + 990] = x
    t = torch.arange(9, dtype=torch.int32)
    dev = whole.to(DEV)[:, offset:offset + 990]
    _check(dev, t.to(DEV), 7)


@pytest.mark.parametrize("rows", [1, 3, 700])
def test_ties_go_to_the_lower_index(rows):
    g = torch.Generator().manual_seed(rows)
    x = torch.randint(-2, 3, (rows, 30001), generator=g).to(torch.bfloat16)
    x[0] = 1.5                       # one value everywhere
    x[-1, ::2] = -0.0                # -0 equals 0
    x[-1, 1::2] = 0.0
    t = torch.full((rows,), 30000, dtype=torch.int32)
    _check(x.to(DEV), t.to(DEV), 32)


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows(rows, dtype):
    """-inf and the type's lowest value as masks; rows of nothing else."""
    g = torch.Generator().manual_seed(rows)
    lowest = torch.finfo(dtype).min
    for mask in (-INF, lowest):
        x = (torch.randn(rows, 5003, generator=g) * 5).to(dtype)
        x[torch.rand(rows, 5003, generator=g) < 0.7] = mask
        x[0] = mask
        t = torch.randint(0, 5003, (rows,), generator=g).to(torch.int32)
        _check(x.to(DEV), t.to(DEV), 9)
        x[0, 4001] = 2.0             # one token left
        _, ent, ids, _ = _check(x.to(DEV), t.to(DEV), 9)
        assert int(ids[0, 0]) == 4001 and float(ent[0]) == 0.0
    x = torch.full((rows, 100), -INF, dtype=dtype)
    x[:, 50:60] = lowest
    _check(x.to(DEV), torch.full((rows,), 55, dtype=torch.int32, device=DEV), 12)


@pytest.mark.parametrize("rows", [2, 650])
def test_nan_and_inf(rows):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 6001, generator=g)
    x[0, 17] = float("nan")
    x[0, 5000] = float("nan")
    x[1, 3] = INF
    t = torch.zeros(rows, dtype=torch.int32)
    lp, ent, ids, top = _check(x.to(DEV), t.to(DEV), 4)
    assert ids[0, :2].tolist() == [17, 5000] and int(ids[1, 0]) == 3
    assert bool(lp[:2].isnan().all()) and bool(ent[:2].isnan().all())


def test_token_outside_the_vocabulary():
    x = torch.randn(3, 100, device=DEV)
    lp, _, _, _ = ops.token_logprobs(x, torch.tensor([-1, 100, 5], dtype=torch.int32, device=DEV))
    assert lp.isnan().tolist() == [True, True, False]


@pytest.mark.parametrize("rows", [1, 640])
@pytest.mark.parametrize("order", ["ascending", "descending", "few_places"])
def test_hard_orders(rows, order):
    """Orders that crowd the largest values: into the last or first places, or
    into the strided places that a few threads read."""
    n = 100003
    x = torch.randn(rows, n, generator=torch.Generator().manual_seed(1))
    if order == "ascending":
        x[0] = torch.linspace(-5, 5, n)
    elif order == "descending":
        x[0] = torch.linspace(5, -5, n)
    else:
        i = torch.arange(n)
        for period in (256 * 4, 512 * 4, 1024 * 4):
            place = i % period
            hot = place < 19 * 4
            x[0] = torch.where(hot, 10 + i / n, x[0])
    t = torch.zeros(rows, dtype=torch.int32)
    _check(x.to(DEV), t.to(DEV), 20)


def test_wide_spread_of_logits():
    x = torch.randn(3, 20000, generator=torch.Generator().manual_seed(3)) * 1e4
    x[1] = x[1] * 1e30
    _check(x.to(DEV), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), 5)


def test_repeatable_streams_and_empty():
    g = torch.Generator().manual_seed(9)
    x = (torch.randn(6, 128256, generator=g) * 3).to(torch.bfloat16).to(DEV)
    t = torch.randint(0, 128256, (6,), generator=g).to(torch.int32).to(DEV)
    ws = ops.GemmWorkspace(DEV, max_floats=16, max_counters=2)
    a = ops.token_logprobs(x, t, 20, workspace=ws)
    for _ in range(3):
        b = ops.token_logprobs(x, t, 20, workspace=ws)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    torch.cuda.synchronize()
    assert int(ws.counters.count_nonzero()) == 0
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = ops.token_logprobs(x, t, 20)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    e = ops.token_logprobs(x[:0], t[:0], 3)
    assert [tuple(v.shape) for v in e] == [(0,), (0,), (0, 3), (0, 3)]


def test_refusals():
    x = torch.randn(2, 50, device=DEV)
    t = torch.zeros(2, dtype=torch.int32, device=DEV)
    for a in ((x.double(), t, 1), (x.t(), t, 1), (x, t.long(), 1), (x, t[:1], 1), (x, t, 33),
              (x, t, -1), (x[:, :4], t, 5), (x, t.cpu(), 1), (x.cpu(), t, 1)):
        with pytest.raises((RuntimeError, ValueError)):
            ops.token_logprobs(*a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("k", [0, 1, 20])
def test_many_rows(dtype, k):
    g = torch.Generator().manual_seed(k)
    x = (torch.randn(1301, 5003, generator=g) * 3).to(dtype)
    t = torch.randint(0, 5003, (1301,), generator=g).to(torch.int32)
    _check(x.to(DEV), t.to(DEV), k)


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("k", [2, 32])
def test_largest_values_all_in_a_few_places(rows, k):
    """More values over the bound than fit: all of one thread in 32's, and (one row)
    all of a few slices'."""
    g = torch.Generator().manual_seed(k + rows)
    x = torch.randn(rows, 131072, generator=g).to(torch.bfloat16)
    chunk = torch.arange(131072) // 8
    x[:, chunk % 32 == 5] += 40.0
    t = torch.randint(0, 131072, (rows,), generator=g).to(torch.int32)
    _check(x.to(DEV), t.to(DEV), k)
    if rows == 1:
        v = 1200000
        slices = ops.ext().token_logprobs_plan(1, v, 4)[0]
        x = torch.randn(1, v, generator=g)
        x[:, torch.arange(v) // (-(-v // slices)) % 32 == 3] -= 60.0
        _check(x.to(DEV), t.to(DEV), k)


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", [-1e8, -1e9, -1e10, -1e12, -1e20, -1e28, -1e29, -7e29, -1e30,
                                  -1e35])
def test_large_finite_masks(rows, dtype, mask):
    """Whole runs of a row at a large negative number, as masks leave them: their
    probability is 0, and the others are as without them."""
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, 20001, generator=g) * 5).to(dtype)
    x[:, :12000] = mask             # most threads see nothing else
    x[torch.rand(rows, 20001, generator=g) < 0.3] = mask
    x[:, 20000] = mask
    if rows > 1:
        x[1] = mask                 # every token alike
        x[2] = mask
        x[2, 777] = -3.0            # one token left
    t = torch.randint(0, 20001, (rows,), generator=g).to(torch.int32)
    _check(x.to(DEV), t.to(DEV), 9)


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [1e7, 1e8, 4e8, 6e8, 1e9, 2e9, 1e10, 1e20, 1e28, 2e29])
def test_rows_of_large_logits(rows, dtype, top):
    """Maxima of either sign far from 0, alone, in a few equal values, and with
    neighbours at the distance of the type's numbers there."""
    g = torch.Generator().manual_seed(int(top) % 1000)
    x = torch.randn(rows, 9003, generator=g) * 3
    x = torch.where(torch.rand(rows, 9003, generator=g) < 0.5, -top * (1.5 + x.abs()), x)
    x[0] = -top * (1 + torch.rand(9003, generator=g))
    x[0, [5, 4000, 9002]] = -top
    if rows > 1:
        x[1, [17, 5000]] = top
        x[2] = top * (1 - torch.rand(9003, generator=g) * 1e-6)
        x[3] = -top * (1 + torch.rand(9003, generator=g) * 1e-6)
    x = x.to(dtype)
    t = torch.randint(0, 9003, (rows,), generator=g).to(torch.int32)
    t[0] = 4000
    _check(x.to(DEV), t.to(DEV), 6)


@pytest.mark.parametrize("rows", [1, 64, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_confident_rows(rows, dtype):
    """One token far over the rest, after values that rise in small steps: a probability
    is at most 1, an entropy at least 0."""
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 30011, generator=g) * 0.3
    top = torch.rand(rows, generator=g) * 40 + 12
    at = torch.randint(0, 30011, (rows,), generator=g)
    # The way up to the maximum, in the places before it that its thread reads.
    for back in range(1, 5):
        i = at - back * 512 * (4 if dtype == torch.float32 else 8)
        x[torch.arange(rows)[i >= 0], i[i >= 0]] = (top - 5 * back)[i >= 0]
    x[torch.arange(rows), at] = top
    x = x.to(dtype)
    lp, ent, _, best = _check(x.to(DEV), at.to(torch.int32).to(DEV), 3)
    assert bool((lp <= 0).all()) and bool((best <= 0).all()) and bool((ent >= 0).all())


@pytest.mark.parametrize("gap", [3.0, 5.0, 8.0, 20.0, 60.0])
def test_certain_token(gap):
    """A token that has all but e^-gap of the probability; rows in many frames."""
    x = torch.zeros(257, 40) - gap
    x[:, 7] = 0.0
    x += torch.linspace(-30, 30, 257)[:, None]
    t = torch.full((257,), 7, dtype=torch.int32)
    lp, ent, _, best = _check(x.to(DEV), t.to(DEV), 2)
    assert bool((lp <= 0).all()) and bool((best <= 0).all()) and bool((ent >= 0).all())
