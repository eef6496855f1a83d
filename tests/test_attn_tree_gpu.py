"""Tree / chain / single-token attention over the bf16 and the 8-bit paged
cache against the 64-bit formula."""
import math

import pytest
import torch

from cascadia_b200 import ops
from cascadia_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


class Problem:
    """A paged cache filled with the sequences' keys; every slot that no
    sequence uses holds NaNs."""

    def __init__(self, cache, hq, hkv, d, lens, nodes, seed=0, tree=True, k_mul=1.0, v_mul=None,
                 layers=2, layer=1, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.cache, self.hq, self.hkv, self.d = cache, hq, hkv, d
        self.lens, self.nodes, self.layer = lens, nodes, layer
        self.scale = 1.0 / math.sqrt(d)
        need = [-(-n // 16) for n in lens]
        nb = sum(need) + spare
        self.k = [torch.randn(n, hkv, d, generator=g) * k_mul for n in lens]
        self.v = [torch.randn(n, hkv, d, generator=g) for n in lens]
        if v_mul is not None:
            self.v = [x * v_mul(x.shape, g) for x in self.v]
        order = torch.randperm(nb, generator=g).tolist()
        self.table = torch.randint(0, nb, (len(lens), max(need + [1]) + 2), generator=g)
        pools = []
        for rows in (self.k, self.v):
            pool = torch.full((layers, nb, hkv, 16, d), float("nan"))
            at = 0
            for b, x in enumerate(rows):
                blocks = order[at:at + need[b]]
                at += need[b]
                self.table[b, :need[b]] = torch.tensor(blocks, dtype=torch.long)
                for i, blk in enumerate(blocks):
                    part = x[16 * i:16 * i + 16]
                    pool[layer, blk, :, :part.shape[0]] = part.transpose(0, 1)
            pools.append(pool)
        self.table = self.table.to(**I32)
        if cache == "fp8":
            (self.kc, self.ks), (self.vc, self.vs) = (ref.quantise_rows(p) for p in pools)
            for c, s in ((self.kc, self.ks), (self.vc, self.vs)):
                c.view(torch.uint8)[s.isnan()] = 0x7f  # unused slots: NaN codes too
            self.kf, self.vf = (ref.dequantise_rows(c, s) for c, s in
                                ((self.kc, self.ks), (self.vc, self.vs)))
            self.ks, self.vs = self.ks.to(DEV), self.vs.to(DEV)
        else:
            self.kc, self.vc = (p.to(torch.bfloat16) for p in pools)
            self.kf, self.vf = self.kc.float(), self.vc.float()
            self.ks = self.vs = None
        self.kc, self.vc = self.kc.to(DEV), self.vc.to(DEV)
        self.starts = [0]
        for n in nodes:
            self.starts.append(self.starts[-1] + n)
        self.masks = None
        if tree:
            self.masks = []
            for n in nodes:
                m = []
                for i in range(n):
                    p = int(torch.randint(max(0, i - 5), i, (1,), generator=g)) if i else -1
                    m.append((m[p] if p >= 0 else 0) | 1 << i)
                self.masks += m
        self.q = torch.randn(self.starts[-1], hq * d, generator=g).to(torch.bfloat16) * 2

    def signed_masks(self):
        if self.masks is None:
            return None
        m = [x - (1 << 64) if x >= 1 << 63 else x for x in self.masks]
        return torch.tensor(m, dtype=torch.int64, device=DEV)

    def run(self, **kw):
        t = self.starts[-1]
        wide = torch.zeros(t, self.hq * self.d + 40, dtype=torch.bfloat16, device=DEV)
        wide[:, 16:16 + self.hq * self.d] = self.q.to(DEV)
        q = wide[:, 16:16 + self.hq * self.d]  # row pitch wider than the row
        out = torch.full((t, self.hq * self.d + 3), 7.0, dtype=torch.bfloat16, device=DEV)
        a = dict(max_nodes=max(self.nodes + [1]))
        a.update(kw)
        ops.attn_tree(q, self.kc, self.vc, self.table, torch.tensor(self.lens, **I32),
                      torch.tensor(self.starts, **I32), out[:, 1:-2], self.layer, self.scale,
                      masks=self.signed_masks(), k_scale=self.ks, v_scale=self.vs, **a)
        assert bool((out[:, 0] == 7).all()) and bool((out[:, -2:] == 7).all())
        return out[:, 1:-2].cpu()

    def rows(self, b):
        need = -(-self.lens[b] // 16)
        at = self.table[b, :need].long().cpu()
        return tuple(p[self.layer][at].permute(0, 2, 1, 3).reshape(-1, self.hkv, self.d)
                     [:self.lens[b]].double() for p in (self.kf, self.vf))

    def check(self, out, skip_rows=()):
        """|error| <= 2^-8 |o| (the bf16 result, 8 bits) + (u + 2 e) A with A =
        sum p |v|, u the rounding of a weight (2^-8 in bf16, 2^-11 in fp16) and e
        the error of a base-2 score: fp32 sums of D products and the folding of
        scales, (D + 16) 2^-24 sum |q k| scale, and 2^-20 for the exponential
        and the running rescale."""
        u = 2.0 ** -11 if self.cache == "fp8" else 2.0 ** -8
        for b, n in enumerate(self.nodes):
            if n == 0:
                continue
            lo, hi = self.starts[b], self.starts[b + 1]
            k, v = self.rows(b)
            if self.lens[b] < n:  # fewer keys than rows: only whole-zero padding rows here
                assert self.lens[b] == 0
                assert bool((out[lo:hi] == 0).all())
                continue
            q = self.q[lo:hi].double().view(n, self.hq, self.d)
            masks = None
            if self.masks is not None:
                masks = [x - (1 << 64) if x >= 1 << 63 else x for x in self.masks[lo:hi]]
            want = ref.tree_attention(q, k, v, self.scale, masks)
            mag = ref.tree_attention(q, k, v.abs(), self.scale, masks)
            big = torch.einsum("qhd,khd->hqk", q.abs(),
                               k.abs().repeat_interleave(self.hq // self.hkv, 1))
            big = big.nan_to_num(0.0).amax(-1).t().unsqueeze(-1) * self.scale
            e = (self.d + 16) * 2.0 ** -24 * big + 2.0 ** -20
            tol = want.abs() * 2.0 ** -8 + (u + 2 * e) * mag + 1e-30
            got = out[lo:hi].double().view(n, self.hq, self.d)
            for i in range(n):
                if lo + i in skip_rows:
                    continue
                bad = (got[i] - want[i]).abs() > tol[i]
                assert not bool(bad.any()) and bool(got[i].isfinite().all()), (
                    b, i, float(((got[i] - want[i]).abs() / tol[i]).max()))


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(3, 3, 64), (8, 1, 128), (16, 1, 64), (12, 4, 128),
                                      (32, 8, 128), (40, 2, 64)])
def test_single_token(cache, hq, hkv, d):
    lens = [1, 2, 15, 16, 17, 0, 33, 129, 700]
    p = Problem(cache, hq, hkv, d, lens, [1] * len(lens), tree=False, seed=d + hq)
    p.check(p.run())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (16, 1, 128), (12, 4, 64)])
@pytest.mark.parametrize("tree", [True, False])
def test_trees_and_chains(cache, hq, hkv, d, tree):
    # Roots only, no context, sequences without rows, 64 nodes, every tail.
    lens = [1, 64, 5, 80, 30, 131, 64, 400, 16]
    nodes = [1, 64, 5, 0, 7, 64, 0, 33, 2]
    p = Problem(cache, hq, hkv, d, lens, nodes, tree=tree, seed=7 * d + hq)
    p.check(p.run())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_wide_rows(cache):
    """64 nodes of 16 heads a kv head: 1024 rows read the same keys."""
    p = Problem(cache, 32, 2, 128, [333, 64, 1000], [64, 64, 61], seed=3)
    p.check(p.run())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_long_chain_without_masks(cache):
    p = Problem(cache, 8, 2, 64, [300, 217], [150, 217], tree=False, seed=5)
    p.check(p.run())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("nodes", [1, 9, 40])
def test_long_context(cache, nodes):
    """One sequence over many pieces, and uneven ones beside it."""
    p = Problem(cache, 8, 2, 128, [20011, 70, 3001], [nodes, 1, nodes], seed=nodes)
    p.check(p.run())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_many_sequences(cache):
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 60, (301,), generator=g).tolist()
    nodes = [int(n > 0) * (1 + n % 3 if n > 3 else 1) for n in lens]
    p = Problem(cache, 4, 1, 64, lens, nodes, seed=9)
    p.check(p.run())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("nodes", [6, 40])
def test_hidden_nodes_may_hold_anything(cache, nodes):
    """A NaN or an infinity in a node's K or V reaches the rows that see the
    node, and no others."""
    p = Problem(cache, 8, 2, 128, [37 + nodes], [nodes], seed=4)
    ctx = 37
    parents = [-1, 0, 0] + [1 + (i % 2) for i in range(nodes - 3)]
    masks = []
    for i, pa in enumerate(parents):
        masks.append((masks[pa] if pa >= 0 else 0) | 1 << i)
    p.masks = masks
    for node, what, where in ((1, float("nan"), "k"), (3, float("inf"), "v")):
        pos = ctx + node
        blk = int(p.table[0, pos // 16])
        for name in (where, where):
            if p.cache == "fp8":
                (p.ks if name == "k" else p.vs)[p.layer, blk, :, pos % 16] = float("nan")
            else:
                (p.kc if name == "k" else p.vc)[p.layer, blk, :, pos % 16, 3] = what
    out = p.run().float().view(nodes, 8, 128)
    sees = [i for i in range(nodes) if masks[i] >> 1 & 1 or masks[i] >> 3 & 1]
    for i in sees:
        assert not bool(out[i, :, 3].isfinite().any()), i
    # The others: as if those nodes were not there at all (their K / V zeroed
    # in the reference, where their weight is zero anyway).
    k_clean = Problem(cache, 8, 2, 128, [37 + nodes], [nodes], seed=4)
    k_clean.masks = masks
    clean = k_clean.run().float().view(nodes, 8, 128)
    k_clean.check(clean.reshape(nodes, -1).to(torch.bfloat16))
    for i in range(nodes):
        if i not in sees:
            assert torch.equal(out[i], clean[i]), i


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_row_that_sees_nothing(cache):
    p = Problem(cache, 4, 2, 128, [5, 21], [5, 4], seed=6)
    p.masks[2] = 0       # no context, empty mask: zeros
    p.masks[5 + 1] = 0   # context only
    out = p.run()
    assert bool((out[2] == 0).all())
    p.check(out)


@pytest.mark.parametrize("nodes", [1, 40])
def test_extreme_scales(nodes):
    """Value rows whose scales span 2^60, zero rows among them, keys and
    queries far from 1."""
    def mul(shape, g):
        e = torch.randint(-30, 31, (shape[0], shape[1], 1), generator=g).float()
        return torch.where(e == 0, torch.zeros_like(e), torch.exp2(e))

    p = Problem("fp8", 8, 2, 128, [300 + nodes], [nodes], seed=8, v_mul=mul, k_mul=1e-3)
    p.q = p.q * 1000
    p.check(p.run())
    p = Problem("fp8", 8, 2, 128, [300 + nodes], [nodes], seed=8, k_mul=1e20)
    p.q = (p.q.float() * 1e-20).to(torch.bfloat16)
    p.check(p.run())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("nodes", [1, 4, 40])
def test_values_of_zero(cache, nodes):
    """A head whose values are all zero (the smallest scale) over a long
    context, alone and beside ordinary heads."""
    p = Problem(cache, 8, 2, 128, [9000, 30 + nodes], [nodes, nodes], seed=18,
                v_mul=lambda shape, g: torch.tensor([0.0, 1.0]).view(1, 2, 1))
    out = p.run()
    p.check(out)
    assert bool((out.view(-1, 2, 4, 128)[:, 0] == 0).all())


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_value_of_one_key_comes_back(cache):
    """A sequence of one key returns its value, to the last bit."""
    p = Problem(cache, 6, 2, 128, [1, 1], [1, 1], tree=False, seed=10)
    out = p.run().view(2, 2, 3, 128)
    for b in range(2):
        _, v = p.rows(b)
        want = v[0].to(torch.bfloat16).unsqueeze(1).expand(2, 3, 128)
        assert torch.equal(out[b], want)


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("nodes", [1, 50])
def test_repeatable_and_workspace_left_clean(cache, nodes):
    p = Problem(cache, 32, 4, 128, [2500, 40 + nodes, 777], [nodes] * 3, seed=12)
    ws = ops.GemmWorkspace(DEV)
    a = p.run(workspace=ws)
    for _ in range(3):
        assert torch.equal(p.run(workspace=ws), a)
    assert int(ws.counters.count_nonzero()) == 0
    # The bound on the rows of a sequence picks the kernel; both are right.
    p.check(p.run(max_nodes=64))


def test_other_stream():
    p = Problem("fp8", 8, 2, 128, [900], [20], seed=13)
    want = p.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = p.run()
    assert torch.equal(got, want)


def test_captured_graph_follows_lengths():
    """A captured call reads lengths and row starts when it is replayed."""
    p = Problem("fp8", 8, 2, 128, [600, 90, 301], [1, 1, 1], tree=False, seed=14)
    lens = torch.tensor([600, 90, 301], **I32)
    starts = torch.tensor([0, 1, 2, 3], **I32)
    q, out = p.q.to(DEV), torch.zeros(3, 1024, dtype=torch.bfloat16, device=DEV)
    ws = ops.GemmWorkspace(DEV)

    def call():
        ops.attn_tree(q, p.kc, p.vc, p.table, lens, starts, out, p.layer, p.scale, k_scale=p.ks,
                      v_scale=p.vs, max_nodes=1, workspace=ws)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
    for now in ([600, 90, 301], [17, 89, 0], [1, 1, 255]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        p.lens = now
        p.check(out.cpu())


def test_offsets_past_32_bits():
    hkv, d, n = 8, 128, 100
    nb = (1 << 32) // (hkv * 16 * d) + 9
    p = Problem("fp8", 16, hkv, d, [n], [3], seed=15, layers=1, layer=0, spare=0)
    kc = torch.empty(1, nb, hkv, 16, d, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    vc = torch.empty_like(kc)
    ks = torch.empty(1, nb, hkv, 16, device=DEV)
    vs = torch.empty_like(ks)
    want = p.run()
    used = p.kc.shape[1]
    for big, small in ((kc, p.kc), (vc, p.vc)):
        big.view(torch.uint8)[:, nb - used:] = small.view(torch.uint8)
    for big, small in ((ks, p.ks), (vs, p.vs)):
        big[:, nb - used:] = small
    p.kc, p.vc, p.ks, p.vs = kc, vc, ks, vs
    p.table = p.table + (nb - used)
    assert torch.equal(p.run(), want)
    p.nodes = [64]  # the bound alone
    assert torch.equal(p.run(max_nodes=3), want)


def test_refusals():
    p = Problem("fp8", 4, 2, 64, [20], [2], seed=16)
    base = dict(q=p.q.to(DEV), k_cache=p.kc, v_cache=p.vc, block_tables=p.table,
                seq_lens=torch.tensor([20], **I32), row_start=torch.tensor([0, 2], **I32),
                out=torch.empty(2, 256, dtype=torch.bfloat16, device=DEV), layer=1, scale=0.125,
                masks=p.signed_masks(), k_scale=p.ks, v_scale=p.vs, max_nodes=2)
    ops.attn_tree(**base)
    bad = [dict(q=base["q"].float()), dict(q=base["q"][:, :192], out=base["out"][:, :192]),
           dict(k_scale=None), dict(v_scale=None), dict(k_scale=p.ks.half()),
           dict(k_cache=p.kc.to(torch.float8_e5m2)), dict(k_cache=p.kc[:, :1]),
           dict(block_tables=p.table.long()), dict(seq_lens=base["seq_lens"].long()),
           dict(row_start=torch.tensor([0], **I32)), dict(masks=base["masks"].int()),
           dict(masks=base["masks"][:1]), dict(max_nodes=65), dict(max_nodes=0), dict(layer=2),
           dict(layer=-1), dict(out=base["out"].float()), dict(out=base["out"][:1]),
           dict(seq_lens=base["seq_lens"].cpu()),
           dict(k_cache=p.kc.to(torch.bfloat16), v_cache=p.vc.to(torch.bfloat16))]
    for kw in bad:
        with pytest.raises(RuntimeError):
            ops.attn_tree(**{**base, **kw})
    with pytest.raises(RuntimeError):  # more sequences than one call takes
        ops.attn_tree(**{**base, **dict(seq_lens=torch.zeros(5000, **I32),
                                        row_start=torch.zeros(5001, **I32),
                                        block_tables=torch.zeros(5000, 2, **I32))})
    small = ops.GemmWorkspace(DEV, max_floats=16, max_counters=1)
    ops.attn_tree(**base, workspace=small)  # grows it
    # No sequences, no rows: nothing to do.
    none = dict(q=base["q"][:0], out=base["out"][:0], seq_lens=base["seq_lens"][:0],
                row_start=torch.zeros(1, **I32), masks=None)
    ops.attn_tree(**{**base, **none})
    wide = torch.zeros(1, 1, 2, 16, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):  # head_dim 256 is not built
        ops.attn_tree(**{**base, **dict(k_cache=wide, v_cache=wide, k_scale=None, v_scale=None,
                                        q=torch.zeros(2, 512, dtype=torch.bfloat16, device=DEV),
                                        out=torch.zeros(2, 512, dtype=torch.bfloat16, device=DEV),
                                        layer=0)})


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,most", [(6, 3, 128, 1), (6, 3, 64, 4), (10, 5, 128, 6)])
def test_pieces_across_sequences(cache, hq, hkv, d, most):
    """Contexts from nothing to some hundred keys: a CTA's piece holds ends, middles and
    whole sequences, with fewer blocks than its warps or many more."""
    g = torch.Generator().manual_seed(31)
    lens = torch.randint(0, 40, (260,), generator=g).tolist()
    lens[::7] = torch.randint(100, 1200, (len(lens[::7]),), generator=g).tolist()
    nodes = [min(n, 1 + i % most) if i % 11 else 0 for i, n in enumerate(lens)]
    p = Problem(cache, hq, hkv, d, lens, nodes, tree=most > 1, seed=d + most)
    p.check(p.run())


def test_refuses_a_misaligned_workspace():
    p = Problem("bf16", 4, 2, 64, [20], [1], seed=4)
    ws = ops.GemmWorkspace(DEV)
    whole = ws.ws
    ws.ws = whole[1:]
    kw = dict(layer=1, scale=0.125, max_nodes=1, workspace=ws)
    args = (p.q.to(DEV), p.kc, p.vc, p.table, torch.tensor([20], **I32),
            torch.tensor([0, 1], **I32), torch.empty(1, 256, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(RuntimeError):
        ops.attn_tree(*args, **kw)
    ws.ws = whole
    ops.attn_tree(*args, **kw)


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,nodes", [(8, 2, 128, 5), (4, 1, 64, 17), (12, 4, 128, 40)])
def test_many_short_jobs_of_odd_tile_counts(cache, hq, hkv, d, nodes):
    """More jobs of one row tile than SMs, of one to three K / V tiles (and some without
    keys): a CTA goes from job to job with the tiles' stages left at either one, and a
    softmax group without a tile of its own at times."""
    g = torch.Generator().manual_seed(nodes)
    lens = [int(torch.randint(128 * t + 1, 128 * t + 129, (1,), generator=g))
            for t in torch.randint(0, 3, (420,), generator=g).tolist()]
    rows = [min(n, nodes) for n in lens]
    lens[::13] = [0] * len(lens[::13])
    rows[::13] = [1] * len(rows[::13])
    p = Problem(cache, hq, hkv, d, lens, rows, seed=nodes)
    a = p.run(max_nodes=64)
    p.check(a)
    for _ in range(20):
        assert torch.equal(p.run(max_nodes=64), a)
    assert ops.read_status(torch.device(DEV)) == 0


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_jobs_of_one_and_two_row_tiles_in_turn(cache):
    """Jobs whose K / V tiles the softmax groups take in turn beside jobs whose tiles
    they share."""
    g = torch.Generator().manual_seed(77)
    lens = torch.randint(64, 520, (330,), generator=g).tolist()
    rows = [(7, 64, 20, 64, 33)[i % 5] for i in range(330)]
    p = Problem(cache, 8, 2, 128, lens, rows, seed=78)
    a = p.run(max_nodes=64)
    p.check(a)
    for _ in range(20):
        assert torch.equal(p.run(max_nodes=64), a)
    assert ops.read_status(torch.device(DEV)) == 0


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("last", [0, 300])
def test_a_softmax_group_without_tiles_keeps_up(cache, last):
    """Job after job of a single K / V tile, all of them one group's, and none at all;
    then one that needs both groups."""
    g = torch.Generator().manual_seed(last)
    lens = torch.randint(5, 129, (900,), generator=g).tolist()
    lens[::9] = [0] * len(lens[::9])
    rows = [5 if n else 1 for n in lens]
    if last:
        lens += [last] * 7
        rows += [40] * 7
    p = Problem(cache, 16, 4, 64, lens, rows, seed=11)
    a = p.run(max_nodes=64)
    p.check(a)
    for _ in range(10):
        assert torch.equal(p.run(max_nodes=64), a)
    assert ops.read_status(torch.device(DEV)) == 0


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("nodes", [1, 5, 40])
@pytest.mark.parametrize("far", [2.0 ** 14, 2.0 ** 25, 2.0 ** 40, 2.0 ** 100])
def test_a_large_value_that_does_not_count(cache, nodes, far):
    """Beside the others' values a key's is far larger, but hidden (a node that only
    itself sees) or of no weight (a score far below the others): the others keep
    their bits."""
    ctx = 150
    for hidden in (True, False):
        if hidden and nodes == 1:
            continue
        at = ctx + 1 if hidden else 70
        p = Problem(cache, 8, 2, 128, [ctx + nodes, 31], [nodes, 1], seed=21,
                    v_mul=lambda shape, g: torch.where(
                        (torch.arange(shape[0]) == at).view(-1, 1, 1), far, 1.0))
        if hidden:
            p.masks[:nodes] = [1 << i | 1 for i in range(nodes)]
        else:
            # Every query has 8 in its first place, this key alone something against it.
            low = -140.0 - 12 * math.log2(far) * (far > 2.0 ** 40)
            p = Problem(cache, 8, 2, 128, [ctx + nodes, 31], [nodes, 1], seed=21,
                        v_mul=lambda shape, g: torch.where(
                            (torch.arange(shape[0]) == at).view(-1, 1, 1), far, 1.0))
            p.q.view(-1, 8, 128)[:, :, 0] = 8.0
            blk, row = int(p.table[0, at // 16]), at % 16
            x = torch.zeros(2, 128)
            x[:, 0] = low
            if cache == "fp8":
                codes, s = ref.quantise_rows(x)
                p.kc.view(torch.uint8)[p.layer, blk, :, row] = codes.view(torch.uint8).to(DEV)
                p.ks[p.layer, blk, :, row] = s.to(DEV)
                p.kf[p.layer, blk, :, row] = ref.dequantise_rows(codes, s)
            else:
                p.kc[p.layer, blk, :, row] = x.to(torch.bfloat16).to(DEV)
                p.kf[p.layer, blk, :, row] = x.to(torch.bfloat16).float()
        p.check(p.run())
        p.check(p.run(max_nodes=64))


def test_tile_kernel_past_32_bits():
    """Rows at the far end of a pool of more than 2^32 codes, read by the tile kernel."""
    hkv, d, n = 8, 128, 300
    nb = (1 << 32) // (hkv * 16 * d) + 40
    p = Problem("fp8", 16, hkv, d, [n, 70], [40, 64], seed=17, layers=1, layer=0, spare=0)
    want = p.run()
    p.check(want)
    pools = []
    used = p.kc.shape[1]
    for small in (p.kc, p.vc):
        big = torch.empty(1, nb, hkv, 16, d, dtype=torch.uint8, device=DEV)
        big[:, nb - used:] = small.view(torch.uint8)
        pools.append(big.view(torch.float8_e4m3fn))
    for small in (p.ks, p.vs):
        big = torch.empty(1, nb, hkv, 16, device=DEV)
        big[:, nb - used:] = small
        pools.append(big)
    p.kc, p.vc, p.ks, p.vs = pools
    p.table = p.table + (nb - used)
    assert torch.equal(p.run(max_nodes=64), want)


def test_tile_kernel_past_32_bits_with_an_infinite_node():
    """The same for the bf16 cache, whose infinities are read a second time."""
    hkv, d, n = 8, 128, 150
    nb = (1 << 32) // (hkv * 16 * d) + 40
    p = Problem("bf16", 16, hkv, d, [n], [40], seed=19, layers=1, layer=0, spare=0)
    blk = int(p.table[0, (n - 37) // 16])  # node 3
    p.vc[0, blk, :, (n - 37) % 16, 5] = float("inf")
    want = p.run()
    sees = torch.tensor([bool(m >> 3 & 1) for m in p.masks])
    got = want.view(40, 16, d)
    assert bool((got[sees][:, :, 5] == float("inf")).all()) and bool(got[~sees].isfinite().all())
    used = p.kc.shape[1]
    pools = []
    for small in (p.kc, p.vc):
        big = torch.empty(1, nb, hkv, 16, d, dtype=torch.bfloat16, device=DEV)
        big[:, nb - used:] = small
        pools.append(big)
    p.kc, p.vc = pools
    p.table = p.table + (nb - used)
    assert torch.equal(p.run(max_nodes=64), want)


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("nodes", [1, 5, 40])
@pytest.mark.parametrize("c,a", [(2.0 ** -9, 1.0), (2.0 ** -9, 0.25), (2.0 ** -9, -0.296875),
                                 (2.0 ** -6, 2.0 ** -5)])
def test_products_are_summed_in_32_bits(cache, nodes, c, a):
    """Two keys that differ by 127 small products beside a product of 448 to 448 000
    times their size: sums of fewer bits would lose them."""
    p = Problem(cache, 4, 1, 128, [2 + nodes], [nodes], seed=23)
    p.masks = [0] * nodes
    p.scale = 1.0
    p.q = torch.full((nodes, 4, 128), a)
    p.q[:, :, 0] = 1.0
    p.q = p.q.view(nodes, 512).to(torch.bfloat16)
    k = torch.zeros(2, 1, 128)
    k[0] = c
    k[:, :, 0] = 448.0
    v = torch.zeros(2, 1, 128)
    v[0] = 1.0
    blk = int(p.table[0, 0])
    for x, pool, full, scale in ((k, p.kc, p.kf, p.ks), (v, p.vc, p.vf, p.vs)):
        for t in range(2):
            if cache == "fp8":
                codes = x[t].to(torch.float8_e4m3fn)
                assert torch.equal(codes.float(), x[t])
                pool.view(torch.uint8)[p.layer, blk, :, t] = codes.view(torch.uint8).to(DEV)
                scale[p.layer, blk, :, t] = 1.0
            else:
                pool[p.layer, blk, :, t] = x[t].to(torch.bfloat16).to(DEV)
            full[p.layer, blk, :, t] = x[t]
    p.check(p.run())
