"""The 8-bit KV cache's kernels: rotation + quantising write, and read-back."""
import math

import pytest
import torch

from cascadia_b200 import ops
from cascadia_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cache(layers, blocks, hkv, d):
    k = torch.zeros(layers, blocks, hkv, 16, d, dtype=torch.uint8, device=DEV)
    ks = torch.ones(layers, blocks, hkv, 16, device=DEV)
    return (k.view(torch.float8_e4m3fn), k.clone().view(torch.float8_e4m3fn), ks, ks.clone())


def _table(max_pos, rot, g):
    ang = torch.rand(max_pos, rot // 2, generator=g) * 6.28
    return torch.cat([ang.cos(), ang.sin()], dim=1)


def _codes_at(cache, layer, slots):
    s = slots.long()
    return cache.view(torch.uint8)[layer, s // 16, :, s % 16].view(cache.dtype).float().cpu()


@pytest.mark.parametrize("tokens", [1, 3, 64, 257])
@pytest.mark.parametrize("hq,hkv,d,rot", [(4, 4, 64, 64), (32, 8, 128, 128), (5, 1, 128, 32),
                                          (7, 3, 64, 16), (8, 2, 256, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_write(tokens, hq, hkv, d, rot, interleaved):
    g = torch.Generator().manual_seed(tokens * 31 + d + rot)
    width = (hq + 2 * hkv) * d
    wide = torch.randn(tokens, width + 24, generator=g).to(torch.bfloat16)
    wide[:, hq * d:] *= torch.exp(2 * torch.randn(tokens, 1, generator=g))
    qkv_cpu = wide[:, 8:8 + width]
    qkv = wide.to(DEV)[:, 8:8 + width]  # a view: row pitch wider than the row
    pos = torch.randint(0, 300, (tokens,), generator=g).to(torch.int32)
    cs = _table(300, rot, g)
    blocks = tokens // 16 + 2
    slots = torch.randperm(blocks * 16, generator=g)[:tokens].to(torch.int32)
    if tokens > 3:
        slots[1] = -1
    k, v, ks, vs = _cache(2, blocks, hkv, d)
    q_out = torch.full((tokens, hq * d), float("nan"), dtype=torch.bfloat16, device=DEV)
    ops.rope_kv_write_fp8(qkv, pos.to(DEV), cs.to(DEV), slots.to(DEV), k, v, ks, vs, 1, hq, hkv, d,
                          rot, interleaved, q_out)
    assert torch.equal(qkv.cpu(), qkv_cpu)  # with q_out the input stays as it was
    x = qkv_cpu.float().view(tokens, hq + 2 * hkv, d)
    y = torch.cat([ref.apply_rope(x[:, :hq + hkv], pos, cs, rot, interleaved), x[:, hq + hkv:]], 1)
    assert torch.equal(q_out.cpu(), y[:, :hq].reshape(tokens, -1).to(torch.bfloat16))
    codes, scales = ref.quantise_rows(y[:, hq:])
    keep = slots >= 0
    for cache, sc, lo in ((k, ks, 0), (v, vs, hkv)):
        assert torch.equal(_codes_at(cache, 1, slots[keep]), codes.float()[keep, lo:lo + hkv])
        s = slots[keep].long()
        assert torch.equal(sc[1].cpu()[s // 16, :, s % 16], scales[keep, lo:lo + hkv])
        # Nothing else is touched: the other layer, other slots, slot -1.
        assert int(cache[0].view(torch.uint8).count_nonzero()) == 0
        untouched = torch.ones(blocks * 16, dtype=torch.bool)
        untouched[s] = False
        assert bool((sc[1].transpose(1, 2).reshape(-1, hkv).cpu()[untouched] == 1).all())
    # In place: the same q, the other heads as they were.
    ops.rope_kv_write_fp8(qkv, pos.to(DEV), cs.to(DEV), slots.to(DEV), k, v, ks, vs, 1, hq, hkv, d,
                          rot, interleaved)
    assert torch.equal(qkv[:, :hq * d], q_out)
    assert torch.equal(qkv[:, hq * d:].cpu(), qkv_cpu[:, hq * d:])


@pytest.mark.parametrize("d", [64, 128])
def test_write_against_64_bits(d):
    """Every stored value is within half an e4m3 step of the 64-bit value:
    2^-4 of it, or half the smallest step 2^-9 of a scale; plus the fp32
    rounding of rotation and scale (2^-21 of the row's largest value)."""
    g = torch.Generator().manual_seed(d)
    t, hq, hkv = 50, 2, 3
    qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * 3).to(torch.bfloat16)
    pos = torch.arange(t, dtype=torch.int32)
    cs = _table(t, d, g)
    k, v, ks, vs = _cache(1, 5, hkv, d)
    slots = torch.randperm(80, generator=g)[:t].to(torch.int32)
    ops.rope_kv_write_fp8(qkv.to(DEV), pos.to(DEV), cs.to(DEV), slots.to(DEV), k, v, ks, vs, 0, hq,
                          hkv, d, d)
    x = qkv.double().view(t, -1, d)
    want_k = ref.apply_rope(x[:, hq:hq + hkv], pos, cs.double(), d)
    for cache, sc, want in ((k, ks, want_k), (v, vs, x[:, hq + hkv:])):
        s = slots.long()
        scale = sc[0].cpu()[s // 16, :, s % 16].double().unsqueeze(-1)
        got = _codes_at(cache, 0, slots).double() * scale
        peak = want.abs().amax(-1, keepdim=True)
        assert torch.allclose(scale, peak / 448, rtol=2.0 ** -20, atol=0)
        tol = torch.maximum(want.abs() / 16, scale * 2.0 ** -10) + peak * 2.0 ** -21
        assert bool(((got - want).abs() <= tol).all())


def test_write_extreme_rows():
    """Zero rows, the smallest and largest bf16 values, and rows with a NaN or
    an infinity (scale NaN, codes 0)."""
    d, hq, hkv = 128, 1, 1
    x = torch.zeros(6, 3, d)
    x[1, 2, 5] = 2.0 ** -133
    x[2, 2, 7] = -3.3895313892515355e38
    x[3, 2, 9] = float("nan")
    x[4, 2, 11] = float("-inf")
    x[5, 2] = torch.linspace(-1, 1, d)
    qkv = x.view(6, -1).to(torch.bfloat16)
    cs = torch.cat([torch.ones(1, 64), torch.zeros(1, 64)], dim=1)
    k, v, ks, vs = _cache(1, 1, hkv, d)
    slots = torch.arange(6, dtype=torch.int32)
    ops.rope_kv_write_fp8(qkv.to(DEV), torch.zeros(6, dtype=torch.int32, device=DEV), cs.to(DEV),
                          slots.to(DEV), k, v, ks, vs, 0, hq, hkv, d, d)
    got_k, got_v = ops.kv_read_fp8(k, v, ks, vs, torch.zeros(1, dtype=torch.int32, device=DEV), 0)
    got = got_v[0, 0, :6].float().cpu()
    assert bool((got_k[0, 0, :6] == 0).all())
    assert bool((got[0] == 0).all())
    assert abs(float(got[1, 5])) <= 2.0 ** -100
    assert float(got[2, 7]) == pytest.approx(-3.3895e38, rel=2.0 ** -7)
    assert bool(got[3].isnan().all()) and bool(got[4].isnan().all())
    assert torch.allclose(got[5], qkv[5, 2 * d:].float(), rtol=1 / 15, atol=2.0 ** -10 / 448 + 1e-6)
    assert bool(vs[0, 0, 0, :3].isfinite().all()) and bool(vs[0, 0, 0, 3:5].isnan().all())


@pytest.mark.parametrize("hkv,d", [(1, 64), (8, 128), (3, 256)])
@pytest.mark.parametrize("n", [1, 5, 67])
def test_read(hkv, d, n):
    g = torch.Generator().manual_seed(n + d)
    codes, scales = ref.quantise_rows(torch.randn(2, 70, hkv, 16, d, generator=g))
    vcodes, vscales = ref.quantise_rows(torch.randn(2, 70, hkv, 16, d, generator=g) * 7)
    blocks = torch.randint(0, 70, (n,), generator=g).to(torch.int32)
    blocks[n // 2] = -1
    out = [torch.full((n, hkv, 16, d), float("nan"), dtype=torch.bfloat16, device=DEV)
           for _ in range(2)]
    ops.kv_read_fp8(codes.to(DEV), vcodes.to(DEV), scales.to(DEV), vscales.to(DEV), blocks.to(DEV),
                    1, out[0], out[1])
    for got, c, s in ((out[0], codes, scales), (out[1], vcodes, vscales)):
        want = ref.dequantise_rows(c[1], s[1])[blocks.clamp_min(0).long()].to(torch.bfloat16)
        want[blocks < 0] = 0
        assert torch.equal(got.cpu(), want)
        wide = c[1].double() * s[1].double().unsqueeze(-1)
        wide = torch.where((blocks < 0)[:, None, None, None], 0.0, wide[blocks.clamp_min(0).long()])
        # one rounding to fp32 (2^-24) and one to bf16 (8 bits: 2^-8)
        assert torch.allclose(got.double().cpu(), wide, rtol=2.0 ** -8 + 2.0 ** -20, atol=0)


def test_empty_calls():
    k, v, ks, vs = _cache(1, 2, 1, 64)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    a, b = ops.kv_read_fp8(k, v, ks, vs, none, 0)
    assert a.shape == (0, 1, 16, 64) and b.shape == a.shape
    ops.rope_kv_write_fp8(torch.zeros(0, 192, dtype=torch.bfloat16, device=DEV), none,
                          torch.zeros(1, 64, device=DEV), none, k, v, ks, vs, 0, 1, 1, 64, 64)
    assert int(k.view(torch.uint8).count_nonzero()) == 0


def test_offsets_past_32_bits():
    """A pool of more than 2^32 codes: rows written and read at its far end."""
    hkv, d = 8, 128
    nb = (1 << 32) // (hkv * 16 * d) + 9
    k = torch.empty(1, nb, hkv, 16, d, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    v = torch.empty_like(k)
    ks = torch.empty(1, nb, hkv, 16, device=DEV)
    vs = torch.empty_like(ks)
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(3, 3 * hkv * d, generator=g).to(torch.bfloat16)
    cs = torch.cat([torch.ones(1, 64), torch.zeros(1, 64)], dim=1)
    blocks = torch.tensor([nb - 1, 0, nb - 3], dtype=torch.int32)
    slots = blocks * 16 + 5
    ops.rope_kv_write_fp8(qkv.to(DEV), torch.zeros(3, dtype=torch.int32, device=DEV), cs.to(DEV),
                          slots.to(DEV), k, v, ks, vs, 0, hkv, hkv, d, d)
    _, got = ops.kv_read_fp8(k, v, ks, vs, blocks.to(DEV), 0)
    codes, scales = ref.quantise_rows(qkv.view(3, 3, hkv, d)[:, 2])
    assert torch.equal(got[:, :, 5].cpu(), ref.dequantise_rows(codes, scales).to(torch.bfloat16))


def test_refusals():
    k, v, ks, vs = _cache(1, 2, 2, 64)
    i32 = dict(dtype=torch.int32, device=DEV)
    qkv = torch.zeros(4, 6 * 64, dtype=torch.bfloat16, device=DEV)
    pos, slots, cs = torch.zeros(4, **i32), torch.zeros(4, **i32), torch.zeros(2, 64, device=DEV)

    def write(**kw):
        a = dict(qkv=qkv, positions=pos, cos_sin=cs, slots=slots, k_cache=k, v_cache=v, k_scale=ks,
                 v_scale=vs, layer=0, hq=2, hkv=2, d=64, rot=64)
        a.update(kw)
        with pytest.raises(RuntimeError):
            ops.rope_kv_write_fp8(**a)

    write(qkv=qkv.float())
    write(qkv=qkv[:, :-64])
    write(qkv=torch.zeros(4, 6 * 64 + 8, dtype=torch.bfloat16, device=DEV)[:, 4:-4])  # 8-byte rows
    write(k_cache=k.to(torch.bfloat16))
    write(k_scale=ks[:, :1])
    write(k_scale=ks.to(torch.float16))
    write(rot=24)
    write(rot=128)
    write(d=32)
    write(layer=1)
    write(layer=-1)
    write(slots=slots.long())
    write(positions=pos[:2])
    write(cos_sin=cs[:, :32])
    write(q_out=torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV))
    write(slots=slots.cpu())
    blocks = torch.zeros(3, **i32)
    out = torch.empty(3, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (dict(blocks=blocks.long()), dict(layer=2), dict(k_out=out.float()),
                dict(v_out=out[:2]), dict(k_scale=ks.double()), dict(v_cache=v[:, :1])):
        a = dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, blocks=blocks, layer=0, k_out=out,
                 v_out=out.clone())
        a.update(bad)
        with pytest.raises(RuntimeError):
            ops.kv_read_fp8(**a)
    assert math.isfinite(float(ks.sum()))  # the device still answers
