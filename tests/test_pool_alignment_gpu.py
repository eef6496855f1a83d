"""Pools, scales and workspaces at addresses that the kernels' wide accesses cannot take
are refused on the host."""
import pytest
import torch

from cascadia_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
POOL = (1, 2, 2, 16, 64)


def _shifted(shape, dtype, by):
    """A contiguous tensor ``by`` elements past an aligned address."""
    n = torch.Size(shape).numel()
    raw = torch.uint8 if dtype == torch.float8_e4m3fn else dtype
    t = torch.zeros(n + 64, dtype=raw, device=DEV)[by:by + n].view(shape)
    assert t.data_ptr() % 16 == by * t.element_size() % 16 and t.is_contiguous()
    return t.view(dtype)


def _attn(k, v, ks, vs):
    q = torch.zeros(2, 256, dtype=torch.bfloat16, device=DEV)
    return ops.attn_tree(q, k, v, torch.zeros(1, 2, **I32), torch.tensor([20], **I32),
                         torch.tensor([0, 2], **I32), torch.empty_like(q), 0, 0.125, k_scale=ks,
                         v_scale=vs, max_nodes=2)


@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_attention_pools(cache):
    fp8 = cache == "fp8"
    dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
    good = _shifted(POOL, dtype, 0)
    scale = _shifted(POOL[:4], torch.float32, 0) if fp8 else None
    _attn(good, good, scale, scale)
    bad = [_shifted(POOL, dtype, by) for by in ((1, 4, 8) if fp8 else (1, 4))]
    for b in bad:
        for k, v in ((b, good), (good, b)):
            with pytest.raises(RuntimeError):
                _attn(k, v, scale, scale)
    _attn(_shifted(POOL, dtype, 16), good, scale, scale)
    if fp8:
        odd = _shifted(POOL[:4], torch.float32, 1)
        for ks, vs in ((odd, scale), (scale, odd)):
            with pytest.raises(RuntimeError):
                _attn(good, good, ks, vs)


def test_write_and_read_pools():
    good = _shifted(POOL, torch.float8_e4m3fn, 0)
    scale = torch.ones(POOL[:4], device=DEV)
    qkv = torch.zeros(3, 6 * 64, dtype=torch.bfloat16, device=DEV)
    pos, cs = torch.zeros(3, **I32), torch.zeros(2, 64, device=DEV)

    def both(k, v):
        ops.rope_kv_write_fp8(qkv, pos, cs, pos, k, v, scale, scale, 0, 2, 2, 64, 64)

    both(good, _shifted(POOL, torch.float8_e4m3fn, 8))
    ops.kv_read_fp8(good, _shifted(POOL, torch.float8_e4m3fn, 8), scale, scale, pos[:1], 0)
    for by in (1, 4, 12):
        odd = _shifted(POOL, torch.float8_e4m3fn, by)
        for k, v in ((odd, good), (good, odd)):
            with pytest.raises(RuntimeError):
                both(k, v)
            with pytest.raises(RuntimeError):
                ops.kv_read_fp8(k, v, scale, scale, pos[:1], 0)


def test_logprobs_workspace():
    x = torch.randn(1, 40000, device=DEV)
    t = torch.zeros(1, **I32)
    ws = ops.GemmWorkspace(DEV)
    whole = ws.ws
    ws.ws = whole[1:]
    with pytest.raises(RuntimeError):
        ops.token_logprobs(x, t, 3, workspace=ws)
    ops.token_logprobs(x.expand(700, -1), t.expand(700).contiguous(), 3, workspace=ws)  # unused
    ws.ws = whole
    ops.token_logprobs(x, t, 3, workspace=ws)
