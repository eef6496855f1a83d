"""Tensors without heads: errors or nothing to do, never a division by zero on the host."""
import pytest
import torch

from cascadia_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def _pool(hkv, dtype=torch.bfloat16):
    raw = torch.uint8 if dtype == torch.float8_e4m3fn else dtype
    return torch.zeros(1, 2, hkv, 16, 64, dtype=raw, device=DEV).view(dtype)


@pytest.mark.parametrize("hkv,width", [(0, 128), (0, 0), (2, 0)])
def test_attention(hkv, width):
    k = _pool(hkv)
    q = torch.zeros(1, width, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):
        ops.attn_tree(q, k, k, torch.zeros(1, 2, **I32), torch.tensor([20], **I32),
                      torch.tensor([0, 1], **I32), torch.empty_like(q), 0, 0.125, max_nodes=1)


def test_write_and_read():
    f8 = torch.float8_e4m3fn
    scale = torch.ones(1, 2, 0, 16, device=DEV)
    k, v = ops.kv_read_fp8(_pool(0, f8), _pool(0, f8), scale, scale, torch.zeros(3, **I32), 0)
    assert k.shape == (3, 0, 16, 64) and v.shape == k.shape
    scale = torch.ones(1, 2, 2, 16, device=DEV)
    qkv = torch.zeros(3, 3 * 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):
        ops.rope_kv_write_fp8(qkv, torch.zeros(3, **I32), torch.zeros(2, 64, device=DEV),
                              torch.zeros(3, **I32), _pool(2, f8), _pool(2, f8), scale, scale, 0,
                              -1, 2, 64, 64)
