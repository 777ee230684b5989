"""Derivatives of the decoding operators that no kernel computes, on the CPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from torsh_b200.ops.kv_cache import kv_cache_write


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8])
def test_cache_writes_refuse_tangents(dtype):
    """What is read back would not carry them."""
    kp, vp = (torch.zeros(2, 1, 16, 8, dtype=dtype) for _ in range(2))
    ks, vs = (torch.zeros(2, 1, 16) if dtype == torch.int8 else None for _ in range(2))
    table, start, k = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.ones(1, 3, 1, 8)
    with fwd.dual_level():
        d = fwd.make_dual(k, k)
        for a, b in ((d, k), (k, d)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                kv_cache_write(a, b, kp, vp, table, start, None, ks, vs)
    assert not kp.any()
    kv_cache_write(k, k, kp, vp, table, start, None, ks, vs)
    assert kp[0, 0, :3].ne(0).all()
