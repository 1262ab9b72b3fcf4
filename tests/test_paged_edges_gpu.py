"""Calls of the paged batch-decode operators at the edges of what their documentation allows.

Roundings as in test_paged_gpu.py: bf16 half a step is 2^-8 of the value, fp32 2^-24.
"""
import pytest

from tests.conftest import has_gpu
from tests.test_paged_gpu import Batch, _no_timeouts  # noqa: F401

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not has_gpu(), reason="no CUDA device")]


# ----------------------------------------------------------------------------- attention
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("B,q,prefix", [(2, 150, 300), (2, 1, 30), (40, 1, 300), (4, 1, 300)])
def test_attn_output_on_any_16_byte_boundary(built_lib, hd, B, q, prefix):
    """An output 16, 32 or 48 bytes into a buffer gets the bits of an aligned one; nothing beside it is written."""
    import torch
    b = Batch(8, 4, hd, 16, prefix, [160] * B, [q] * B, seed=hd + B)
    want = b.call()
    n = want.numel()
    for off in (8, 16, 24):
        flat = torch.full((n + 32,), 7.0, dtype=torch.bfloat16, device="cuda")
        out = flat[off:off + n].view(want.shape)
        assert out.data_ptr() % 32 == (16 if off % 16 else 0)
        b.call(out=out)
        assert torch.equal(out, want)
        assert (flat[:off] == 7.0).all() and (flat[off + n:] == 7.0).all()
