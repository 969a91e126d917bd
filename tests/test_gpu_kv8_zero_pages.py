"""Attention over the 8-bit cache where some pages hold values of zero throughout (their scale is 0): they take part in the sum of the
weights and in nothing else.  Tolerances: those of tests/test_gpu_kv8_weights.py."""
import pytest
import torch

from tests.test_gpu_kv8 import DEV, _gen, _noise_cache, _table
from tests.test_gpu_kv8_weights import BF, F32, _check
from whisper_amd import kv8

pytestmark = pytest.mark.gpu
Z = 0.0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,more", [(1, 2, 0), (1, 1, 100), (24, 2, 0), (200, 112, 0)])      # 16 rows; cut and joined; 32 rows; side by side
@pytest.mark.parametrize("sizes", [(Z, 1e-5, 1e-5), (1e-5, 1e-6, Z), (1e-3, Z, 1e-9, Z), (Z, 1e-37, 1e-37, Z), (1.0, Z, 1e-37), (Z, 1e30, Z), (Z,) * 4, (Z,)])
def test_pages_of_zeros(fmt, dtype, T, H, more, sizes):
    g = _gen(T + H + len(sizes))
    B, D = 2, 64
    sizes = sizes + sizes[-1:] * more
    S = 64 * len(sizes) - 7
    k = torch.randn(B, S, H, D, generator=g, device=DEV)
    v = torch.randn(B, S, H, D, generator=g, device=DEV) * torch.tensor(sizes, device=DEV).repeat_interleave(64)[:S, None, None]
    width = len(sizes)
    c = _noise_cache(g, B * width + 1, H, D, 64, fmt)
    table = _table(g, B, width, c.n_pages)
    kv8.append(c, k, v, table, torch.zeros(B, dtype=torch.int32, device=DEV))
    assert ((c.v_scale[table.long()] == 0) == (torch.tensor(sizes, device=DEV) == 0)[:, None]).all()
    q = (torch.randn(B, T, H, D, generator=g, device=DEV) * 3).to(dtype)
    out, lse = kv8.attention(q, c, table, torch.full((B,), S, dtype=torch.int32, device=DEV), causal=False, return_lse=True)
    _check(out, lse, q, c, table, [S] * B, False, D ** -0.5)
    if not any(sizes):
        assert not out.any()
