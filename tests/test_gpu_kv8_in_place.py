"""Attention over the 8-bit cache into the memory of its queries: the same, bit for bit, in every shape of a call."""
import pytest
import torch

from tests.test_gpu_kv8 import DEV, _filled, _gen
from whisper_amd import kv8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,H,Hkv,D,T", [([1500], 6, 6, 64, 1), ([9000, 70], 8, 2, 128, 5), ([700, 300], 4, 4, 64, 60), ([300, 411, 257, 640], 54, 18, 64, 257)])
def test_output_in_the_place_of_the_queries(dtype, kv, H, Hkv, D, T):
    g = _gen(T + H)
    B = len(kv)
    c, table = _filled(g, B, -(-max(kv) // 64), Hkv, D, 64, "int8", kv)
    ln = torch.tensor(kv, dtype=torch.int32, device=DEV)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype)
    want = kv8.attention(q, c, table, ln)
    got = kv8.attention(q, c, table, ln, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
