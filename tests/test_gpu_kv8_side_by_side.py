"""Attention over the 8-bit cache in calls that fill the chip with 128 (64) rows a workgroup, at least 448 of them with 64 channels, 320 with
128: many rows, ragged rows, V blocks of very different size, one weight beside thousands, poisoned and missing pages.  References and
tolerances are those of the tests of the same names."""
import pytest
import torch

from tests import test_gpu_kv8_many_rows as M
from tests import test_gpu_kv8_ranges as A
from tests.test_gpu_kv8 import DEV, _filled, _gen
from whisper_amd import kv8

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32

# kv lengths                                  H  Hkv  D   P    T  causal
CALLS = [
    ([200, 201, 263, 700, 448, 256, 320, 511], 32, 32, 64, 64, 200, True),
    ([1500] * 4, 40, 10, 64, 16, 400, False),
    ([0, 1, 399, 1111], 40, 10, 64, 16, 400, True),              # rows that see nothing
    ([4500, 3333], 10, 10, 64, 64, 3100, True),
    ([300, 411, 257, 640], 54, 18, 64, 32, 257, True),           # three heads a kv head
    ([140, 130, 1, 1300], 28, 28, 128, 32, 257, True),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kv,H,Hkv,D,P,T,causal", CALLS)
def test_many_rows(fmt, dtype, kv, H, Hkv, D, P, T, causal):
    M.test_many_rows(fmt, dtype, kv, H, Hkv, D, P, T, causal)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_rows(fmt, dtype, causal):
    M.test_ragged_rows(fmt, dtype, causal, [500, 0, 33, 1, 900, 128, 0, 129], [500, 7, 40, 2222, 950, 64, 0, 129], 64, 32, 64, 32)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("sizes", [(1.0, 1e-37, 1.0, 1e30, 1e-37, 1e-30), (1e-37, 1e30, 1e-37, 1.0, 1e-20, 1e-37), (1e-38, 1e-38, 1e-38, 1e-38, 1.0, 1e-38)])
def test_v_blocks_of_very_different_size(fmt, dtype, sizes):
    A.test_v_blocks_of_very_different_size(fmt, dtype, 200, 112, sizes)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("at", [0, 70, 2990])
def test_one_large_weight_beside_thousands_of_small_ones(dtype, at):
    A.test_one_large_weight_beside_thousands_of_small_ones(dtype, 200, 112, at)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_poisoned_blocks_and_missing_pages_reach_only_the_rows_that_see_them(dtype):
    g = _gen(22)
    B, H, D, T, kv = 4, 64, 64, 250, 400
    c, table = _filled(g, B, 7, H, D, 64, "int8", [kv] * B)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype)
    ln = torch.full((B,), kv, dtype=torch.int32, device=DEV)
    clean = kv8.attention(q, c, table, ln)
    c.v_scale[table[0, 4].long(), 1] = float("nan")          # positions 256 .. of sequence 0, head 1
    table[2, 5] = c.n_pages                                   # positions 320 .. of sequence 2
    out = kv8.attention(q, c, table, ln)
    at = torch.arange(kv - T, kv, device=DEV)
    assert torch.isnan(out[0, at >= 256, 1]).all() and torch.isnan(out[2, at >= 320]).all()
    clean[0, at >= 256, 1], clean[2, at >= 320] = 0, 0
    out[0, at >= 256, 1], out[2, at >= 320] = 0, 0
    assert torch.equal(out, clean)


def test_captured_with_lengths_that_change():
    g = _gen(23)
    B, H, Hkv, D, T, longest = 3, 40, 10, 64, 512, 1500
    c, table = _filled(g, B, 24, Hkv, D, 64, "e4m3", [longest] * B)
    ln = torch.full((B,), longest, dtype=torch.int32, device=DEV)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv8.attention(q, c, table, ln)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, lse = kv8.attention(q, c, table, ln, return_lse=True)
    for kv in ([longest, 50, 700], [0, 512, 1499], [64, 1, 1408]):
        ln.copy_(torch.tensor(kv, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        graph.replay()
        want, want_lse = kv8.attention(q, c, table, ln, return_lse=True)
        assert torch.equal(held, want) and torch.equal(lse, want_lse)
        torch.cuda.synchronize()
        M._check(held, lse, q, c, table, kv, "e4m3", True, D ** -0.5)
