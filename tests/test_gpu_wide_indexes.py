"""Positions, lengths and token ids given in 64 bits mean what they say: one that 32 bits do not hold lies behind every table and outside every
vocabulary, not at what is left of it when its upper half is cut off."""
import pytest
import torch

from tests.test_gpu_kv8 import DEV, _filled, _gen
from tests.test_gpu_verify import _check, _inputs
from whisper_amd import kv8

pytestmark = pytest.mark.gpu
FAR = [1 << 32, (1 << 32) + 5, (1 << 31) + 7, (1 << 62) + 1, -(1 << 32) + 3]


@pytest.mark.parametrize("far", FAR)
def test_positions_and_lengths(far):
    g = _gen(3)
    c, table = _filled(g, 2, 3, 2, 64, 64, "int8", [100, 100])
    x = torch.randn(2, 4, 2, 64, generator=g, device=DEV)
    at = torch.tensor([far, 20], dtype=torch.int64, device=DEV)
    own = table[0].long()
    before = [t[own].view(torch.uint8).clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    kv8.append(c, x, x, table, at)
    for t, b in zip((c.k, c.v, c.k_scale, c.v_scale), before):
        assert torch.equal(t[own].view(torch.uint8), b)
    k, v = kv8.read(c, table, at, 4, dtype=torch.float32)
    assert torch.isnan(k[0]).all() and torch.isnan(v[0]).all() and (k[1] - x[1]).abs().max() < 0.1
    out, lse = kv8.attention(x, c, table, at, causal=False, return_lse=True)
    if far > 0:
        assert torch.isnan(out[0]).all()
    else:
        assert not out[0].any() and (lse[0] == -float("inf")).all()
    assert torch.equal(out[1], kv8.attention(x, c, table, at.clamp(-1, 20).int(), causal=False)[1])
    # rows packed to such an end belong to no sequence
    out = torch.full((8, 2, 64), 7.0, device=DEV)
    start = torch.tensor([0, 4, far], dtype=torch.int64, device=DEV)
    kv8.attention(x.flatten(0, 1), c, table, torch.tensor([50, 50], device=DEV), tok_start=start, out=out)
    assert not (out[:4] == 7.0).any() and (out[4:] == 7.0).all()


@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_token_ids(far, temperature):
    x, _, d, u = _inputs(4, 6, 3, 500, torch.float32, False)
    d = x[:, :3].argmax(-1)
    d[1:, 0] += far - far % (1 << 32) if far % (1 << 32) < 500 else far          # another id with the same lower half
    u[:, :3] = 0.0
    n = torch.tensor([3, 3, 3, far, 3, 3], device=DEV)
    acc, _ = _check(x, d, u, n_drafted=n, temperature=temperature)
    assert acc.tolist() == [3, 0, 0, 0, 0, 0]
