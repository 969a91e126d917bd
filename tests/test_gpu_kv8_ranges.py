"""Attention over the 8-bit cache where magnitudes differ by what f32 can hold: V blocks from 1e-37 to 1e30 beside one another, one
large weight beside thousands of small ones, positions before the first.

Tolerances: those of many rows (tests/test_gpu_kv8_many_rows.py); a result below f32's normal range is off by half its fixed step,
2^-150, more -- in bf16 2^-134 -- and so is the product it comes from (2^-150)."""
import pytest
import torch

from tests.test_gpu_kv8 import DEV, U, _gen, _halves, _noise_cache, _table
from whisper_amd import kv8

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _check(out, lse, q, c, table, S, fmt, scale):
    hk, hv = _halves(c)
    D = c.head_dim
    for b in range(q.shape[0]):
        k, v = (torch.from_numpy(h.tokens(table[b].tolist(), c.page, S)).to(DEV) for h in (hk, hv))
        vs = c.v_scale[table[b].long()].double().repeat_interleave(c.page, 0)[:S]
        for h in range(q.shape[2]):
            qh, kh, vh = q[b, :, h].double(), k[:, h].contiguous(), v[:, h].contiguous()
            s = qh @ kh.t().contiguous() * scale
            l = torch.logsumexp(s, 1)
            p = torch.exp(s - l[:, None])
            o, pv = p @ vh, p @ vh.abs()
            A = (qh.abs() @ kh.abs().t().contiguous() * abs(scale)).amax(1)
            rel = U * (2 * (D + 16) * A + 8 * (A + 1) + S / 16 + 64 + 127)        # 127: the largest |log2| of a V scale, in the exponent
            tol = rel[:, None] * pv + U * o.abs() + 2.0 ** -149
            if q.dtype == BF:
                small = 2.0 ** -25 * S * (p * vs[None, :, h]).amax(1) * (127 if fmt == "int8" else 448)
                tol = tol + (2.0 ** -11 * pv + small[:, None]) * (1 + 2.0 ** -8) + 2.0 ** -8 * o.abs() * (1 + 2.0 ** -8) + 2.0 ** -134
            err = (out[b, :, h].double() - o).abs()
            bad = ~(err <= tol)
            assert not bad.any(), (b, h, bad.nonzero()[:4].tolist(), float(err.max()), float((err / tol).max()))
            assert ((lse[b, :, h].double() - l).abs() <= rel + 4 * U * (l.abs() + 1)).all()


def _cache(g, fmt, k, v):
    B, S, H, D = k.shape
    width = -(-S // 64)
    c = _noise_cache(g, B * width + 1, H, D, 64, fmt)
    table = _table(g, B, width, c.n_pages)
    kv8.append(c, k, v, table, torch.zeros(B, dtype=torch.int32, device=DEV))
    return c, table, torch.full((B,), S, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H", [(1, 2), (24, 2), (200, 96)])             # keys shared by waves (16 and 32 rows), rows side by side
@pytest.mark.parametrize("sizes", [(1e-37,) * 6, (1.0, 1e-37, 1.0, 1e30, 1e-37, 1e-30), (1e-37, 1e30, 1e-37, 1.0, 1e-20, 1e-37),
                                   (1e-38, 1e-38, 1e-38, 1e-38, 1.0, 1e-38)])
def test_v_blocks_of_very_different_size(fmt, dtype, T, H, sizes):
    """A token's share of the sum of weights does not depend on how large its value is."""
    g = _gen(T + H)
    B, D = 2, 64
    S = 64 * len(sizes) - 7
    k = torch.randn(B, S, H, D, generator=g, device=DEV)
    v = torch.randn(B, S, H, D, generator=g, device=DEV) * torch.tensor(sizes, device=DEV).repeat_interleave(64)[:S, None, None]
    q = (torch.randn(B, T, H, D, generator=g, device=DEV) * 3).to(dtype)
    c, table, ln = _cache(g, fmt, k, v)
    out, lse = kv8.attention(q, c, table, ln, causal=False, return_lse=True)
    _check(out, lse, q, c, table, S, fmt, D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H", [(1, 2), (24, 2), (200, 96)])
@pytest.mark.parametrize("at", [0, 70, 2990])
def test_one_large_weight_beside_thousands_of_small_ones(dtype, T, H, at):
    """Together the small ones count as much: 3000 of 2^-11 .. 2^-13 of the largest."""
    g = _gen(31 + T)
    B, D, S = 2, 64, 3000
    k = torch.zeros(B, S, H, D, device=DEV)
    k[..., 0] = -1 - torch.rand(B, S, H, generator=g, device=DEV) * 0.2
    k[:, at, :, 0] = 0.0
    v = torch.randn(B, S, H, D, generator=g, device=DEV).abs()
    v[:, at] *= 0.1
    q = torch.zeros(B, T, H, D, device=DEV)
    q[..., 0] = 7.7
    c, table, ln = _cache(g, "int8", k, v)
    out, lse = kv8.attention(q.to(dtype), c, table, ln, causal=False, scale=1.0, return_lse=True)
    _check(out, lse, q.to(dtype), c, table, S, "int8", 1.0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_positions_before_the_first(dtype):
    """An append skips them, a read gives NaN there, a negative length sees nothing."""
    g = _gen(41)
    c = _noise_cache(g, 4, 2, 64, 16, "int8")
    table = torch.tensor([[1, 2]], dtype=torch.int32, device=DEV)
    x = torch.randn(1, 30, 2, 64, generator=g, device=DEV).to(dtype)
    kv8.append(c, x, x, table, torch.tensor([-19], dtype=torch.int32, device=DEV))
    d = _noise_cache(_gen(41), 4, 2, 64, 16, "int8")
    kv8.append(d, x[:, 19:].contiguous(), x[:, 19:].contiguous(), table, torch.tensor([0], dtype=torch.int32, device=DEV))
    for a, b in ((c.k, d.k), (c.v, d.v), (c.k_scale, d.k_scale), (c.v_scale, d.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    got = kv8.read(c, table, torch.tensor([-19], dtype=torch.int32, device=DEV), 30, dtype=dtype)
    want = kv8.read(d, table, torch.tensor([0], dtype=torch.int32, device=DEV), 11, dtype=dtype)
    for y, w in zip(got, want):
        assert torch.isnan(y[0, :19]).all() and torch.equal(y[0, 19:], w[0])
    out, lse = kv8.attention(x, c, table, torch.tensor([-5], dtype=torch.int32, device=DEV), return_lse=True)
    assert not out.any() and (lse == -float("inf")).all()
