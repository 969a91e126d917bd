"""Attention over the 8-bit cache where the weights that make the result are small beside the largest one: a key that holds nearly all
of a row's weight and has no value (an attention sink), and scores spread over hundreds.

The reference is 64-bit arithmetic on the cache's own values.  With u = 2^-24 an output element is off by at most
    u * [ 2 (D + 16) A  +  8 (A + 1)  +  S / 16 + 64 + 127 ] * sum p|v|  +  u |o|
(A = the row's largest scale * sum |q||k|; a score is off by at most (D + 16) u A and enters numerator and sum; 8 (A + 1) for the
exponential and its argument; S / 16 + 64 for the longest chain of additions; 127 for the logarithm of a V scale in the exponent).  The
weights of bf16 queries are two bf16 planes: the first is off by 2^-8 of the weight, the second by 2^-8 of that, 2^-16 sum p|v|
altogether, and the result is rounded to bf16, 2^-8 |o|.  Nothing in this depends on the largest weight: a row whose largest weight
meets a value of zero has its result from the others, to the same relative error -- as long as f32 holds them: weights, and planes of
them, below 2^-126 of the largest weight * V scale are 0.  At most three planes of S weights are lost so, times codes of up to `top`:
2^-124 S top max(vs) more.  Results below f32's normal range are off by half a step of it, 2^-150, and so is the product they come from
(in bf16 by 2^-134)."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv8 import CASES, DEV, U, _filled, _gen, _halves, _noise_cache, _table
from whisper_amd import kv8

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _check(out, lse, q, c, table, kv, causal, scale):
    hk, hv = _halves(c)
    D, G = c.head_dim, q.shape[2] // c.n_kv_heads
    for b, S in enumerate(kv):
        if S == 0:
            assert not out[b].any() and (lse[b] == -float("inf")).all()
            continue
        k, v = (torch.from_numpy(np.ascontiguousarray(h.tokens(table[b].tolist(), c.page, S))).to(DEV) for h in (hk, hv))
        n = q.shape[1]
        ends = torch.arange(n, device=DEV) + (S - n + 1) if causal else torch.full((n,), S, device=DEV)
        hide = torch.arange(S, device=DEV)[None, :] >= ends[:, None]
        some = ~hide.all(1)
        for h in range(q.shape[2]):
            qh, kh, vh = q[b, :, h].double(), k[:, h // G].contiguous(), v[:, h // G].contiguous()
            s = (qh @ kh.t().contiguous() * scale).masked_fill(hide, -float("inf"))
            l = torch.logsumexp(s, 1)
            p = torch.exp(s - torch.where(some, l, 0.0)[:, None])
            o, pv = p @ vh, p @ vh.abs()
            A = (qh.abs() @ kh.abs().t().contiguous() * abs(scale)).masked_fill(hide, 0.0).amax(1)
            rel = U * (2 * (D + 16) * A + 8 * (A + 1) + S / 16 + 64 + 127)
            lost = 2.0 ** -124 * S * (127 if c.k.dtype == torch.int8 else 448) * float(c.v_scale[table[b, : -(-S // c.page)].long(), h // G].max())
            tol = rel[:, None] * pv + U * o.abs() + lost + 2.0 ** -149
            if q.dtype == BF:
                tol = tol + 2.0 ** -16 * pv * (1 + 2.0 ** -8) + 2.0 ** -8 * o.abs() * (1 + 2.0 ** -8) + 2.0 ** -134
            err = (out[b, :, h].double() - o).abs()
            bad = ~(err <= tol)
            assert not bad.any(), (b, h, bad.nonzero()[:4].tolist(), float(err.max()), float((err / tol).max()))
            assert (lse[b, ~some, h] == -float("inf")).all()
            assert ((lse[b, some, h].double() - l[some]).abs() <= (rel + 4 * U * (l.abs() + 1))[some]).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,S", [(1, 2, 1500), (1, 1, 9000), (24, 2, 3000), (200, 112, 700)])      # 16 rows; cut and joined; 32 rows; side by side
@pytest.mark.parametrize("gap", [10, 17.5, 30, 60])
def test_a_key_with_all_the_weight_and_no_value(fmt, dtype, T, H, S, gap):
    g = _gen(int(gap) + T)
    B, D = 2, 64
    k = torch.zeros(B, S, H, D, device=DEV)
    k[..., 0] = -1 - 0.2 * torch.rand(B, S, H, generator=g, device=DEV)
    k[:, 70, :, 0] = 0.0
    v = torch.randn(B, S, H, D, generator=g, device=DEV) + 0.5
    v[:, 70] = 0.0
    width = -(-S // 64)
    c = _noise_cache(g, B * width + 1, H, D, 64, fmt)
    table = _table(g, B, width, c.n_pages)
    kv8.append(c, k, v, table, torch.zeros(B, dtype=torch.int32, device=DEV))
    q = torch.zeros(B, T, H, D, device=DEV)
    q[..., 0] = gap
    q = q.to(dtype)
    out, lse = kv8.attention(q, c, table, torch.full((B,), S, dtype=torch.int32, device=DEV), causal=False, scale=1.0, return_lse=True)
    _check(out, lse, q, c, table, [S] * B, False, 1.0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("spread", [1.0, 12.0])
@pytest.mark.parametrize("kv,H,Hkv,D,P,T,causal", CASES + [([1500] * 4, 40, 10, 64, 16, 400, False), ([140, 130, 1, 1300], 48, 48, 128, 32, 257, True)])
def test_attention_to_the_rounding_of_the_result(fmt, dtype, spread, kv, H, Hkv, D, P, T, causal):
    g = _gen(sum(kv) + H + D + T + 1)
    B, width = len(kv), max(1, (max(kv) + P - 1) // P) + 1
    c, table = _filled(g, B, width, Hkv, D, P, fmt, kv)
    q = (torch.randn(B, T, H, D, generator=g, device=DEV) * spread).to(dtype)
    out, lse = kv8.attention(q, c, table, torch.tensor(kv, dtype=torch.int32, device=DEV), causal=causal, return_lse=True)
    _check(out, lse, q, c, table, kv, causal, D ** -0.5)
