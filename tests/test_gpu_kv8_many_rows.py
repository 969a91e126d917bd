"""GPU parity of attention over the 8-bit cache where many rows share a sequence's keys: prompts, and batches that fill the chip with
row tiles (four waves side by side); and ragged rows over sequences long enough to be cut and joined.

The reference is 64-bit arithmetic on the cache's own values.  With u = 2^-24 an output element of f32 queries is off by at most
    u * [ 2 (D + 16) A  +  8 (A + 1)  +  S / 16 + 64 ] * sum p|v|   +  u |o|
(A = the row's largest scale * sum |q||k|; a score is off by at most (D + 16) u A and enters numerator and sum; 8 (A + 1) for the
exponential and its argument; S / 16 + 64 for the longest chain of additions).  bf16 queries add the rounding of each weight to f16,
2^-11 of it and 2^-25 of the largest weight * V scale where it runs out of exponent (over S keys and codes of up to 127 or 448), and the
rounding of the result, 2^-8 |o|."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv8 import DEV, U, _filled, _gen, _halves
from whisper_amd import kv8

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def _check(out, lse, q, c, table, kv, fmt, causal, scale, start=None):
    """out, lse, q: [B, T, ...], or [N, ...] with `start` as a list."""
    hk, hv = _halves(c)
    for b, S in enumerate(kv):
        rows = slice(start[b], start[b + 1]) if start else b
        qb, ob, lb = q[rows].double(), out[rows].double(), lse[rows].double()
        n, H, D = qb.shape
        if n == 0:
            continue
        if S == 0:
            assert not ob.any() and (lb == -float("inf")).all()
            continue
        pages = table[b].tolist()
        k, v = _cuda(hk.tokens(pages, c.page, S)), _cuda(hv.tokens(pages, c.page, S))
        vs = float(c.v_scale[table[b, : -(-S // c.page)].long()].max())
        ends = torch.arange(n, device=DEV) + (S - n + 1) if causal else torch.full((n,), S, device=DEV)
        sees = torch.arange(S, device=DEV)[None, :] < ends[:, None]
        some = sees.any(1)
        G = H // c.n_kv_heads
        for h in range(H):
            kh, vh = k[:, h // G].contiguous(), v[:, h // G].contiguous()
            qh = qb[:, h].contiguous()
            s = (qh @ kh.t().contiguous() * scale).masked_fill(~sees, -float("inf"))
            l = torch.logsumexp(s, 1)
            p = torch.exp(s - torch.where(some, l, 0.0)[:, None])
            o, pv = p @ vh, p @ vh.abs()
            A = (qh.abs() @ kh.abs().t().contiguous() * abs(scale)).masked_fill(~sees, 0.0).amax(1)
            rel = U * (2 * (D + 16) * A + 8 * (A + 1) + S / 16 + 64)
            tol = rel[:, None] * pv + U * o.abs()
            if q.dtype == BF:
                small = 2.0 ** -25 * S * p.amax(1) * vs * (127 if fmt == "int8" else 448)
                tol = tol + (2.0 ** -11 * pv + small[:, None]) * (1 + 2.0 ** -8) + 2.0 ** -8 * o.abs() * (1 + 2.0 ** -8)
            err = (ob[:, h] - o).abs()
            bad = ~(err <= tol)
            assert not bad.any(), (b, h, bad.nonzero()[:4].tolist(), float(err.max()), float((err / tol.clamp_min(1e-300)).max()))
            assert (lb[~some, h] == -float("inf")).all() and not ob[~some, h].any()
            assert ((lb[some, h] - l[some]).abs() <= (rel + 4 * U * (l.abs() + 1))[some]).all()


# kv lengths                            H  Hkv  D   P    T  causal    -- 128 rows (f32 of 128 channels 64) a workgroup, 384 or more
MANY = [
    ([200, 201, 263, 700, 448, 256, 320, 511], 24, 24, 64, 64, 200, True),
    ([1500] * 4, 32, 8, 64, 16, 400, False),
    ([0, 1, 399, 1111], 32, 8, 64, 16, 400, True),               # rows that see nothing; a table longer than one look at 64 pages
    ([140, 130, 1, 1300], 48, 48, 128, 32, 257, True),
    ([70, 65, 64, 63], 96, 96, 128, 256, 33, False),
    ([4500, 3333], 8, 8, 64, 64, 3100, True),
    ([129] * 12, 32, 32, 64, 128, 129, True),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kv,H,Hkv,D,P,T,causal", MANY)
def test_many_rows(fmt, dtype, kv, H, Hkv, D, P, T, causal):
    g = _gen(sum(kv) + H + D + T)
    B, width = len(kv), (max(kv) + P - 1) // P + 1
    c, table = _filled(g, B, width, Hkv, D, P, fmt, kv)
    ln = torch.tensor(kv, dtype=torch.int32, device=DEV)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype)
    for scale in (D ** -0.5, -0.1):
        out, lse = kv8.attention(q, c, table, ln, causal=causal, scale=scale, return_lse=True)
        _check(out, lse, q, c, table, kv, fmt, causal, scale)
        assert torch.equal(out, kv8.attention(q, c, table, ln, causal=causal, scale=scale))


RAGGED = [
    # tokens                              keys                                      H  Hkv  D   P
    ([500, 0, 33, 1, 900, 128, 0, 129], [500, 7, 40, 2222, 950, 64, 0, 129], 32, 16, 64, 32),      # 64 keys for 128 tokens
    ([8 * (i % 2) + i % 3 for i in range(300)], [5 * i % 700 for i in range(300)], 16, 2, 64, 16),     # more than 256 sequences
    ([300, 0, 700, 65], [300, 0, 4700, 1065], 32, 32, 128, 64),
    ([20, 0, 3], [5000, 100, 2600], 8, 2, 128, 64),                                                 # few rows: keys cut and joined
    ([9, 0, 1, 30, 0], [2300, 0, 4097, 30, 11], 6, 3, 64, 128),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,kv,H,Hkv,D,P", RAGGED)
def test_ragged_rows(fmt, dtype, causal, n, kv, H, Hkv, D, P):
    g = _gen(sum(kv) + H + D)
    B, width = len(kv), (max(kv) + P - 1) // P
    c, table = _filled(g, B, width, Hkv, D, P, fmt, kv)
    start = [0] + list(np.cumsum(n))
    N = start[-1] + 3                                        # rows behind the last sequence stay as they are
    q = torch.randn(N, H * D + 4, generator=g, device=DEV).to(dtype)[:, 4:].view(N, H, D)     # not 16-byte aligned in bf16
    out = torch.full((N, H, D), 7.0, dtype=dtype, device=DEV)
    _, lse = kv8.attention(q, c, table, torch.tensor(kv, dtype=torch.int32, device=DEV), causal=causal, return_lse=True, out=out,
                           tok_start=torch.tensor(start, dtype=torch.int32, device=DEV))
    assert (out[start[-1]:] == 7.0).all()
    _check(out, lse, q, c, table, kv, fmt, causal, D ** -0.5, [int(x) for x in start])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_poisoned_blocks_and_missing_pages_reach_only_the_rows_that_see_them(dtype):
    g = _gen(21)
    B, H, D, T, kv = 4, 64, 64, 250, 400
    c, table = _filled(g, B, 7, H, D, 64, "e4m3", [kv] * B)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype)
    ln = torch.full((B,), kv, dtype=torch.int32, device=DEV)
    clean = kv8.attention(q, c, table, ln)
    assert torch.isfinite(clean).all()
    c.k_scale[table[0, 4].long(), 1] = float("nan")          # positions 256 .. of sequence 0, head 1
    c.v_scale[table[1, 0].long(), 0] = float("inf")          # positions 0 .. of sequence 1, head 0
    table[2, 5] = 1 << 29                                     # positions 320 .. of sequence 2
    ln[3] = 1000                                              # behind the table: causal rows all see the missing pages
    out = kv8.attention(q, c, table, ln)
    at = torch.arange(kv - T, kv, device=DEV)
    assert torch.isnan(out[0, at >= 256, 1]).all() and torch.equal(out[0, at < 256, 1], clean[0, at < 256, 1])
    others = [h for h in range(H) if h != 1]
    assert torch.equal(out[0][:, others], clean[0][:, others])
    assert not torch.isfinite(out[1, :, 0]).any() and torch.equal(out[1, :, 1:], clean[1, :, 1:])
    assert torch.isnan(out[2, at >= 320]).all() and torch.equal(out[2, at < 320], clean[2, at < 320])
    assert torch.isnan(out[3]).all()


@pytest.mark.parametrize("packed", [False, True])
def test_tables_far_wider_than_their_sequences(packed):
    """One long sequence among many short ones, under a table that could hold half a million tokens: the scratch for its parts is
    bounded, so its keys are cut more coarsely."""
    g = _gen(51)
    B, T, H, Hkv, D, P, kv = 128, 8, 4, 1, 64, 256, [90 + i % 50 for i in range(127)] + [20000]
    c, table = _filled(g, B, 79, Hkv, D, P, "int8", kv)
    wide = torch.full((B, 2000), -1, dtype=torch.int32, device=DEV)
    wide[:, :79] = table
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(BF)
    start = [T * i for i in range(B + 1)] if packed else None
    kw = {"tok_start": torch.tensor(start, dtype=torch.int32, device=DEV)} if packed else {}
    x = q.flatten(0, 1) if packed else q
    out, lse = kv8.attention(x, c, wide, torch.tensor(kv, dtype=torch.int32, device=DEV), return_lse=True, **kw)
    _check(out, lse, x, c, wide, kv, "int8", True, D ** -0.5, start)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kv,H,Hkv,D,T", [([100, 2500, 0, 64], 6, 2, 64, 1), ([100, 900], 15, 3, 64, 7), ([9000, 77], 7, 1, 128, 3),
                                          ([300, 411, 257, 640], 48, 16, 64, 257), ([500, 130], 36, 12, 128, 600)])
def test_query_heads_in_threes_fives_and_sevens(dtype, causal, kv, H, Hkv, D, T):
    """Heads a kv head that are no power of two, in every shape of a call."""
    g = _gen(H + D + T)
    B, P = len(kv), 64
    c, table = _filled(g, B, max(1, -(-max(kv) // P)), Hkv, D, P, "e4m3", kv)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype)
    out, lse = kv8.attention(q, c, table, torch.tensor(kv, dtype=torch.int32, device=DEV), causal=causal, return_lse=True)
    _check(out, lse, q, c, table, kv, "e4m3", causal, D ** -0.5)


def test_two_graphs_of_cut_sequences_with_lengths_that_change():
    """Each graph has its own parts; lengths, tables and queries are read when it is replayed."""
    g = _gen(61)
    B, H, Hkv, D, P, T, longest = 3, 8, 2, 128, 64, 2, 9000
    c, table = _filled(g, B, 141, Hkv, D, P, "int8", [longest] * B)
    ln = torch.tensor([longest, 50, 4000], dtype=torch.int32, device=DEV)
    qs = [torch.randn(B, T, H, D, generator=g, device=DEV).to(BF) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv8.attention(qs[0], c, table, ln)
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(kv8.attention(q, c, table, ln, return_lse=True))
    for kv in ([longest, 50, 4000], [0, 8999, 1], [70, 2112, 2113], [8192, 8192, 8192]):
        ln.copy_(torch.tensor(kv, dtype=torch.int32))
        for q in qs:
            q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        for x in graphs:
            x.replay()
        for q, (out, lse) in zip(qs, held):
            want, want_lse = kv8.attention(q, c, table, ln, return_lse=True)
            assert torch.equal(out, want) and torch.equal(lse, want_lse)
            torch.cuda.synchronize()
            _check(out, lse, q, c, table, kv, "int8", True, D ** -0.5)
