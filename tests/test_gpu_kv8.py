"""GPU parity of the 8-bit paged key/value cache against the 64-bit restatement in tests/kv8_oracle.py.

Append and read are exact: the codes follow from the definition whatever the order of evaluation, a value is one product.
Attention: with u = 2^-24 the f32 kernel's error of an output element is at most
    u * [ 2 (D + 16) A  +  8 (A + 1)  +  S / 16 + 64 ] * sum p|v|   +  u |o|
A = the row's largest scale * sum |q||k| (a score is a sum of D products, each sum and the scaling off by at most (D + 16) u A;
a score enters the numerator and the sum, hence 2), 8 (A + 1) for the exponential and its argument, S / 16 + 64 for the
longest chain of additions over the S keys (keys are dealt to lanes of at least 16).  bf16 adds the rounding of the
probabilities that enter the product, eps/2 sum p|v|, and of the result, eps/2 |o|, eps/2 = 2^-8."""
import math

import numpy as np
import pytest
import torch

from tests import kv8_oracle as R
from whisper_amd import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    x = torch.randn(shape, generator=g, device=DEV)
    return x * (1 + 5 * (torch.rand(shape[-1], generator=g, device=DEV) < 0.1))


def _noise_cache(g, pages, heads, dim, page, fmt):
    """A cache full of leftovers: any bytes, any scales, NaN among both."""
    c = kv8.KV8Cache.allocate(pages, heads, dim, page, fmt, DEV)
    for x in (c.k, c.v):
        x.view(torch.uint8).copy_(torch.randint(0, 256, x.shape, generator=g, device=DEV, dtype=torch.int32))
    for s in (c.k_scale, c.v_scale):
        s.copy_(torch.randn(s.shape, generator=g, device=DEV))
        s[::2] = float("nan")
    return c


def _table(g, B, width, pages):
    return torch.randperm(pages, generator=g, device=DEV)[: B * width].view(B, width).to(torch.int32)


def _halves(c):
    return R.Half(c.k, c.k_scale, False), R.Half(c.v, c.v_scale, True)


def _seqs(x, tok_start=None):
    x = x.detach().float().cpu().numpy().astype(np.float64)
    if tok_start is None:
        return list(x)
    t = tok_start.cpu().tolist()
    return [x[a:b] for a, b in zip(t, t[1:])]


def _same(c, want_k, want_v):
    """Scales bit for bit and the value of every code whose value is specified (the codes of a poisoned block are not)."""
    for (codes, scale, tr), want in zip(((c.k, c.k_scale, False), (c.v, c.v_scale, True)), (want_k, want_v)):
        got = R.Half(codes, scale, tr)
        assert np.array_equal(got.s, want.s, equal_nan=True)
        said = ~np.isinf(want.c)
        assert np.array_equal(got.c[said], want.c[said], equal_nan=True)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,P,H,T,pos", [(64, 64, 3, 1, [0, 5, 63, 64, 200]), (64, 16, 2, 37, [0, 1, 15, 16, 40]),
                                         (128, 32, 1, 70, [0, 31, 33, 64, 2]), (64, 128, 2, 300, [0, 127, 1, 128, 64]),
                                         (128, 256, 1, 2, [255, 0, 254, 1, 511])])
def test_append_is_exact(fmt, dtype, D, P, H, T, pos):
    g = _gen(D + P + T)
    B, width = len(pos), (max(pos) + T + P - 1) // P
    c = _noise_cache(g, B * width + 2, H, D, P, fmt)
    table = _table(g, B, width, c.n_pages)
    at = torch.tensor(pos, dtype=torch.int32, device=DEV)
    # earlier tokens first, so that the call under test meets blocks with scales of their own (small values: some have to grow)
    first = _randn(g, int(sum(pos)), H, D).to(dtype) * 0.3
    start = torch.tensor([0] + list(np.cumsum(pos)), dtype=torch.int32, device=DEV)
    want_k, want_v = _halves(c)
    kv8.append(c, first, -first, table, torch.zeros_like(at), tok_start=start)
    R.append(want_k, fmt, _seqs(first, start), table.tolist(), [0] * B)
    R.append(want_v, fmt, _seqs(-first, start), table.tolist(), [0] * B)
    _same(c, want_k, want_v)
    k, v = _randn(g, B, T, H, D).to(dtype), _randn(g, B, T, H, D).to(dtype)
    kv8.append(c, k, v, table, at)
    R.append(want_k, fmt, _seqs(k), table.tolist(), pos)
    R.append(want_v, fmt, _seqs(v), table.tolist(), pos)
    _same(c, want_k, want_v)
    # and read back: every token so far, rounded once
    n = [p + T for p in pos]
    start = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32, device=DEV)
    got = kv8.read(c, table, torch.zeros_like(at), sum(n), tok_start=start, dtype=dtype)
    for x, half in zip(got, (want_k, want_v)):
        ref = np.concatenate([half.tokens(table[b].tolist(), P, n[b]) for b in range(B)])
        assert torch.equal(x.cpu(), torch.from_numpy(ref).float().to(dtype))
    some = kv8.read(c, table, at, T, dtype=dtype)
    for x, whole in zip(some, got):
        for b in range(B):
            assert torch.equal(x[b], whole[int(start[b]) + pos[b]: int(start[b]) + n[b]])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_token_by_token_growth_is_exact_and_stays_close(fmt):
    """Blocks whose values keep growing: every token of 70 is stored alone.  Errors of int8 stay within one and a half steps of the
    final scale (half a step when stored, at most one for all re-roundings: 1/2 + 1/4 + ... of it), of e4m3 within half a step of
    the value, or of the smallest step where the scale has left it behind."""
    g = _gen(3)
    P, D, H = 64, 64, 2
    c = _noise_cache(g, 4, H, D, P, fmt)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    x = _randn(g, 1, 70, H, D) * torch.logspace(-3, 1, 70, device=DEV)[None, :, None, None]
    want_k, want_v = _halves(c)
    for t in range(70):
        kv8.append(c, x[:, t:t + 1], x[:, t:t + 1], table, torch.tensor([t], dtype=torch.int32, device=DEV))
        for half in (want_k, want_v):
            R.append(half, fmt, _seqs(x[:, t:t + 1]), table.tolist(), [t])
    _same(c, want_k, want_v)
    k, v = kv8.read(c, table, torch.zeros(1, dtype=torch.int32, device=DEV), 70, dtype=torch.float32)
    for got, scale in ((k, c.k_scale), (v, c.v_scale)):
        s = scale[table[0].long()][torch.arange(70, device=DEV) // P][None, :, :, None]
        err = (got - x).abs()
        if fmt == "int8":
            assert (err <= 1.5 * s * (1 + 1e-5)).all()
        else:
            assert (err <= x.abs() * 2.0 ** -4 + 1.5 * s * 2.0 ** -10).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_zeros_tiny_huge_and_non_finite(fmt):
    g = _gen(4)
    P, D, H = 16, 64, 4
    c = _noise_cache(g, 4, H, D, P, fmt)
    table = torch.tensor([[3, 1, 0]], dtype=torch.int32, device=DEV)
    x = torch.zeros(1, 40, H, D, device=DEV)
    x[0, :, 1] = 1e-42                               # below the smallest normal number
    x[0, :, 2] = torch.randn(40, D, generator=g, device=DEV) * 1e37
    x[0, 5, 2, 0], x[0, 20, 2, 1] = 3.4e38, -3.4e38
    x[0, :, 3] = torch.randn(40, D, generator=g, device=DEV)
    x[0, 20, 3, 7], x[0, 21, 3, 8] = float("nan"), float("inf")
    want_k, want_v = _halves(c)
    for t0, t1 in ((0, 3), (3, 17), (17, 40)):
        kv8.append(c, x[:, t0:t1], x[:, t0:t1], table, torch.tensor([t0], dtype=torch.int32, device=DEV))
        for half in (want_k, want_v):
            R.append(half, fmt, _seqs(x[:, t0:t1]), table.tolist(), [t0])
    _same(c, want_k, want_v)
    assert math.isnan(float(c.k_scale[1, 3])) and math.isfinite(float(c.k_scale[0, 3]))
    # a block of zeros takes the scale of what comes after; a poisoned one is clean again once begun anew
    y = torch.randn(1, 8, H, D, generator=g, device=DEV)
    kv8.append(c, y, y, table, torch.tensor([40], dtype=torch.int32, device=DEV))
    kv8.append(c, y, y, table, torch.tensor([16], dtype=torch.int32, device=DEV))
    for half in (want_k, want_v):
        R.append(half, fmt, _seqs(y), table.tolist(), [40])
        R.append(half, fmt, _seqs(y), table.tolist(), [16])
    _same(c, want_k, want_v)
    assert math.isfinite(float(c.k_scale[1, 3]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_packed_strided_misaligned_and_empty_sequences(dtype):
    g = _gen(5)
    P, D, H = 32, 64, 2
    n, pos = [5, 0, 33, 1, 0], [30, 7, 0, 31, 64]
    c = _noise_cache(g, 16, H, D, P, "int8")
    table = _table(g, 5, 3, 16)
    start = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32, device=DEV)
    # rows of a fused q|k|v product, with rows behind the last sequence; and the same shifted by one element
    fused = _randn(g, sum(n) + 4, 3 * H * D + 8).to(dtype)
    for off in (0, 1):
        k = fused[:, off + H * D: off + 2 * H * D].view(-1, H, D)
        v = fused[:, off + 2 * H * D: off + 3 * H * D].view(-1, H, D)
        want_k, want_v = _halves(c)
        kv8.append(c, k, v, table, torch.tensor(pos, dtype=torch.int32, device=DEV), tok_start=start)
        R.append(want_k, "int8", _seqs(k, start), table.tolist(), pos)
        R.append(want_v, "int8", _seqs(v, start), table.tolist(), pos)
        _same(c, want_k, want_v)


def test_pages_that_do_not_exist_are_skipped():
    g = _gen(6)
    P, D, H = 16, 64, 1
    c = _noise_cache(g, 3, H, D, P, "e4m3")
    before = [x.view(torch.uint8).clone() for x in (c.k, c.v)]
    table = torch.tensor([[0, -1, 3], [1 << 30, 2, -(1 << 30)]], dtype=torch.int32, device=DEV)
    x = _randn(g, 2, 64, H, D)                       # 64 tokens: also past the three columns of the table
    want_k, want_v = _halves(c)
    kv8.append(c, x, x, table, torch.zeros(2, dtype=torch.int32, device=DEV))
    for half in (want_k, want_v):
        R.append(half, "e4m3", _seqs(x), table.tolist(), [0, 0])
    _same(c, want_k, want_v)
    assert torch.equal(c.k.view(torch.uint8)[1], before[0][1]) and torch.equal(c.v.view(torch.uint8)[1], before[1][1])
    k, v = kv8.read(c, table, torch.zeros(2, dtype=torch.int32, device=DEV), 64, dtype=torch.float32)
    for got in (k, v):
        assert torch.isnan(got[0, 16:]).all() and torch.isfinite(got[0, :16]).all()
        assert torch.isnan(got[1, :16]).all() and torch.isfinite(got[1, 16:32]).all() and torch.isnan(got[1, 32:]).all()
    # attention: rows that see only good pages are right, the others NaN
    q = _randn(g, 2, 20, 1, D)
    out = kv8.attention(q, c, table, torch.tensor([20, 0], dtype=torch.int32, device=DEV))
    assert torch.isfinite(out[0, :16]).all() and torch.isnan(out[0, 16:]).all() and not out[1].any()
    # a length behind the table
    out = kv8.attention(q[:, :1].contiguous(), c, table, torch.tensor([16, 49], dtype=torch.int32, device=DEV), causal=False)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()


def _filled(g, B, width, H, D, P, fmt, kv):
    """A cache whose sequences hold kv[b] tokens, everything else leftovers."""
    c = _noise_cache(g, B * width + 1, H, D, P, fmt)
    table = _table(g, B, width, c.n_pages)
    start = torch.tensor([0] + list(np.cumsum(kv)), dtype=torch.int32, device=DEV)
    x = _randn(g, int(sum(kv)), H, D)
    y = _randn(g, int(sum(kv)), H, D)
    kv8.append(c, x, y, table, torch.zeros(B, dtype=torch.int32, device=DEV), tok_start=start)
    return c, table


def _check_attention(out, lse, q, c, table, kv, causal, scale, tok_start=None):
    hk, hv = _halves(c)
    bf = q.dtype == torch.bfloat16
    worst = 0.0
    outs, lses = _seqs(out, tok_start), _seqs(lse, tok_start) if lse is not None else None
    for b, qs in enumerate(_seqs(q, tok_start)):
        pages = table[b].tolist()
        k, v = hk.tokens(pages, c.page, kv[b]), hv.tokens(pages, c.page, kv[b])
        o, l, pv, A = R.attention(qs, k, v, causal, scale)
        S, D = kv[b], c.head_dim
        rel = U * (2 * (D + 16) * A + 8 * (A + 1) + S / 16 + 64)
        tol = rel[..., None] * pv + U * np.abs(o)
        if bf:
            tol = tol + 2.0 ** -8 * (pv * (1 + 2.0 ** -8) + np.abs(o))
        bad = ~(np.abs(outs[b] - o) <= tol)
        assert not bad.any(), (b, np.argwhere(bad)[:4], np.abs(outs[b] - o).max(), float((np.abs(outs[b] - o) / np.maximum(tol, 1e-30)).max()))
        if len(o):
            worst = max(worst, float((np.abs(outs[b] - o) / np.maximum(tol, 1e-30)).max()))
        if lses is not None:
            fine = np.isfinite(l)
            assert np.array_equal(fine, np.isfinite(lses[b])) and (lses[b][~fine] == -np.inf).all()
            assert (np.abs(lses[b][fine] - l[fine]) <= (rel + 4 * U * (np.abs(l) + 1))[fine]).all()
    return worst


CASES = [
    # B kv lengths                       H  Hkv D   P    T  causal
    ([1500, 1500], 6, 6, 64, 64, 1, False),
    ([1, 2, 15, 16, 17, 63, 64, 65, 448], 2, 2, 64, 16, 1, True),
    ([0, 1, 130, 257], 4, 2, 64, 64, 1, False),
    ([5, 64, 700, 2049], 8, 2, 128, 32, 5, True),
    ([3, 33, 1000], 8, 1, 64, 128, 3, True),
    ([170, 171, 300], 3, 3, 64, 64, 170, True),
    ([1500, 37], 4, 2, 128, 64, 90, False),
    ([513, 400, 512], 4, 4, 64, 256, 130, True),
    ([9000], 4, 1, 64, 64, 2, True),
    ([4, 2, 0, 90], 2, 1, 64, 16, 6, True),             # more query tokens than keys: rows that see nothing
    ([600], 32, 2, 64, 64, 7, False),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,H,Hkv,D,P,T,causal", CASES)
def test_attention(fmt, dtype, kv, H, Hkv, D, P, T, causal):
    g = _gen(sum(kv) + H + D + T)
    B, width = len(kv), max(1, (max(kv) + P - 1) // P) + 1
    c, table = _filled(g, B, width, Hkv, D, P, fmt, kv)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype)
    out, lse = kv8.attention(q, c, table, torch.tensor(kv, dtype=torch.int32, device=DEV), causal=causal, return_lse=True)
    _check_attention(out, lse, q, c, table, kv, causal, D ** -0.5)
    again = kv8.attention(q, c, table, torch.tensor(kv, dtype=torch.int32, device=DEV), causal=causal)
    assert torch.equal(out, again)                       # no order of arrival in the result


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_packed_strided_and_rows_behind_the_last(dtype, causal):
    g = _gen(11)
    n, kv, H, Hkv, D, P = [7, 0, 150, 1, 64, 0, 2], [40, 9, 150, 333, 500, 0, 1], 4, 2, 64, 32
    c, table = _filled(g, 7, 17, Hkv, D, P, "int8", kv)
    start = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32, device=DEV)
    N = sum(n) + 5
    for off in (0, 3):                                    # a slice of a fused product; and one that is not 16-byte aligned
        q = torch.randn(N, 2 * H * D + 8, generator=g, device=DEV).to(dtype)[:, off: off + H * D].view(N, H, D)
        out = torch.full((N, H, D), 7.0, dtype=dtype, device=DEV)
        got, lse = kv8.attention(q, c, table, torch.tensor(kv, dtype=torch.int32, device=DEV), tok_start=start, causal=causal, scale=0.2,
                                 return_lse=True, out=out)
        assert got.data_ptr() == out.data_ptr() and (out[sum(n):] == 7.0).all()
        _check_attention(out[: sum(n)], lse[: sum(n)], q, c, table, kv, causal, 0.2, start)
        fresh = kv8.attention(q, c, table, torch.tensor(kv, dtype=torch.int32, device=DEV), tok_start=start, causal=causal, scale=0.2)
        assert torch.equal(fresh[: sum(n)], out[: sum(n)])


@pytest.mark.parametrize("T", [1, 40])
def test_poisoned_blocks_reach_only_the_rows_that_see_them(T):
    g = _gen(12)
    kv, P, D = [200, 200], 64, 64
    c, table = _filled(g, 2, 4, 2, D, P, "e4m3", kv)
    q = torch.randn(2, T, 2, D, generator=g, device=DEV)
    ln = torch.tensor(kv, dtype=torch.int32, device=DEV)
    clean = kv8.attention(q, c, table, ln)
    c.k_scale[table[0, 3].long(), 1] = float("nan")       # positions 192 .. of sequence 0, head 1
    c.v_scale[table[1, 0].long(), 0] = float("inf")
    out = kv8.attention(q, c, table, ln)
    sees = torch.arange(200 - T, 200, device=DEV) >= 192
    assert torch.isnan(out[0, sees, 1]).all() and torch.equal(out[0, ~sees, 1], clean[0, ~sees, 1])
    assert torch.equal(out[0, :, 0], clean[0, :, 0]) and torch.equal(out[1, :, 1], clean[1, :, 1])
    assert not torch.isfinite(out[1, :, 0]).any()


def test_one_huge_score_and_equal_scores():
    """A score far above the rest (the others underflow), and all scores equal (the mean of the values)."""
    P, D = 64, 64
    c = kv8.KV8Cache.allocate(4, 1, D, P, "int8", DEV)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    k = torch.zeros(1, 130, 1, D, device=DEV)
    k[0, 77] = 127.0
    v = torch.arange(130, device=DEV).float()[None, :, None, None].expand(1, 130, 1, D)
    kv8.append(c, k, v, table, torch.zeros(1, dtype=torch.int32, device=DEV))
    ln = torch.tensor([130], dtype=torch.int32, device=DEV)
    vals = kv8.read(c, table, torch.zeros(1, dtype=torch.int32, device=DEV), 130, dtype=torch.float32)[1]
    for sign in (1.0, -1.0):
        q = torch.full((1, 1, 1, D), sign * 100.0, device=DEV)
        out, lse = kv8.attention(q, c, table, ln, causal=False, scale=1.0, return_lse=True)
        keep = torch.ones(130, device=DEV, dtype=torch.bool)
        keep[77] = False
        ref = vals[0, 77] if sign > 0 else vals[0, keep].mean(0)
        assert torch.allclose(out[0, 0], ref, rtol=1e-5, atol=0)
        assert abs(float(lse) - (100.0 * 127 * D if sign > 0 else math.log(129))) <= 1e-6 * 100 * 127 * D
    q = torch.zeros(1, 3, 1, D, device=DEV)
    out = kv8.attention(q, c, table, ln, causal=True)
    for t in range(3):
        assert torch.allclose(out[0, t], vals[0, : 128 + t].mean(0), rtol=1e-5, atol=0)


def test_offsets_past_32_bits():
    """Pages that begin 4 GiB and more into the cache."""
    P, D, H = 256, 128, 16
    pages = (9 << 29) // (P * D * H) + 8                 # 4.5 GiB of codes in each half
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GiB")
    c = kv8.KV8Cache.allocate(pages, H, D, P, "e4m3", DEV)
    g = _gen(13)
    table = torch.tensor([[pages - 1, 3], [pages - 2, pages // 2 + 1]], dtype=torch.int32, device=DEV)
    small = kv8.KV8Cache.allocate(4, H, D, P, "e4m3", DEV)
    near = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    k, v = _randn(g, 2, 300, H, D).bfloat16(), _randn(g, 2, 300, H, D).bfloat16()
    zero, ln = torch.zeros(2, dtype=torch.int32, device=DEV), torch.tensor([300, 260], dtype=torch.int32, device=DEV)
    kv8.append(c, k, v, table, zero)
    kv8.append(small, k, v, near, zero)
    for T in (1, 70):
        q = torch.randn(2, T, H, D, generator=g, device=DEV).bfloat16()
        assert torch.equal(kv8.attention(q, c, table, ln), kv8.attention(q, small, near, ln))
    for a, b in zip(kv8.read(c, table, zero, 300), kv8.read(small, near, zero, 300)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_decoding_with_drafted_tokens_and_rollback(fmt):
    """The operators as a server uses them: a prompt is stored and attended, then rounds of one to four drafted tokens are appended
    and attended, some taken back (the next append overwrites them).  Checked against the 64-bit restatement each round."""
    g = _gen(14)
    B, H, Hkv, D, P = 3, 8, 4, 64, 32
    c = _noise_cache(g, 32, Hkv, D, P, fmt)
    table = _table(g, B, 8, 32)
    want_k, want_v = _halves(c)
    pos = [0] * B
    for step, (n, back) in enumerate([(70, 0), (1, 0), (4, 3), (4, 1), (1, 0), (3, 3), (2, 0), (60, 0)]):
        k, v = _randn(g, B, n, Hkv, D).bfloat16(), _randn(g, B, n, Hkv, D).bfloat16()
        q = torch.randn(B, n, H, D, generator=g, device=DEV).bfloat16()
        kv8.append(c, k, v, table, torch.tensor(pos, dtype=torch.int32, device=DEV))
        R.append(want_k, fmt, _seqs(k), table.tolist(), pos)
        R.append(want_v, fmt, _seqs(v), table.tolist(), pos)
        _same(c, want_k, want_v)
        ln = [p + n for p in pos]
        out = kv8.attention(q, c, table, torch.tensor(ln, dtype=torch.int32, device=DEV))
        _check_attention(out, None, q, c, table, ln, True, D ** -0.5)
        pos = [p + n - (back if b != 1 else 0) for b, p in enumerate(pos)]


def test_captured_and_replayed_beside_eager_calls():
    g = _gen(15)
    B, H, Hkv, D, P, kv = 4, 8, 4, 64, 64, [900, 17, 448, 300]
    c, table = _filled(g, B, 16, Hkv, D, P, "int8", kv)
    k, v = _randn(g, B, 1, Hkv, D).bfloat16(), _randn(g, B, 1, Hkv, D).bfloat16()
    q = torch.randn(B, 1, H, D, generator=g, device=DEV).bfloat16()
    pos = torch.tensor(kv, dtype=torch.int32, device=DEV)

    def step():
        kv8.append(c, k, v, table, pos)
        return kv8.attention(q, c, table, pos + 1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        k.copy_(_randn(g, B, 1, Hkv, D))
        pos.copy_(torch.tensor([m + 3 * i for m in kv], dtype=torch.int32))
        graph.replay()
        got = held.clone()
        assert torch.equal(got, step())
        torch.cuda.synchronize()
        _check_attention(got, None, q, c, table, [m + 3 * i + 1 for m in kv], True, D ** -0.5)


def test_two_streams_at_once():
    g = _gen(16)
    kv, D = [5000, 4100], 64
    c, table = _filled(g, 2, 80, 2, D, 64, "e4m3", kv)
    ln = torch.tensor(kv, dtype=torch.int32, device=DEV)
    qs = [torch.randn(2, 1, 4, D, generator=g, device=DEV).bfloat16() for _ in range(2)]
    ref = [kv8.attention(q, c, table, ln) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(kv8.attention(qs[i], c, table, ln))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[i]) for i in range(2) for o in outs[i])
