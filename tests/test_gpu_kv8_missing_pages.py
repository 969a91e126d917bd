"""Attention over the 8-bit cache with tables that name pages which do not exist, where the pages that do exist hold leftovers that are no
numbers: only rows that see a missing page are NaN, the others have their result to the last bit."""
import pytest
import torch

from tests.test_gpu_kv8 import DEV, _filled, _gen
from tests.test_gpu_kv8_weights import BF, F32, _check
from whisper_amd import kv8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("P", [16, 32, 64, 256])
@pytest.mark.parametrize("B,T,H,D", [(2, 8, 2, 64), (2, 30, 2, 64), (1, 100, 2, 128), (4, 250, 64, 64), (4, 250, 40, 128)])      # keys shared: 16, 32 rows, of 128 channels; side by side
@pytest.mark.parametrize("after", [0, 40])
def test_rows_that_do_not_see_a_missing_page_are_not_touched_by_it(dtype, P, B, T, H, D, after):
    g = _gen(P + T + H)
    kv = 512 + after
    c, table = _filled(g, B, -(-kv // P), H, D, P, "e4m3", [kv] * B)
    # page 0 to whoever can do without it: it holds e4m3's NaN throughout, and is what a careless lookup of no page would read
    spare = [p for p in range(c.n_pages) if p not in set(table.flatten().tolist())][0]
    for x in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale):
        x[spare] = x[0]
    table[table == 0] = spare
    for x in (c.k, c.v):
        x.view(torch.uint8)[0] = 0x7f
    c.k_scale[0] = c.v_scale[0] = 1.0
    ln = torch.full((B,), kv, dtype=torch.int32, device=DEV)
    q = torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype)
    clean, lse = kv8.attention(q, c, table, ln, return_lse=True)
    _check(clean, lse, q, c, table, [kv] * B, True, D ** -0.5)
    at = torch.arange(kv - T, kv, device=DEV)
    # the last token's page is none; then one inside the rows' range; then one that all see
    for page in ((kv - 1) // P, (kv - T // 2) // P, 0):
        for none in (-1, c.n_pages, 1 << 30):
            holed = table.clone()
            holed[0, page] = none
            out, l = kv8.attention(q, c, holed, ln, return_lse=True)
            sees = at >= page * P
            assert torch.isnan(out[0, sees]).all() and torch.isnan(l[0, sees]).all()
            assert torch.equal(out[0, ~sees], clean[0, ~sees]) and torch.equal(l[0, ~sees], lse[0, ~sees])
            assert torch.equal(out[1:], clean[1:])
    # rows that end inside a block whose other pages are none: the entries behind the sequences' ends name nothing
    for less in (T, T + 1):
        short = ln - less
        wide = torch.cat([table, torch.full((B, 3), -1, dtype=torch.int32, device=DEV)], 1)
        want, wl = kv8.attention(q, c, table, short, return_lse=True)
        cut = wide.clone()
        cut[:, -(-(kv - less) // P):] = -1
        out, l = kv8.attention(q, c, cut, short, return_lse=True)
        assert torch.equal(out, want) and torch.equal(l, wl) and torch.isfinite(out).all()
