"""What the 8-bit cache's operators and the draft verification refuse, and how: no GPU is touched."""
import ctypes as C

import pytest
import torch

from whisper_amd import kv8
from whisper_amd import lib as L
from whisper_amd.speculative import verify_draft


def _cache(fmt="int8", pages=4, heads=2, page=16, dim=64):
    return kv8.KV8Cache.allocate(pages, heads, dim, page, fmt, device="cpu")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_allocate_describes_the_layout(fmt):
    c = _cache(fmt)
    assert c.k.shape == (4, 2, 16, 64) and c.v.shape == (4, 2, 64, 16) and c.k_scale.shape == (4, 2)
    assert (c.n_pages, c.n_kv_heads, c.page, c.head_dim) == (4, 2, 16, 64)
    assert not c.k.view(torch.uint8).any() and not c.v_scale.any()


def test_cache_tensors_are_checked():
    c = _cache()
    with pytest.raises(ValueError, match="fmt"):
        kv8.KV8Cache.allocate(1, 1, fmt="int4", device="cpu")
    with pytest.raises(ValueError, match="codes"):
        kv8.KV8Cache(c.k.float(), c.v, c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="transposed"):
        kv8.KV8Cache(c.k, c.k, c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="scales"):
        kv8.KV8Cache(c.k, c.v, c.k_scale[:3], c.v_scale)
    with pytest.raises(ValueError, match="contiguous"):
        kv8.KV8Cache(c.k.transpose(2, 3).contiguous().transpose(2, 3), c.v, c.k_scale, c.v_scale)


def test_wrong_shapes_and_types_are_refused():
    c = _cache()
    table, pos = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    x = torch.zeros(3, 5, 2, 64)
    for args, word in (((x[:2], x[:2], table, pos), "sequences"), ((x.half(), x.half(), table, pos), "float32 or bfloat16"),
                       ((x[..., :32], x, table, pos), "float32 or bfloat16"), ((x, x[:, :4], table, pos), "alike"),
                       ((x[:, :, :1], x[:, :, :1], table, pos), "heads"), ((x, x, table.long(), pos), "page table"),
                       ((x, x, table[:, :0], pos), "page table"), ((x, x, table, pos[:2]), "pos"), ((x, x, table, pos.float()), "pos")):
        with pytest.raises(ValueError, match=word):
            kv8.append(c, *args)
    with pytest.raises(ValueError, match="tok_start"):
        kv8.append(c, x[0], x[0], table, pos, tok_start=pos)
    with pytest.raises(ValueError, match="query heads"):
        kv8.attention(torch.zeros(3, 1, 3, 64), c, table, pos)
    with pytest.raises(ValueError, match="kv_len"):
        kv8.attention(torch.zeros(3, 1, 4, 64), c, table, pos[:1])
    with pytest.raises(ValueError, match="out must"):
        kv8.attention(torch.zeros(3, 1, 4, 64), c, table, pos, out=torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="count"):
        kv8.read(c, table, pos, -1)
    # right shapes, no GPU: refused before the library is reached
    for call in (lambda: kv8.append(c, x, x, table, pos), lambda: kv8.read(c, table, pos, 2),
                 lambda: kv8.attention(torch.zeros(3, 1, 4, 64), c, table, pos)):
        with pytest.raises(L.UwError, match="GPU"):
            call()


def test_library_refuses_before_any_gpu_call():
    lib = L.load()
    good = dict(k=64, v=64, k_scale=64, v_scale=64, n_pages=4, n_kv_heads=2, page=16, head_dim=64, format=L.UW_KV8_INT8)
    tok = dict(data=64, seq_stride=128, tok_stride=128, head_stride=64, n_tok=3, tok_start=None, B=3, T=1)

    def rc(cache=None, t=None, dtype=L.UW_DTYPE_BF16, heads=2, table=64, width=1, ln=64):
        c, x = L.UwKv8Cache(**{**good, **(cache or {})}), L.UwKv8Tokens(**{**tok, **(t or {})})
        out = []
        out.append(lib.uw_kv8_append(C.byref(c), dtype, C.byref(x), C.byref(x), table, width, ln, None))
        out.append(lib.uw_kv8_read(C.byref(c), dtype, C.byref(x), C.byref(x), table, width, ln, None))
        out.append(lib.uw_kv8_attention(C.byref(c), dtype, C.byref(x), C.byref(x), None, heads, table, width, ln, 1, 0.125, None, None))
        return out

    def refused(word, **kw):
        assert all(r != 0 for r in rc(**kw)), (word, kw)
        assert word.encode() in lib.uw_last_error(), lib.uw_last_error()

    refused("null cache", cache={"k": None})
    refused("format", cache={"format": 2})
    refused("tokens", cache={"page": 48})
    refused("head_dim", cache={"head_dim": 96})
    refused("pages", cache={"n_pages": 0})
    refused("aligned", cache={"v": 72})
    refused("dtype", dtype=7)
    refused("sequences", t={"B": 0})
    refused("null data", t={"data": None})
    refused("rows", t={"n_tok": 4})
    refused("multiples", t={"tok_stride": 130})
    refused("null page table", table=None)
    refused("null page table", width=0)
    c, x = L.UwKv8Cache(**good), L.UwKv8Tokens(**tok)
    assert lib.uw_kv8_attention(C.byref(c), 1, C.byref(x), C.byref(x), None, 3, 64, 1, 64, 1, 0.125, None, None) != 0
    assert b"query heads" in lib.uw_last_error()
    y = L.UwKv8Tokens(**{**tok, "B": 1, "T": 3})
    assert lib.uw_kv8_append(C.byref(c), 1, C.byref(x), C.byref(y), 64, 1, 64, None) != 0 and b"same tokens" in lib.uw_last_error()
    # nothing to do is no error
    z = L.UwKv8Tokens(**{**tok, "T": 0, "n_tok": 0})
    assert lib.uw_kv8_append(C.byref(c), 1, C.byref(z), C.byref(z), 64, 1, 64, None) == 0


def test_verify_draft_refuses():
    t, d, u = torch.zeros(2, 4, 10), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 4)
    for kw, word in ((dict(target=t[0]), "target"), (dict(target=t.half()), "target"), (dict(target=t[:, :0]), "empty"),
                     (dict(drafted=d[:, :2]), "drafted"), (dict(drafted=d.float()), "drafted"), (dict(uniforms=None), "uniforms"),
                     (dict(uniforms=u[:, :3]), "uniforms"), (dict(draft=t), "draft"), (dict(draft=t[:, :3].bfloat16()), "draft"),
                     (dict(n_drafted=torch.zeros(3, dtype=torch.int32)), "n_drafted"), (dict(temperature=-1.0), "temperature"),
                     (dict(temperature=float("inf")), "temperature"), (dict(temperature=0.5, probs=True), "temperature")):
        args = {"target": t, "drafted": d, "uniforms": u, **kw}
        with pytest.raises(ValueError, match=word):
            verify_draft(**args)
    with pytest.raises(L.UwError, match="GPU"):
        verify_draft(t, d, u)
    lib = L.load()
    assert lib.uw_verify_draft(0, None, 0, 0, None, 0, 0, None, None, None, 1, 1, 1, 1.0, 0, None, None, None, None) != 0
    assert lib.uw_verify_draft(3, 64, 0, 0, None, 0, 0, 64, None, 64, 1, 1, 1, 1.0, 0, 64, 64, 64, None) != 0
    assert lib.uw_verify_draft(0, 66, 0, 0, None, 0, 0, 64, None, 64, 1, 1, 1, 1.0, 0, 64, 64, 64, None) != 0
    assert b"misaligned" in lib.uw_last_error()
