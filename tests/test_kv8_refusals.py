"""What the 8-bit cache's operators and the draft verification refuse, and how: no GPU is touched."""
import pytest
import torch

from whisper_amd import kv8
from whisper_amd import lib as L
from whisper_amd.speculative import _ARGS, verify_draft


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
                       ((x[..., :32], x[..., :32], table, pos), "float32 or bfloat16"), ((x, x[:, :4], table, pos), "alike"),
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
    """The C entries check every size before they touch the GPU; the addresses here are none."""
    lib = L.load()
    good = dict(k=64, v=64, ks=64, vs=64, n_pages=4, heads=2, page=16, dim=64, fmt=L.UW_KV8_INT8, r=0, table=64, len=64, start=0,
                n_tok=3, width=1, B=3, T=1, dtype=L.UW_DTYPE_BF16, x=64, sB=128, sT=128, sH=64, y=64, yB=128, yT=128, yH=64)
    last = dict(lse=0, ws=0, ws_bytes=0, n_heads=2, causal=1, scale=0.125, r2=0)

    def calls(**kw):
        a = {**good, **{k: v for k, v in kw.items() if k in good}}
        vals = list(a.values())
        store = kv8._CACHE.pack(*vals[:10]) + kv8._STORE.pack(*vals[10:])
        attend = kv8._CACHE.pack(*vals[:10]) + kv8._ATTEND.pack(*vals[10:], *{**last, **{k: v for k, v in kw.items() if k in last}}.values())
        return (lambda: lib.uw_kv8_append(store, None), lambda: lib.uw_kv8_read(store, None), lambda: lib.uw_kv8_attention(attend, None),
                lambda: lib.uw_kv8_attention_workspace_bytes(attend))

    def refused(word, which=range(4), **kw):
        for i in which:
            rc = calls(**kw)[i]()
            assert (rc == -1) if i == 3 else rc > 0, (word, i, rc)
            assert word.encode() in lib.uw_last_error(), (i, lib.uw_last_error())

    refused("null cache", k=0)
    refused("format", fmt=2)
    refused("tokens", page=48)
    refused("head_dim", dim=96)
    refused("pages", n_pages=0)
    refused("aligned", v=72)
    refused("dtype", dtype=7)
    refused("sequences", B=0)
    refused("null data", x=0)
    refused("rows are not", n_tok=4)
    refused("too many rows", n_tok=1 << 40, start=64)
    refused("multiples", sT=130)
    refused("multiples", y=72)
    refused("null page table", table=0)
    refused("null page table", width=0)
    refused("columns", width=1 << 24)
    refused("query heads", (2, 3), n_heads=3)
    refused("workspace", (2,), width=4096)                    # long enough to be split over workgroups, and no workspace
    assert calls(width=4096)[3]() > 0
    refused("workspace", (2,), width=4096, ws=64, ws_bytes=16)
    for call in calls(T=0, n_tok=0)[:3]:                      # nothing to do is no error
        assert call() == 0
    for fn in (lib.uw_kv8_append, lib.uw_kv8_read, lib.uw_kv8_attention):
        assert fn(None, None) > 0 and b"null arguments" in lib.uw_last_error()


def test_cross_cache_refuses():
    from whisper_amd.config import dims_for
    from whisper_amd.engine import Engine
    with pytest.raises(ValueError, match="cross_cache"):
        Engine(dims_for("micro"), {}, cross_cache="int4")
    lib = L.load()
    assert lib.uw_ctx_cross_cache(None, L.UW_KV8_INT8) > 0 and b"null context" in lib.uw_last_error()


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
    good = dict(target=64, sB=20, sN=10, draft=0, dB=0, dN=0, drafted=64, n_drafted=0, uniforms=64, accepted=64, tokens=64, ws=0, ws_bytes=0,
                dtype=0, B=1, N=1, V=10, temperature=1.0, probs=0)
    for kw, word in ((dict(target=0), "null"), (dict(tokens=0), "null"), (dict(drafted=0), "null"), (dict(dtype=3), "dtype"), (dict(V=0), "V 0"),
                     (dict(N=-1), "N -1"), (dict(B=0), "B 0"), (dict(uniforms=0), "uniforms"), (dict(temperature=-0.5), "temperature"),
                     (dict(temperature=float("nan")), "temperature"), (dict(temperature=0.5, probs=1), "temperature"),
                     (dict(target=66), "misaligned"), (dict(draft=65), "misaligned")):
        args = _ARGS.pack(*{**good, **kw}.values())
        assert lib.uw_verify_draft(args, None) > 0 and word.encode() in lib.uw_last_error(), (kw, lib.uw_last_error())
        assert lib.uw_verify_draft_workspace_bytes(args) == -1
    args = _ARGS.pack(*good.values())
    assert lib.uw_verify_draft_workspace_bytes(args) > 0
    for ws in (dict(), dict(ws=72, ws_bytes=1 << 20), dict(ws=64, ws_bytes=16)):
        assert lib.uw_verify_draft(_ARGS.pack(*{**good, **ws}.values()), None) > 0 and b"workspace" in lib.uw_last_error()
    assert lib.uw_verify_draft(_ARGS.pack(*{**good, "B": 1 << 20, "V": 51865}.values()), None) > 0 and b"too many rows" in lib.uw_last_error()
    assert lib.uw_verify_draft(None, None) > 0


def test_attention_scratch_stays_small():
    """Parts of cut sequences take at most 256 MB, whatever the table could hold."""
    from whisper_amd import kv8
    seen = set()
    for B, T, heads, kv_heads, D, P, width in ((1, 1, 8, 1, 128, 64, 2000), (256, 4, 8, 1, 128, 256, 2000), (1, 2048, 8, 1, 128, 64, 8000),
                                               (64, 1, 32, 8, 64, 16, 100000), (3, 200, 12, 12, 64, 64, 5000), (8, 5, 32, 8, 128, 64, 513)):
        dims = kv8._CACHE_DIMS.pack(1000, kv_heads, P, D, 0, 0)
        for packed in (False, True):
            n = kv8._workspace_bytes(dims, B * T, width, B, 0 if packed else T, 1, packed, heads)
            assert 0 <= n <= 256 << 20
            seen.add(n > 0)
    assert seen == {False, True}
