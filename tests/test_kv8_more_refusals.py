"""More of what the 8-bit cache's operators refuse: no GPU is touched."""
import pytest
import torch

from whisper_amd import kv8
from whisper_amd import lib as L


def _cache():
    return kv8.KV8Cache.allocate(4, 2, 64, 16, "int8", device="cpu")


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, -1e300])
def test_scales_that_are_no_f32_numbers(scale):
    c, table, ln = _cache(), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="scale"):
        kv8.attention(torch.zeros(1, 1, 2, 64), c, table, ln, scale=scale)
    with pytest.raises(L.UwError, match="GPU"):
        kv8.attention(torch.zeros(1, 1, 2, 64), c, table, ln, scale=-3.4e38)


def test_library_refuses_such_scales_too():
    lib = L.load()
    a = (64, 64, 64, 64, 4, 2, 16, 64, L.UW_KV8_INT8, 0, 64, 64, 0, 3, 1, 3, 1, L.UW_DTYPE_BF16, 64, 128, 128, 64, 64, 128, 128, 64, 0, 0, 0, 2, 1)
    for scale in (float("nan"), float("inf"), -float("inf")):
        args = kv8._CACHE.pack(*a[:10]) + kv8._ATTEND.pack(*a[10:], scale, 0)
        assert lib.uw_kv8_attention(args, None) > 0 and b"scale" in lib.uw_last_error()
        assert lib.uw_kv8_attention_workspace_bytes(args) == -1


def test_the_tensors_of_a_cache_stay():
    """The operators hold on to the addresses of the tensors that a cache was made of: another tensor in their place would not be what is used."""
    c = _cache()
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    assert c.k.shape == (4, 2, 16, 64) and c.v.shape == (4, 2, 64, 16) and c.k_scale.shape == c.v_scale.shape == (4, 2)


def test_an_output_that_lies_across_the_queries():
    """Rows that are written while others are still to be read; the queries' own memory, row by row the same, is fine, and so is memory beside it."""
    c, table, ln = _cache(), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    buf = torch.zeros(3 * 2 * 2 * 64 * 2)
    q = buf[:768].view(3, 2, 2, 64)
    for out in (buf[64:832].view(3, 2, 2, 64), buf[704:1472].view(3, 2, 2, 64)):
        with pytest.raises(ValueError, match="overlap"):
            kv8.attention(q, c, table, ln, out=out)
    fused = buf.view(3, 2, 2, 128)[..., :64]
    with pytest.raises(ValueError, match="overlap"):
        kv8.attention(fused, c, table, ln, out=buf[:768].view(3, 2, 2, 64))
    for out in (q, buf[768:].view(3, 2, 2, 64)):
        with pytest.raises(L.UwError, match="GPU"):
            kv8.attention(q, c, table, ln, out=out)
