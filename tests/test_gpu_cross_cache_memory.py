"""An 8-bit cross cache that does not fit leaves the context as it was: nothing allocated, every call as before, and the next try free to
succeed."""
import pytest
import torch

from tests.test_gpu_cross_cache import DEV, HEADS, _model, _states
from whisper_amd import engine as E
from whisper_amd import lib as L

pytestmark = pytest.mark.gpu


def _all_but(least, most):
    """A tensor, never written, that leaves so much memory."""
    for spare in range(least, most + 1, 1 << 28):
        try:
            return torch.empty(torch.cuda.mem_get_info()[0] - spare, dtype=torch.uint8, device=DEV)
        except torch.OutOfMemoryError:
            continue
    pytest.skip("the free memory cannot be had in one piece")


def test_a_cache_that_does_not_fit_leaves_nothing_behind():
    if torch.cuda.mem_get_info()[0] < 140 << 30:
        pytest.skip("needs 140 GiB")
    dims, sd = _model()
    windows = 4096                                   # codes of 3.2 GB beside a few MB of scales and tables
    eng = E.Engine(dims, sd, dtype="bf16", max_batch=windows, align_heads=HEADS)
    enc = _states("int8", 2, dims.d_model, 1)
    ids, pos = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    eng.cross_kv(2, enc)
    plain = eng.decode_step(ids, pos)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held = eng.device_bytes
    hog = _all_but(1 << 30, 2 << 30)
    for _ in range(2):
        with pytest.raises(L.UwError, match="memory"):
            L.check(eng.lib.uw_ctx_cross_cache(eng.ctx, L.UW_KV8_INT8))
        assert eng.device_bytes == held
        assert torch.equal(eng.decode_step(ids, pos), plain)          # no error left for the next call to find
    del hog
    torch.cuda.empty_cache()
    L.check(eng.lib.uw_ctx_cross_cache(eng.ctx, L.UW_KV8_INT8))
    grown = eng.device_bytes
    assert grown > held + (3 << 30)
    eng.cross_kv(2, enc)
    assert (eng.decode_step(ids, pos) - plain).abs().max() <= 4e-3    # the bound of the other tests of exactly quantised states
    for fmt in (-1, L.UW_KV8_E4M3):
        L.check(eng.lib.uw_ctx_cross_cache(eng.ctx, fmt))
        assert eng.device_bytes == grown                              # off and on again, in either format: the same memory
    eng.close()
