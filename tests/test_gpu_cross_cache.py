"""Decode steps over the 8-bit cross-attention cache (Engine(cross_cache=...)).  The cross K and V projections are the identity
and the encoder states lie on the format's own grid with every block's largest value at its top, so that quantising them loses
nothing: the 8-bit engine must then agree with the plain one to the rounding of the arithmetic itself."""
import numpy as np
import pytest
import torch

from whisper_amd import engine as E
from whisper_amd import lib as L
from whisper_amd.config import dims_for
from whisper_amd.weights import synthetic_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS = [(0, 1), (1, 0), (1, 1)]
SOT, EOT, TS = 824, 823, (924, 1023)


def _model():
    dims = dims_for("micro")
    sd = synthetic_state_dict(dims, seed=3, std=0.06)
    for name in list(sd):
        if "encoder_attn.k_proj" in name or "encoder_attn.v_proj" in name:
            sd[name] = torch.eye(dims.d_model) if name.endswith("weight") else torch.zeros_like(sd[name])
    return dims, sd


def _states(fmt, B, d, seed):
    """[B, 1500, d]: multiples of 2^-7 up to 127 (int8), or e4m3 codes times 2^-9; each 64 x 64 block holds its top value."""
    g = torch.Generator().manual_seed(seed)
    if fmt == "int8":
        x = torch.randint(-127, 128, (B, 1500, d), generator=g).float()
        x[:, ::64, ::64] = 127.0
        return (x * 2.0 ** -7).to(DEV)
    x = (torch.randn(B, 1500, d, generator=g) * 60).to(torch.float8_e4m3fn).float()
    x[:, ::64, ::64] = 448.0
    return (x * 2.0 ** -9).to(DEV)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,B", [("f32", 3), ("bf16", 20), ("bf16", 140)])
def test_exactly_quantised_states_decode_alike(fmt, dtype, B):
    dims, sd = _model()
    enc = _states(fmt, B, dims.d_model, B)
    plain = E.Engine(dims, sd, dtype=dtype, max_batch=B, align_heads=HEADS)
    small = E.Engine(dims, sd, dtype=dtype, max_batch=B, align_heads=HEADS, cross_cache=fmt)
    assert small.device_bytes > plain.device_bytes
    prompts = [[SOT, 825, 826, TS[0]] + [5 + b % 7] * (b % 3) for b in range(B)]
    out, steps = [], []
    for eng in (plain, small):
        eng.cross_kv(B, enc)
        ids = torch.tensor([[SOT, 825, 826]] * B, dtype=torch.int32)
        eng.decoder_forward(ids)
        steps.append(eng.decode_step(torch.arange(B, dtype=torch.int32) % 50, torch.full((B,), 3, dtype=torch.int32)))
        res = eng.decode_greedy(prompts, 40, EOT, SOT, *TS)
        n = int(res["n_text"].max())
        out.append((res, eng.attn_rows(B, n)))
    # Tolerances: one logits row is a chain of layers whose arithmetic is the plain engine's but for the order of the attention sums.
    # f32: the bound the cached steps are held to against the oracle.  bf16: an attention output goes on as hi + lo planes (2^-16) after
    # sums whose inputs are bf16 (q) and, in the 8-bit kernel, weights in f16 (2^-12 of each, over a mean of values below 1): 2^-12 is
    # what the step's hidden state can differ by per layer relative to its attention term, and logits are sums of 128 such terms with
    # weights of 0.06: 2 layers * 2^-12 * 128 * 0.06 < 4e-3
    tol = 1e-4 if dtype == "f32" else 4e-3
    assert (steps[0] - steps[1]).abs().max() <= tol
    (a, ra), (b, rb) = out
    if dtype == "f32":
        for key in ("new_tokens", "n_new", "text_ids", "n_text", "status"):
            assert torch.equal(a[key], b[key]), key
        for w in range(B):
            k = int(a["n_text"][w])
            assert (ra[w, :, :k] - rb[w, :, :k]).abs().max() <= 1e-6      # probabilities: the bound of the plain rows
            assert torch.allclose(rb[w, :, :k].sum(-1), torch.ones(len(HEADS), k, device=DEV), atol=1e-5)
    else:
        # tokens may part where two logits are closer than the tolerance; the first text row is before that
        for w in range(B):
            if int(a["n_text"][w]) and int(b["n_text"][w]):
                assert (ra[w, :, 0] - rb[w, :, 0]).abs().max() <= 2e-4
    # off again: bit for bit the plain engine
    L.check(small.lib.uw_ctx_cross_cache(small.ctx, -1))
    small.cross_kv(B, enc)
    res = small.decode_greedy(prompts, 40, EOT, SOT, *TS)
    for key in ("new_tokens", "n_new", "text_ids", "n_text"):
        assert torch.equal(res[key], a[key])
    plain.close(), small.close()


def test_a_switched_context_asks_for_the_cross_kv_again():
    dims, sd = _model()
    eng = E.Engine(dims, sd, dtype="bf16", max_batch=2, align_heads=HEADS)
    enc = _states("int8", 2, dims.d_model, 1)
    eng.cross_kv(2, enc)
    ids, pos = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    first = eng.decode_step(ids, pos)
    L.check(eng.lib.uw_ctx_cross_cache(eng.ctx, L.UW_KV8_INT8))
    with pytest.raises(L.UwError, match="uw_cross_kv"):
        eng.decode_step(ids, pos)
    eng.cross_kv(2, enc)
    assert (eng.decode_step(ids, pos) - first).abs().max() <= 4e-3
    # a position outside the context leaves the window's logits alone, as ever
    pos[1] = -1
    assert torch.isfinite(eng.decode_step(ids, pos)).all()
    with pytest.raises(L.UwError, match="format"):
        L.check(eng.lib.uw_ctx_cross_cache(eng.ctx, 5))
    eng.close()


def test_whole_windows_through_the_pool():
    """Audio to boundaries with the 8-bit cache, several batches in flight: the same as one engine alone."""
    from whisper_amd.parallel import EnginePool
    dims = dims_for("micro")
    sd = synthetic_state_dict(dims, seed=0, std=0.06)
    rng = np.random.default_rng(0)
    audio = torch.from_numpy((0.1 * rng.standard_normal((2, 480000))).astype(np.float32)).to(DEV)
    n = torch.tensor([480000, 200000], dtype=torch.int32)
    prompts = [[SOT, 825, 826, TS[0]]] * 2
    args = (audio, n, prompts, 24, EOT, SOT, *TS)
    eng = E.Engine(dims, sd, dtype="bf16", max_batch=2, align_heads=HEADS, cross_cache="int8")
    want = eng.transcribe_windows(*args)
    with EnginePool(dims, sd, inflight=2, dtype="bf16", max_batch=2, align_heads=HEADS, cross_cache="int8") as pool:
        futures = [pool.transcribe_windows_async(*args) for _ in range(4)]
        for f in futures:
            got = f.result()
            for key in ("new_tokens", "n_new", "text_ids", "n_text", "boundaries"):
                assert torch.equal(got[key].cpu(), want[key].cpu()), key
    assert (want["n_new"] > 0).all() and (want["boundaries"][:, 0] >= 0).all()
    eng.close()
