"""GPU draft verification against the 64-bit restatement: whole numbers, equal."""
import numpy as np
import pytest
import torch

from tests import kv8_oracle as R
from whisper_amd.speculative import verify_draft

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(seed, B, N, V, dtype, probs, spread=2.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.randn(B, N + 1, V, generator=g, device=DEV) * spread
    x += 8.0 * (torch.rand(B, N + 1, V, generator=g, device=DEV) < 3.0 / V)
    y = x[:, :N] + 0.5 * torch.randn(B, N, V, generator=g, device=DEV)
    drafted = torch.where(torch.rand(B, N, generator=g, device=DEV) < 0.6, y.argmax(-1),
                          torch.randint(0, V, (B, N), generator=g, device=DEV)).to(torch.int32) if N else torch.zeros(B, 0, dtype=torch.int32, device=DEV)
    if probs:
        x, y = torch.softmax(x, -1), torch.softmax(y, -1)
    return x.to(dtype), y.to(dtype), drafted, torch.rand(B, N + 1, generator=g, device=DEV)


def _np(x):
    return None if x is None else x.detach().to("cpu", torch.float64).numpy()


def _check(target, drafted, u, draft=None, n_drafted=None, temperature=1.0, probs=False):
    acc, tok = verify_draft(target, drafted, u, draft=draft, n_drafted=n_drafted, temperature=temperature, probs=probs)
    ra, rt = R.verify(_np(target), drafted.cpu().numpy(), _np(u), _np(draft), None if n_drafted is None else n_drafted.cpu().numpy(),
                      temperature, probs)
    assert acc.cpu().tolist() == ra.tolist()
    assert tok.cpu().tolist() == rt.tolist()
    return acc, tok


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("mode", ["logits", "cool", "probs", "greedy"])
@pytest.mark.parametrize("B,N,V", [(1, 4, 51865), (9, 3, 1000), (40, 7, 4097), (2, 1, 130001), (3, 0, 777), (300, 2, 65), (5, 2, 1)])
def test_verify(dtype, with_draft, mode, B, N, V):
    probs = mode == "probs"
    x, y, d, u = _inputs(B + V, B, N, V, dtype, probs)
    t = {"logits": 1.0, "cool": 0.7, "probs": 1.0, "greedy": 0.0}[mode]
    _check(x, d, u, draft=y if with_draft else None, temperature=t, probs=probs)
    n = torch.arange(B, device=DEV, dtype=torch.int32) % (N + 3) - 1          # also -1 and N + 1: clamped
    _check(x, d, u, draft=y if with_draft else None, n_drafted=n, temperature=t, probs=probs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_with_strides_and_odd_bases(dtype):
    """The drafted positions cut out of all positions' logits, and rows that start at odd addresses."""
    B, N, V = 3, 4, 999
    x, y, d, u = _inputs(1, B, N + 6, V, dtype, False)
    _check(x[:, 5: 6 + N], d[:, :N].contiguous(), u[:, : N + 1].contiguous(), draft=y[:, 2: 2 + N])
    flat = torch.randn(B * (N + 1) * 1003 + 3, device=DEV).to(dtype)
    for off in (1, 2, 3):
        z = flat[off: off + B * (N + 1) * 1003].view(B, N + 1, 1003)[:, :, :V]
        _check(z, d[:, :N].contiguous(), u[:, : N + 1].contiguous())
        _check(z, d[:, :N].contiguous(), u[:, : N + 1].contiguous(), temperature=0.0)
    _check(x[:, :5].transpose(1, 2).contiguous().transpose(1, 2), d[:, :4].contiguous(), u[:, :5].contiguous())
    _check(x[:1, :1].expand(B, N + 1, V), d[:, :N].contiguous(), u[:, : N + 1].contiguous())


def test_borders_and_empty_mass():
    """Probabilities that are whole fractions: a draw on a border takes the token behind it, tokens without mass are never drawn."""
    V = 300
    p = torch.zeros(7, 2, V, device=DEV)
    p[:, :, 3], p[:, :, 200], p[:, :, 299] = 0.25, 0.25, 0.5
    d = torch.full((7, 1), 10, dtype=torch.int32, device=DEV)          # p = 0: rejected, the residual is p itself
    u = torch.tensor([[0.0, x] for x in (0.0, 0.2499999, 0.25, 0.4999999, 0.5, 0.75, 0.99999994)], device=DEV)
    acc, tok = _check(p, d, u, probs=True)
    assert acc.tolist() == [0] * 7 and tok[:, 0].tolist() == [3, 3, 200, 200, 299, 299, 299]
    # acceptance: u * q < p, strictly
    q = torch.zeros(7, 1, V, device=DEV)
    q[:, :, 3] = 0.5
    d = torch.full((7, 1), 3, dtype=torch.int32, device=DEV)
    u = torch.tensor([[x, 0.0] for x in (0.0, 0.25, 0.4999999, 0.5, 0.5000001, 0.75, 0.99)], device=DEV)
    acc, tok = _check(p, d, u, draft=q, probs=True)
    assert acc.tolist() == [1, 1, 1, 0, 0, 0, 0]
    assert tok[3].tolist() == [200, -1]                                # residual: 3 has none left
    # a drafter that is certain, of a token the target is certain of: accepted; of one that is alone with the mass but not whole
    one = torch.zeros(1, 2, V, device=DEV)
    one[:, :, 7] = 0.5
    acc, tok = _check(one, torch.tensor([[7]], dtype=torch.int32, device=DEV), torch.tensor([[0.5, 0.3]], device=DEV), probs=True)
    assert acc.tolist() == [0] and tok.tolist() == [[7, -1]]           # the residual is empty: drawn from the row itself
    # q above p everywhere: the residual is empty too
    acc, tok = _check(p[:1], d[:1], torch.tensor([[0.9, 0.6]], device=DEV), draft=p[:1, :1] * 2, probs=True)
    assert acc.tolist() == [0] and tok[0, 0] == 299
    # no mass at all
    acc, tok = _check(torch.zeros(1, 2, V, device=DEV), d[:1], u[:1], probs=True)
    assert tok.tolist() == [[-1, -1]]


def test_equal_rows_accept_whatever_the_number():
    x, _, d, u = _inputs(8, 16, 5, 5003, torch.float32, False)
    u[:, :5] = 0.99999994
    d = torch.multinomial(torch.softmax(x[:, :5], -1).view(-1, 5003), 1).view(16, 5).to(torch.int32)
    acc, _ = verify_draft(x, d, u, draft=x[:, :5].contiguous())
    assert acc.tolist() == [5] * 16


@pytest.mark.parametrize("temperature", [1.0, 0.0])
@pytest.mark.parametrize("V", [257, 51865])
def test_masked_and_broken_rows(temperature, V):
    inf, nan = float("inf"), float("nan")
    x, y, d, u = _inputs(9, 8, 2, V, torch.float32, False)
    x[0, :, : V // 2] = -inf                       # masked tokens
    x[1, 1, V // 3] = nan                          # a broken row
    x[2, 0] = -inf                                 # nothing left
    x[3, 0, V - 1] = inf
    x[4] = -3.4028234663852886e38                  # the type's lowest value throughout
    x[5, :, :] = -3.4028234663852886e38
    x[5, :, 5] = 0.0
    d[6, 0], d[7, 1] = -1, V                       # no token of the vocabulary
    d[5] = 5
    d[1, 0] = int(x[1, 0].argmax())
    u[1, 0] = 0.0
    acc, tok = _check(x, d, u, temperature=temperature)
    assert acc[1] == 1 and tok[1, 1] == -1         # kept up to the broken row, no token from it
    assert acc[6] == 0 and acc[7] <= 1 and acc[5] == 2 and tok[5].tolist() == [5, 5, 5]
    if temperature:
        y[0, 0, 3] = nan                           # a drafter's broken row rejects and gives no token
        _check(x, d, u, draft=y, temperature=temperature)


def test_greedy_takes_the_lowest_of_equal_scores():
    x = torch.zeros(3, 2, 5000, device=DEV, dtype=torch.bfloat16)
    x[0, 0, 4999] = x[0, 0, 17] = x[0, 0, 2500] = 3.0
    x[1, 0, 4096:] = 1.0
    d = torch.tensor([[17], [4096], [0]], dtype=torch.int32, device=DEV)
    acc, tok = _check(x, d, None, temperature=0.0)
    assert acc.tolist() == [1, 1, 1] and tok.tolist() == [[17, 0], [4096, 0], [0, 0]]


def test_tokens_are_distributed_as_the_target():
    """Exact, not sampled: over a fine grid of both random numbers the first token's frequencies are the target's probabilities.
    A grid of n numbers counts an interval to within one of n, and a token's outcomes are at most three intervals of either."""
    V, n = 4, 128
    p = torch.tensor([0.5, 0.125, 0.25, 0.125], device=DEV)
    q = torch.tensor([0.25, 0.5, 0.125, 0.125], device=DEV)
    grid = (torch.arange(n, device=DEV) + 0.5) / n
    u = torch.stack(torch.meshgrid(grid, grid, indexing="ij"), -1).view(-1, 2)
    freq = torch.zeros(V, device=DEV)
    for tok in range(V):
        d = torch.full((n * n, 1), tok, dtype=torch.int32, device=DEV)
        acc, out = verify_draft(p.expand(n * n, 2, V), d, u.contiguous(), draft=q.expand(n * n, 1, V), probs=True)
        freq += q[tok] * torch.bincount(out[:, 0].long(), minlength=V) / (n * n)
    assert (freq - p).abs().max() <= 3.0 / n


def test_captured_and_replayed_beside_eager_calls():
    x, y, d, u = _inputs(21, 6, 3, 51865, torch.float32, False)
    run = lambda: verify_draft(x, d, u, draft=y)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        a, b, dd, uu = _inputs(30 + i, 6, 3, 51865, torch.float32, False)
        x.copy_(a), y.copy_(b), d.copy_(dd), u.copy_(uu)
        graph.replay()
        got = [t.clone() for t in held]
        assert all(torch.equal(s, t) for s, t in zip(got, run()))
        torch.cuda.synchronize()


def test_greedy_verification_of_an_engine():
    """A prompt plus drafted tokens through one decoder pass, its logits verified: what the engine itself decodes greedily is accepted
    up to the first token that was changed, and the token behind is the engine's own."""
    from whisper_amd import engine as E
    from whisper_amd.config import dims_for
    from whisper_amd.weights import synthetic_state_dict
    dims = dims_for("micro")
    eng = E.Engine(dims, synthetic_state_dict(dims, seed=0, std=0.06), dtype="f32", max_batch=2)
    g = torch.Generator(device=DEV)
    g.manual_seed(0)
    enc = torch.randn(2, 1500, dims.d_model, generator=g, device=DEV)
    eng.cross_kv(2, enc)
    prompt = [824, 825, 826, 924]
    res = eng.decode_greedy([prompt, prompt], 14, 823, 824, 924, 1023)
    n = min(int(m) for m in res["n_new"])
    assert n >= 6
    own = res["new_tokens"][:, :n].clone()
    drafted = own[:, :5].clone()
    drafted[1, 3] = (drafted[1, 3] + 1) % 800
    ids = torch.cat([torch.tensor([prompt, prompt], device=DEV, dtype=torch.int32), drafted], 1)
    logits = eng.decoder_forward(ids, logits_all=True)["logits_all"][:, len(prompt) - 1:]
    acc, tok = verify_draft(logits, drafted, temperature=0.0)
    assert acc.tolist() == [5, 3]
    assert tok[0].tolist() == own[0, :6].tolist() and tok[1].tolist() == own[1, :4].tolist() + [-1, -1]
    # and with a temperature: what is accepted and drawn follows the same rows
    u = torch.rand(2, 6, generator=g, device=DEV)
    _check(logits, drafted, u, temperature=0.9)
    eng.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [8, 9, 17, 40])
@pytest.mark.parametrize("mode", ["logits", "probs", "greedy"])
def test_many_drafted_tokens(dtype, N, mode):
    """A drafter that agrees up to a position of its own in every window: acceptance runs past eight positions, the last included."""
    B, V = N + 1, 501
    x, _, d, u = _inputs(70 + N, B, N, V, dtype, False)
    d = x[:, :N].argmax(-1).to(torch.int32)
    y = x[:, :N].clone()
    for b in range(N):
        y[b, b] = -1.0                                   # flat there,
        x[b, b, d[b, b].long()] = -60.0                  # and the target has turned away from that token
    t = 0.0 if mode == "greedy" else 1.0
    if mode == "probs":
        x, y = torch.softmax(x.float(), -1).to(dtype), torch.softmax(y.float(), -1).to(dtype)
    acc, _ = _check(x, d, u, draft=y, temperature=t, probs=mode == "probs")
    if mode != "greedy":
        assert acc.tolist() == list(range(N + 1))
    _check(x, d, u, temperature=t, probs=mode == "probs")


@pytest.mark.parametrize("temperature", [1e-30, 1e-4, 0.05, 30.0, 1e6, 3e38])
@pytest.mark.parametrize("with_draft", [False, True])
def test_extreme_temperatures_and_masked_scores(temperature, with_draft):
    """From arg-max to uniform over what is not masked; scores of -inf and of the type's lowest value are never drawn."""
    B, N, V = 24, 3, 9001
    x, y, d, u = _inputs(5, B, N, V, torch.float32, False)
    for z in (x, y):
        z[..., 1000:6000] = -float("inf")
        z[..., 8000:] = torch.finfo(torch.float32).min if temperature < 1e5 else -float("inf")
    d = torch.where((d >= 1000) & (d < 6000), d % 1000, d).to(torch.int32)
    _, tok = _check(x, d, u, draft=y if with_draft else None, temperature=temperature)
    got = tok[tok >= 0]
    assert not ((got >= 1000) & (got < 6000)).any()
