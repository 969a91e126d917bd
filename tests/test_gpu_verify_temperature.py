"""Draft verification takes its temperature as it is given, in 64 bits: numbers that fall between what it and its rounding to 32 bits
would decide, many draws from one row, and temperatures that 32 bits do not hold.  Whole numbers, equal to the 64-bit restatement's."""
import numpy as np
import pytest
import torch

from tests.test_gpu_verify import DEV, _check, _inputs
from whisper_amd.speculative import verify_draft

pytestmark = pytest.mark.gpu


def _p(x, t):
    e = np.exp((x - x.max()) / t)
    return e / e.sum()


def _same(got, want):
    """Equal whole numbers; else where they are not (a diff of thousands would be of no use, and takes minutes)."""
    got = got.cpu().numpy()
    at = np.nonzero(got != np.asarray(want))[0]
    assert not at.size, (at.size, len(got), at[:5].tolist(), got[at[:5]].tolist(), np.asarray(want)[at[:5]].tolist())


def _between(a, b):
    """An f32 number strictly between a and b, away from both by 1e-10 of them -- a hundred times what the kernel's exponentials are off by --, or None."""
    u = np.float32((a + b) / 2)
    lo, hi = min(a, b), max(a, b)
    return u if lo * (1 + 1e-10) < float(u) < hi * (1 - 1e-10) else None


@pytest.mark.parametrize("t", [0.6, 0.7, 0.8, 1.3])
def test_numbers_between_the_temperature_and_its_f32(t):
    rounded = float(np.float32(t))
    assert rounded != t
    V = 4001
    g = torch.Generator().manual_seed(int(t * 10))
    x = torch.randn(V, generator=g) * 4
    p, r = _p(x.double().numpy(), t), _p(x.double().numpy(), rounded)
    # acceptance: u < p(d)
    found = [(d, u) for d in range(V) for u in [_between(p[d], r[d])] if u is not None]
    assert len(found) > 100
    B = len(found)
    target = x.to(DEV).expand(B, 2, V)
    drafted = torch.tensor([[d] for d, _ in found], dtype=torch.int32, device=DEV)
    u = torch.tensor([[float(n), 0.5] for _, n in found], dtype=torch.float32, device=DEV)
    acc, _ = verify_draft(target, drafted, u, temperature=t)
    _same(acc, [int(float(n) < p[d]) for d, n in found])
    # drawing: the first token whose cumulative weight exceeds u
    cp, cr = np.cumsum(p), np.cumsum(r)
    draws = [n for a, b in zip(cp[:-1], cr[:-1]) for n in [_between(a, b)] if n is not None]
    assert len(draws) > 20
    B = len(draws)
    u = torch.tensor(draws, dtype=torch.float32, device=DEV)[:, None]
    _, tok = verify_draft(x.to(DEV).expand(B, 1, V), torch.zeros(B, 0, dtype=torch.int32, device=DEV), u, temperature=t)
    _same(tok[:, 0], np.searchsorted(cp, np.array(draws, np.float64) * cp[-1], side="right"))


@pytest.mark.parametrize("t", [0.6, 0.8])
def test_twenty_thousand_draws(t):
    B, V = 20000, 51865
    x, _, _, _ = _inputs(77, 1, 0, V, torch.float32, False, spread=2.5)
    u = torch.rand(B, 1, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    _, tok = verify_draft(x.expand(B, 1, V), torch.zeros(B, 0, dtype=torch.int32, device=DEV), u, temperature=t)
    c = np.cumsum(_p(x[0, 0].double().cpu().numpy(), t))
    _same(tok[:, 0], np.searchsorted(c, u[:, 0].double().cpu().numpy() * c[-1], side="right"))


@pytest.mark.parametrize("t", [5e-324, 1e-200, 1e-50, 1e39, 1e200, 1.7e308])
@pytest.mark.parametrize("with_draft", [False, True])
def test_temperatures_outside_f32(t, with_draft):
    """Next to 0 the arg-max stands and is drawn -- with random numbers still, so equal maxima share --, far up all that is not masked is alike."""
    x, y, d, u = _inputs(6, 12, 3, 5003, torch.float32, False)
    for z in (x, y):
        z[..., 1000:2000] = -float("inf")
    x[3, :, 7] = x[3, :, 4999] = 50.0
    d[3] = 7
    d = torch.where((d >= 1000) & (d < 2000), d % 1000, d).to(torch.int32)
    _check(x, d, u, draft=y if with_draft else None, temperature=t)
