"""Plain 64-bit restatement of the 8-bit paged cache's operators and of draft verification, sequence by sequence in numpy."""
import math

import numpy as np
import torch

TOP = {"int8": 127.5, "e4m3": 448.0}


def e4m3_round(y):
    y = np.clip(np.asarray(y, np.float64), -448.0, 448.0)
    _, e = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.rint(y / step) * step


def code_round(y, fmt):
    return np.clip(np.rint(y), -127, 127) if fmt == "int8" else e4m3_round(y)


def base_scale(amax, fmt):
    if amax == 0:
        return np.float32(0)
    if fmt == "int8":
        return max(np.float32(amax) * np.float32(1 / 127), np.float32(2.0 ** -126))
    m, e = math.frexp(float(amax) / 448.0)
    return np.float32(2.0 ** max(e - 1 if m == 0.5 else e, -126))


def growth(amax, s, fmt):
    need = float(amax) / (TOP[fmt] * float(s))
    if not need > 1.0:
        return 0
    m, e = math.frexp(need)
    return e - 1 if m == 0.5 else e


class Half:
    """One half (K or V) of a cache as code VALUES [pages, heads, P, D] f64 and scales f32 [pages, heads]."""

    def __init__(self, codes, scale, transposed):
        x = codes.detach().cpu()
        x = (x.to(torch.float64) if x.dtype == torch.int8 else x.to(torch.float32).to(torch.float64)).numpy()
        self.c = np.swapaxes(x, 2, 3).copy() if transposed else x.copy()
        self.s = scale.detach().cpu().numpy().copy()

    def append(self, fmt, x, page, r0):
        """x [n, heads, D] f64 into rows r0.. of a page."""
        for h in range(x.shape[1]):
            v = x[:, h]
            old = self.s[page, h]
            if not np.isfinite(v).all() or (r0 > 0 and not np.isfinite(old)):
                self.s[page, h] = np.nan
                self.c[page, h, r0:r0 + len(v)] = np.inf          # no code is inf: "unspecified"; under the scale the values are NaN
                continue
            amax = np.abs(v).max()
            if r0 == 0 or old <= 0:          # no scale is negative: leftovers of a page that was never written count as zeros
                s = base_scale(amax, fmt)
            else:
                k = growth(amax, old, fmt)
                s = np.float32(np.ldexp(np.float64(old), k))
                if k:
                    self.c[page, h, :r0] = code_round(self.c[page, h, :r0] * np.ldexp(1.0, -k), fmt)
            r = np.float64(np.float32(1) / s) if s > 0 else 0.0
            self.c[page, h, r0:r0 + len(v)] = code_round(v * r, fmt)
            self.s[page, h] = s

    def tokens(self, pages, P, n):
        """Values [n, heads, D] of a sequence's first n tokens; NaN where the page is none."""
        out = np.full((n, *self.c.shape[1:2], self.c.shape[3]), np.nan)
        for i in range(0, n, P):
            page = pages[i // P] if i // P < len(pages) else -1
            if 0 <= page < len(self.c):
                m = min(P, n - i)
                with np.errstate(invalid="ignore"):
                    out[i:i + m] = np.swapaxes(self.c[page] * self.s[page].astype(np.float64)[:, None, None], 0, 1)[:m]
        return out


def append(half, fmt, x_seqs, table, pos):
    """x_seqs: per sequence [n, heads, D] f64."""
    n_pages, _, P, _ = half.c.shape
    for b, x in enumerate(x_seqs):
        t = 0
        while t < len(x):
            p = int(pos[b]) + t
            m = min(P - p % P, len(x) - t)
            page = table[b][p // P] if p // P < len(table[b]) else -1
            if 0 <= page < n_pages:
                half.append(fmt, x[t:t + m], page, p % P)
            t += m


def attention(q, k, v, causal, scale):
    """q [n, H, D], k, v [S, Hkv, D] f64 -> out, lse, sum of p|v|, the largest sum of |q||k| scale, the spread of the scores."""
    n, H, D = q.shape
    S, G = k.shape[0], H // k.shape[1]
    out, lse, pv = np.zeros((n, H, D)), np.full((n, H), -np.inf), np.zeros((n, H, D))
    reach = np.zeros((n, H))
    for t in range(n):
        lim = max(0, S - n + t + 1) if causal else S
        if lim == 0:
            continue
        for h in range(H):
            kk, vv = k[:lim, h // G], v[:lim, h // G]
            with np.errstate(invalid="ignore"):
                s = kk @ q[t, h] * scale
                m = s.max()
                e = np.exp(s - m)
                z = e.sum()
                out[t, h], lse[t, h] = (e / z) @ vv, m + np.log(z)
                pv[t, h] = (e / z) @ np.abs(vv)
                reach[t, h] = (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale)
    return out, lse, pv, reach


def verify(target, drafted, u, draft, n_drafted, temperature, probs):
    """target [B, N+1, V], draft [B, N, V] or None (f64 numpy); returns accepted, tokens."""
    B, R, V = target.shape
    N = R - 1
    acc_out, tok_out = np.zeros(B, np.int32), np.full((B, N + 1), -1, np.int32)

    def dist(x):
        if probs:
            return x
        with np.errstate(invalid="ignore"):
            e = np.exp((x - x.max()) / temperature)
            return e / e.sum()

    for b in range(B):
        n = N if n_drafted is None else min(max(int(n_drafted[b]), 0), N)
        a = 0
        nxt = -1
        if temperature == 0:
            while True:
                x = target[b, a]
                nxt = -1 if np.isnan(x).any() else int(np.argmax(x))
                if a < n and nxt >= 0 and nxt == drafted[b, a]:
                    a += 1
                    continue
                break
        else:
            while a < n:
                d = int(drafted[b, a])
                if not 0 <= d < V:
                    break
                qd = 1.0 if draft is None else dist(draft[b, a])[d]
                if not float(u[b, a]) * qd < dist(target[b, a])[d]:
                    break
                a += 1
            p = dist(target[b, a])
            w = p
            if a < n:
                if draft is not None:
                    w = np.where(np.isnan(p - dist(draft[b, a])), np.nan, np.maximum(p - dist(draft[b, a]), 0))
                elif 0 <= drafted[b, a] < V:
                    w = p.copy()
                    w[drafted[b, a]] = 0
            if w.sum() == 0:
                w = p
            if np.isfinite(w.sum()) and w.sum() > 0:
                c = np.cumsum(w)
                over = np.nonzero(c > float(u[b, N]) * c[-1])[0]
                nxt = int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])
        acc_out[b] = a
        tok_out[b, :a] = drafted[b, :a]
        tok_out[b, a] = nxt
    return acc_out, tok_out
