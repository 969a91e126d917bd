"""Speculative decoding: verification of drafted tokens against the target model's scores, from given random numbers (C ABI:
uw_verify_draft in include/uw_hip.h).  The scores are what `Engine.decoder_forward(ids, logits_all=True)` returns for the drafted
positions: one pass of the decoder scores all of them."""
from __future__ import annotations

from functools import lru_cache
from struct import Struct
from typing import Optional, Tuple

import torch

from . import lib as L
from .kv8 import _call, narrowed

_DTYPES = {torch.float32: L.UW_DTYPE_F32, torch.bfloat16: L.UW_DTYPE_BF16}
_ARGS = Struct("@P2q P2q 5P Pq 4idi4x")        # uw_verify_args


def _ints(x: torch.Tensor, shape, what: str, dev: int) -> torch.Tensor:
    if x.shape != shape or x.dtype not in (torch.int32, torch.int64) or x.get_device() != dev:
        raise ValueError(f"{what} must be int32 {list(shape)} beside target, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x if x.dtype is torch.int32 and x.is_contiguous() else narrowed(x)


@lru_cache(maxsize=4096)
def _workspace_bytes(dtype: int, B: int, N: int, V: int, greedy: bool, probs: bool, with_draft: bool) -> int:
    """Scratch of a call of these sizes (they alone decide: the addresses here are none)."""
    need = L.load().uw_verify_draft_workspace_bytes(_ARGS.pack(64, 0, 0, 64 if with_draft else 0, 0, 0, 64, 0, 64, 64, 64, 0, 0, dtype, B, N, V,
                                                               0.0 if greedy else 1.0, 1 if probs else 0))
    if need < 0:
        L.check(1)
    return (need + 15) // 16 * 16


def verify_draft(target: torch.Tensor, drafted: torch.Tensor, uniforms: Optional[torch.Tensor] = None,
                 draft: Optional[torch.Tensor] = None, n_drafted: Optional[torch.Tensor] = None, temperature: float = 1.0,
                 probs: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which of the drafted tokens the target model accepts, and the token that follows them.

    target [B, N + 1, V]: the target's logits at the drafted positions and the one behind (or probabilities, with probs=True);
    drafted i32 [B, N]; uniforms f32 [B, N + 1] in [0, 1): column i decides about token i, the last draws the next token.
    draft [B, N, V]: the drafter's logits (probabilities); None for a drafter that is certain of its tokens.  n_drafted i32 [B]:
    how many of the N columns hold a token (default all).  temperature 0 is greedy verification: a token stands while it is the
    arg-max of its row; uniforms and draft are not used.

    Returns accepted i32 [B] and tokens i32 [B, N + 1]: the accepted tokens, then the next token, then -1.  The tokens are
    distributed as if drawn from the target alone.  A next token of -1 says that its row held a NaN or no mass
    (greedy: a NaN)."""
    shape = target.shape
    if len(shape) != 3 or target.dtype not in _DTYPES:
        raise ValueError(f"target must be float32 or bfloat16 [B, N + 1, V], got {target.dtype} {tuple(shape)}")
    if 0 in shape:
        raise ValueError(f"empty target {tuple(shape)}")
    B, N, V = shape[0], shape[1] - 1, shape[2]
    dev = target.get_device()
    if not 0.0 <= temperature < float("inf"):
        raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    greedy = temperature == 0.0
    if probs and not greedy and temperature != 1.0:
        raise ValueError("probabilities take no temperature: apply it before the softmax")
    drafted = _ints(drafted, (B, N), "drafted", dev)
    if n_drafted is not None:
        n_drafted = _ints(n_drafted, (B,), "n_drafted", dev)
    if draft is not None:
        if draft.shape != (B, N, V) or draft.dtype != target.dtype or draft.get_device() != dev:
            raise ValueError(f"draft must be {target.dtype} [{B}, {N}, {V}] beside target, got {draft.dtype} {tuple(draft.shape)} on {draft.device}")
        if draft.stride(2) != 1:
            draft = draft.contiguous()
    if not greedy:
        if uniforms is None or uniforms.shape != (B, N + 1) or uniforms.dtype != torch.float32 or uniforms.get_device() != dev:
            raise ValueError(f"uniforms must be float32 [{B}, {N + 1}] beside target")
        uniforms = uniforms.contiguous()
    if dev < 0:
        raise L.UwError("target is not on a GPU: this operator runs on MI355X only (no CPU fallback)")
    st = target.stride()
    if st[2] != 1:
        target = target.contiguous()
        st = target.stride()
    accepted, tokens = drafted.new_empty(B), drafted.new_empty((B, N + 1))
    if draft is None or greedy:
        at, dB, dN = 0, 0, 0
    else:
        at, (dB, dN, _) = draft.data_ptr(), draft.stride()
    dtype = _DTYPES[target.dtype]
    need = _workspace_bytes(dtype, B, N, V, greedy, probs, at != 0)
    ws = drafted.new_empty(need // 4)
    _call(L.load().uw_verify_draft, _ARGS.pack(
        target.data_ptr(), st[0], st[1], at, dB, dN, drafted.data_ptr(), 0 if n_drafted is None else n_drafted.data_ptr(),
        0 if greedy else uniforms.data_ptr(), accepted.data_ptr(), tokens.data_ptr(), ws.data_ptr(), need, dtype, B, N, V, temperature,
        1 if probs else 0), dev)
    return accepted, tokens
