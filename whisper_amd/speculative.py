"""Speculative decoding: verification of drafted tokens against the target model's scores, from given random numbers (C ABI:
uw_verify_draft in include/uw_hip.h).  The scores are what `Engine.decoder_forward(ids, logits_all=True)` returns for the drafted
positions: one pass of the decoder scores all of them."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import lib as L

_DTYPES = {torch.float32: L.UW_DTYPE_F32, torch.bfloat16: L.UW_DTYPE_BF16}


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
    distributed as if drawn from the target alone.  A next token of -1 says that its row held a NaN or no mass."""
    if target.dim() != 3 or target.dtype not in _DTYPES:
        raise ValueError(f"target must be float32 or bfloat16 [B, N + 1, V], got {target.dtype} {tuple(target.shape)}")
    B, rows, V = target.shape
    N, dev = rows - 1, target.device
    if B == 0 or rows == 0 or V == 0:
        raise ValueError(f"empty target {tuple(target.shape)}")
    if not 0.0 <= temperature < float("inf"):
        raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    if probs and temperature not in (0.0, 1.0):
        raise ValueError("probabilities take no temperature: apply it before the softmax")
    if drafted.shape != (B, N) or drafted.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"drafted must be int32 [{B}, {N}], got {drafted.dtype} {tuple(drafted.shape)}")
    if draft is not None and (draft.shape != (B, N, V) or draft.dtype != target.dtype):
        raise ValueError(f"draft must be {target.dtype} [{B}, {N}, {V}], got {draft.dtype} {tuple(draft.shape)}")
    if temperature > 0.0 and (uniforms is None or uniforms.shape != (B, N + 1) or uniforms.dtype != torch.float32):
        raise ValueError(f"uniforms must be float32 [{B}, {N + 1}]")
    if n_drafted is not None and (n_drafted.shape != (B,) or n_drafted.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"n_drafted must be int32 [{B}]")
    for name, t in (("drafted", drafted), ("uniforms", uniforms), ("draft", draft), ("n_drafted", n_drafted)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, target on {dev}")
    if not target.is_cuda:
        raise L.UwError("target is not on a GPU: this operator runs on MI355X only (no CPU fallback)")
    if target.stride(2) != 1:
        target = target.contiguous()
    if draft is not None and draft.stride(2) != 1:
        draft = draft.contiguous()
    drafted = drafted.to(torch.int32).contiguous()
    if uniforms is not None:
        uniforms = uniforms.contiguous()
    if n_drafted is not None:
        n_drafted = n_drafted.to(torch.int32).contiguous()
    accepted = torch.empty((B,), dtype=torch.int32, device=dev)
    tokens = torch.empty((B, N + 1), dtype=torch.int32, device=dev)
    lib = L.load()
    need = lib.uw_verify_draft_workspace_bytes(B, N, V)
    ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
    ds = draft.stride() if draft is not None else (0, 0, 0)
    with torch.cuda.device(dev):
        L.check(lib.uw_verify_draft(_DTYPES[target.dtype], target.data_ptr(), target.stride(0), target.stride(1), L.ptr(draft), ds[0], ds[1],
                                    drafted.data_ptr(), L.ptr(n_drafted), L.ptr(uniforms), B, N, V, float(temperature), int(probs),
                                    accepted.data_ptr(), tokens.data_ptr(), L.ptr(ws), L.stream_handle()))
    return accepted, tokens
