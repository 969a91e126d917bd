"""Key/value cache in 8 bits: pages of tokens with a scale for each page and head, and the operators on it -- `append`, `read`
and `attention` (C ABI: uw_kv8_* in include/uw_hip.h, which states the cache's layout and every rule).

A token takes half of its bf16 size, so decoding, which is bound by the stream of cached keys and values, moves half the bytes.
Calls run on the tensors' device and its current stream, do not synchronise and may be captured into a graph."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import lib as L

_FORMATS = {"int8": (L.UW_KV8_INT8, torch.int8), "e4m3": (L.UW_KV8_E4M3, torch.float8_e4m3fn)}
_FORMAT_OF = {torch.int8: L.UW_KV8_INT8, torch.float8_e4m3fn: L.UW_KV8_E4M3}
_DTYPES = {torch.float32: L.UW_DTYPE_F32, torch.bfloat16: L.UW_DTYPE_BF16}
_UNIT = {torch.float32: 4, torch.bfloat16: 8}        # elements in 16 bytes


class KV8Cache:
    """The four tensors of a cache: k [pages, kv heads, page, head_dim] and v [pages, kv heads, head_dim, page] (int8 or
    float8_e4m3fn), k_scale and v_scale f32 [pages, kv heads]."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "_c")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dim() != 4 or k.dtype not in _FORMAT_OF or v.dtype != k.dtype:
            raise ValueError(f"codes must be int8 or float8_e4m3fn tensors of four dimensions, got {k.dtype} {tuple(k.shape)} and {v.dtype}")
        n, h, p, d = k.shape
        if v.shape != (n, h, d, p):
            raise ValueError(f"v must be [{n}, {h}, {d}, {p}] (transposed inside the page), got {tuple(v.shape)}")
        if k_scale.shape != (n, h) or v_scale.shape != (n, h) or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError(f"scales must be float32 [{n}, {h}]")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("cache tensors must be contiguous")
        if not (k.device == v.device == k_scale.device == v_scale.device):
            raise ValueError("cache tensors must be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._c = L.UwKv8Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, h, p, d, _FORMAT_OF[k.dtype])

    @classmethod
    def allocate(cls, n_pages: int, n_kv_heads: int, head_dim: int = 64, page: int = 64, fmt: str = "int8",
                 device="cuda:0") -> "KV8Cache":
        """An empty cache; fmt "int8" (finer for well-spread values) or "e4m3" (finer for blocks with outliers)."""
        if fmt not in _FORMATS:
            raise ValueError(f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")
        dt = _FORMATS[fmt][1]
        codes = torch.zeros((2, n_pages, n_kv_heads, page * head_dim), dtype=torch.uint8, device=device).view(dt)
        scales = torch.zeros((2, n_pages, n_kv_heads), dtype=torch.float32, device=device)
        return cls(codes[0].view(n_pages, n_kv_heads, page, head_dim), codes[1].view(n_pages, n_kv_heads, head_dim, page),
                   scales[0], scales[1])

    n_pages = property(lambda self: self.k.shape[0])
    n_kv_heads = property(lambda self: self.k.shape[1])
    page = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])


def _index(x: torch.Tensor, n: Optional[int], what: str, device) -> torch.Tensor:
    if x.dtype not in (torch.int32, torch.int64) or x.dim() != 1 or (n is not None and x.shape[0] != n):
        raise ValueError(f"{what} must be an int32 tensor" + (f" of {n} elements" if n is not None else ""))
    if x.device != device:
        raise ValueError(f"{what} is on {x.device}, the cache on {device}")
    return x if x.dtype == torch.int32 and x.is_contiguous() else x.to(torch.int32).contiguous()


def _tokens(x: torch.Tensor, what: str, cache: KV8Cache, B: int, tok_start) -> Tuple[torch.Tensor, "L.UwKv8Tokens"]:
    """x [B, T, heads, head_dim], or [N, heads, head_dim] with tok_start -> the tensor to keep alive and its description."""
    dims = 3 if tok_start is not None else 4
    if x.dim() != dims or x.shape[-1] != cache.k.shape[3] or x.dtype not in _DTYPES:
        raise ValueError(f"{what} must be float32 or bfloat16 " + ("[rows, heads, " if dims == 3 else "[B, T, heads, ")
                         + f"{cache.k.shape[3]}], got {x.dtype} {tuple(x.shape)}")
    if dims == 4 and x.shape[0] != B:
        raise ValueError(f"{what} holds {x.shape[0]} sequences, the page table {B}")
    if x.device != cache.k.device:
        raise ValueError(f"{what} is on {x.device}, the cache on {cache.k.device}")
    st, unit = x.stride(), _UNIT[x.dtype]
    if st[-1] != 1 or x.data_ptr() % 16 or st[-2] % unit or st[-3] % unit or (dims == 4 and st[0] % unit):
        x = x.contiguous()                       # rows the kernels cannot fetch in 16-byte pieces
        st = x.stride()
        if x.data_ptr() % 16:
            x = x.clone()
    if dims == 4:
        return x, L.UwKv8Tokens(x.data_ptr(), st[0], st[1], st[2], x.shape[0] * x.shape[1], None, B, x.shape[1])
    return x, L.UwKv8Tokens(x.data_ptr(), 0, st[0], st[1], x.shape[0], tok_start.data_ptr(), B, 0)


def _table(table: torch.Tensor, cache: KV8Cache) -> torch.Tensor:
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous() or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"the page table must be a contiguous int32 tensor [B, blocks], got {table.dtype} {tuple(table.shape)}")
    if table.device != cache.k.device:
        raise ValueError(f"the page table is on {table.device}, the cache on {cache.k.device}")
    return table


def _on_gpu(cache: KV8Cache) -> None:
    if not cache.k.is_cuda:
        raise L.UwError("the cache is not on a GPU: these operators run on MI355X only (no CPU fallback)")


def append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, pos: torch.Tensor,
           tok_start: Optional[torch.Tensor] = None) -> None:
    """Stores new keys and values behind the pos[b] tokens that sequence b has: k, v [B, T, kv heads, head_dim], or
    [N, kv heads, head_dim] of sequences packed one behind the other with tok_start [B + 1].  table i32 [B, blocks]."""
    table = _table(table, cache)
    B = table.shape[0]
    pos = _index(pos, B, "pos", table.device)
    if tok_start is not None:
        tok_start = _index(tok_start, B + 1, "tok_start", table.device)
    k, ck = _tokens(k, "k", cache, B, tok_start)
    v, cv = _tokens(v, "v", cache, B, tok_start)
    if k.shape != v.shape or k.dtype != v.dtype or k.shape[-2] != cache.k.shape[1]:
        raise ValueError(f"k and v must be alike, with {cache.k.shape[1]} heads: got {tuple(k.shape)} and {tuple(v.shape)}")
    _on_gpu(cache)
    with torch.cuda.device(table.device):
        L.check(L.load().uw_kv8_append(C.byref(cache._c), _DTYPES[k.dtype], C.byref(ck), C.byref(cv), table.data_ptr(),
                                       table.shape[1], pos.data_ptr(), L.stream_handle()))


def read(cache: KV8Cache, table: torch.Tensor, first: torch.Tensor, n_tok: int, tok_start: Optional[torch.Tensor] = None,
         dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of cached tokens: n_tok of each sequence from position first[b] on -> k, v [B, n_tok, kv heads, head_dim]; with
    tok_start [B + 1], tok_start[b + 1] - tok_start[b] of sequence b, n_tok rows altogether -> [n_tok, kv heads, head_dim] (rows
    behind tok_start[B] are zero)."""
    table = _table(table, cache)
    B, dev = table.shape[0], table.device
    first = _index(first, B, "first", dev)
    if dtype not in _DTYPES or n_tok < 0:
        raise ValueError(f"float32 or bfloat16 and a count, got {dtype} and {n_tok}")
    heads = (cache.k.shape[1], cache.k.shape[3])
    if tok_start is not None:
        tok_start = _index(tok_start, B + 1, "tok_start", dev)
    _on_gpu(cache)
    if tok_start is not None:
        k, v = torch.zeros((2, n_tok, *heads), dtype=dtype, device=dev)
    else:
        k, v = torch.empty((2, B, n_tok, *heads), dtype=dtype, device=dev)
    k, ck = _tokens(k, "k", cache, B, tok_start)
    v, cv = _tokens(v, "v", cache, B, tok_start)
    with torch.cuda.device(dev):
        L.check(L.load().uw_kv8_read(C.byref(cache._c), _DTYPES[dtype], C.byref(ck), C.byref(cv), table.data_ptr(), table.shape[1],
                                     first.data_ptr(), L.stream_handle()))
    return k, v


def attention(q: torch.Tensor, cache: KV8Cache, table: torch.Tensor, kv_len: torch.Tensor, tok_start: Optional[torch.Tensor] = None,
              causal: bool = True, scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """softmax(scale * q . K) V over the first kv_len[b] cached tokens of each sequence.  q [B, T, heads, head_dim], or
    [N, heads, head_dim] with tok_start [B + 1]; heads a multiple of the cache's (grouped heads lie side by side).  causal: the
    last of a sequence's n query tokens sees kv_len[b] keys, the one before one less, and so on; a token that sees none gives 0.
    scale defaults to head_dim ** -0.5 (pass 1.0 for queries scaled before).  Returns the output (in `out`, contiguous and shaped
    like q, if given; its rows behind tok_start[B] are left as they were) and, with return_lse, f32 log-sum-exp
    [..., heads]."""
    table = _table(table, cache)
    B, dev = table.shape[0], table.device
    kv_len = _index(kv_len, B, "kv_len", dev)
    if tok_start is not None:
        tok_start = _index(tok_start, B + 1, "tok_start", dev)
    q, cq = _tokens(q, "q", cache, B, tok_start)
    heads = q.shape[-2]
    if heads % cache.k.shape[1]:
        raise ValueError(f"{heads} query heads over {cache.k.shape[1]} cached heads")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev) if tok_start is None else torch.zeros(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous, 16-byte aligned and like q")
    _on_gpu(cache)
    out, co = _tokens(out, "out", cache, B, tok_start)
    lse = None
    if return_lse:
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev)
        if tok_start is not None:
            lse.fill_(float("-inf"))
    lib = L.load()
    need = lib.uw_kv8_attention_workspace_bytes(C.byref(cache._c), heads, B, cq.n_tok, cq.T, table.shape[1])
    ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
    with torch.cuda.device(dev):
        L.check(lib.uw_kv8_attention(C.byref(cache._c), _DTYPES[q.dtype], C.byref(cq), C.byref(co), L.ptr(lse), heads, table.data_ptr(),
                                     table.shape[1], kv_len.data_ptr(), int(causal), q.shape[-1] ** -0.5 if scale is None else float(scale),
                                     L.ptr(ws), L.stream_handle()))
    return (out, lse) if return_lse else out
