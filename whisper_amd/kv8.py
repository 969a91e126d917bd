"""Key/value cache in 8 bits: pages of tokens with a scale for each page and head, and the operators on it -- `append`, `read`
and `attention` (C ABI: uw_kv8_* in include/uw_hip.h, which states the cache's layout and every rule).

A token takes half of its bf16 size, so decoding, which is bound by the stream of cached keys and values, moves half the bytes.
Calls run on the tensors' device and its current stream, do not synchronise and may be captured into a graph."""
from __future__ import annotations

from functools import lru_cache
from struct import Struct
from typing import Optional, Tuple

import torch

from . import lib as L

_FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_FORMAT_OF = {torch.int8: L.UW_KV8_INT8, torch.float8_e4m3fn: L.UW_KV8_E4M3}
_DTYPES = {torch.float32: L.UW_DTYPE_F32, torch.bfloat16: L.UW_DTYPE_BF16}

_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16
_F32_MAX = torch.finfo(torch.float32).max
# the argument structures of the C ABI behind their uw_kv8_cache
_CACHE = Struct("@4P6i")
_CACHE_DIMS = Struct("@6i")
_ADDRESSES = 32                                  # bytes of a uw_kv8_cache in front of its sizes
_STORE = Struct("@3Pq4i P3q P3q")
_ATTEND = Struct("@3Pq4i P3q P3q 2Pq2ifi")


class KV8Cache:
    """The four tensors of a cache: k [pages, kv heads, page, head_dim] and v [pages, kv heads, head_dim, page] (int8 or
    float8_e4m3fn), k_scale and v_scale f32 [pages, kv heads].  A cache keeps the tensors it was made of."""

    __slots__ = ("_tensors", "_ks", "_c", "_dev", "_h", "_d")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        dtype = k.dtype
        fmt = _FORMAT_OF.get(dtype)
        if fmt is None or v.dtype is not dtype or k.dim() != 4:
            raise ValueError(f"codes must be int8 or float8_e4m3fn tensors of four dimensions, got {k.dtype} {tuple(k.shape)} and {v.dtype}")
        n, h, p, d = k.shape
        if v.shape != (n, h, d, p):
            raise ValueError(f"v must be [{n}, {h}, {d}, {p}] (transposed inside the page), got {tuple(v.shape)}")
        if k_scale.shape != (n, h) or v_scale.shape != (n, h) or k_scale.dtype is not _F32 or v_scale.dtype is not _F32:
            raise ValueError(f"scales must be float32 [{n}, {h}]")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("cache tensors must be contiguous")
        dev = k.get_device()
        if v.get_device() != dev or k_scale.get_device() != dev or v_scale.get_device() != dev:
            raise ValueError("cache tensors must be on one device")
        self._tensors, self._ks = (k, v, k_scale, v_scale), k_scale
        self._c = _CACHE.pack(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, h, p, d, fmt, 0)
        self._dev, self._h, self._d = dev, h, d

    @classmethod
    def allocate(cls, n_pages: int, n_kv_heads: int, head_dim: int = 64, page: int = 64, fmt: str = "int8",
                 device="cuda:0") -> "KV8Cache":
        """An empty cache; fmt "int8" (finer for well-spread values) or "e4m3" (finer for blocks with outliers)."""
        if fmt not in _FORMATS:
            raise ValueError(f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")
        codes = torch.zeros((2, n_pages, n_kv_heads, page * head_dim), dtype=torch.uint8, device=device).view(_FORMATS[fmt])
        scales = torch.zeros((2, n_pages, n_kv_heads), dtype=torch.float32, device=device)
        return cls(codes[0].view(n_pages, n_kv_heads, page, head_dim), codes[1].view(n_pages, n_kv_heads, head_dim, page),
                   scales[0], scales[1])

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])
    n_pages = property(lambda self: self.k.shape[0])
    n_kv_heads = property(lambda self: self.k.shape[1])
    page = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])


# The checks come in an order that lets a sound argument through with the fewest questions: a call's arguments cost as much time as its
# kernel when there is little to do.
def narrowed(x: torch.Tensor) -> torch.Tensor:
    """Whole numbers as contiguous int32; of 64 bits, those that 32 do not hold become the outermost that they do."""
    return (x.clamp(-(1 << 31), (1 << 31) - 1) if x.dtype is torch.int64 else x).to(_I32).contiguous()


def _index(x: torch.Tensor, n: int, what: str, dev: int) -> torch.Tensor:
    if x.dtype is _I32 and x.dim() == 1 and x.numel() == n and x.get_device() == dev and x.is_contiguous():
        return x
    if x.shape != (n,) or x.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what} must be an int32 tensor of {n} elements, got {x.dtype} {tuple(x.shape)}")
    if x.get_device() != dev:
        raise ValueError(f"{what} is on {x.device}, not on the cache's device")
    return narrowed(x)


def _tokens(x: torch.Tensor, shape: torch.Size, what: str, cache: KV8Cache, B: int, packed: bool):
    """x [B, T, heads, head_dim], or [N, heads, head_dim] if packed -> the tensor to keep alive, its type and (address, strides)."""
    st, dtype = x.stride(), x.dtype
    code, unit = (L.UW_DTYPE_BF16, 7) if dtype is _BF16 else (L.UW_DTYPE_F32, 3) if dtype is _F32 else (-1, 0)
    if len(st) != (3 if packed else 4) or code < 0 or shape[-1] != cache._d:
        raise ValueError(f"{what} must be float32 or bfloat16 " + ("[rows, heads, " if packed else "[B, T, heads, ")
                         + f"{cache._d}], got {dtype} {tuple(shape)}")
    if not packed and shape[0] != B:
        raise ValueError(f"{what} holds {shape[0]} sequences, the page table {B}")
    if x.get_device() != cache._dev:
        raise ValueError(f"{what} is on {x.device}, not on the cache's device")
    at = x.data_ptr()
    if st[-1] != 1 or at & 15 or (st[-2] | st[-3] | st[0]) & unit:      # unit: elements in 16 bytes, less one
        x = x.clone(memory_format=torch.contiguous_format)      # rows the kernels cannot fetch in 16-byte pieces
        st, at = x.stride(), x.data_ptr()
    return x, code, ((at, 0, st[0], st[1]) if packed else (at, st[0], st[1], st[2]))


def _table(table: torch.Tensor, cache: KV8Cache) -> Tuple[int, int]:
    B, width = table.shape if table.dim() == 2 else (0, 0)
    if not B or not width or table.dtype is not _I32 or not table.is_contiguous():
        raise ValueError(f"the page table must be a contiguous int32 tensor [B, blocks], got {table.dtype} {tuple(table.shape)}")
    if table.get_device() != cache._dev:
        raise ValueError(f"the page table is on {table.device}, not on the cache's device")
    return B, width


# the current stream's handle: what torch.cuda.current_stream(dev).cuda_stream answers, without making a Stream object (2.7 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(fn, args: bytes, dev: int) -> None:
    if torch.cuda.current_device() == dev:
        rc = fn(args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(args, _raw_stream(dev))
    if rc:
        L.check(rc)


def _on_gpu(cache: KV8Cache) -> None:
    if cache._dev < 0:
        raise L.UwError("the cache is not on a GPU: these operators run on MI355X only (no CPU fallback)")


def append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, pos: torch.Tensor,
           tok_start: Optional[torch.Tensor] = None) -> None:
    """Stores new keys and values behind the pos[b] tokens that sequence b has: k, v [B, T, kv heads, head_dim], or
    [N, kv heads, head_dim] of sequences packed one behind the other with tok_start [B + 1].  table i32 [B, blocks]."""
    B, width = _table(table, cache)
    dev = cache._dev
    pos = _index(pos, B, "pos", dev)
    packed = tok_start is not None
    if packed:
        tok_start = _index(tok_start, B + 1, "tok_start", dev)
    shape = k.shape
    if shape != v.shape or k.dtype != v.dtype or len(shape) < 3 or shape[-2] != cache._h:
        raise ValueError(f"k and v must be alike, with {cache._h} heads: got {k.dtype} {tuple(shape)} and {v.dtype} {tuple(v.shape)}")
    k, dtype, ck = _tokens(k, shape, "k", cache, B, packed)
    v, _, cv = _tokens(v, shape, "v", cache, B, packed)
    _on_gpu(cache)
    n, T = (shape[0], 0) if packed else (B * shape[1], shape[1])
    _call(L.load().uw_kv8_append, cache._c + _STORE.pack(table.data_ptr(), pos.data_ptr(), tok_start.data_ptr() if packed else 0, n, width,
                                                         B, T, dtype, *ck, *cv), dev)


def read(cache: KV8Cache, table: torch.Tensor, first: torch.Tensor, n_tok: int, tok_start: Optional[torch.Tensor] = None,
         dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of cached tokens: n_tok of each sequence from position first[b] on -> k, v [B, n_tok, kv heads, head_dim]; with
    tok_start [B + 1], tok_start[b + 1] - tok_start[b] of sequence b, n_tok rows altogether -> [n_tok, kv heads, head_dim] (rows
    behind tok_start[B] are not written)."""
    B, width = _table(table, cache)
    dev = cache._dev
    first = _index(first, B, "first", dev)
    if dtype not in _DTYPES or n_tok < 0:
        raise ValueError(f"float32 or bfloat16 and a count, got {dtype} and {n_tok}")
    packed = tok_start is not None
    if packed:
        tok_start = _index(tok_start, B + 1, "tok_start", dev)
    _on_gpu(cache)
    h, d = cache._h, cache._d
    k = cache._ks.new_empty((n_tok, h, d) if packed else (B, n_tok, h, d), dtype=dtype)
    v = torch.empty_like(k)
    st = (0, h * d, d) if packed else (n_tok * h * d, h * d, d)
    _call(L.load().uw_kv8_read, cache._c + _STORE.pack(table.data_ptr(), first.data_ptr(), tok_start.data_ptr() if packed else 0,
                                                       n_tok if packed else B * n_tok, width, B, 0 if packed else n_tok, _DTYPES[dtype],
                                                       k.data_ptr(), *st, v.data_ptr(), *st), dev)
    return k, v


@lru_cache(maxsize=4096)
def _workspace_bytes(dims: bytes, n: int, width: int, B: int, T: int, dtype: int, packed: bool, heads: int) -> int:
    """Scratch of a call of these sizes (they alone decide: the addresses here are none)."""
    need = L.load().uw_kv8_attention_workspace_bytes(_CACHE.pack(64, 64, 64, 64, *_CACHE_DIMS.unpack(dims)) + _ATTEND.pack(
        64, 64, 64 if packed else 0, n, width, B, T, dtype, 64, 0, 0, 0, 64, 0, 0, 0, 0, 0, 0, heads, 0, 1.0, 0))
    if need < 0:
        L.check(1)
    return (need + 15) // 16 * 16


def attention(q: torch.Tensor, cache: KV8Cache, table: torch.Tensor, kv_len: torch.Tensor, tok_start: Optional[torch.Tensor] = None,
              causal: bool = True, scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """softmax(scale * q . K) V over the first kv_len[b] cached tokens of each sequence.  q [B, T, heads, head_dim], or
    [N, heads, head_dim] with tok_start [B + 1]; heads a multiple of the cache's (grouped heads lie side by side).  causal: the
    last of a sequence's n query tokens sees kv_len[b] keys, the one before one less, and so on; a token that sees none gives 0.
    scale defaults to head_dim ** -0.5 (pass 1.0 for queries scaled before).  Returns the output (in `out`, contiguous and shaped
    like q, if given; q itself will do) and, with return_lse, f32 log-sum-exp [..., heads].  Rows behind tok_start[B] are not written."""
    B, width = _table(table, cache)
    dev = cache._dev
    kv_len = _index(kv_len, B, "kv_len", dev)
    packed = tok_start is not None
    if packed:
        tok_start = _index(tok_start, B + 1, "tok_start", dev)
    shape = q.shape
    q, dtype, cq = _tokens(q, shape, "q", cache, B, packed)
    heads, d = shape[-2], cache._d
    if heads % cache._h or heads == 0:
        raise ValueError(f"{heads} query heads over {cache._h} cached heads")
    if scale is None:
        scale = d ** -0.5
    elif not abs(scale) <= _F32_MAX:
        raise ValueError(f"scale must be a finite f32 number, got {scale}")
    if out is not None and (out.shape != shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous() or out.data_ptr() & 15):
        raise ValueError("out must be contiguous, 16-byte aligned and like q")
    if out is not None and out.numel() and not (out.data_ptr() == q.data_ptr() and q.is_contiguous()):
        span = 1 + sum((n - 1) * s for n, s in zip(shape, q.stride()))
        if q.data_ptr() < out.data_ptr() + out.numel() * q.element_size() and out.data_ptr() < q.data_ptr() + span * q.element_size():
            raise ValueError("out must not overlap q (but may be q itself, if that is contiguous)")
    _on_gpu(cache)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)
    n, T = (shape[0], 0) if packed else (B * shape[1], shape[1])
    lse = cache._ks.new_empty((n, heads) if packed else (B, T, heads)) if return_lse else None
    need = _workspace_bytes(cache._c[_ADDRESSES:], n, width, B, T, dtype, packed, heads)
    ws = cache._ks.new_empty(need // 4) if need else None
    _call(L.load().uw_kv8_attention, cache._c + _ATTEND.pack(
        table.data_ptr(), kv_len.data_ptr(), tok_start.data_ptr() if packed else 0, n, width, B, T, dtype, *cq, out.data_ptr(), T * heads * d,
        heads * d, d, lse.data_ptr() if return_lse else 0, ws.data_ptr() if need else 0, need, heads, 1 if causal else 0,
        float(scale), 0), dev)
    return (out, lse) if return_lse else out
