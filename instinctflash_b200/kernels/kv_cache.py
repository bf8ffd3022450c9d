"""A paged key/value cache in 8 bits, with a scale for each page and head, and attention over it.

What ``rope.qkv_split`` leaves in 16 bits goes into the cache with ``cache_append``; ``cache_attention`` reads the codes
as they are.  Half the bytes of a 16-bit cache, which are what a step of one token a sequence waits for.

    pages   k, v [pages, heads, page_tokens, head_dim] e4m3;  k_scale, v_scale [pages, heads] float32
    table   [batch, max_pages] int32: the pages of a sequence in order, ``page_tokens`` tokens each

Masks leave a query the keys below a limit of its own.  Query token t of n of a sequence of length L (which counts the new
tokens) stands at position p = L - n + t and sees the keys j with

    j < L                                    ``causal=False``
    j < L and (j <= p or j < prefix)         ``causal=True``

The reference has no counterpart; head order, scaling and workspaces follow ``attention``.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from ._common import E4M3, launch, native, same_device

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_HEAD_DIMS = (64, 128, 256)


@dataclass
class KVCache8:
    k: torch.Tensor        # [pages, heads, page_tokens, head_dim] e4m3
    v: torch.Tensor
    k_scale: torch.Tensor  # [pages, heads] float32: a code stands for code * scale
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, heads: int, page_tokens: int, head_dim: int, device) -> "KVCache8":
        codes = [torch.zeros(pages, heads, page_tokens, head_dim, device=device, dtype=E4M3) for _ in range(2)]
        return cls(*codes, *(torch.zeros(pages, heads, device=device) for _ in range(2)))


def attention_workspace(device, nbytes: int = 16 << 20) -> torch.Tensor:
    """Scratch of ``cache_attention`` for calls that run one after the other.  It has to start at zero and is handed back
    that way where it matters; any size is right, a larger one lets more GPU multiprocessors share a long sequence."""
    return torch.zeros(nbytes, device=device, dtype=torch.uint8)


def _cache(cache):
    k = cache.k
    if not isinstance(k, torch.Tensor) or k.ndim != 4 or k.dtype != E4M3:
        raise ValueError("cache.k must be an e4m3 [pages, heads, page_tokens, head_dim] tensor")
    if k.device.type != "cuda":
        raise ValueError("cache.k must live on a CUDA device; this path has no CPU implementation")
    pages, heads, page_tokens, head_dim = k.shape
    if head_dim not in _HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
    if page_tokens < 16 or page_tokens > 256 or page_tokens % 16:
        raise ValueError(f"page_tokens must be a multiple of 16, at most 256, got {page_tokens}")
    if cache.v.shape != k.shape or cache.v.dtype != E4M3 or not k.is_contiguous() or not cache.v.is_contiguous():
        raise ValueError("cache.k and cache.v must be contiguous e4m3 tensors of one shape")
    for name in ("k_scale", "v_scale"):
        t = getattr(cache, name)
        if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads) or not t.is_contiguous():
            raise ValueError(f"cache.{name} must be a contiguous float32 [{pages}, {heads}] tensor")
    same_device(k, v=cache.v, k_scale=cache.k_scale, v_scale=cache.v_scale)
    return pages, heads, page_tokens, head_dim


def _ints(t, name, shape, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.ndim != len(shape) or t.device != device \
            or any(n is not None and t.shape[i] != n for i, n in enumerate(shape)) or (t.numel() > 0 and t.stride(-1) != 1
                                                                                    and t.shape[-1] > 1):
        raise ValueError(f"{name} must be an int32 tensor of shape {[n if n is not None else 'any' for n in shape]} on {device}, "
                         "contiguous in its last dimension")
    return t


def _heads(t, name, batch, heads, head_dim, dtypes, device):
    if not isinstance(t, torch.Tensor) or t.ndim != 4 or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a [batch, tokens, heads, head_dim] tensor of one of {tuple(dtypes)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if (batch is not None and t.shape[0] != batch) or (heads is not None and t.shape[2] != heads) or t.shape[3] != head_dim:
        raise ValueError(f"{name} has shape {tuple(t.shape)}")
    if t.stride(3) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return t


def cache_append(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, *,
                 counts: torch.Tensor | None = None) -> None:
    """Write ``k``, ``v`` [B, T, heads, head_dim] (float32, bfloat16 or float16) at positions ``start[b] + t``.

    A page's scale becomes the least power of two that brings its largest value to 448 or below, and never less than it
    was: what the page holds below ``start[b]`` is rescaled where the scale grows (exactly, but for codes that fall below
    2^-6).  A page whose first token is written starts afresh.  Values that are not finite become NaN codes and do not
    enter the scale.  ``counts`` [B] int32: only the first ``counts[b]`` tokens of a row are there.  Tokens whose page lies
    beyond the table, or whose entry is no page of the cache, are dropped, and so is a row with a negative start.  A page must
    belong to one sequence of the call, in one place of its table, and what it holds at and above ``start[b] + counts[b]`` is not
    kept up."""
    if native.cache_append(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, table, start, counts):
        return
    pages, heads, page_tokens, head_dim = _cache(cache)
    dev = cache.k.device
    _heads(k, "k", None, heads, head_dim, _FLOATS, dev)
    B, T = k.shape[:2]
    _heads(v, "v", B, heads, head_dim, (k.dtype,), dev)
    if v.shape[1] != T:
        raise ValueError("k and v must have the same number of tokens")
    _ints(table, "table", (B, None), dev)
    _ints(start, "start", (B,), dev)
    _ints(counts, "counts", (B,), dev)
    launch("iflb200_cache_append", cache.k, k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0),
           v.stride(1), v.stride(2), _lib.dtype_code(k.dtype), B, T, heads, head_dim, cache.k.data_ptr(), cache.v.data_ptr(),
           cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages, page_tokens, table.data_ptr(), table.stride(0),
           table.shape[1], start.data_ptr(), _lib.ptr(counts))


def cache_attention(q: torch.Tensor, cache: KVCache8, table: torch.Tensor, lens: torch.Tensor, out: torch.Tensor, *,
                    causal: bool = True, prefix: torch.Tensor | None = None, softcap: float = 0.0,
                    slopes: torch.Tensor | None = None, scale: float | None = None, q_lens: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """out [B, T, heads_q, head_dim] = attention of ``q`` (the same shape, bfloat16 or float16) over the cache.

    Query head i reads head ``i // (heads_q // heads)``.  ``lens`` [B] int32 are the sequences' lengths with the new
    tokens.  Scores are ``scale`` (head_dim ** -0.5) * q.k, then ``softcap * tanh(score / softcap)`` where that is not 0,
    then minus ``slopes[i] * |p - j|`` (float32 [heads_q]), then masked (see above; ``prefix`` [B] int32).

    ``q_lens`` [B] int32: only the first ``q_lens[b]`` tokens of a row are there; the rows of ``out`` behind them are left
    as they were.  A query that sees no key gets zeros.  A length above what the table holds counts as what it holds;
    tokens of a page that is no page of the cache are masked.  Keys and values that a query does not see may hold
    anything.  A value scale is 0 (the page's values are zeros) or lies between 2^-60 and 2^60, those of a sequence's pages within
    2^96 of one another, where 0 counts as 2^-60.  More than 2^6 among them costs time: many rows take a pass over the keys for each
    2^6 that has pages.  ``out`` must not overlap itself, nor ``q`` unless it is ``q``.

    Scores and all sums are float32.  The weights enter the product as float16: 2^-11 off each, or 2^-28 of the row's largest
    probability where that is more; an element of a bfloat16 ``q`` is off by 2^-40 of its row's largest at most (where that is 2^-111
    at least).  A table holds 2^30 tokens of a sequence at most, a call B up to 65535 and T * heads_q up to eight million.

    ``workspace``: see ``attention_workspace``; without one a sequence is not shared among multiprocessors.  How far it is shared
    goes by what the table holds, not by ``lens``: a table no wider than the longest sequence is the fastest (one sequence of 2048
    tokens, 8 heads of 128: 1.4 times the time in a table 16 times as wide)."""
    if native.cache_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, lens, out, causal, prefix, softcap,
                              slopes, scale, q_lens, workspace):
        return out
    pages, heads, page_tokens, head_dim = _cache(cache)
    dev = cache.k.device
    _heads(q, "q", None, None, head_dim, (torch.bfloat16, torch.float16), dev)
    B, T, heads_q = q.shape[:3]
    _heads(out, "out", B, heads_q, head_dim, (q.dtype,), dev)
    if out.shape[1] != T:
        raise ValueError("out must have the shape of q")
    if heads < 1 or heads_q % heads or heads_q < 1:
        raise ValueError("heads_q must be a multiple of the cache's heads")
    _ints(table, "table", (B, None), dev)
    _ints(lens, "lens", (B,), dev)
    _ints(q_lens, "q_lens", (B,), dev)
    _ints(prefix, "prefix", (B,), dev)
    if prefix is not None and not causal:
        raise ValueError("prefix goes with causal=True: without it every key is seen")
    f32 = torch.finfo(torch.float32)
    if not (softcap == 0.0 or f32.tiny <= softcap <= f32.max):
        raise ValueError("softcap must be 0 (none) or a positive, finite, normal float32 number")
    if scale is not None and not abs(scale) <= f32.max:
        raise ValueError("scale must be a finite float32 number")
    if slopes is not None and (slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads_q,) or not slopes.is_contiguous()):
        raise ValueError(f"slopes must be a contiguous float32 [{heads_q}] tensor")
    if workspace is not None and (workspace.dtype != torch.uint8 or workspace.ndim != 1 or not workspace.is_contiguous()
                                  or workspace.data_ptr() % 16):
        raise ValueError("workspace must be a contiguous 16-byte aligned uint8 vector")
    same_device(cache.k, slopes=slopes, workspace=workspace)
    launch("iflb200_cache_attention", cache.k, q.data_ptr(), _lib.dtype_code(q.dtype), q.stride(0), q.stride(1), q.stride(2),
           cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages, page_tokens,
           head_dim, table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(), _lib.ptr(q_lens), _lib.ptr(prefix),
           _lib.ptr(slopes), B, T, heads_q, heads, float(head_dim ** -0.5 if scale is None else scale), float(softcap),
           int(bool(causal)), out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), _lib.ptr(workspace),
           workspace.numel() if workspace is not None else 0)
    return out
