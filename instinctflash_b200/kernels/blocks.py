"""FP8 linear with a scale for each block: 1 x 128 activations, 128 x 128 weights.

Beside the per-token / per-channel path of ``fp8`` and ``norm``: one large channel takes precision only
from the 128 columns of its block, not from its whole row.  The calls of a layer are the same:
``block_quant`` where activations are produced (with ``act`` behind a fused ``[gate | up]`` projection),
``block_linear`` for the projection.

    q[m, k] = e4m3(v[m, k] * (448 / amax)),  q_scale[m, b] = amax / 448     amax over the 128 columns of block b
    out[m, n] = sum_b a_scale[m, b] * w.scale[n // 128, b] * sum_{k in b} a[m, k] * w[n, k]  (+ bias[n])

The reference has no counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from ._common import E4M3, launch, ld, native, rows, same_device
from .activation import GELU_TANH, SILU

BLOCK = 128
FP8_MAX = 448.0
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def blocks_of(n: int) -> int:
    return -(-n // BLOCK)


@dataclass
class BlockWeight:
    w: torch.Tensor                   # [N, K] e4m3, K contiguous
    scale: torch.Tensor               # [ceil(N / 128), ceil(K / 128)] float32: amax of the block / 448
    bias: torch.Tensor | None = None  # [N] float32 or bfloat16

    @property
    def shape(self):
        return tuple(self.w.shape)


def quantize_weight_blocks(w: torch.Tensor, bias: torch.Tensor | None = None, device=None) -> BlockWeight:
    """Pack ``w`` [N, K] (any float dtype) with one scale per 128 x 128 block on ``device``.

    Load-time work, plain torch, the arithmetic of ``fp8.quantize_weight`` block by block:
    scale = max(amax, 1e-12) / 448, codes = e4m3_rn(clamp(w / scale)).
    """
    if w.ndim != 2:
        raise ValueError(f"weight must be [N, K], got shape {tuple(w.shape)}")
    N, K = w.shape
    target = device if device is not None else w.device
    padded = torch.zeros(blocks_of(N) * BLOCK, blocks_of(K) * BLOCK, device=target, dtype=torch.float32)
    padded[:N, :K] = w.to(device=target, dtype=torch.float32)
    tiles = padded.view(blocks_of(N), BLOCK, blocks_of(K), BLOCK)
    scale = tiles.abs().amax(dim=(1, 3)).clamp_min(1e-12) / FP8_MAX
    codes = (tiles / scale[:, None, :, None]).clamp_(-FP8_MAX, FP8_MAX).view_as(padded)[:N, :K].to(E4M3).contiguous()
    packed_bias = None if bias is None else bias.to(device=target, dtype=torch.float32).contiguous()
    return BlockWeight(codes, scale.contiguous(), packed_bias)


def block_scales(M: int, K: int, device) -> torch.Tensor:
    """A [M, ceil(K / 128)] tensor for activation scales, stored block by block: the layout ``block_linear`` reads
    fastest (neighbouring tokens' scales of one block side by side)."""
    return torch.empty(blocks_of(K), M, device=device, dtype=torch.float32).t()


def _scales(t, name, M, K, device, written):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != (M, blocks_of(K)):
        raise ValueError(f"{name} must be a float32 [{M}, {blocks_of(K)}] tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if written and not (t.stride(0) >= t.stride(1) * t.shape[1] and t.stride(1) >= 1
                        or t.stride(1) >= t.stride(0) * t.shape[0] and t.stride(0) >= 1):
        raise ValueError(f"{name} must not overlap itself")
    return t


def block_quant(x: torch.Tensor, q: torch.Tensor, q_scale: torch.Tensor, *, act: int | None = None) -> None:
    """``x`` [M, K] (float32, bfloat16 or float16) to ``q`` [M, K] e4m3 and ``q_scale`` [M, ceil(K / 128)] float32.

    With ``act`` (``GELU_TANH`` or ``SILU``) ``x`` is [M, 2K], ``[gate | up]``, and what is quantised is
    ``act(gate) * up`` in float32.  Any K, any row strides; ``q_scale`` in either order (see ``block_scales``).
    A block's maximum counts as at least 1e-8; an infinity or NaN makes its block's scale infinite or NaN."""
    if native.block_quant(x, q, q_scale, -1 if act is None else act):
        return
    if act not in (None, GELU_TANH, SILU):
        raise ValueError("act must be None, GELU_TANH (0) or SILU (1)")
    rows(x, "x", _FLOATS)
    rows(q, "q", (E4M3,))
    M, width = x.shape
    if act is not None and width % 2:
        raise ValueError("a [gate | up] input has an even width")
    K = width if act is None else width // 2
    if tuple(q.shape) != (M, K):
        raise ValueError(f"q must be [{M}, {K}], got {tuple(q.shape)}")
    if M > 1 and q.stride(0) < K:
        raise ValueError("q must not overlap itself")
    _scales(q_scale, "q_scale", M, K, x.device, True)
    same_device(x, q=q)
    launch("iflb200_block_quant", x, x.data_ptr(), _lib.dtype_code(x.dtype), ld(x), M, K, -1 if act is None else int(act),
           q.data_ptr(), ld(q), q_scale.data_ptr(), q_scale.stride(0), q_scale.stride(1))


def block_linear(a: torch.Tensor, a_scale: torch.Tensor, w: BlockWeight, out: torch.Tensor, *,
                 bias: torch.Tensor | None = None, use_weight_bias: bool = True) -> torch.Tensor:
    """out[M, N] (float32, bfloat16 or float16) = the block-scaled product of ``a`` [M, K] e4m3 and ``w``.

    K and N multiples of 16, rows 16-byte aligned.  All sums are float32 and the result is rounded once.
    ``a_scale`` [M, ceil(K / 128)] with any strides.  ``bias`` overrides ``w.bias`` (float32 or bfloat16).
    As for ``fp8.gemm``: with at most 2048 rows ``w.w`` must not be an output of the kernel enqueued directly before."""
    b = bias if bias is not None else (w.bias if use_weight_bias else None)
    if native.block_linear(a, a_scale, w.w, w.scale, b, out):
        return out
    rows(a, "a", (E4M3,))
    rows(w.w, "w.w", (E4M3,))
    M, K = a.shape
    N, Kw = w.w.shape
    if K != Kw:
        raise ValueError(f"a is [M, {K}] but the weight is [{N}, {Kw}]")
    if K % 16 or N % 16:
        raise ValueError("FP8 GEMM input/output dimensions must be multiples of 16")
    rows(out, "out", _FLOATS)
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out must be [{M}, {N}], got {tuple(out.shape)}")
    _scales(a_scale, "a_scale", M, K, a.device, False)
    if w.scale.dtype != torch.float32 or tuple(w.scale.shape) != (blocks_of(N), blocks_of(K)) or not w.scale.is_contiguous():
        raise ValueError(f"w.scale must be a contiguous float32 [{blocks_of(N)}, {blocks_of(K)}] tensor")
    if b is not None and (b.dtype not in (torch.float32, torch.bfloat16) or b.numel() != N or not b.is_contiguous()):
        raise ValueError("bias must be a contiguous float32 or bfloat16 vector of N elements")
    same_device(a, w=w.w, w_scale=w.scale, out=out, bias=b)
    launch("iflb200_block_linear", a, a.data_ptr(), ld(a), w.w.data_ptr(), ld(w.w), M, N, K, a_scale.data_ptr(),
           a_scale.stride(0), a_scale.stride(1), w.scale.data_ptr(), _lib.ptr(b),
           _lib.dtype_code(b.dtype) if b is not None else _lib.F32, out.data_ptr(), _lib.dtype_code(out.dtype), ld(out))
    return out
