"""What the block-scaled operators decide on the host: packing, refusals before any launch, plain forms' own arithmetic."""
import ctypes
import math

import pytest
import torch

import block_ref as ref
from instinctflash_b200 import _lib
from instinctflash_b200.kernels import blocks, kv_cache

E4M3 = torch.float8_e4m3fn


def test_weight_packing_covers_ragged_edges():
    w = torch.randn(200, 300, generator=torch.Generator().manual_seed(0))
    w[130:, 260:] = 0.0
    w[0, 0] = 100.0
    packed = blocks.quantize_weight_blocks(w, torch.ones(200, dtype=torch.float64))
    assert packed.shape == (200, 300) and packed.scale.shape == (2, 3) and packed.bias.dtype == torch.float32
    for n in range(2):
        for k in range(3):
            tile = w[128 * n:128 * n + 128, 128 * k:128 * k + 128]
            scale = torch.clamp(tile.abs().max(), min=1e-12) / 448.0
            assert packed.scale[n, k] == scale
            want = (tile / scale).clamp(-448, 448).to(E4M3)
            assert torch.equal(packed.w[128 * n:128 * n + 128, 128 * k:128 * k + 128].view(torch.uint8), want.view(torch.uint8))
    with pytest.raises(ValueError):
        blocks.quantize_weight_blocks(w[0])


def test_scale_layout():
    s = blocks.block_scales(5, 300, "cpu")
    assert s.shape == (5, 3) and s.stride() == (1, 5)


def test_power_of_two_of_the_reference():
    for amax in (448.0, 448.0001, 224.0, 1.0, 3e38, 1e-9):
        s = ref.power_of_two(amax)
        assert max(amax, 1e-8) / s <= 448.0 * (1 + 2 ** -22) and max(amax, 1e-8) / s > 224.0 * (1 - 2 ** -22)
    assert ref.power_of_two(448.0) == 1.0 and ref.power_of_two(449.0) == 2.0 and ref.power_of_two(0.0) == 2.0 ** -35


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 256)
    q, s = torch.empty(4, 256, dtype=E4M3), torch.empty(4, 2)
    with pytest.raises(ValueError, match="CUDA"):
        blocks.block_quant(x, q, s)
    with pytest.raises(ValueError, match="CUDA"):
        blocks.block_linear(q, s, blocks.quantize_weight_blocks(torch.randn(32, 256)), torch.empty(4, 32))
    cache = kv_cache.KVCache8.empty(2, 1, 16, 64, "cpu")
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.cache_append(cache, torch.randn(1, 1, 1, 64), torch.randn(1, 1, 1, 64), one.view(1, 1), one)
    with pytest.raises(ValueError, match="CUDA"):
        q16 = torch.randn(1, 1, 1, 64).half()
        kv_cache.cache_attention(q16, cache, one.view(1, 1), one, q16.clone())


def test_entry_points_reject_bad_arguments_before_any_launch():
    lib = _lib.lib()
    p = ctypes.c_void_p(4096)  # never dereferenced
    F32, BF16 = 0, 1

    def quant(x=p, dt=BF16, ld=256, M=4, K=256, act=-1, q=p, ldq=256, qs=p, r=1, b=4):
        return lib.iflb200_block_quant(x, dt, ld, M, K, act, q, ldq, qs, r, b, None)
    assert quant(M=0) == 0 and quant(K=0) == 0
    assert quant(x=None) == -1 and quant(ld=255) == -1 and quant(act=0) == -1 and quant(act=2) == -1 and quant(ldq=200) == -1
    assert quant(dt=5) == -4 and quant(M=-1) == -1 and quant(r=-1) == -1

    def linear(a=p, lda=256, w=p, ldw=256, M=4, N=64, K=256, sa=p, r=1, b=4, sw=p, bias=None, bt=F32, out=p, dt=BF16, ldo=64):
        return lib.iflb200_block_linear(a, lda, w, ldw, M, N, K, sa, r, b, sw, bias, bt, out, dt, ldo, None)
    assert linear(M=0) == 0 and linear(N=0) == 0
    assert linear(K=0) == -2 and linear(K=24) == -2 and linear(N=40) == -2
    assert linear(a=ctypes.c_void_p(8)) == -3 and linear(lda=264) == -3 and linear(ldo=68) == -3
    assert linear(sa=None) == -1 and linear(sw=None) == -1 and linear(lda=128) == -1 and linear(ldo=32) == -1 and linear(b=-4) == -1
    assert linear(dt=7) == -4 and linear(bias=p, bt=2) == -4

    for ok in ((0, 0, 0), (1, 128, 8), (2, 128, 1), (2, 16, 0)):
        assert lib.iflb200_block_linear_set_form(*ok) == 0
    for bad in ((3, 0, 0), (1, 144, 0), (2, 24, 0), (2, 0, 2), (1, 0, 9), (-1, 0, 0)):
        assert lib.iflb200_block_linear_set_form(*bad) == -1
    assert lib.iflb200_block_linear_set_form(0, 0, 0) == 0

    def append(dt=BF16, B=1, T=1, H=1, D=64, k=p, pages=4, P=16, table=p, mp=2, start=p, codes=p):
        return lib.iflb200_cache_append(k, 64, 64, 64, p, 64, 64, 64, dt, B, T, H, D, codes, p, p, p, pages, P, table, mp, mp, start,
                                        None, None)
    assert append(B=0) == 0 and append(T=0) == 0 and append(pages=0) == 0 and append(mp=0) == 0
    assert append(D=96) == -2 and append(P=24) == -2 and append(P=512) == -2 and append(B=1 << 17) == -2
    assert append(dt=9) == -4 and append(k=None) == -1 and append(start=None) == -1 and append(codes=ctypes.c_void_p(4104)) == -3

    def attend(dt=BF16, B=1, T=1, HQ=2, H=1, D=64, q=p, pages=4, P=16, table=p, mp=2, lens=p, prefix=None, scale=1.0, cap=0.0, causal=1,
               ws=None, wb=0):
        return lib.iflb200_cache_attention(q, dt, 64, 64, 64, p, p, p, p, pages, P, D, table, mp, mp, lens, None, prefix, None, B, T, HQ,
                                           H, scale, cap, causal, p, 64, 64, 64, ws, wb, None)
    assert attend(B=0) == 0 and attend(T=0) == 0
    assert attend(HQ=3, H=2) == -2 and attend(D=80) == -2 and attend(P=8) == -2 and attend(mp=1 << 30) == -2
    assert attend(T=1 << 28) == -2 and attend(T=1 << 30, HQ=4) == -2 and attend(B=1 << 16) == -2
    assert attend(dt=F32) == -4 and attend(q=None) == -1 and attend(lens=None) == -1 and attend(table=None) == -1
    assert attend(prefix=p, causal=0) == -1 and attend(cap=-1.0) == -1 and attend(cap=math.nan) == -1 and attend(scale=math.nan) == -1
    assert attend(ws=ctypes.c_void_p(4104), wb=8192) == -3 and attend(wb=-1) == -1
    assert [lib.iflb200_cache_attention_set_form(f) for f in (0, 1, 2, 0, 3, -1)] == [0, 0, 0, 0, -1, -1]
