"""Sizes of the block-scaled operators and the 8-bit cache that take a kernel through all its rings, refills and ranges."""
import pytest
import torch

import block_ref as ref
import test_gpu_blocks as linear
import test_gpu_kv_cache as cached
from instinctflash_b200 import _lib
from instinctflash_b200.kernels import blocks, kv_cache
from instinctflash_b200.kernels.activation import GELU_TANH, SILU
from util import code_steps

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("act", [GELU_TANH, SILU])
@pytest.mark.parametrize("M,K,dtype", [(816, 16384, torch.bfloat16), (333, 5001, torch.float32), (2050, 1024, torch.float16)])
def test_gated_quantiser_of_many_rows(M, K, dtype, act):
    x = linear.activations(M, 2 * K, dtype, 4)
    q, s = linear.run_quant(x, K, act)
    qr, sr = ref.quant(x, act)
    # as for few rows: the activation by ex2 (2 ulp), a division (2 ulp) and six roundings; gelu's 1 + tanh is a sum near 1
    assert ((s.cpu() - sr).abs() <= sr * 2.0 ** -20 + 1e-9).all()
    steps = code_steps(q, qr)
    assert steps.max() <= 1 and (steps != 0).float().mean() < 5e-3


@pytest.mark.parametrize("form,tokens,splits", [(0, 0, 0), (1, 128, 1), (2, 128, 1), (2, 80, 1)])
def test_linear_of_many_tiles_and_many_steps(form, tokens, splits):
    a, sa, w = linear.operands(1500, 4880, 2832, 6)     # three to six tiles a CTA (or pair) of 23 K steps: three batches of scales
    out = torch.full((1500, 4880), float("nan"), device=DEV, dtype=torch.bfloat16)
    assert _lib.lib().iflb200_block_linear_set_form(form, tokens, splits) == 0
    try:
        blocks.block_linear(a, sa, w, out)
    finally:
        _lib.lib().iflb200_block_linear_set_form(0, 0, 0)
    linear.check_linear(a, sa, w, out)


@pytest.mark.parametrize("T,D,P", [(1, 64, 16), (2, 128, 48), (1, 256, 256)])
def test_long_sequences_that_are_not_shared(T, D, P):
    """More than sixteen tiles a warp: pages are looked up afresh on the way, some of them missing."""
    q, cache, table = cached.scene(2, T, 4, 2, D, P, 9000)
    table[0, 5::37], table[1, table.shape[1] // 2] = -1, 1 << 30
    lens = cached.ints(9000, 2049)
    cached.check_attention(q, cache, table, lens)
    cached.check_attention(q, cache, table, lens, causal=False, slopes=torch.full((4,), 2.0 ** -10, device=DEV))


@pytest.mark.parametrize("B,T,HQ,H,D", [(130, 1, 8, 8, 64), (65, 3, 34, 17, 128), (13, 100, 160, 80, 64)])
def test_more_sequences_and_heads_than_tickets(B, T, HQ, H, D):
    """Over 1024 (sequence, head, row tile) units with a workspace."""
    q, cache, table = cached.scene(B, T, HQ, H, D, 16, 112)
    lens = torch.randint(T, 112, (B,), device=DEV, generator=cached.gen(1), dtype=torch.int32)
    # (the reference is slow: of many rows all are there for one sequence only)
    q_lens = torch.full((B,), T, device=DEV, dtype=torch.int32) if T <= 3 else cached.ints(*([100] + [1] * (B - 1)))
    cached.check_attention(q, cache, table, lens, kv_cache.attention_workspace(DEV), q_lens=q_lens)


@pytest.mark.parametrize("T,D", [(1, 128), (1, 256), (40, 64)])
def test_tables_much_wider_than_the_sequences(T, D):
    q, cache, table = cached.scene(3, T, 8, 2, D, 32, 900)
    wide = torch.full((3, 4096), -1, device=DEV, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    lens = cached.ints(900, 128, 517)
    for nbytes in (1 << 20, 16 << 20):
        cached.check_attention(q, cache, wide, lens, kv_cache.attention_workspace(DEV, nbytes))
