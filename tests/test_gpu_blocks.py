"""Block-scaled quantiser and linear against their definitions."""
import pytest
import torch

import block_ref as ref
from instinctflash_b200 import _lib
from instinctflash_b200.kernels import blocks
from instinctflash_b200.kernels.activation import GELU_TANH, SILU
from util import code_steps, i32, u8

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def activations(rows, width, dtype, seed=0):
    x = torch.randn(rows, width, device=DEV, generator=gen(seed))
    x[:, ::37] *= 20.0
    return x.to(dtype)


def run_quant(x, K, act=None, block_major=True):
    M = x.shape[0]
    q = torch.zeros(M, K, device=DEV, dtype=E4M3)
    s = blocks.block_scales(M, K, DEV) if block_major else torch.empty(M, blocks.blocks_of(K), device=DEV)
    blocks.block_quant(x, q, s, act=act)
    return q, s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 127), (3, 128), (2, 129), (50, 1024), (7, 300), (33, 2056), (301, 4096)])
def test_quant_is_the_stated_arithmetic(M, K, dtype):
    x = activations(M, K, dtype, M + K)
    q, s = run_quant(x, K, block_major=M % 2 == 0)
    qr, sr = ref.quant(x)
    assert torch.equal(i32(s), i32(sr))
    assert torch.equal(u8(q), u8(qr))


@pytest.mark.parametrize("act", [GELU_TANH, SILU])
@pytest.mark.parametrize("M,K,dtype", [(1, 16, torch.bfloat16), (5, 130, torch.float16), (50, 4096, torch.bfloat16), (9, 512, torch.float32)])
def test_gated_quant(M, K, dtype, act):
    x = activations(M, 2 * K, dtype, 3)
    q, s = run_quant(x, K, act)
    qr, sr = ref.quant(x, act)
    # the activation by ex2 (2 ulp), a division (2 ulp) and six roundings; gelu's 1 + tanh is a sum near 1
    assert ((s.cpu() - sr).abs() <= sr * 2.0 ** -20 + 1e-9).all()
    steps = code_steps(q, qr)
    assert steps.max() <= 1 and (steps != 0).float().mean() < 5e-3


def test_quant_of_strided_rows_and_unaligned_columns():
    base = activations(9, 700, torch.bfloat16)
    for x in (base[:, 4:516], base[::2, 1:258], base[3:4, 8:136]):
        q, s = run_quant(x, x.shape[1])
        qr, sr = ref.quant(x)
        assert torch.equal(u8(q), u8(qr)) and torch.equal(i32(s), i32(sr))
    wide = torch.zeros(9, 1024, device=DEV, dtype=E4M3)   # strided codes: what lies beside them stays
    s = blocks.block_scales(9, 384, DEV)
    blocks.block_quant(base[:, :384], wide[:, 128:512], s)
    assert torch.equal(u8(wide[:, 128:512]), u8(ref.quant(base[:, :384])[0]))
    assert not u8(wide[:, :128]).any() and not u8(wide[:, 512:]).any()


def test_what_is_not_finite_stays_in_its_block():
    x = activations(4, 512, torch.float32)
    x[0, 5], x[1, 130], x[2, 300] = float("nan"), float("inf"), 0.0
    x[3, 384:] = 0.0
    q, s = run_quant(x, 512)
    clean = x.clone()
    clean[0, :128] = 0.0
    clean[1, 128:256] = 0.0
    qr, sr = ref.quant(clean)
    assert s[0, 0].isnan() and s[1, 1].isinf()
    assert q.float()[0, :128].isnan().all() and q.float()[1, 130].isnan() and (q.float()[1, 131:256] == 0).all()
    keep = torch.ones(4, 4, dtype=torch.bool)
    keep[0, 0] = keep[1, 1] = False
    assert torch.equal(s.cpu()[keep], sr[keep])
    cols = keep.repeat_interleave(128, dim=1)
    assert torch.equal(u8(q)[cols], u8(qr)[cols])


# ------------------------------------------------------------------ linear

def operands(M, N, K, seed=0):
    g = gen(seed)
    a = (torch.randn(M, K, device=DEV, generator=g) * 100).clamp_(-448, 448).to(E4M3)
    w = (torch.randn(N, K, device=DEV, generator=g) * 100).clamp_(-448, 448).to(E4M3)
    sa = torch.rand(blocks.blocks_of(K), M, device=DEV, generator=g).t() * 0.1 + 1e-3
    sw = torch.rand(blocks.blocks_of(N), blocks.blocks_of(K), device=DEV, generator=g) * 0.01 + 1e-4
    return a, sa, blocks.BlockWeight(w, sw)


def check_linear(a, sa, w, out, bias=None):
    y, mag = ref.linear(a, sa, w.w, w.scale, bias)
    K = a.shape[1]
    # fp32 sums of K products, two scales a block and a bias, then one rounding to the output's type (and its
    # subnormals' step)
    tol = mag * (K + 2 * blocks.blocks_of(K) + 4) * 2.0 ** -24 + y.abs() * torch.finfo(out.dtype).eps / 2 + torch.finfo(out.dtype).tiny
    bad = (out.double() - y).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


SHAPES = [(1, 16, 16), (1, 128, 128), (2, 272, 144), (5, 144, 400), (17, 128, 8192), (50, 2560, 1024), (64, 1024, 4096),
          (128, 512, 256), (129, 272, 2096), (257, 144, 128), (333, 2576, 2096), (816, 1040, 640), (1030, 256, 2048)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(M, N, K, dtype):
    a, sa, w = operands(M, N, K, M)
    out = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    blocks.block_linear(a, sa, w, out)
    check_linear(a, sa, w, out)


@pytest.mark.parametrize("form,tokens,splits", [(1, 16, 1), (1, 48, 2), (1, 128, 1), (1, 64, 4), (1, 16, 8), (1, 112, 8), (2, 16, 1),
                                                (2, 80, 1), (2, 128, 1)])
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (33, 400, 1040), (150, 256, 1152), (270, 2320, 384)])
def test_every_form_of_the_linear(M, N, K, form, tokens, splits):
    a, sa, w = operands(M, N, K, 7)
    lib = _lib.lib()
    assert lib.iflb200_block_linear_set_form(form, tokens, splits) == 0
    try:
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
            blocks.block_linear(a, sa, w, out)
            check_linear(a, sa, w, out)
    finally:
        lib.iflb200_block_linear_set_form(0, 0, 0)


def test_linear_of_many_tiles():
    a, sa, w = operands(2304, 5120, 256, 1)     # more tiles than CTAs: the ring and the accumulators go round
    out = torch.empty(2304, 5120, device=DEV, dtype=torch.bfloat16)
    blocks.block_linear(a, sa, w, out)
    check_linear(a, sa, w, out)


@pytest.mark.parametrize("bias_type", [torch.float32, torch.bfloat16])
def test_linear_bias_strides_and_scale_orders(bias_type):
    M, N, K = 75, 304, 1168
    a, sa, w = operands(M, N, K, 2)
    bias = torch.randn(N, device=DEV, generator=gen(5)).to(bias_type) * 50
    wide_a = torch.zeros(M, K + 32, device=DEV, dtype=E4M3)
    wide_a[:, 16:K + 16] = a
    wide_w = torch.zeros(N, K + 48, device=DEV, dtype=E4M3)
    wide_w[:, 32:K + 32] = w.w
    room = torch.zeros(M + 2, N + 64, device=DEV, dtype=torch.float16)
    out = room[1:-1, 32:N + 32]
    blocks.block_linear(wide_a[:, 16:K + 16], sa.contiguous(), blocks.BlockWeight(wide_w[:, 32:K + 32], w.scale, bias), out)
    check_linear(a, sa, w, out, bias)
    assert not room[0].any() and not room[-1].any() and not room[:, :32].any() and not room[:, N + 32:].any()
    plain = torch.empty(M, N, device=DEV, dtype=torch.float16)
    blocks.block_linear(a, sa, blocks.BlockWeight(w.w, w.scale, bias), plain, use_weight_bias=False)
    check_linear(a, sa, w, plain)
    one = torch.full((1, 1), 0.25, device=DEV).expand(M, blocks.blocks_of(K))   # one scale for all: stride 0
    blocks.block_linear(a, one, w, plain)
    check_linear(a, one, w, plain)


def test_a_nan_code_stays_in_its_row():
    a, sa, w = operands(40, 256, 640, 3)
    clean = torch.empty(40, 256, device=DEV)
    blocks.block_linear(a, sa, w, clean)
    u8v = a.view(torch.uint8)
    u8v[11, 600] = 0x7F
    out = torch.empty(40, 256, device=DEV)
    blocks.block_linear(a, sa, w, out)
    assert out[11].isnan().all()
    keep = torch.arange(40, device=DEV) != 11
    assert torch.equal(out[keep], clean[keep])


def test_linear_repeats_itself_and_replays():
    a, sa, w = operands(50, 1024, 4096, 4)      # ranges of K shared in clusters
    out = torch.empty(50, 1024, device=DEV)
    blocks.block_linear(a, sa, w, out)
    first = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        blocks.block_linear(a, sa, w, out)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_weight_packing_and_a_gated_mlp():
    """quantise -> gate_up -> gated quantiser -> down, against 64 bits on the same codes."""
    M, hidden, ffn = 37, 512, 1024
    x = activations(M, hidden, torch.bfloat16, 8)
    gu = blocks.quantize_weight_blocks(torch.randn(2 * ffn, hidden, device=DEV, generator=gen(9)) * 0.05)
    down = blocks.quantize_weight_blocks(torch.randn(hidden, ffn, device=DEV, generator=gen(10)) * 0.05)
    back = gu.w.float() * gu.scale.repeat_interleave(128, 0).repeat_interleave(128, 1)
    assert back.isfinite().all() and gu.scale.shape == (16, 4)
    q, s = run_quant(x, hidden)
    raw = torch.empty(M, 2 * ffn, device=DEV, dtype=torch.bfloat16)
    blocks.block_linear(q, s, gu, raw)
    check_linear(q, s, gu, raw)
    h, hs = run_quant(raw, ffn, SILU)
    hr, hsr = ref.quant(raw, SILU)
    assert code_steps(h, hr).max() <= 1
    y = torch.empty(M, hidden, device=DEV, dtype=torch.bfloat16)
    blocks.block_linear(h, hs, down, y)
    check_linear(h, hs, down, y)


def test_empty_and_refused():
    a, sa, w = operands(4, 64, 256)
    out = torch.empty(4, 64, device=DEV, dtype=torch.bfloat16)
    blocks.block_linear(a[:0], sa[:0], w, out[:0])
    blocks.block_quant(out[:0], a[:0, :64], torch.empty(0, 1, device=DEV))
    for args in ((a, sa[:, :1], w, out), (a, sa.double(), w, out), (a[:, :240], sa, w, out), (a, sa, w, out[:, :48]),
                 (a.float(), sa, w, out), (a, sa, blocks.BlockWeight(w.w, w.scale.t().contiguous().t()[:, :1]), out),
                 (a.cpu(), sa, w, out)):
        with pytest.raises(ValueError):
            blocks.block_linear(*args)
    with pytest.raises(ValueError, match="multiples of 16"):
        blocks.block_linear(a[:, :24], sa[:, :1], blocks.BlockWeight(w.w[:, :24], w.scale[:, :1].contiguous()), out)
    with pytest.raises(RuntimeError, match="alignment"):
        odd = torch.empty(4 * 72 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(4, 72)[:, :64]
        blocks.block_linear(a, sa, w, odd)
    x = torch.randn(4, 256, device=DEV)
    q = torch.empty(4, 256, device=DEV, dtype=E4M3)
    for bad in (lambda: blocks.block_quant(x, q, torch.empty(4, 1, device=DEV)), lambda: blocks.block_quant(x, q[:, :128], torch.empty(4, 2, device=DEV)),
                lambda: blocks.block_quant(x, q[:, :128], torch.empty(4, 1, device=DEV), act=5),
                lambda: blocks.block_quant(x, q, torch.empty(1, 2, device=DEV).expand(4, 2)),
                lambda: blocks.block_quant(x.double(), q, torch.empty(4, 2, device=DEV)),
                lambda: blocks.block_quant(x[:, :255], q[:, :127], torch.empty(4, 1, device=DEV), act=SILU)):
        with pytest.raises(ValueError):
            bad()
