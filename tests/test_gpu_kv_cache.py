"""The 8-bit paged cache and attention over it, against their definitions."""
import math

import pytest
import torch

import block_ref as ref
from instinctflash_b200 import _lib
from instinctflash_b200.kernels import blocks, kv_cache, rope
from util import u8

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def pool(pages, heads, page, D, seed=0, nan=False):
    g = gen(seed)
    cache = kv_cache.KVCache8.empty(pages, heads, page, D, DEV)
    for name in ("k", "v"):
        codes = (torch.randn(pages, heads, page, D, device=DEV, generator=g) * 100).clamp_(-448, 448).to(E4M3)
        getattr(cache, name).copy_(codes)
        scale = torch.exp2(torch.randint(-9, -5, (pages, heads), device=DEV, generator=g).float())
        getattr(cache, name + "_scale").copy_(scale)
    return cache


def table_of(B, per, pages, seed=0):
    return (torch.randperm(pages - 1, device=DEV, generator=gen(seed))[: B * per] + 1).to(torch.int32).reshape(B, per)


def ints(*v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


# ------------------------------------------------------------------ append

def check_append(cache, k, v, table, start, counts=None):
    want = [ref.append(c, s, x, table, start, counts) for c, s, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v))]
    kv_cache.cache_append(cache, k, v, table, start, counts=counts)
    for (codes, scale), c, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert torch.equal(s.cpu().double(), scale)
        got = c.cpu().double()
        assert torch.equal(got.isnan(), codes.isnan())
        assert torch.equal(got.nan_to_num(0.0), codes.nan_to_num(0.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,H,D,P,starts", [
    (1, 1, 1, 64, 16, (0,)), (3, 1, 2, 128, 64, (0, 63, 64)), (2, 5, 3, 256, 16, (14, 31)), (2, 70, 1, 64, 32, (1, 90)),
    (1, 300, 2, 128, 48, (7,)), (4, 33, 2, 64, 256, (0, 255, 240, 256))])
def test_append(B, T, H, D, P, starts, dtype):
    per = (max(starts) + T + P - 1) // P + 1
    pages = B * per + 2
    cache = pool(pages, H, P, D, T)
    g = gen(T + 1)
    k = (torch.randn(B, T, H, D, device=DEV, generator=g) * torch.tensor([1.0, 40.0, 1e-3, 9.0], device=DEV)[:B, None, None, None]).to(dtype)
    v = torch.randn(B, T, H, D, device=DEV, generator=g).to(dtype)
    table = table_of(B, per, pages)
    check_append(cache, k, v, table, ints(*starts))


def test_append_one_by_one_lets_scales_grow():
    cache = pool(3, 2, 16, 64)
    table = ints(2).view(1, 1)
    for i, size in enumerate((1e-3, 1.0, 0.5, 448.0, 449.0, 3.0, 1e4)):
        k = torch.full((1, 1, 2, 64), size, device=DEV, dtype=torch.float32)
        check_append(cache, k, -k, table, ints(i))
    # what was written first has moved to the scale of the largest, 2^5, without losing more than codes below 2^-6 lose
    assert cache.k_scale[2].tolist() == [32.0, 32.0]
    assert cache.k[2, 0, 1, 0].float() * 32.0 == 1.0 and cache.v[2, 1, 3, 5].float() * 32.0 == -448.0


def test_append_counts_padding_and_places_that_are_no_page():
    P, D, H = 16, 64, 2
    cache = pool(6, H, P, D, 3)
    T = 40
    k = torch.randn(5, T, H, D, device=DEV, generator=gen(1)).to(torch.bfloat16)
    table = ints(1, 2, -1, 99, 3, 0x7FFFFFFF, 4, -7, 5, 5, 5, 5, 0, 0, 0).view(5, 3)
    table[3] = ints(5, -1, -1)
    table[4] = ints(-1, -1, -1)
    # rows: into the missing third page; a page out of range first; past the table; no token; all pages missing
    check_append(cache, k, k + 1, table, ints(2, 3, 20, 6, 0), ints(T, T + 5, T, 0, T))
    check_append(cache, k[:1], k[:1], table[:1], ints(-4))
    check_append(cache, k[:, :0], k[:, :0], table, ints(0, 0, 0, 0, 0))


def test_append_of_what_is_not_finite_or_nothing():
    cache = pool(2, 1, 16, 64)
    k = torch.randn(1, 6, 1, 64, device=DEV, generator=gen(2))
    k[0, 0, 0, 3], k[0, 1, 0, 4], k[0, 2, 0, 5] = math.nan, math.inf, -math.inf
    v = torch.zeros_like(k)
    check_append(cache, k, v, ints(1).view(1, 1), ints(0))
    assert cache.k[1, 0].float()[:6].isnan().sum() == 3 and cache.v_scale[1, 0] == 2.0 ** -35
    huge = torch.full((1, 2, 1, 64), 3.0e38, device=DEV)
    check_append(cache, huge, huge, ints(1).view(1, 1), ints(6))


def test_append_of_strided_and_unaligned_rows():
    cache = pool(8, 2, 16, 64)
    base = torch.randn(2, 21, 5, 200, device=DEV, generator=gen(4)).to(torch.float16)
    table = table_of(2, 3, 8)
    check_append(cache, base[:, :, 1:3, 8:72], base[:, :, 2:4, 16:80], table, ints(3, 9))
    check_append(cache, base[:, 1::2, ::4, 3:67], base[:, 1::2, ::4, 70:134], table, ints(30, 5))


# ------------------------------------------------------------------ attention

def check_attention(q, cache, table, lens, workspace=None, out=None, **kw):
    """Every form of the operator against the reference; returns the result of the one that the rule takes."""
    out = torch.full_like(q, 7.5) if out is None else out
    before = out.clone()
    names = dict(softcap="cap")
    want, written, tol = ref.attend(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, lens, eps=torch.finfo(q.dtype).eps,
                                    **{names.get(n, n): x for n, x in kw.items()})
    want, tol = want[written], tol[written]
    for form in (1, 2, 0):
        out.copy_(before)
        assert _lib.lib().iflb200_cache_attention_set_form(form) == 0
        try:
            kv_cache.cache_attention(q, cache, table, lens, out, workspace=workspace, **kw)
        finally:
            _lib.lib().iflb200_cache_attention_set_form(0)
        got = out.cpu().double()
        assert torch.equal(got[~written], before.cpu().double()[~written]), f"form {form}: rows that are not there were written"
        got = got[written]
        assert torch.equal(got.isnan(), want.isnan()), f"form {form}: NaN in other places"
        off = ((got - want).abs() - tol).nan_to_num(-1.0)
        assert off.numel() == 0 or off.max() <= 0, f"form {form}: {float(off.max())} outside at {(off > 0).nonzero()[0].tolist()}"
    return out


def scene(B, T, HQ, H, D, P, capacity, dtype=torch.bfloat16, seed=0):
    per = -(-capacity // P)
    pages = B * per + 2
    cache = pool(pages, H, P, D, seed)
    q = torch.randn(B, T, HQ, D, device=DEV, generator=gen(seed + 1)).to(dtype)
    return q, cache, table_of(B, per, pages, seed + 2)


def spoil(cache, table, lens):
    """NaN codes and NaN scales wherever no token of a sequence is."""
    pages, H, P, D = cache.k.shape
    used = torch.zeros(pages, P, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        j = torch.arange(min(max(n, 0), table.shape[1] * P))
        used[table[b].cpu().long()[j // P], j % P] = True
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        raw = codes.view(torch.uint8)
        raw[~used.to(DEV)[:, None, :, None].expand_as(raw)] = 0x7F
        scale[~used.any(1).to(DEV)] = math.nan


GEOMETRY = [(1, 1, 1, 1, 64, 16, 40), (2, 1, 8, 1, 256, 64, 300), (3, 1, 8, 2, 128, 32, 500), (2, 3, 5, 1, 64, 16, 90), (2, 7, 4, 4, 128, 16, 64),
            (1, 2, 16, 1, 128, 48, 1000), (2, 20, 8, 2, 64, 128, 260), (1, 50, 8, 1, 256, 32, 300), (1, 70, 4, 2, 128, 64, 200)]


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,T,HQ,H,D,P,capacity", GEOMETRY)
def test_attention(B, T, HQ, H, D, P, capacity, causal, shared):
    dtype = torch.float16 if T % 2 else torch.bfloat16
    q, cache, table = scene(B, T, HQ, H, D, P, capacity, dtype)
    lens = torch.randint(T, capacity + 1, (B,), device=DEV, generator=gen(9), dtype=torch.int32)
    lens[0] = capacity - 1
    spoil(cache, table, lens)
    check_attention(q, cache, table, lens, kv_cache.attention_workspace(DEV) if shared else None, causal=causal)


@pytest.mark.parametrize("T,HQ,H,D", [(1, 8, 2, 128), (9, 4, 1, 64), (33, 8, 1, 256), (40, 8, 2, 128)])
def test_attention_cap_slopes_prefix_and_scale(T, HQ, H, D):
    q, cache, table = scene(2, T, HQ, H, D, 32, 150)
    lens = ints(150, T + 3)
    spoil(cache, table, lens)
    slopes = torch.exp2(-torch.arange(HQ, device=DEV).float())
    ws = kv_cache.attention_workspace(DEV)
    check_attention(q, cache, table, lens, ws, softcap=5.0)
    check_attention(q, cache, table, lens, ws, softcap=300.0, slopes=slopes)
    check_attention(q, cache, table, lens, ws, slopes=slopes, causal=False, scale=0.3)
    check_attention(q, cache, table, lens, ws, prefix=ints(140, 2), slopes=slopes)
    check_attention(q, cache, table, lens, ws, prefix=ints(-3, 10 ** 6), scale=-0.05)


@pytest.mark.parametrize("T,D", [(4, 64), (24, 128), (80, 64), (80, 256)])
def test_rows_that_are_not_there_and_rows_that_see_nothing(T, D):
    q, cache, table = scene(5, T, 4, 2, D, 16, 100)
    # no key at all; fewer keys than queries (the first see none); negative; more than the table holds; a padded row
    lens = ints(0, T - 2, -5, 1000, 60)
    spoil(cache, table, lens)
    out = check_attention(q, cache, table, lens, kv_cache.attention_workspace(DEV), q_lens=ints(T, T, T, 2, 0))
    assert (out[0] == 0).all() and (out[1, :2] == 0).all() and (out[4] == 7.5).all()
    check_attention(q, cache, table, lens, causal=False, q_lens=ints(1, -1, 0, 10 ** 6, T))


def test_pages_that_are_none_are_masked():
    q, cache, table = scene(2, 2, 4, 1, 64, 32, 300)
    lens = ints(300, 31)
    table[0, 3], table[0, 9], table[1, 0] = -1, 10 ** 9, cache.k.shape[0]
    out = check_attention(q, cache, table, lens, kv_cache.attention_workspace(DEV))
    assert (out[1] == 0).all()


@pytest.mark.parametrize("T,D", [(6, 64), (6, 256), (70, 128)])
def test_nan_reaches_the_rows_that_see_it_and_no_others(T, D):
    q, cache, table = scene(1, T, 4, 1, D, 16, 120)
    lens = ints(120)
    place = 120 - 3       # the last three queries see it
    page, slot = int(table[0, place // 16]), place % 16
    cache.v.view(torch.uint8)[page, 0, slot, 5] = 0xFF
    out = check_attention(q, cache, table, lens)
    assert out[0, -3:, :, 5].isnan().all() and out.isnan().sum() == 3 * 4
    cache.v.view(torch.uint8)[page, 0, slot, 5] = 0
    cache.k.view(torch.uint8)[page, 0, slot, 5] = 0x7F
    out = check_attention(q, cache, table, lens)
    assert out[0, -3:].isnan().all() and not out[0, :-3].isnan().any()
    cache.k.view(torch.uint8)[page, 0, slot, 5] = 0
    q[0, 1, 2, 7], q[0, 2, 1, 3] = math.nan, math.inf
    out = check_attention(q, cache, table, lens)
    assert out[0, 1, 2].isnan().all() and out.isnan().any(dim=3).sum() <= 2


@pytest.mark.parametrize("T", [1, 5, 90])
def test_scales_far_apart_and_large_scores(T):
    q, cache, table = scene(1, T, 8, 1, 128, 16, 400)
    lens = ints(400)
    used = table[0].long()
    cache.v_scale[used, 0] = torch.exp2(torch.linspace(-30, 20, used.numel(), device=DEV).round())
    check_attention(q, cache, table, lens, kv_cache.attention_workspace(DEV))
    cache.v_scale[used, 0] = torch.exp2(torch.linspace(20, -30, used.numel(), device=DEV).round())
    cache.v_scale[used[3], 0] = 0.0
    cache.v_scale[used[0], 0] = 0.0
    check_attention(q, cache, table, lens)
    # the last pages decide: their values come through whatever went before
    cache.k_scale[used, 0] = 2.0 ** -7
    cache.k_scale[used[-1], 0] = 8.0
    check_attention(q, cache, table, lens)
    check_attention(q * 3e4 if q.dtype == torch.bfloat16 else q, cache, table, lens, scale=1e-6)


@pytest.mark.parametrize("T,D", [(1, 128), (5, 64), (2, 256), (90, 128), (90, 256)])
def test_pages_with_a_value_scale_of_zero(T, D):
    """Their keys count, their values are zeros (a NaN stays one), and the others' small values keep their bits."""
    q, cache, table = scene(1, T, 4, 1, D, 16, 300)
    used = table[0].long()
    cache.v_scale[used, 0] = 2.0 ** -20
    cache.v_scale[used[0::3], 0] = 0.0
    check_attention(q, cache, table, ints(300), kv_cache.attention_workspace(DEV))
    u8(cache.v)[used[3], 0, 2, 7] = 0x7F
    u8(cache.v)[used[-1], 0, 9, 11] = 0xFF
    cache.v_scale[used[-1], 0] = 0.0
    check_attention(q, cache, table, ints(300))
    cache.v_scale[used, 0] = 0.0
    check_attention(q, cache, table, ints(299), kv_cache.attention_workspace(DEV))


@pytest.mark.parametrize("low", [0.0, 6.0, 12.0, 14.0, 16.0, 20.0])
@pytest.mark.parametrize("high", [16.0, 20.0, 26.0, 30.0, 60.0, 120.0])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_that_jump(D, low, high):
    """Weights 2^0 on the first keys, then 2^low, then 2^high, each with values in columns of its own."""
    q = torch.zeros(1, 2, 8, D, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    cache = kv_cache.KVCache8.empty(20, 1, 16, D, DEV)
    table = (torch.arange(16, device=DEV) + 2).to(torch.int32).view(1, 16)
    k, v = torch.zeros(256, D, device=DEV), torch.zeros(256, D, device=DEV)
    v[:128, 3] = 1.0
    for at, exponent in ((130, low), (140, low), (170, high), (200, high - 9.0), (250, high)):
        k[at, 0] = exponent
        v[at, at % 64] = 448.0
    for codes, x in ((cache.k, k), (cache.v, v)):
        codes[2:18, 0] = x.view(16, 16, D).to(E4M3)
    cache.k_scale.fill_(1.0)
    cache.v_scale.fill_(1.0)
    check_attention(q, cache, table, ints(256), scale=math.log(2.0), causal=False)


def test_wide_range_of_q_and_its_strides():
    q, cache, table = scene(2, 3, 8, 2, 128, 16, 100)
    lens = ints(100, 64)
    big = torch.zeros(2, 5, 9, 264, device=DEV, dtype=torch.bfloat16)
    big[:, 1:4, 1:, 8:136] = q * torch.exp2(torch.arange(128, device=DEV) % 11 - 8.0)
    out = torch.full((2, 3, 8, 300), 7.5, device=DEV, dtype=torch.bfloat16)
    check_attention(big[:, 1:4, 1:, 8:136], cache, table, lens, out=out[..., 100:228])
    assert (out[..., :100] == 7.5).all() and (out[..., 228:] == 7.5).all()
    check_attention(big[:, 1:4, 1:, 7:135], cache, table, lens, out=out[..., 101:229])
    tq = torch.empty(8, 128, 2, 3, device=DEV, dtype=torch.bfloat16).permute(2, 3, 0, 1)
    assert tq.stride(3) != 1
    with pytest.raises(ValueError):
        kv_cache.cache_attention(tq, cache, table, lens, q.clone())


def test_one_workspace_for_calls_of_every_geometry():
    ws = kv_cache.attention_workspace(DEV, 3 << 20)
    for seed, (B, T, HQ, H, D, P, cap) in enumerate([(1, 1, 8, 1, 128, 64, 4000), (5, 1, 8, 2, 64, 16, 700), (1, 3, 4, 4, 256, 32, 900)] * 2):
        q, cache, table = scene(B, T, HQ, H, D, P, cap, seed=seed)
        lens = torch.randint(T, cap + 1, (B,), device=DEV, generator=gen(seed), dtype=torch.int32)
        check_attention(q, cache, table, lens, ws)
    assert not ws[:4096].any()


@pytest.mark.parametrize("nbytes", [0, 16, 4096, 4100, 20000, 70000])
def test_any_size_of_workspace(nbytes):
    q, cache, table = scene(2, 1, 8, 2, 128, 16, 900)
    room = torch.full((nbytes + 4096,), 0, device=DEV, dtype=torch.uint8)
    room[nbytes:] = 0xAB
    check_attention(q, cache, table, ints(900, 500), room[:nbytes])
    assert (room[nbytes:] == 0xAB).all()


def test_offsets_beyond_32_bits():
    pages, P, D = 70000, 256, 256      # 4.6 GB of codes each
    cache = kv_cache.KVCache8(*(torch.zeros(pages, 1, P, D, device=DEV, dtype=E4M3) for _ in range(2)),
                              *(torch.ones(pages, 1, device=DEV) for _ in range(2)))
    k = torch.randn(1, 600, 1, D, device=DEV, generator=gen(1)).to(torch.bfloat16)
    v = torch.randn(1, 600, 1, D, device=DEV, generator=gen(2)).to(torch.bfloat16)
    table = ints(pages - 1, pages - 3, pages - 2).view(1, 3)
    kv_cache.cache_append(cache, k, v, table, ints(0))
    small = kv_cache.KVCache8(cache.k[-3:], cache.v[-3:], cache.k_scale[-3:], cache.v_scale[-3:])
    want = [ref.append(torch.zeros(3, 1, P, D), torch.ones(3, 1), x, ints(2, 0, 1).view(1, 3), ints(0)) for x in (k, v)]
    assert torch.equal(small.k.cpu().double(), want[0][0]) and torch.equal(small.v_scale.cpu().double(), want[1][1])
    for T in (1, 40):
        q = torch.randn(1, T, 2, D, device=DEV, generator=gen(3)).to(torch.bfloat16)
        a, b = torch.empty_like(q), torch.empty_like(q)
        kv_cache.cache_attention(q, cache, table, ints(600), a)
        kv_cache.cache_attention(q, small, ints(2, 0, 1).view(1, 3), ints(600), b)
        assert torch.equal(a, b)
    assert not cache.k[:-3].view(torch.uint8).any()


@pytest.mark.parametrize("T", [1, 80])
def test_empty_tables_caches_and_sequences(T):
    q, cache, table = scene(2, T, 8, 2, 64, 16, 100)
    ws = kv_cache.attention_workspace(DEV)
    for c, t, lens in ((cache, table[:, :0], ints(50, 0)), (cache, table, ints(0, -3)),
                       (kv_cache.KVCache8.empty(0, 2, 16, 64, DEV), table, ints(100, 7))):
        for form in (1, 2, 0):
            _lib.lib().iflb200_cache_attention_set_form(form)
            out = torch.full_like(q, 7.5)
            try:
                kv_cache.cache_attention(q, c, t, lens, out, workspace=ws, causal=False)
            finally:
                _lib.lib().iflb200_cache_attention_set_form(0)
            assert (out == 0).all()
    k = torch.randn(2, T, 2, 64, device=DEV)
    kv_cache.cache_append(kv_cache.KVCache8.empty(0, 2, 16, 64, DEV), k, k, table, ints(0, 0))
    kv_cache.cache_append(cache, k, k, table[:, :0], ints(0, 0))


@pytest.mark.parametrize("T,D", [(1, 128), (7, 256), (60, 128)])
def test_output_over_q_and_the_same_bits_every_time(T, D):
    q, cache, table = scene(3, T, 8, 2, D, 16, 1200)
    lens, ws = ints(1200, 64, 700), kv_cache.attention_workspace(DEV)
    first = kv_cache.cache_attention(q, cache, table, lens, torch.empty_like(q), workspace=ws)
    for _ in range(5):
        x = q.clone()
        kv_cache.cache_attention(x, cache, table, lens, x, workspace=ws)
        assert torch.equal(x, first)


def test_two_streams_at_once_with_a_workspace_each():
    scenes = [scene(1, t, 8, 2, 128, 16, 1500, seed=t) for t in (1, 40)]
    lens = ints(1500)
    ws = [kv_cache.attention_workspace(DEV) for _ in scenes]
    want = [kv_cache.cache_attention(q, c, t, lens, torch.empty_like(q), workspace=w) for (q, c, t), w in zip(scenes, ws)]
    outs = [torch.empty_like(q) for q, _, _ in scenes]
    streams = [torch.cuda.Stream() for _ in scenes]
    torch.cuda.synchronize()
    for _ in range(10):
        for (q, c, t), w, o, s in zip(scenes, ws, outs, streams):
            with torch.cuda.stream(s):
                kv_cache.cache_attention(q, c, t, lens, o, workspace=w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_without_the_call_extension(monkeypatch):
    """The same through ctypes."""
    q, cache, table = scene(2, 3, 8, 2, 128, 16, 300)
    twin = kv_cache.KVCache8(*(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    k = torch.randn(2, 3, 2, 128, device=DEV, generator=gen(1))
    kw = dict(softcap=20.0, slopes=torch.rand(8, device=DEV), prefix=ints(5, 0), q_lens=ints(3, 2), workspace=kv_cache.attention_workspace(DEV))
    outs = []
    for c in (cache, twin):
        kv_cache.cache_append(c, k, k, table, ints(90, 17), counts=ints(3, 1))
        outs.append(kv_cache.cache_attention(q, c, table, ints(93, 18), torch.zeros_like(q), **kw))
        for name in ("cache_append", "cache_attention"):
            monkeypatch.setattr(kv_cache.native, name, lambda *a: False)
    assert torch.equal(outs[0], outs[1]) and torch.equal(u8(cache.k), u8(twin.k)) and torch.equal(cache.v_scale, twin.v_scale)


def test_captured_steps_follow_lengths_and_share_a_workspace():
    """A decode step (append, attend) captured once and replayed as the sequences grow; a second graph with the same
    workspace in between."""
    B, HQ, H, D, P = 3, 8, 2, 128, 16
    q, cache, table = scene(B, 1, HQ, H, D, P, 200)
    other = kv_cache.KVCache8(cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone())
    ws = kv_cache.attention_workspace(DEV)
    k, v = (torch.randn(B, 1, H, D, device=DEV, generator=gen(i)).to(torch.bfloat16) for i in (5, 6))
    start, lens = ints(20, 100, 190), ints(21, 101, 191)
    outs = [torch.empty_like(q) for _ in range(2)]

    def step(c, o):
        kv_cache.cache_append(c, k, v, table, start)
        kv_cache.cache_attention(q, c, table, lens, o, workspace=ws)

    graphs = []
    for c, o in zip((cache, other), outs):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(c, o)
        graphs.append(graph)
    for i in range(4):
        k.normal_(generator=gen(10 + i))
        v.normal_(generator=gen(20 + i))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want, _, tol = ref.attend(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, lens, eps=2.0 ** -7)
        assert ((outs[0].cpu().double() - want).abs() <= tol).all()
        assert torch.equal(outs[0], outs[1])
        start += 1
        lens += 1


def test_on_a_stream_of_its_own():
    q, cache, table = scene(1, 1, 8, 1, 128, 64, 3000)
    lens = ints(3000)
    ws = kv_cache.attention_workspace(DEV)
    want = torch.empty_like(q)
    kv_cache.cache_attention(q, cache, table, lens, want, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(64 << 20, device=DEV)
        cache.k.copy_(cache.k.clone())
        big.sin_()
        out = torch.empty_like(q)
        kv_cache.cache_attention(q, cache, table, lens, out, workspace=ws)
    side.synchronize()
    assert torch.equal(out, want)


def test_a_layer_from_projection_to_projection():
    """Fused QKV projection, split with rotary, cache, attention, output projection: each step against 64 bits on what
    the step before it left."""
    B, T, HQ, H, D, hidden, P = 2, 9, 4, 2, 64, 256, 16
    g = gen(0)
    x = torch.randn(B * T, hidden, device=DEV, generator=g).to(torch.bfloat16)
    width = (HQ + 2 * H) * D
    wqkv = blocks.quantize_weight_blocks(torch.randn(width, hidden, device=DEV, generator=g) * 0.06)
    wo = blocks.quantize_weight_blocks(torch.randn(hidden, HQ * D, device=DEV, generator=g) * 0.06)
    q8, s8 = torch.empty(B * T, hidden, device=DEV, dtype=E4M3), blocks.block_scales(B * T, hidden, DEV)
    blocks.block_quant(x, q8, s8)
    raw = torch.empty(B * T, width, device=DEV, dtype=torch.bfloat16)
    blocks.block_linear(q8, s8, wqkv, raw)
    want, mag = ref.linear(q8, s8, wqkv.w, wqkv.scale)
    assert ((raw.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * 300 * 2.0 ** -24).all()
    q, k, v = (torch.empty(B * T, n, D, device=DEV, dtype=torch.bfloat16) for n in (HQ, H, H))
    pos = torch.arange(T, device=DEV).float().repeat(B)[:, None].contiguous()
    rope.qkv_split(raw, q, k, v, heads_q=HQ, heads_kv=H, head_dim=D, inv_freq=rope.rope_inv_freq(D, 10000.0, DEV), pos=pos)
    cache = pool(7, H, P, D)
    table = table_of(B, 3, 7)
    start = ints(0, 20)
    check_append(cache, k.view(B, T, H, D), v.view(B, T, H, D), table, start)
    out = torch.empty(B, T, HQ, D, device=DEV, dtype=torch.bfloat16)
    check_attention(q.view(B, T, HQ, D), cache, table, start + T, kv_cache.attention_workspace(DEV), out=out, prefix=ints(4, 0))
    o8, os8 = torch.empty(B * T, HQ * D, device=DEV, dtype=E4M3), blocks.block_scales(B * T, HQ * D, DEV)
    blocks.block_quant(out.view(B * T, HQ * D), o8, os8)
    y = torch.empty(B * T, hidden, device=DEV, dtype=torch.bfloat16)
    blocks.block_linear(o8, os8, wo, y)
    want, mag = ref.linear(o8, os8, wo.w, wo.scale)
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * 300 * 2.0 ** -24).all()


def test_refusals():
    q, cache, table = scene(2, 1, 4, 2, 64, 16, 64)
    lens, out = ints(3, 4), torch.empty_like(q)
    att = lambda **kw: kv_cache.cache_attention(**{**dict(q=q, cache=cache, table=table, lens=lens, out=out), **kw})  # noqa: E731
    for kw in (dict(q=q.float()), dict(out=out.half()), dict(lens=lens.long()), dict(lens=lens[:1]), dict(table=table[:1]),
               dict(table=table.long()), dict(q=q[:, :, :3], out=out[:, :, :3]), dict(q=q[..., :32], out=out[..., :32]),
               dict(prefix=lens, causal=False), dict(prefix=lens.float()), dict(softcap=-1.0), dict(softcap=math.nan),
               dict(slopes=torch.ones(3, device=DEV)), dict(slopes=torch.ones(4, device=DEV).half()), dict(q_lens=lens[:1]),
               dict(workspace=torch.zeros(4096, device=DEV)), dict(workspace=torch.zeros(4112, device=DEV, dtype=torch.uint8)[1:]),
               dict(lens=lens.cpu()), dict(q=q.cpu())):
        with pytest.raises(ValueError):
            att(**kw)
    odd = kv_cache.KVCache8.empty(4, 2, 16, 64, DEV)
    for name, bad in (("k", odd.k.float()), ("v", odd.v[:3]), ("k_scale", odd.k_scale.half()), ("v_scale", odd.v_scale[:, :1])):
        broken = kv_cache.KVCache8(**{**odd.__dict__, name: bad})
        with pytest.raises(ValueError):
            att(cache=broken)
        with pytest.raises(ValueError):
            kv_cache.cache_append(broken, q[:, :, :2], q[:, :, :2], table, lens)
    for shape in ((4, 2, 24, 64), (4, 2, 16, 96), (4, 2, 512, 64)):
        with pytest.raises(ValueError):
            att(cache=kv_cache.KVCache8.empty(*shape, DEV))
    new = torch.randn(2, 3, 2, 64, device=DEV)
    for args in ((new, new.half(), table, lens), (new, new[:, :2], table, lens), (new[:, :, :1], new[:, :, :1], table, lens),
                 (new, new, table[:1], lens), (new, new, table, lens.long()), (new.double(), new.double(), table, lens)):
        with pytest.raises(ValueError):
            kv_cache.cache_append(cache, *args)
    assert kv_cache.cache_attention(q[:, :0], cache, table, lens, out[:, :0]).shape[1] == 0
