"""Attention over the 8-bit cache where weights, value scales, queries or positions cover a wide range: every key's share of the
result within the error that the kernels' arithmetic leaves it, not only the largest ones'."""
import math

import pytest
import torch

from instinctflash_b200 import _lib
from instinctflash_b200.kernels import kv_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
FORMS = (1, 2, 0)


def ints(*v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def cache_of(k, v, ks, vs, page, order=None):
    """A cache of one sequence from rows [keys, heads, D] and scales [pages, heads]; its pages lie in ``order``."""
    n, H, D = k.shape
    pages = n // page
    order = torch.arange(pages, device=DEV) if order is None else order
    cache = kv_cache.KVCache8.empty(pages, H, page, D, DEV)
    for codes, x in ((cache.k, k), (cache.v, v)):
        codes[order] = x.view(pages, page, H, D).transpose(1, 2).to(E4M3)
    cache.k_scale[order], cache.v_scale[order] = ks, vs
    return cache, order.to(torch.int32).view(1, pages)


def plain(q, cache, table, n, scale, flush, causal=True, slopes=None, first=0):
    """Result in 64 bits for one sequence of ``n`` keys (those ahead of ``first`` have no weight), and the error allowed: scores in
    fp32, weights as f16 (half a step, 2^-11 of each, or ``flush`` of the row's largest below f16's normal range), one rounding of the
    result."""
    T, HQ, D = q.shape[1:]
    H, P = cache.k.shape[1:3]
    j = torch.arange(first, n, device=DEV)
    page = table[0].long()[j // P]
    p = torch.arange(n - T, n, device=DEV)
    out, tol = torch.zeros(T, HQ, D, device=DEV, dtype=torch.float64), torch.zeros(T, HQ, D, device=DEV, dtype=torch.float64)
    for i in range(HQ):
        h = i * H // HQ
        key = cache.k[page, h, j % P].double() * cache.k_scale[page, h].double()[:, None]
        val = cache.v[page, h, j % P].double() * cache.v_scale[page, h].double()[:, None]
        x = q[0, :, i].double()
        s, mag = x @ key.t() * scale, x.abs() @ key.abs().t() * abs(scale)
        err = mag * (D + 8) * 2.0 ** -24
        if q.dtype == torch.bfloat16:   # q as f16, its largest element at 2^15 or above: half a step of f16's subnormals is 2^-25, so each
            err = err + 2.0 ** -40 * x.abs().amax(1, keepdim=True) * key.abs().sum(1) * abs(scale)   # element is off by 2^-40 of it at most
        if slopes is not None:
            bias = slopes[i].double() * (p[:, None] - j).abs()
            s, err = s - bias, err + bias * 2.0 ** -22
        err = err + s.abs() * 2.0 ** -22 + 2.0 ** -21     # to base 2, less the maximum, ex2
        if causal:
            s = s.masked_fill(j[None] > p[:, None], -math.inf)
        w = torch.softmax(s, 1)
        err = torch.where(w > 0, err, 0.0)
        o = w @ val
        share = torch.where(w > 0, w * (2.0 ** -11 + 2 * err) + flush * w.amax(1, keepdim=True), 0.0)
        f16 = 2.0 ** -25 if q.dtype == torch.float16 else 0.0          # half of its least step
        out[:, i] = o
        tol[:, i] = share @ val.abs() + (w * 2 * err).sum(1, keepdim=True) * o.abs() + torch.finfo(q.dtype).eps / 2 * o.abs() + f16
    return out, tol


def check(q, cache, table, n, scale, flush, workspaces=(0, 16 << 20), forms=FORMS, **kw):
    first = kw.pop("first", 0)
    want, tol = plain(q, cache, table, n, scale, flush, first=first, **kw)
    for nbytes in workspaces:
        for form in forms:
            out = torch.full_like(q, math.nan)
            assert _lib.lib().iflb200_cache_attention_set_form(form) == 0
            try:
                kv_cache.cache_attention(q, cache, table, ints(n), out, scale=scale,
                                         workspace=kv_cache.attention_workspace(DEV, nbytes) if nbytes else None, **kw)
            finally:
                _lib.lib().iflb200_cache_attention_set_form(0)
            got = out[0].double()
            assert torch.equal(got.isnan(), want.isnan()), f"form {form}, workspace {nbytes}: NaN in other places"
            off = ((got - want).abs() - tol).nan_to_num(-1.0)
            assert off.max() <= 0, f"form {form}, workspace {nbytes}: {float(off.max())} outside at {(off > 0).nonzero()[0].tolist()}"


def rows_of(D, T=1, heads=4, dtype=torch.bfloat16):
    """Queries that take columns 0 and 1 of the keys as they are: scores to base 2 with a scale of log 2."""
    q = torch.zeros(1, T, heads, D, device=DEV, dtype=dtype)
    q[..., :2] = 1.0
    return q


# A weight keeps f16's eleven bits down to 2^-24 of the row's largest (normal f16 with the largest at 2^10) and half a step of f16's
# subnormals, 2^-25 / 2^10, below; twice that where a step's weights move to a larger maximum after they were rounded.
FLUSH = 2.0 ** -34


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("place", [0, 2000, 4095])
@pytest.mark.parametrize("depth", [12.0, 18.0, 22.0, 24.0, 26.0, 28.0])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_long_tail_of_small_weights(D, depth, place, dtype):
    """One key with nearly all the weight and no value in the tail's columns, 4095 keys 2^-depth below it that alone have some."""
    n, g = 4096, torch.Generator(device=DEV).manual_seed(int(depth))
    k, v = torch.zeros(n, 1, D, device=DEV), torch.zeros(n, 1, D, device=DEV)
    k[:, 0, 1] = torch.randint(-11, 1, (n,), device=DEV, generator=g) / 16.0
    v[:, 0, 2:34] = torch.rand(n, 32, device=DEV, generator=g) * 300.0 + 100.0
    v[:, 0, 34:] = torch.randn(n, D - 34, device=DEV, generator=g) * 100.0
    k[place], v[place] = 0.0, 0.0
    k[place, 0, 0], v[place, 0, 1] = depth, 448.0
    lift = torch.full((n // 64, 1), 2.0 ** 6, device=DEV)
    cache, table = cache_of(k, v, torch.ones_like(lift), lift, 64)
    check(rows_of(D, dtype=dtype), cache, table, n, math.log(2.0), FLUSH)


# Value scales within 2^6 of one another share the running maximum (2^-35 of it is then 2^-29 of the row's largest probability, in units
# of the page's own values), others have one of their own; twice that as above.
FAR = 2.0 ** -28


def scaled_cache(D, page, scales, seed, heads=1, depth=0.0):
    """Pages with the given value scales (to base 2; None: zero), each with values in every sixteenth column only, so that a column has
    nothing but its own pages'.  The page with the largest scale has a key 2^depth above the rest."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = len(scales)
    n = pages * page
    k, v = torch.zeros(n, heads, D, device=DEV), torch.zeros(n, heads, D, device=DEV)
    k[:, :, 1] = torch.randint(-12, 1, (n, heads), device=DEV, generator=g) / 8.0
    for i in range(pages):
        own = torch.arange(i % 16, D, 16, device=DEV)
        v[i * page:(i + 1) * page, :, own] = torch.rand(page, heads, own.numel(), device=DEV, generator=g) * 400.0 + 40.0
    vs = torch.tensor([0.0 if s is None else 2.0 ** s for s in scales], device=DEV)[:, None].expand(pages, heads)
    k[int(vs[:, 0].argmax()) * page + 3, :, 0] = depth
    return cache_of(k, v, torch.ones(pages, heads, device=DEV), vs, page, torch.randperm(pages, device=DEV, generator=g)), n


@pytest.mark.parametrize("gap", [5, 8, 15, 20, 26, 40, 60, 96])
@pytest.mark.parametrize("large_first", [False, True])
@pytest.mark.parametrize("T,D,page", [(1, 64, 16), (1, 128, 64), (2, 256, 32), (90, 128, 16), (90, 256, 128), (90, 64, 256)])
def test_pages_with_value_scales_far_apart(T, D, page, large_first, gap):
    """A page with a large scale leaves the others their values, in the columns where it has none."""
    half = [-gap / 2] * (640 // page) + [gap / 2] * (640 // page)
    (cache, table), n = scaled_cache(D, page, half[::-1] if large_first else half, gap)
    check(rows_of(D, T), cache, table, n, math.log(2.0), FAR)
    (cache, table), n = scaled_cache(D, page, (half * 3)[::-1] if large_first else half * 3, gap, depth=16.0)
    check(rows_of(D, T), cache, table, n, math.log(2.0), FAR)


@pytest.mark.parametrize("T,D,page", [(1, 64, 16), (3, 128, 32), (1, 256, 16), (70, 128, 16), (70, 64, 48), (70, 256, 16)])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_value_scales_over_their_whole_range(T, D, page, order):
    scales = [-48 + 3 * i for i in range(33)] + [None] * 3
    if order == "falling":
        scales.reverse()
    if order == "mixed":
        scales = [scales[i * 11 % 36] if i % 2 else scales[-1 - i] for i in range(36)]
    (cache, table), n = scaled_cache(D, page, scales, 3, heads=2, depth=4.0)
    check(rows_of(D, T, 8), cache, table, n, math.log(2.0), FAR)
    check(rows_of(D, T, 8), cache, table, n - page // 2, math.log(2.0), FAR, slopes=torch.full((8,), 2.0 ** -9, device=DEV))


def test_value_scales_far_apart_in_f16():
    for T in (1, 80):
        (cache, table), n = scaled_cache(128, 16, [0, -9, 3, -8, 0, -6, -9, None] * 6, 5, depth=8.0)
        check(rows_of(128, T, dtype=torch.float16), cache, table, n, math.log(2.0), FAR)


@pytest.mark.parametrize("T,D", [(1, 64), (1, 128), (1, 256), (70, 128), (70, 256)])
@pytest.mark.parametrize("ratio", [10, 18, 24, 30])
def test_a_large_element_of_q_where_keys_have_none(T, D, ratio):
    """The other elements decide the scores: they keep their bits beside it."""
    g = torch.Generator(device=DEV).manual_seed(ratio)
    n = 640
    k, v = (torch.randn(n, 2, D, device=DEV, generator=g) * 60.0 for _ in range(2))
    k[..., 5] = 0.0
    for dtype in (torch.bfloat16, torch.float16):
        if dtype == torch.float16 and ratio > 24:
            continue
        low = 1.0 if dtype == torch.bfloat16 else 2.0 ** (14 - ratio)
        q = (torch.randn(1, T, 8, D, device=DEV, generator=g) * low).to(dtype)
        q[..., 5] = low * 2.0 ** ratio
        one = torch.ones(n // 16, 2, device=DEV)
        cache, table = cache_of(k, v, one / 60.0, one / 60.0, 16)
        check(q, cache, table, n, 3.0 * D ** -0.5 / low, FAR)


@pytest.mark.parametrize("T", [1, 3, 80])
def test_distances_of_far_positions(T):
    """Slopes count whole tokens beyond 2^24, where float32 has every second one only: a sequence of a few pages over and over."""
    n, D, page = (1 << 24) + 1003, 64, 256
    g = torch.Generator(device=DEV).manual_seed(T)
    k, v = (torch.randn(8 * page, 1, D, device=DEV, generator=g) * 60.0 for _ in range(2))
    one = torch.ones(8, 1, device=DEV)
    cache, _ = cache_of(k, v, one / 600.0, one / 60.0, page)
    table = (torch.arange(-(-n // page), device=DEV) % 8).to(torch.int32).view(1, -1)
    q = torch.randn(1, T, 2, D, device=DEV, generator=g).to(torch.bfloat16)
    slopes = torch.tensor([1.0, 0.25], device=DEV)
    # (4000 tokens back a key has less than e^-900)
    check(q, cache, table, n, 0.125, FAR, workspaces=(16 << 20,), forms=(1, 2), slopes=slopes, first=n - 4096)


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 256)])
def test_one_token_at_a_time_by_a_warp_repeats_itself(D, page):
    """Steps of one token, whose page's scale grows at every one: the codes of the page follow one old and one new scale."""
    sizes = torch.exp2(torch.arange(page, device=DEV) % 24 - 12.0)
    k = torch.randn(64, page, 2, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)) * sizes[:, None, None]
    table = torch.arange(64, device=DEV, dtype=torch.int32).view(64, 1)
    caches = [kv_cache.KVCache8.empty(64, 2, page, D, DEV) for _ in range(3)]
    for c in caches:
        for i in range(page):
            kv_cache.cache_append(c, k[:, i:i + 1], -k[:, i:i + 1], table, torch.full((64,), i, device=DEV, dtype=torch.int32))
        assert torch.equal(c.k_scale, c.v_scale) and torch.equal(c.k.view(torch.uint8) & 0x7F, c.v.view(torch.uint8) & 0x7F)
        assert torch.equal(c.k.view(torch.uint8), caches[0].k.view(torch.uint8))
    amax = k.abs().amax(dim=(1, 3))
    assert ((amax / caches[0].k_scale <= 448.0) & (amax / caches[0].k_scale > 224.0)).all()
    # every code within half a step of the largest scale's for each time that it moved: it moves exactly, or below the subnormals
    back = caches[0].k.float() * caches[0].k_scale[:, :, None, None]
    off = (back - k.transpose(1, 2)).abs()
    assert (off <= k.transpose(1, 2).abs() * 2.0 ** -4 + caches[0].k_scale[:, :, None, None] * 2.0 ** -10 * 2).all()


def test_scalars_that_are_no_normal_numbers_are_refused():
    one = torch.ones(1, 1, device=DEV)
    cache, table = cache_of(torch.ones(16, 1, 64, device=DEV), torch.ones(16, 1, 64, device=DEV), one, one, 16)
    q = rows_of(64)
    for kw in (dict(softcap=math.inf), dict(softcap=1e-39), dict(softcap=1e39), dict(softcap=-1e-39), dict(scale=math.inf), dict(scale=-1e39),
               dict(scale=math.nan)):
        with pytest.raises(ValueError):
            kv_cache.cache_attention(q, cache, table, ints(16), torch.empty_like(q), **kw)
    for cap in (1.2e-38, 3e38):   # the ends of what is taken: scores of about the cap, and scores as they are
        out = kv_cache.cache_attention(q, cache, table, ints(16), torch.empty_like(q), softcap=cap, scale=0.01)
        assert (out == 1.0).all()
