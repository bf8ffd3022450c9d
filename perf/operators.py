"""The block-scaled 8-bit operators as their users call them, for timing and for comparison.

``quant``    activations to e4m3 with a scale for each row and 128 columns, plain or behind a gated activation
``linear``   product of such activations with a weight that has a scale for each 128 x 128 block
``append``   new keys and values written into an 8-bit paged cache with a scale for each page and head
``attend``   attention of one or many query tokens a sequence over that cache

With ``own`` false ``run`` computes the operators in elementary torch operations in 32 bits; with ``own`` true it
calls the package.  Page 0 of every cache is the null page: no table entry in use names it.
"""
import math

import torch

own = False

DEV = "cuda"
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 128


def listed():
    return [
        # input of an action-expert projection, one episode's 50 tokens: all latency
        dict(name="quant_expert", op="quant", M=50, K=1024, dtype="bf16", gated=False),
        # [gate | up] of the vision-language prefix's feed-forward, on the way to its down projection
        dict(name="quant_gated_prefix", op="quant", M=816, K=16384, dtype="bf16", gated=True),
        # fused QKV projection of the expert: the smallest product
        dict(name="linear_expert", op="linear", M=50, N=2560, K=1024, out="bf16", bias=False),
        # an odd number of vision-language tokens, a depth that ends inside a block, biased
        dict(name="linear_ragged", op="linear", M=333, N=2576, K=2096, out="f16", bias=True),
        # gate_up of the prefix: three images and 48 text tokens
        dict(name="linear_prefix", op="linear", M=816, N=32768, K=2048, out="bf16", bias=False),
        # first feed-forward projection of a video diffusion block, all tokens of a request: the largest
        dict(name="linear_video", op="linear", M=4680, N=14336, K=5120, out="bf16", bias=True),
        # one new token for each of 32 sequences, some pages' scales grow
        dict(name="append_step", op="append", B=32, T=1, heads=8, D=128, page=64, context=4000, dtype="bf16"),
        # prompts of up to 2048 tokens for eight sequences, from wherever their last page ends
        dict(name="append_prompts", op="append", B=8, T=2048, heads=8, D=128, page=64, context=100, dtype="f16"),
        # one token behind the prefix at the expert's heads: the smallest attention
        dict(name="attend_token", op="attend", B=1, T=1, heads_q=8, heads=1, D=256, page=64, context=866, dtype="bf16",
             causal=True, prefix=False, cap=0.0, slopes=False),
        # a serving step of 32 sequences of ragged lengths up to 8192, grouped heads
        dict(name="attend_step", op="attend", B=32, T=1, heads_q=32, heads=8, D=128, page=64, context=8192, dtype="bf16",
             causal=True, prefix=False, cap=50.0, slopes=False),
        # the action tokens of eight episodes over prefix and themselves, every one seeing all
        dict(name="attend_expert", op="attend", B=8, T=50, heads_q=8, heads=1, D=256, page=32, context=866, dtype="f16",
             causal=False, prefix=False, cap=0.0, slopes=False),
        # a chunk of a long prompt behind what the cache has, its first tokens a prefix that sees itself both ways
        dict(name="attend_chunk", op="attend", B=1, T=2048, heads_q=32, heads=8, D=128, page=64, context=8192, dtype="bf16",
             causal=True, prefix=True, cap=0.0, slopes=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("quant", "linear", "linear", "append", "attend", "attend", "attend"))
    if op == "quant":
        gated = rng.random() < 0.5
        return dict(op=op, M=_log_int(rng, 1, 4096), K=16 * _log_int(rng, 1, 500) if gated else _log_int(rng, 16, 8192),
                    dtype=rng.choice(("bf16", "f16", "f32")), gated=gated)
    if op == "linear":
        while True:
            c = dict(op=op, M=_log_int(rng, 1, 4600), N=16 * _log_int(rng, 1, 1024), K=16 * _log_int(rng, 4, 512),
                     out=rng.choice(("bf16", "f16", "f32")), bias=rng.random() < 0.5)
            if c["M"] * c["N"] * c["K"] > 1 << 18:
                return c
    heads, D, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 256)), rng.choice((16, 32, 64, 128))
    if op == "append":
        T = _log_int(rng, 1, 2048)
        return dict(op=op, B=_log_int(rng, 1, max(1, min(64, 12000 // T))), T=T, heads=heads, D=D, page=page,
                    context=_log_int(rng, 1, 4096), dtype=rng.choice(("bf16", "f16", "f32")))
    T = rng.choice((1, 1, _log_int(rng, 2, 1500)))
    group = rng.choice((1, 2, 4, 5, 8, 16))
    while heads * group > 32:
        group //= 2
    causal = rng.random() < 0.7
    while True:
        B, context = _log_int(rng, 1, 48), _log_int(rng, 16, 32768)
        if T <= context and B * context * heads * D <= 1 << 27 and B * T * heads * group * context <= 1 << 28:
            return dict(op=op, B=B, T=T, heads_q=heads * group, heads=heads, D=D, page=page, context=context,
                        dtype=rng.choice(("bf16", "bf16", "f16")), causal=causal, prefix=causal and rng.random() < 0.4,
                        cap=rng.choice((0.0, 0.0, 30.0)), slopes=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs

def _activations(gen, rows, width, dtype):
    x = torch.randn(rows, width, device=DEV, generator=gen)
    x[:, torch.randperm(width, device=DEV, generator=gen)[: max(1, width // 100)]] *= 20.0
    return x.to(dtype)


def _codes(gen, *shape):
    """Codes of values whose block has its maximum near the end of the range, as a quantiser leaves them."""
    return (torch.randn(*shape, device=DEV, generator=gen) * 100.0).clamp_(-448.0, 448.0).to(E4M3)


def _uniform(gen, lo, hi, *shape):
    return torch.rand(*shape, device=DEV, generator=gen) * (hi - lo) + lo


def _blocks(n):
    return -(-n // BLOCK)


def _paged(gen, case, room):
    """A pool with a few pages more than the sequences use, its pages in random order, and the table."""
    B, H, D, P = case["B"], case["heads"], case["D"], case["page"]
    per = -(-room // P)
    pages = 1 + B * per + 3
    table = (torch.randperm(pages - 1, device=DEV, generator=gen)[: B * per] + 1).to(torch.int32).reshape(B, per)
    return dict(table=table, k=_codes(gen, pages, H, P, D), v=_codes(gen, pages, H, P, D)), pages


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(op=case["op"])
    if case["op"] == "quant":
        M, K = case["M"], case["K"]
        s |= dict(x=_activations(gen, M, K * (2 if case["gated"] else 1), TYPES[case["dtype"]]), act=1 if case["gated"] else None,
                  q=torch.empty(M, K, device=DEV, dtype=E4M3), scale=torch.empty(_blocks(K), M, device=DEV).t())
    elif case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s |= dict(a=_codes(gen, M, K), a_scale=_uniform(gen, 0.005, 0.02, _blocks(K), M).t(), w=_codes(gen, N, K),
                  w_scale=_uniform(gen, 1e-4, 4e-4, _blocks(N), _blocks(K)),
                  bias=torch.randn(N, device=DEV, generator=gen) if case["bias"] else None,
                  out=torch.empty(M, N, device=DEV, dtype=TYPES[case["out"]]))
    elif case["op"] == "append":
        B, T, H, D = (case[n] for n in ("B", "T", "heads", "D"))
        pool, pages = _paged(gen, case, case["context"] + T)
        # powers of two, as this operator leaves them; some are below what the new tokens need
        exponent = torch.randint(-8, -5, (2, pages, H), device=DEV, generator=gen)
        start = torch.randint(0, case["context"] + 1, (B,), device=DEV, generator=gen, dtype=torch.int32)
        s |= pool | dict(k_scale=torch.exp2(exponent[0].float()), v_scale=torch.exp2(exponent[1].float()), start=start,
                         new_k=_activations(gen, B * T * H, D, TYPES[case["dtype"]]).reshape(B, T, H, D),
                         new_v=torch.randn(B, T, H, D, device=DEV, generator=gen).to(TYPES[case["dtype"]]))
    else:
        B, T, D, HQ = case["B"], case["T"], case["D"], case["heads_q"]
        pool, pages = _paged(gen, case, case["context"])
        low = max(T, case["context"] // 4)   # lengths of a batch differ; one sequence has the longest
        lens = torch.randint(low, case["context"] + 1, (B,), device=DEV, generator=gen, dtype=torch.int32)
        lens[0] = case["context"]
        dtype = TYPES[case["dtype"]]
        s |= pool | dict(k_scale=_uniform(gen, 0.0075, 0.0125, pages, case["heads"]),
                         v_scale=_uniform(gen, 0.0075, 0.0125, pages, case["heads"]), lens=lens,
                         q=torch.randn(B, T, HQ, D, device=DEV, generator=gen).to(dtype),
                         out=torch.zeros(B, T, HQ, D, device=DEV, dtype=dtype), causal=case["causal"], cap=case["cap"],
                         prefix=(lens - T + T // 4).to(torch.int32) if case["prefix"] else None,
                         slopes=torch.exp2(-8.0 * torch.arange(1, HQ + 1, device=DEV) / HQ) * 0.25 if case["slopes"] else None,
                         workspace=torch.zeros(48 << 20, device=DEV, dtype=torch.uint8))
    return s


# ------------------------------------------------------------------ plain forms, 32 bits

def _plain_quant(s):
    v = s["x"].float()
    if s["act"] is not None:
        g, u = v.chunk(2, dim=1)
        v = g / (1.0 + torch.exp(-g)) * u
    M, K = v.shape
    padded = torch.zeros(M, _blocks(K) * BLOCK, device=DEV)
    padded[:, :K] = v
    padded = padded.reshape(M, -1, BLOCK)
    amax = padded.abs().amax(dim=2).clamp_min(1e-8)
    q = (padded * (448.0 / amax)[:, :, None]).clamp(-448.0, 448.0).reshape(M, -1)[:, :K].to(E4M3)
    return q, amax / 448.0


def _plain_linear(s):
    K = s["a"].shape[1]
    N = s["w"].shape[0]
    a = s["a"].float() * s["a_scale"].repeat_interleave(BLOCK, dim=1)[:, :K]
    w = s["w"].float() * s["w_scale"].repeat_interleave(BLOCK, dim=0)[:N].repeat_interleave(BLOCK, dim=1)[:, :K]
    y = a @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["out"].dtype)


def _power_of_two(amax):
    """Least power of two that brings ``amax`` to 448 or below."""
    m, e = torch.frexp(amax.clamp_min(1e-8))
    return torch.ldexp(torch.ones_like(m), torch.where(m <= 0.875, e - 9, e - 8))


def _plain_append(s):
    B, T, H, D = s["new_k"].shape
    P = s["k"].shape[2]
    spans = (T + P - 2) // P + 1
    start = s["start"].long()
    first = start // P
    place = (first[:, None] + torch.arange(spans, device=DEV))[:, :, None] * P + torch.arange(P, device=DEV)   # [B, spans, P]
    t = place - start[:, None, None]
    new = (t >= 0) & (t < T)
    touched = new.any(dim=2)
    index = (first[:, None] + torch.arange(spans, device=DEV)).clamp_max(s["table"].shape[1] - 1)
    page = torch.where(touched, s["table"].long().gather(1, index), 0)                                          # 0: the null page
    began = place[:, :, 0] < start[:, None]

    def one(codes, scale, values):
        rows = torch.arange(B, device=DEV)[:, None, None]
        x = values[rows, t.clamp(0, T - 1)].float().permute(0, 1, 3, 2, 4)                                      # [B, spans, H, P, D]
        fresh = new[:, :, None, :, None]
        need = _power_of_two(torch.where(fresh, x.abs(), 0.0).amax(dim=(3, 4)))
        old = torch.where(began[:, :, None], scale[page], 0.0)
        now = torch.maximum(old, need)
        kept = codes[page].float()
        before = (t < 0)[:, :, None, :, None]
        kept = torch.where(before, kept * (old / now)[..., None, None], kept)
        full = torch.where(fresh, x / now[..., None, None], kept).to(E4M3)
        codes.view(torch.uint8)[page] = full.view(torch.uint8)
        scale[page] = now

    one(s["k"], s["k_scale"], s["new_k"])
    one(s["v"], s["v_scale"], s["new_v"])


def _plain_attend(s):
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    B, T, HQ, D = q.shape
    H, P = s["k"].shape[1:3]
    S, G = table.shape[1] * P, HQ // H

    def gathered(codes, scale):
        return (codes[table].float() * scale[table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(B, H, S, D)

    x = q.float().reshape(B, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * T, D)
    score = ((x @ gathered(s["k"], s["k_scale"]).transpose(2, 3)) / math.sqrt(D)).reshape(B, H, G, T, S)
    if s["cap"]:
        score = s["cap"] * torch.tanh(score / s["cap"])
    j = torch.arange(S, device=DEV)
    place = (lens[:, None] - T + torch.arange(T, device=DEV))[:, :, None]     # [B, T, 1]
    if s["slopes"] is not None:
        score = score - s["slopes"].reshape(1, H, G, 1, 1) * (place - j).abs().float()[:, None, None]
    seen = (j < lens[:, None, None]).expand(B, T, S)
    if s["causal"]:
        near = j <= place
        if s["prefix"] is not None:
            near = near | (j < s["prefix"].long()[:, None, None])
        seen = seen & near
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(dim=-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(score - top)
    p = (p / p.sum(dim=-1, keepdim=True).clamp_min(1e-37)).reshape(B, H, G * T, S)
    o = (p @ gathered(s["v"], s["v_scale"])).reshape(B, H, G, T, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, HQ, D).to(q.dtype)


# ------------------------------------------------------------------ one pass

def _own(s):
    if s["op"] in ("quant", "linear"):
        from instinctflash_b200.kernels import blocks
        if s["op"] == "quant":
            blocks.block_quant(s["x"], s["q"], s["scale"], act=s["act"])
            return s["q"], s["scale"]
        if "weight" not in s:
            s["weight"] = blocks.BlockWeight(s["w"], s["w_scale"], s["bias"])
        return blocks.block_linear(s["a"], s["a_scale"], s["weight"], s["out"])
    from instinctflash_b200.kernels import kv_cache
    if "cache" not in s:
        s["cache"] = kv_cache.KVCache8(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "append":
        kv_cache.cache_append(s["cache"], s["new_k"], s["new_v"], s["table"], s["start"])
        return None
    return kv_cache.cache_attention(s["q"], s["cache"], s["table"], s["lens"], s["out"], causal=s["causal"], prefix=s["prefix"],
                                    softcap=s["cap"], slopes=s["slopes"], workspace=s["workspace"])


def run(state):
    if own:
        out = _own(state)
    else:
        out = {"quant": _plain_quant, "linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[state["op"]](state)
    if state["op"] == "append":   # all pages but the null page
        return state["k"][1:], state["v"][1:], state["k_scale"][1:], state["v_scale"][1:]
    return out


def work(case):
    if case["op"] == "quant":
        M, K = case["M"], case["K"]
        n = M * K * (2 if case["gated"] else 1)
        return {"bytes": n * SIZE[case["dtype"]] + M * K + 4 * M * _blocks(K), "flops": 4 * n}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K + N * K + 4 * _blocks(K) * (M + _blocks(N)) + SIZE[case["out"]] * M * N + (4 * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    if case["op"] == "append":
        n = 2 * case["B"] * case["T"] * case["heads"] * case["D"]
        return {"bytes": n * (SIZE[case["dtype"]] + 1) + 8 * case["B"] * case["heads"] * (1 + case["T"] // case["page"]), "flops": 3 * n}
    # lengths lie between a quarter of the context and all of it, the first sequence's at the end
    B, T, S = case["B"], case["T"], case["context"]
    low = max(T, S // 4)
    keys = S + (B - 1) * (low + S) / 2
    seen = T * keys - (B * T * (T - 1) / 2 if case["causal"] else 0)
    return {"bytes": 2 * keys * case["heads"] * case["D"] + 2 * 2 * B * T * case["heads_q"] * case["D"]
            + 8 * case["heads"] * keys / case["page"], "flops": 4 * seen * case["heads_q"] * case["D"]}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        x = s["x"].double()
        K = case["K"]
        if case["gated"]:
            x = x[:, :K] * torch.sigmoid(x[:, :K]) * x[:, K:]
        q, scale = [], []
        for at in range(0, K, BLOCK):
            piece = x[:, at:at + BLOCK]
            scale.append(piece.abs().max(dim=1).values.clamp_min(1e-8) / 448.0)
            q.append(piece / scale[-1][:, None])
        return torch.cat(q, 1), torch.stack(scale, 1)
    if op == "linear":
        y = torch.zeros(case["M"], case["N"], device=DEV, dtype=torch.float64)
        rows = torch.arange(case["N"], device=DEV) // BLOCK
        for b, at in enumerate(range(0, case["K"], BLOCK)):
            part = s["a"][:, at:at + BLOCK].double() @ s["w"][:, at:at + BLOCK].double().t()
            y += part * s["a_scale"][:, b].double()[:, None] * s["w_scale"][rows, b].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "append":
        B, T, P = case["B"], case["T"], case["page"]
        if B * (T / P + 1) > 6000:
            return None
        start, table = s["start"].tolist(), s["table"].tolist()
        outs = []
        for codes, scale, values in ((s["k"], s["k_scale"], s["new_k"]), (s["v"], s["v_scale"], s["new_v"])):
            codes, scale = codes.double(), scale.double()
            for b in range(B):
                at = start[b]
                while at < start[b] + T:
                    n = min(P - at % P, start[b] + T - at)
                    x = values[b, at - start[b]:at - start[b] + n].double().transpose(0, 1)          # [H, n, D]
                    page, slot = table[b][at // P], at % P
                    m, e = torch.frexp(x.abs().amax(dim=(1, 2)).clamp_min(1e-8) / 448.0)   # m in [1/2, 1)
                    need = torch.exp2((e - (m == 0.5).int()).double())
                    if slot:
                        need = torch.maximum(need, scale[page])
                        codes[page, :, :slot] *= (scale[page] / need)[:, None, None]
                    scale[page] = need
                    codes[page, :, slot:slot + n] = x / need[:, None, None]
                    at += n
            outs.append((codes[1:], scale[1:]))
        return outs[0][0], outs[1][0], outs[0][1], outs[1][1]
    B, T, HQ, D, H, P = (case[n] for n in ("B", "T", "heads_q", "D", "heads", "page"))
    out = torch.zeros(B, T, HQ, D, device=DEV, dtype=torch.float64)
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, : -(-n // P)].long()
        keys = s["k"][pages].double() * s["k_scale"][pages].double()[:, :, None, None]
        vals = s["v"][pages].double() * s["v_scale"][pages].double()[:, :, None, None]
        j = torch.arange(n, device=DEV)
        at = n - T + torch.arange(T, device=DEV)
        hidden = torch.zeros(T, n, device=DEV, dtype=torch.bool)
        if case["causal"]:
            hidden = j[None, :] > at[:, None]
            if case["prefix"]:
                hidden &= j[None, :] >= int(s["prefix"][b])
        for h in range(HQ):
            kh = keys[:, h * H // HQ].reshape(-1, D)[:n]
            z = s["q"][b, :, h].double() @ kh.t() * D ** -0.5
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if case["slopes"]:
                z -= s["slopes"][h].double() * (at[:, None] - j[None, :]).abs()
            z.masked_fill_(hidden, -math.inf)
            out[b, :, h] = torch.softmax(z, dim=1) @ vals[:, h * H // HQ].reshape(-1, D)[:n]
    return out
