"""Plain forms of the block-scaled operators in 64 bits (whole numbers and powers of two where a result is exact)."""
import math

import torch

E4M3 = torch.float8_e4m3fn
BLOCK = 128


def blocks_of(n):
    return -(-n // BLOCK)


def quant(x, act=None):
    """Codes and scales of ``block_quant`` on the CPU: the stated fp32 operations, IEEE division included."""
    v = x.cpu().float()
    if act is not None:
        g, u = v.double().chunk(2, dim=1)
        if act == 1:
            v = g * torch.sigmoid(g) * u
        else:
            v = torch.nn.functional.gelu(g, approximate="tanh") * u
        v = v.float()
    M, K = v.shape
    padded = torch.zeros(M, blocks_of(K) * BLOCK)
    padded[:, :K] = v
    tiles = padded.view(M, -1, BLOCK)
    amax = torch.maximum(tiles.abs().amax(dim=2), torch.tensor(1e-8))
    inv = torch.tensor(448.0) / amax
    codes = (tiles * inv[..., None]).clamp(-448, 448).view(M, -1)[:, :K].to(E4M3)
    return codes, amax / torch.tensor(448.0)


def linear(a, a_scale, w, w_scale, bias=None):
    """Result and the sum of the terms' magnitudes, which rounding errors are relative to."""
    M, K = a.shape
    N = w.shape[0]
    sa = a_scale.double().repeat_interleave(BLOCK, dim=1)[:, :K]
    sw = w_scale.double().repeat_interleave(BLOCK, dim=0)[:N].repeat_interleave(BLOCK, dim=1)[:, :K]
    ad, wd = a.double() * sa, w.double() * sw
    y, mag = ad @ wd.t(), ad.abs() @ wd.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag


def power_of_two(amax):
    """Least power of two that brings amax (a float) to 448 or below."""
    m, e = math.frexp(max(amax, float(torch.tensor(1e-8))) / 448.0)
    return 2.0 ** (e - 1 if m == 0.5 else e)


def append(codes, scale, values, table, start, counts=None):
    """New ``codes`` (float64 tensor of what they stand for as e4m3 values, NaN kept) and ``scale`` after the call."""
    codes, scale = codes.cpu().double(), scale.cpu().double()
    values = values.cpu().double()
    pages, H, P, D = codes.shape
    for b in range(values.shape[0]):
        n = values.shape[1] if counts is None else min(max(int(counts[b]), 0), values.shape[1])
        at, end = int(start[b]), int(start[b]) + n
        if at < 0:
            continue
        first = at
        while at < end:
            slot, step = at % P, min(P - at % P, end - at)
            page = int(table[b, at // P]) if at // P < table.shape[1] else -1
            if 0 <= page < pages:
                for h in range(H):
                    x = values[b, at - first:at - first + step, h]
                    fin = x[x.isfinite()].abs()
                    need = power_of_two(float(fin.max()) if fin.numel() else 0.0)
                    if slot:
                        old = float(scale[page, h])
                        need = max(need, old)
                        codes[page, h, :slot] = (codes[page, h, :slot] * (old / need)).float().to(E4M3).double()
                    scale[page, h] = need
                    y = torch.where(x.isfinite(), x, math.nan) / need
                    codes[page, h, slot:slot + step] = y.float().to(E4M3).double()
            at += step
    return codes, scale


def attend(q, k, v, ks, vs, table, lens, causal=True, prefix=None, cap=0.0, slopes=None, scale=None, q_lens=None, eps=0.0):
    """Output (NaN rows kept), rows that are written, and the error that the stated arithmetic may leave: weights as f16
    (half a step, 2^-11 of each; absolute 2^-25 below its normal range), fp32 scores, the output rounded with ``eps`` (f16: or by half of its least step)."""
    B, T, HQ, D = q.shape
    pages, H, P, _ = k.shape
    out, tol = torch.zeros(B, T, HQ, D, dtype=torch.float64), torch.zeros(B, T, HQ, D, dtype=torch.float64)
    written = torch.zeros(B, T, dtype=torch.bool)
    scale = D ** -0.5 if scale is None else scale
    q, k, v, ks, vs = (x.cpu().double() for x in (q, k, v, ks, vs))
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * P))
        nq = T if q_lens is None else min(max(int(q_lens[b]), 0), T)
        written[b, :nq] = True
        j = torch.arange(n)
        page = table[b].cpu().long()[j // P] if n else torch.zeros(0, dtype=torch.long)
        there = (page >= 0) & (page < pages)
        safe = page.clamp(0, max(pages - 1, 0))
        for t in range(nq):
            p = n - nq + t
            seen = there.clone()
            if causal:
                seen &= (j <= p) | (j < (int(prefix[b]) if prefix is not None else 0))
            if not seen.any():
                continue
            jj, pg = j[seen], safe[seen]
            for hq in range(HQ):
                h = hq * H // HQ
                key = k[pg, h, jj % P] * ks[pg, h][:, None]
                val = v[pg, h, jj % P] * vs[pg, h][:, None]
                x = q[b, t, hq]
                s = (key @ x) * scale
                mag = (key.abs() @ x.abs()) * abs(scale)
                err = mag * (D + 8) * 2.0 ** -24
                if cap:
                    s = cap * torch.tanh(s / cap)
                    err = err + cap * 2.0 ** -21
                if slopes is not None:
                    bias = float(slopes[hq]) * (p - jj).abs().double()
                    s, err = s - bias, err + bias * 2.0 ** -22
                err = err + s.abs() * 2.0 ** -22 + 2.0 ** -21   # to base 2, less the maximum, ex2
                w = torch.softmax(s, 0)
                o = w @ val
                share = w * (2.0 ** -11 + 2 * err) + 2.0 ** -19 * w.max()
                out[b, t, hq] = o
                tol[b, t, hq] = share @ val.abs() + (w * 2 * err).sum() * o.abs() + eps / 2 * o.abs() + 2.0 ** -25
    return out, written, tol
