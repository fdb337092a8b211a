"""64-bit oracles of the operators around the 4-bit cache: rotary positions,
the quantiser, the cache's rows and pages, and attention over them.  Test
infrastructure, never imported by the product.  Everything runs on CPU tensors
in float64; comparisons with the 16-bit outputs of the kernels are the tests'."""

from __future__ import annotations

import math
from fractions import Fraction

import torch

GROUP = 64


def rotary64(x, positions, inv_freq, sections, interleaved, inverse=False):
    """x [B, N, H, d] turned by positions [axes, B, N] * inv_freq [pairs]; float64."""
    x, pos, inv = x.double(), positions.double(), inv_freq.double()
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    angle = torch.stack([pos[a] * inv[j] for j, a in enumerate(axis)], -1)[:, :, None, :]
    c, s = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
    rot = 2 * len(axis)
    out = x.clone()
    a_idx = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b_idx = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    a, b = x[..., a_idx], x[..., b_idx]
    out[..., a_idx] = a * c - b * s
    out[..., b_idx] = b * c + a * s
    return out


def round_fraction(x: Fraction, dtype) -> float:
    """x rounded once to a 16-bit type, halves to even (no overflow)."""
    if x == 0:
        return 0.0
    bits, low = (11, -24) if dtype == torch.float16 else (8, -133)
    e = math.floor(math.log2(abs(float(x)))) if abs(x) > Fraction(1, 1 << 1000) else low
    while abs(x) >= Fraction(2) ** (e + 1):
        e += 1
    while abs(x) < Fraction(2) ** e:
        e -= 1
    step = Fraction(2) ** max(e - bits + 1, low)
    n = x / step
    f = n.numerator // n.denominator
    rest = n - f
    if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and f % 2):
        f += 1
    return float(f * step)


def quantise_exact(x, dtype):
    """(codes, s, m) of x [..., d] in exact arithmetic (python fractions; slow):
    codes int [..., d], s and m float64 [..., d / 64]."""
    flat = x.double().reshape(-1, GROUP)
    codes, steps, mins = [], [], []
    for row in flat.tolist():
        f = [Fraction(v) for v in row]
        low, high = min(f), max(f)
        s = Fraction(round_fraction((high - low) / 15, dtype))
        steps.append(float(s))
        mins.append(float(low))
        out = []
        for v in f:
            c = 0
            if s != 0:
                q = (v - low) / s
                c = q.numerator // q.denominator
                rest = q - c
                if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and c % 2):
                    c += 1
                c = min(c, 15)
            out.append(c)
        codes.append(out)
    shape = x.shape[:-1]
    groups = x.shape[-1] // GROUP
    return (torch.tensor(codes).reshape(*shape, -1), torch.tensor(steps, dtype=torch.float64).reshape(*shape, groups),
            torch.tensor(mins, dtype=torch.float64).reshape(*shape, groups))


def quantise64(x, dtype):
    """As quantise_exact, in float64 (exact for operands of similar size)."""
    g = x.double().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    s = ((high - low) / 15).to(dtype).double()
    q = (g - low[..., None]) / torch.where(s > 0, s, torch.ones_like(s))[..., None]
    codes = torch.where(s[..., None] > 0, q.round().clamp(0, 15), torch.zeros_like(q))
    return codes.flatten(-2).long(), s, low


def pack_rows(codes, s, m, dtype):
    """uint8 rows [..., d / 2 + d / 16]."""
    c = codes.to(torch.uint8)
    packed = c[..., 0::2] | (c[..., 1::2] << 4)
    params = torch.stack([s, m], -1).to(dtype).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([packed, params], -1)


def unpack_rows(rows, dtype):
    """(codes, s, m) of uint8 rows: int64 [..., d], float64 [..., d / 64] twice."""
    d = rows.shape[-1] * 16 // 9
    packed = rows[..., : d // 2]
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).long()
    params = rows[..., d // 2:].contiguous().view(dtype).double().unflatten(-1, (-1, 2))
    return codes, params[..., 0], params[..., 1]


def sequence_rows(cache, page_table, b, length):
    """Rows of one sequence, uint8 [2, length, heads, row]."""
    page = cache.shape[3]
    pages = page_table[b, : -(-length // page)].long()
    rows = cache[pages]  # [n, heads, 2, page, row]
    return rows.permute(2, 0, 3, 1, 4).flatten(1, 2)[:, :length]


def attention64(q, cache, page_table, kv_lens, causal=False, scale=None, new_lens=None):
    """O, lse and the terms of an error bound, in float64, for q [B, N, H, d].

    Returns (o, lse, weight, reach): weight [B, N, H, d] = sum_t p_t (s' c' + |m'|),
    reach [B, N, H] = the largest scale * sum |q| (s c + |m|) of a visible token."""
    B, N, H, d = q.shape
    hk = cache.shape[1]
    dtype = q.dtype
    scale = 1 / math.sqrt(d) if scale is None else scale
    o = torch.zeros(B, N, H, d, dtype=torch.float64)
    weight, reach = torch.zeros_like(o), torch.zeros(B, N, H, dtype=torch.float64)
    lse = torch.full((B, H, N), -math.inf, dtype=torch.float64)
    for b in range(B):
        length = int(kv_lens[b])
        fresh = N if new_lens is None else int(new_lens[b])
        rows = sequence_rows(cache, page_table, b, length)
        spread = []
        for r in rows:
            c, s, m = unpack_rows(r, dtype)
            part = c.double() * s.repeat_interleave(GROUP, -1)
            spread.append((part, m.repeat_interleave(GROUP, -1)))
        (kc, km), (vc, vm) = spread
        for n in range(fresh):
            see = min(length, max(0, length - fresh + n + 1)) if causal else length
            if see == 0:
                continue
            for h in range(H):
                j = h // (H // hk)
                x = q[b, n, h].double()
                score = (kc[:see, j] + km[:see, j]) @ x * scale
                top = score.max()
                p = torch.exp(score - top)
                lse[b, h, n] = top + torch.log(p.sum())
                p = p / p.sum()
                o[b, n, h] = p @ (vc[:see, j] + vm[:see, j])
                weight[b, n, h] = p @ (vc[:see, j] + vm[:see, j].abs())
                reach[b, n, h] = ((kc[:see, j] + km[:see, j].abs()) @ x.abs()).max() * scale
    return o, lse, weight, reach
