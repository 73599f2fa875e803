"""Plain 64-bit forms of a drafted step's operators, and their error bounds."""

from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24                                   # half a step of fp32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half the least subnormal


def rounded(x: torch.Tensor, err: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """How far a result may be off that is off by ``err`` before its one rounding."""
    return err + (x.abs() + err) * HALF[dtype] + TINY[dtype]


def norm_rope(x: torch.Tensor, weight: torch.Tensor | None, eps: float | None,
              pos: torch.Tensor, freq: torch.Tensor, sections: list[int] | None, layout: str
              ) -> tuple[torch.Tensor, torch.Tensor]:
    """(result, error bound before its rounding) of x (B, H, S, D), 64 bits on the CPU.

    A normed value: D / 16 + 5 roundings of a sum of squares that count half in
    its root, the root's own two, two products: (D / 32 + 8) u of |y|.  The
    angle's fraction of a turn is rounded to fp32 at 1/2 turn at most: pi u,
    and 2^-24 turns, 2 pi u, of the product of far positions; sine and cosine
    2 u each: 14 u.  The rotation adds two products and a sum: 3 u."""
    B, H, S, D = x.shape
    y = x.double()
    if eps is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    n = freq.shape[0]
    p = pos if sections is not None else pos[None]
    axis = [a for a, c in enumerate(sections or [n]) for _ in range(c)]
    ang = torch.stack([p[a].double() * f for a, f in zip(axis, freq.double())], -1)  # (B, S, n)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    i = torch.arange(n)
    lo, hi = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    out, mag = y.clone(), y.abs()
    out[..., lo] = y[..., lo] * c - y[..., hi] * s
    out[..., hi] = y[..., hi] * c + y[..., lo] * s
    both = mag[..., lo] + mag[..., hi]
    mag[..., lo], mag[..., hi] = both, both
    return out, (D / 32 + 8 + 14 + 3) * U32 * mag


def verify(tokens: list[list[int]], target: torch.Tensor, draft: torch.Tensor | None,
           u: torch.Tensor, lens: list[int]) -> tuple[list[list[int]], list[int]]:
    """Tokens and accepted counts by the definition, a sequence at a time, 64 bits."""
    outs, counts = [], []
    N, V = u.shape[1] - 1, target.shape[2]
    for b, n in enumerate(lens):
        n = max(0, min(n, N))
        m = 0
        while m < n:
            t = tokens[b][m]
            if not 0 <= t < V:
                break
            q = 1.0 if draft is None else float(draft[b, m, t])
            if not float(u[b, m]) * q < float(target[b, m, t]):
                break
            m += 1
        p = torch.nan_to_num(target[b, m].double(), nan=0.0).clamp(min=0)
        w = p
        if m < n:
            w = target[b, m].double()
            if draft is not None:
                w = w - draft[b, m].double()
            elif 0 <= tokens[b][m] < V:
                w = w.clone()
                w[tokens[b][m]] -= 1.0
            w = torch.nan_to_num(w, nan=0.0).clamp(min=0)
            w = w if float(w.sum()) > 0 else p
        total = w.cumsum(0)
        past = (total > float(u[b, N]) * float(total[-1])).nonzero()
        some = (w > 0).nonzero()
        drawn = int(past[0]) if len(past) else int(some[-1]) if len(some) else -1
        outs.append(tokens[b][:m] + [drawn] + [-1] * (N - m))
        counts.append(m)
    return outs, counts


def window_attention(q: torch.Tensor, rows: list[tuple[torch.Tensor, torch.Tensor]],
                     lens: list[int], qlens: list[int], window: int | None, sinks: int,
                     scale: float, weight_half: float) -> tuple[torch.Tensor, ...]:
    """(out, lse, their error bounds) of q (B, H, S, D) over each sequence's
    K and V rows, (Hkv, n, D) in 64 bits; query i at lens - qlens + i.

    A score: D products' sum, its scale's and its row's rounding, D u S with
    S = scale sum |q||k|; its exponential's argument rounded twice at its size
    and the base's: 8 u |s|, with 2 u of its own and 2 u for each of up to n
    rescales: all of it twice, in the weight and in their sum.  A weight enters
    the product with v rounded to ``weight_half`` at most, and n products' sum
    and the division add (n + 4) u."""
    B, H, S, D = q.shape
    out = torch.zeros((B, H, S, D), dtype=torch.float64)
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64)
    eo, el = torch.zeros_like(out), torch.zeros((B, H, S), dtype=torch.float64)
    for b, (n, m) in enumerate(zip(lens, qlens)):
        k, v = rows[b]
        G = H // k.shape[0]
        j = torch.arange(k.shape[1])
        for i in range(m):
            p = n - m + i
            seen = j <= p
            if window is not None:
                seen &= (p - j < window) | (j < sinks)
            ks, vs = k[:, seen].repeat_interleave(G, 0), v[:, seen].repeat_interleave(G, 0)
            if ks.shape[1] == 0:
                continue
            qi = q[b, :, i].double().unsqueeze(1)
            s = (qi * ks).sum(-1) * scale                                   # (H, keys)
            size = (qi.abs() * ks.abs()).sum(-1) * abs(scale)
            z = torch.logsumexp(s, -1)
            w = torch.exp(s - z.unsqueeze(-1))
            w = torch.where(torch.isneginf(z).unsqueeze(-1), 0.0, w)
            keys = ks.shape[1]
            ds = ((D + 2) * U32 * size + 8 * U32 * s.abs()).amax(-1)
            out[b, :, i] = (w.unsqueeze(-1) * vs).sum(1)
            lse[b, :, i] = z
            rel = 2 * (ds + (2 + 2 * min(keys, 64)) * U32) + weight_half + (keys + 4) * U32
            eo[b, :, i] = rel.unsqueeze(-1) * (w.unsqueeze(-1) * vs.abs()).sum(1)
            el[b, :, i] = ds + (2 * min(keys, 64) + keys + 4) * U32 + 4 * U32 * z.abs()
    return out, lse, eo, el
