"""Plain 64-bit forms of the paged-cache operators, and their error bounds."""

from __future__ import annotations

import torch

CACHE_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


class Cache:
    """A paged cache on the CPU with random rows, its block table and lengths.

    ``lens`` are the sequences' lengths; pages are dealt in a random order, -1
    behind each sequence's last one, and every row that no sequence owns
    holds NaN (as do the rows behind a sequence's end in its last page)."""

    def __init__(self, lens: list[int], Hkv: int, D: int, page: int, kind: str, seed: int = 0,
                 room: int = 0, spare: int = 2, std: float = 1.0) -> None:
        g = torch.Generator().manual_seed(seed)
        self.lens, self.Hkv, self.D, self.page, self.kind = lens, Hkv, D, page, kind
        need = [-(-(n + room) // page) for n in lens]
        self.P = sum(need) + spare
        order = torch.randperm(self.P, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.P, Hkv, page, D)
        dt = CACHE_DTYPES[kind]
        self.ks = self.vs = None
        if kind == "e4m3":
            self.k, self.v = ((torch.randn(shape, generator=g) * 120).clamp(-448, 448).to(dt)
                              for _ in range(2))
            self.ks, self.vs = (torch.rand(shape[:3], generator=g) * 0.01 * std + 0.001
                                for _ in range(2))
        else:
            self.k, self.v = ((torch.randn(shape, generator=g) * std).to(dt) for _ in range(2))
        owned = torch.zeros((self.P, page), dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(n):
                owned[self.table[b, j // page], j % page] = True
        hole = ~owned.view(self.P, 1, page).expand(self.P, Hkv, page)
        for x in (self.k, self.v):
            raw = x.view(torch.uint8) if kind == "e4m3" else x
            raw[hole] = 0x7F if kind == "e4m3" else float("nan")
        if self.ks is not None:
            self.ks[hole] = self.vs[hole] = float("nan")

    def rows(self, x: torch.Tensor, scale: torch.Tensor | None, b: int, n: int) -> torch.Tensor:
        """The first n rows of sequence b of a cache tensor, (Hkv, n, D) in 64 bits."""
        j = torch.arange(n)
        pg = self.table[b, j // self.page].long()
        out = x.double()[pg, :, j % self.page]
        if scale is not None:
            out = out * scale.double()[pg, :, j % self.page].unsqueeze(-1)
        return out.transpose(0, 1)

    def to(self, dev: torch.device, layout: str = "hnd") -> dict:
        """The cache on the GPU: "hnd" (pages, Hkv, page, D) contiguous, "nhd" a
        view of (pages, page, Hkv, D), "both" slices of (pages, 2, Hkv, page, D)."""
        if layout == "nhd":
            k, v = (x.permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3)
                    for x in (self.k, self.v))
        elif layout == "both":
            raw = [x.view(torch.uint8) if self.kind == "e4m3" else x for x in (self.k, self.v)]
            kv = torch.stack(raw, dim=1).to(dev).view(self.k.dtype)
            k, v = kv[:, 0], kv[:, 1]
        else:
            k, v = self.k.to(dev), self.v.to(dev)
        f32 = (lambda s: None if s is None else s.to(dev))
        return {"k_cache": k, "v_cache": v, "block_table": self.table.to(dev),
                "k_scale": f32(self.ks), "v_scale": f32(self.vs)}


def decode(q: torch.Tensor, c: Cache, lens: list[int], scale: float
           ) -> tuple[torch.Tensor, torch.Tensor, list[torch.Tensor], torch.Tensor, torch.Tensor]:
    """(out (B, H, D), lse (B, H), weights per sequence (H, n), error bounds of
    the fp32 kernels: of out before its rounding (B, H, D), of lse (B, H)).

    The bounds count roundings of u = 2^-24.  A score is a sum of D exact
    products: D u sum|q k| scale, two more for the scale and the row's, and
    its exponential's argument is rounded twice at the score's size: ds =
    (D + 4) u S + 4 u |s|, S = scale sum|q||k|.  A weight is off by ds, the
    exponential's own 2 u and its share of the running maximum's rescales (n
    of them at most, 2 u each); so is the sum.  Before the product with v a
    weight has 16 bits or more: 2^-16.  So out is off by 2 (ds + 2 n u + 2^-16)
    sum p|v|, and a sum of n products adds n u of it."""
    B, H, D = q.shape
    u = 2.0 ** -24
    out, lse = torch.zeros(B, H, D, dtype=torch.float64), torch.full((B, H), -float("inf"),
                                                                    dtype=torch.float64)
    eo, el = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    ws = []
    G = H // c.Hkv
    for b, n in enumerate(lens):
        if n == 0:
            ws.append(torch.zeros(H, 0, dtype=torch.float64))
            continue
        k = c.rows(c.k, c.ks, b, n).repeat_interleave(G, 0)          # (H, n, D)
        v = c.rows(c.v, c.vs, b, n).repeat_interleave(G, 0)
        qb = q[b].double().unsqueeze(1)
        s = (qb * k).sum(-1) * scale
        S = (qb.abs() * k.abs()).sum(-1) * abs(scale)
        lse[b] = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[b].unsqueeze(-1))
        ds = ((D + 4) * u * S + 4 * u * s.abs()).amax(-1)
        out[b] = (p.unsqueeze(-1) * v).sum(1)
        eo[b] = (2 * (ds + 2 * n * u + 2.0 ** -16) + n * u).unsqueeze(-1) * \
            (p.unsqueeze(-1) * v.abs()).sum(1)
        el[b] = ds + 2 * n * u + 8 * u * (1 + lse[b].abs())
        ws.append(p)
    return out, lse, ws, eo, el


def keep(w: torch.Tensor, n: int, budget: int, recent: int) -> list[int]:
    """The positions of one (sequence, head) that stay, rising."""
    if n <= budget:
        return list(range(n))
    old = n - recent
    x = [float("inf") if v != v else v + 0.0 for v in w[:old].tolist()]
    nan = [v != v for v in w[:old].tolist()]
    order = sorted(range(old), key=lambda i: (not nan[i], -x[i], i))
    return sorted(order[:budget - recent]) + list(range(old, n))
