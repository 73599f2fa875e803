"""Calls of ``paged_attention`` over wide block tables, against 64 bits.

How a call is launched goes by its rows (tokens times query heads of a kv head)
and by the table's places, not by the lengths in it.  More than 128 rows of a
kv head, up to 128 dims, over 2048 places or more run eight waves a workgroup,
as every long prompt does; so do they over fewer where the row tiles of all
sequences are 256 or more.  A table widened by entries that are no page takes
short sequences, which a definition in 64 bits can follow, down that path."""

from __future__ import annotations

import math

import torch

import _drafts
import _paged
from repercep_runtime_amd import ops

Q_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PLACES = 2048


def kinds(kind: str) -> tuple[str, str]:
    """(queries' type, the cache's) of "bf16", "fp16", "bf16-e4m3", "fp16-e4m3"."""
    return tuple(kind.split("-")) if "-" in kind else (kind, kind)


def queries(B: int, H: int, S: int, D: int, dtype: str, seed: int = 0, std: float = 1.0
            ) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, H, S, D), generator=g) * std).to(Q_DTYPES[dtype])


def widen(c: _paged.Cache, places: int = PLACES) -> _paged.Cache:
    """The cache with a table of at least ``places`` positions, -1 behind its own."""
    entries = max(c.table.shape[1], -(-places // c.page))
    table = torch.full((c.table.shape[0], entries), -1, dtype=torch.int32)
    table[:, :c.table.shape[1]] = c.table
    c.table = table
    return c


def held(c: _paged.Cache, n: list[int]) -> list[tuple[torch.Tensor, torch.Tensor]]:
    """The first n rows of each sequence, K and V."""
    return [tuple(c.rows(x, s, b, m) for x, s in ((c.k, c.ks), (c.v, c.vs)))
            for b, m in enumerate(n)]


def definition(q: torch.Tensor, rows: list[tuple[torch.Tensor, torch.Tensor]], lens: list[int],
               qlens: list[int], window: int | None, sinks: int, scale: float,
               weight_half: float, gone: tuple[int, ...] = ()) -> tuple[torch.Tensor, ...]:
    """``_drafts.window_attention`` of rows that are finite, all tokens of a
    sequence at a time (a masked weight of 0 meets no infinity); the positions
    ``gone`` are no rows."""
    B, H, S, D = q.shape
    u = _drafts.U32
    out = torch.zeros((B, H, S, D), dtype=torch.float64)
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64)
    eo, el = torch.zeros_like(out), torch.zeros((B, H, S), dtype=torch.float64)
    for b, (n, m) in enumerate(zip(lens, qlens)):
        k, v = rows[b]
        if m == 0 or k.shape[1] == 0:
            continue
        G = H // k.shape[0]
        k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
        p = (n - m + torch.arange(m))[:, None]
        j = torch.arange(k.shape[1])[None]
        seen = j <= p
        if window is not None:
            seen &= (p - j < min(window, 2 ** 62)) | (j < min(sinks, 2 ** 62))
        seen[:, [at for at in gone if at < k.shape[1]]] = False
        kt = k.transpose(1, 2).contiguous()
        qb = q[b, :, :m].double()
        s = torch.matmul(qb, kt) * scale
        size = torch.matmul(qb.abs(), kt.abs()) * abs(scale)
        s = s.masked_fill(~seen, -math.inf)
        z = torch.logsumexp(s, -1)
        w = torch.exp(s - z.unsqueeze(-1)).masked_fill(torch.isneginf(z).unsqueeze(-1), 0.0)
        keys = seen.sum(-1)
        ds = ((D + 2) * u * size + 8 * u * s.abs()).masked_fill(~seen, 0.0).amax(-1)
        near = 2 * keys.clamp(max=64)
        rel = 2 * (ds + (2 + near) * u) + weight_half + (keys + 4) * u
        out[b, :, :m] = torch.matmul(w, v)
        lse[b, :, :m] = z
        eo[b, :, :m] = rel.unsqueeze(-1) * torch.matmul(w, v.abs())
        el[b, :, :m] = ds + (near + keys + 4) * u + 4 * u * z.abs()
    return out, lse, eo, el


def call(c: _paged.Cache, q: torch.Tensor, lens: list[int], qlens: list[int] | None,
         gpu: torch.device, layout: str = "hnd", qview: torch.Tensor | None = None, **kw
         ) -> tuple[torch.Tensor, torch.Tensor]:
    i32 = (lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=gpu))
    return ops.paged_attention(qview if qview is not None else q.to(gpu), seq_lens=i32(lens),
                               q_lens=i32(qlens), return_lse=True, **c.to(gpu, layout), **kw)


def compare(got: tuple[torch.Tensor, torch.Tensor], want: tuple[torch.Tensor, ...]) -> None:
    """Within the bounds where the definition is finite, its infinities and
    NaNs elsewhere."""
    out, lse = (x.cpu().double() for x in got)
    x, z, eo, el = want
    dtype = got[0].dtype
    fine = x.isfinite()
    assert torch.equal(out.isnan(), x.isnan())
    assert torch.equal(out[x.isinf()], x[x.isinf()])
    bound = _drafts.rounded(x, eo, dtype)
    off = (out - x).abs()
    assert bool((off <= bound)[fine].all()), float((off / bound)[fine].max())
    none = torch.isneginf(z)
    assert torch.equal(torch.isneginf(lse), none)
    there = ~none & z.isfinite()
    assert bool(((lse - z).abs() <= el + z.abs() * _drafts.U32)[there].all())


def check(c: _paged.Cache, q: torch.Tensor, lens: list[int], qlens: list[int] | None,
          gpu: torch.device, window: int | None = None, sinks: int = 0,
          scale: float | None = None, weight_half: float | None = None, exact=definition, **kw
          ) -> tuple[torch.Tensor, torch.Tensor]:
    """Runs the call and compares.  The rows past the last page that a sequence
    has are no rows, whatever its length says."""
    B, H, S, D = q.shape
    got = call(c, q, lens, qlens, gpu, window=window, sinks=sinks, scale=scale, **kw)
    ns = [max(0, n) for n in lens]
    ql = [max(0, min(S, m)) for m in (qlens if qlens is not None else [S] * B)]
    rows = held(c, [min(n, c.lens[b]) for b, n in enumerate(ns)])
    compare(got, exact(q, rows, ns, ql, window, sinks, 1 / math.sqrt(D) if scale is None else scale,
                       _drafts.HALF[q.dtype] if weight_half is None else weight_half))
    return got
