"""Attention of several new tokens over a paged cache, on the GPU against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import _drafts
import _paged
from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu
Q_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def queries(B: int, H: int, S: int, D: int, dtype: str, seed: int = 0, std: float = 1.0
            ) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, H, S, D), generator=g) * std).to(Q_DTYPES[dtype])


def check(c: _paged.Cache, q: torch.Tensor, lens: list[int], qlens: list[int] | None, gpu,
          window: int | None = None, sinks: int = 0, scale: float | None = None,
          layout: str = "hnd", qview: torch.Tensor | None = None, **kw) -> torch.Tensor:
    """Runs the call and compares: a weight may be rounded to 16 bits of q's type."""
    B, H, S, D = q.shape
    out, lse = ops.paged_attention(
        qview if qview is not None else q.to(gpu), seq_lens=torch.tensor(lens, dtype=torch.int32, device=gpu),
        q_lens=None if qlens is None else torch.tensor(qlens, dtype=torch.int32, device=gpu),
        window=window, sinks=sinks, scale=scale, return_lse=True, **c.to(gpu, layout), **kw)
    ql = [max(0, min(S, m)) for m in (qlens if qlens is not None else [S] * B)]
    ns = [max(0, n) for n in lens]
    cap = c.table.shape[1] * c.page
    rows = [tuple(c.rows(x, s, b, min(n, cap)) for x, s in ((c.k, c.ks), (c.v, c.vs)))
            for b, n in enumerate(ns)]
    want, wlse, eo, el = _drafts.window_attention(
        q, rows, ns, ql, window, sinks, 1 / math.sqrt(D) if scale is None else scale,
        _drafts.HALF[q.dtype])
    bound = _drafts.rounded(want, eo, q.dtype)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).nan_to_num(nan=9e9).max())
    none = torch.isneginf(wlse)
    assert torch.equal(torch.isneginf(lse.cpu()), none)
    off = (lse.cpu().double() - wlse)[~none].abs()
    assert bool((off <= el[~none] + wlse[~none].abs() * _drafts.U32).all())
    return out


CASES = [  # B, H, Hkv, D, S, lens, qlens, window, sinks, page
    (1, 1, 1, 32, 1, [1], None, None, 0, 16),
    (2, 4, 2, 64, 1, [65, 1], None, 16, 2, 16),
    (2, 4, 4, 128, 3, [70, 3], [3, 1], None, 0, 16),
    (3, 8, 2, 128, 6, [300, 6, 129], [6, 0, 4], 100, 4, 16),
    (1, 5, 1, 128, 8, [513], None, 64, 65, 32),
    (2, 16, 2, 64, 5, [200, 130], [5, 2], None, 0, 64),
    (1, 8, 8, 256, 2, [97], None, 33, 1, 16),
    (2, 6, 2, 256, 20, [150, 33], [20, 17], 40, 8, 16),
    (1, 4, 2, 128, 100, [100], None, None, 0, 16),
    (2, 8, 1, 64, 70, [170, 71], [70, 33], 50, 3, 32),
    (1, 2, 1, 128, 300, [411], None, 128, 64, 128),
    (1, 1, 1, 32, 257, [600], None, 1, 0, 16),
    (1, 3, 3, 64, 33, [40], None, 7, 40, 16),
    (2, 4, 4, 32, 130, [130, 131], [130, 129], None, 0, 16),
]


@pytest.mark.parametrize("kind", ["bf16", "fp16", "bf16-e4m3", "fp16-e4m3"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_definition(case: tuple, kind: str, gpu: torch.device) -> None:
    B, H, Hkv, D, S, lens, qlens, window, sinks, page = case
    dtype, cache = kind.split("-") if "-" in kind else (kind, kind)
    c = _paged.Cache(lens, Hkv, D, page, cache, seed=S)
    check(c, queries(B, H, S, D, dtype, seed=H), lens, qlens, gpu, window, sinks)


@pytest.mark.parametrize("page", [1, 2, 8, 256])
@pytest.mark.parametrize("S", [3, 90])
def test_page_sizes(page: int, S: int, gpu: torch.device) -> None:
    for kind in ("bf16", "e4m3"):
        c = _paged.Cache([150, 91], 2, 64, page, kind, seed=page)
        check(c, queries(2, 4, S, 64, "bf16"), [150, 91], [S, 2], gpu, 60, 5)


@pytest.mark.parametrize("layout", ["nhd", "both"])
def test_layouts_and_strides(layout: str, gpu: torch.device) -> None:
    for S in (4, 70):
        c = _paged.Cache([140, 75], 2, 128, 16, "fp16", seed=2)
        q = queries(2, 8, S, 128, "fp16")
        wide = torch.zeros((2, S, 8, 136), dtype=torch.float16, device=gpu)
        wide[..., 8:] = q.to(gpu).permute(0, 2, 1, 3)
        room = torch.full((2, 8, S, 160), 3.0, dtype=torch.float16, device=gpu)
        check(c, q, [140, 75], None, gpu, layout=layout, qview=wide[..., 8:].permute(0, 2, 1, 3),
              out=room[..., 8:136])
        assert bool((room[..., :8] == 3.0).all()) and bool((room[..., 136:] == 3.0).all())


@pytest.mark.parametrize("S", [2, 80])
def test_lengths_at_the_edges(S: int, gpu: torch.device) -> None:
    """Sequences without rows, with fewer rows than new tokens, past their table,
    with negative and too large numbers of tokens."""
    c = _paged.Cache([64, 64, 64, 64, 64], 2, 64, 16, "bf16", seed=3)
    lens = [0, 1, -4, 64, 64]
    check(c, queries(5, 4, S, 64, "bf16"), lens, [S, S, S, 1 << 30, -3], gpu)
    check(c, queries(5, 4, S, 64, "bf16"), [0, 1, 5, 70, 64], None, gpu, window=12, sinks=3)


@pytest.mark.parametrize("S", [3, 90])
def test_windows_and_sinks_past_every_length(S: int, gpu: torch.device) -> None:
    """Also where tokens stand before the first row."""
    c = _paged.Cache([600, 64, 64], 2, 64, 16, "bf16", seed=4)
    q = queries(3, 4, S, 64, "bf16")
    for window, sinks in ((2 ** 31 - 1, 2 ** 31 - 1), (2 ** 62, 0), (7, 2 ** 32)):
        check(c, q, [600, 2, 64], None, gpu, window, sinks)


@pytest.mark.parametrize("S", [3, 90])
def test_largest_lengths(S: int, gpu: torch.device) -> None:
    """Tokens far behind the table's last position see all of its rows."""
    c = _paged.Cache([64, 64], 2, 64, 16, "bf16", seed=5)
    check(c, queries(2, 4, S, 64, "bf16"), [2 ** 31 - 1, 2 ** 31 - 1], [S, 1], gpu)
    check(c, queries(2, 4, S, 64, "bf16"), [2 ** 31 - 1, 64], None, gpu, window=9, sinks=3)


@pytest.mark.parametrize("S", [3, 66])
def test_given_away_pages(S: int, gpu: torch.device) -> None:
    """Pages between the sinks and the window that no token sees: their entries
    are -1 or another's, their rows NaN."""
    n, window, sinks, page = 400, 50, 20, 16
    c = _paged.Cache([n], 1, 64, page, "bf16", seed=4)
    q = queries(1, 4, S, 64, "bf16")
    want = check(c, q, [n], None, gpu, window, sinks)
    first = (n - S - window + 1) // page
    for i in range(2, first):
        pg = int(c.table[0, i])
        c.k[pg] = c.v[pg] = float("nan")
        if i % 2:
            c.table[0, i] = -1 if i % 4 == 1 else c.P + 5
    f = c.to(gpu)
    out = ops.paged_attention(q.to(gpu), seq_lens=torch.tensor([n], dtype=torch.int32, device=gpu),
                              window=window, sinks=sinks, **f)
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("S", [1, 5, 70])
def test_missing_pages_hold_no_rows(S: int, kind: str, gpu: torch.device) -> None:
    """An entry that is no page, inside the keys that are seen."""
    n = 150
    c = _paged.Cache([n], 2, 64, 16, kind, seed=5)
    q = queries(1, 4, S, 64, "fp16" if kind == "fp16" else "bf16")
    gone = int(c.table[0, 4])
    c.table[0, 4] = -1
    out = ops.paged_attention(q.to(gpu), seq_lens=torch.tensor([n], dtype=torch.int32, device=gpu),
                              **c.to(gpu))
    c.table[0, 4] = gone
    k, v = (c.rows(x, s, 0, n) for x, s in ((c.k, c.ks), (c.v, c.vs)))
    for i in range(S):
        p = n - S + i
        seen = [j for j in range(p + 1) if j // 16 != 4]
        ks, vs = k[:, seen].repeat_interleave(2, 0), v[:, seen].repeat_interleave(2, 0)
        s = (q[0, :, i].double().unsqueeze(1) * ks).sum(-1) / 8
        w = torch.softmax(s, -1).unsqueeze(-1)
        want, size = (w * vs).sum(1), (w * vs.abs()).sum(1)
        err = size * (_drafts.HALF[q.dtype] + 2.0 ** -12)     # 64 products a score: 2^-15 or so
        off = (out[0, :, i].cpu().double() - want).abs()
        assert bool((off <= _drafts.rounded(want, err, q.dtype)).all())


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("S", [4, 70])
def test_infinite_values(S: int, kind: str, value: float, gpu: torch.device) -> None:
    """An infinity or NaN in V reaches the tokens that see its row, in its
    column, and no others."""
    n, window, H, Hkv, D = 130, 40, 4, 2, 64
    c = _paged.Cache([n], Hkv, D, 16, kind, seed=6)
    q = queries(1, H, S, D, kind, std=0.3)
    base = check(c, q, [n], None, gpu, window, 3).cpu()
    spots = [(n - 2, 7), (n - S - 20, 40), (1, 13)]           # (position, column)
    for j, d in spots:
        c.v[int(c.table[0, j // 16]), 1, j % 16, d] = value
    out = ops.paged_attention(q.to(gpu), seq_lens=torch.tensor([n], dtype=torch.int32, device=gpu),
                              window=window, sinks=3, **c.to(gpu)).cpu()
    hit = torch.zeros((1, H, S, D), dtype=torch.bool)
    for j, d in spots:
        for i in range(S):
            p = n - S + i
            if j <= p and (p - j < window or j < 3):
                hit[0, 2:, i, d] = True
    got = out[hit]
    assert bool((torch.isnan(got) if value != value else got == value).all())
    # what is finite is as accurate as before (another order of the same sums)
    off = (out.double() - base.double()).abs()[~hit]
    assert bool((off <= 4 * _drafts.HALF[q.dtype] * (1 + base.double().abs()[~hit])).all())


@pytest.mark.parametrize("S", [2, 80])
def test_infinite_keys_and_queries(S: int, gpu: torch.device) -> None:
    """A NaN in K or q spoils the tokens that see it only; scores of -inf weigh
    nothing, and nothing else gives zeros and -inf."""
    n, H, D = 100, 2, 64
    c = _paged.Cache([n], 1, D, 16, "bf16", seed=7)
    q = queries(1, H, S, D, "bf16").abs()
    c.k[int(c.table[0, (n - 1) // 16]), 0, (n - 1) % 16, 5] = float("nan")
    q[0, 1, 0, 3] = float("nan")
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    bad = ops.paged_attention(q.to(gpu), seq_lens=lens, **c.to(gpu)).cpu().isnan()
    want = torch.zeros_like(bad)
    want[0, :, S - 1] = True
    want[0, 1, 0] = True
    assert torch.equal(bad, want)
    c.k[...] = float("-inf")
    q[0, 1, 0, 3] = 1.0
    out, lse = ops.paged_attention(q.to(gpu), seq_lens=lens, return_lse=True, **c.to(gpu))
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("S", [2, 80])
def test_largest_values(S: int, dtype: str, gpu: torch.device) -> None:
    """Values near the type's largest do not overflow on the way."""
    n, D = 200, 64
    c = _paged.Cache([n], 1, D, 16, dtype, seed=8)
    big = float(torch.finfo(Q_DTYPES[dtype]).max)
    c.v = torch.where(c.v.isnan(), c.v, torch.full_like(c.v, big))
    out = ops.paged_attention(queries(1, 2, S, D, dtype).to(gpu),
                              seq_lens=torch.tensor([n], dtype=torch.int32, device=gpu),
                              **c.to(gpu)).cpu().double()
    # weights that add up to 1 but for the 16-bit rounding of each
    assert bool((out >= big * (1 - 2 * _drafts.HALF[Q_DTYPES[dtype]])).all())


@pytest.mark.parametrize("S", [1, 70])
def test_many_small_weights(S: int, gpu: torch.device) -> None:
    """8000 weights of 2^-19 of the largest each add 2^-6 of it in all: none is
    lost in fp16."""
    n, D = 8064, 64
    c = _paged.Cache([n], 1, D, 64, "fp16", seed=9)
    c.k = torch.where(c.k.isnan(), c.k, torch.zeros_like(c.k))
    c.v = torch.where(c.v.isnan(), c.v, torch.ones_like(c.v))
    pg, at = int(c.table[0, 0]), 0
    q = torch.zeros((1, 1, S, D), dtype=torch.float16)
    q[..., 0] = 19 * math.log(2.0)
    c.k[pg, 0, at, 0] = 1.0
    c.v[pg, 0, at] = 0.0
    check(c, q, [n], None, gpu, scale=1.0)


def test_scales_and_steep_scores(gpu: torch.device) -> None:
    """Scales of either sign and 0; scores far apart, the largest first or last."""
    for S in (3, 70):
        for kind in ("bf16", "e4m3"):
            c = _paged.Cache([190], 2, 64, 16, kind, seed=10)
            q = queries(1, 4, S, 64, "bf16")
            for scale in (-0.2, 0.0, 1e-3, 2.0):
                check(c, q, [190], None, gpu, scale=scale)


@pytest.mark.parametrize("S", [4, 64])
def test_hint_changes_the_split_only(S: int, gpu: torch.device) -> None:
    """Long sequences in one and in many parts, ragged, some without keys in some parts."""
    lens, m = [5000, 40, 2600], [S, min(S, 40), 1]
    c = _paged.Cache(lens, 1, 64, 64, "bf16", seed=11)
    q = queries(3, 2, S, 64, "bf16")
    for hint in (None, 1, 700, 5000):
        check(c, q, lens, m, gpu, max_seq_len=hint)
    check(c, q, lens, m, gpu, window=3000, sinks=70)


def test_many_ragged_sequences(gpu: torch.device) -> None:
    """More sequences than lanes, some long enough for several parts."""
    lens = [1 + 7 * i % 50 for i in range(70)]
    lens[0], lens[37], lens[69] = 2100, 1500, 1100
    c = _paged.Cache(lens, 1, 64, 64, "bf16", seed=15)
    check(c, queries(70, 2, 2, 64, "bf16"), lens, [i % 3 for i in range(70)], gpu)
    check(c, queries(70, 20, 2, 64, "bf16"), lens, None, gpu, window=1050, sinks=2)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("D,S,G", [(64, 10, 4), (128, 100, 2), (256, 9, 4), (256, 70, 2)])
def test_row_tiles_of_long_sequences(D: int, S: int, G: int, kind: str, gpu: torch.device) -> None:
    """Several row tiles and several parts of the keys, the last tile not full."""
    n = 4200
    c = _paged.Cache([n], 1, D, 32, kind, seed=16, std=0.7)
    q = queries(1, G, S, D, "fp16" if kind == "fp16" else "bf16")
    check(c, q, [n], [S - 1], gpu)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "bf16-e4m3", "fp16-e4m3"])
@pytest.mark.parametrize("D", [32, 128, 256])
def test_chunks_in_short_parts(D: int, kind: str, gpu: torch.device) -> None:
    """A chunk after four parts' keys, beside a sequence that leaves parts empty;
    a prompt of its own in two."""
    dtype, cache = kind.split("-") if "-" in kind else (kind, kind)
    c = _paged.Cache([1105, 90], 2, D, 16, cache, seed=D)
    check(c, queries(2, 4, 70, D, dtype), [1105, 90], [70, 41], gpu)
    check(c, queries(2, 4, 70, D, dtype), [1105, 90], [70, 41], gpu, window=700, sinks=33)
    check(c, queries(2, 4, 280, D, dtype), [1105, 90], [280, 90], gpu)


def test_one_token_as_decode(gpu: torch.device) -> None:
    """Without a window one token's attention is ``paged_attention_decode``'s, to rounding."""
    for kind in ("bf16", "fp16", "e4m3"):
        c = _paged.Cache([700, 33], 2, 128, 16, kind, seed=12)
        q = queries(2, 8, 1, 128, "fp16" if kind == "fp16" else "bf16").to(gpu)
        lens = torch.tensor([700, 33], dtype=torch.int32, device=gpu)
        f = c.to(gpu)
        x = ops.paged_attention(q, seq_lens=lens, **f).double()
        y = ops.paged_attention_decode(q, seq_lens=lens, **f).double()
        # each within its own bound of the same number; both round it once
        h = _drafts.HALF[q.dtype]
        assert bool(((x - y).abs() <= 4 * h * y.abs() + h).all())


def test_shared_pages(gpu: torch.device) -> None:
    """Candidates that share a prompt's pages and own their last ones."""
    c = _paged.Cache([64, 64, 64], 2, 64, 16, "bf16", seed=13)
    c.table[1:, :2] = c.table[0, :2]
    check(c, queries(3, 4, 5, 64, "bf16"), [64, 60, 50], None, gpu)


def test_other_stream_and_graph(gpu: torch.device) -> None:
    """Several replays, each against the eager result, lengths changed between
    (a length past a sequence's own rows reads the NaNs behind them)."""
    for S, heads in ((2, 4), (80, 4)):
        c = _paged.Cache([900, 500], 2, 64, 16, "bf16", seed=14)
        f = c.to(gpu)
        q = queries(2, heads, S, 64, "bf16").to(gpu)
        lens = torch.tensor([900, 500], dtype=torch.int32, device=gpu)
        call = (lambda: ops.paged_attention(q, seq_lens=lens, window=300, sinks=4, **f))
        want = call()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = call()
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for n in (850, 200, 333):
            lens.fill_(n)
            q.mul_(0.9)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.allclose(got, call(), rtol=0, atol=0, equal_nan=True)


def test_empty(gpu: torch.device) -> None:
    c = _paged.Cache([20], 2, 64, 16, "bf16")
    f = c.to(gpu)
    q = torch.zeros((1, 4, 0, 64), dtype=torch.bfloat16, device=gpu)
    lens = torch.tensor([20], dtype=torch.int32, device=gpu)
    assert ops.paged_attention(q, seq_lens=lens, **f).shape == (1, 4, 0, 64)
