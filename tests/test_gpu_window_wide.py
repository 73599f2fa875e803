"""Attention of long prompts over a paged cache, eight waves a workgroup (at 256
dims four), on the GPU against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import _drafts
import _paged
import _wide
from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "fp16", "bf16-e4m3", "fp16-e4m3"]

CASES = [  # B, H, Hkv, D, S, lens, qlens, window, sinks, page
    # within a window: several row tiles, none of them split
    (1, 2, 1, 32, 300, [411], None, 128, 64, 16),
    (2, 8, 2, 64, 150, [700, 150], [150, 33], 100, 4, 32),
    (1, 4, 2, 128, 300, [640], None, 64, 65, 64),
    (1, 3, 3, 64, 257, [300], None, 1, 0, 16),
    (2, 4, 4, 128, 130, [130, 400], [129, 130], 7, 200, 16),
    (2, 3, 1, 128, 90, [2100, 90], None, 300, 33, 128),
    # every key: up to eight parts, most of them without a key
    (1, 5, 1, 32, 33, [90], None, None, 0, 16),
    (2, 4, 2, 64, 100, [100, 300], [100, 7], None, 0, 16),
    (1, 2, 1, 128, 280, [1105], None, None, 0, 16),
    (1, 2, 1, 64, 600, [2111], [599], None, 0, 64),
    # four waves, tiles of 32 keys
    (2, 4, 2, 256, 150, [400, 90], [150, 33], 70, 40, 16),
    (1, 2, 1, 256, 140, [1105], None, None, 0, 32),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_definition(case: tuple, kind: str, gpu: torch.device) -> None:
    B, H, Hkv, D, S, lens, qlens, window, sinks, page = case
    dtype, cache = _wide.kinds(kind)
    c = _wide.widen(_paged.Cache(lens, Hkv, D, page, cache, seed=S))
    q = _wide.queries(B, H, S, D, dtype, seed=H)
    got = _wide.check(c, q, lens, qlens, gpu, window, sinks)
    again = _wide.call(c, q, lens, qlens, gpu, window=window, sinks=sinks)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_every_number_of_key_tiles(D: int, kind: str, gpu: torch.device) -> None:
    """136 workgroups or more, too many to be split: sequences of one tile of 64 keys
    to six, some with fewer rows than tokens; then as many over a narrow table."""
    dtype, cache = _wide.kinds(kind)
    lens = [1 + 20 * i for i in range(17)]
    lens[3], lens[6] = 64, 128
    qlens = [min(70, 3 + 11 * i) for i in range(17)]
    c = _wide.widen(_paged.Cache(lens, 8, D, 16, cache, seed=D))
    q = _wide.queries(17, 16, 70, D, dtype, seed=D)
    _wide.check(c, q, lens, qlens, gpu)
    _wide.check(c, q, lens, None, gpu, 90, 5)
    if D == 64:
        lens = [1 + 5 * i for i in range(32)]
        c = _paged.Cache(lens, 8, D, 16, cache, seed=D)
        _wide.check(c, _wide.queries(32, 16, 70, D, dtype), lens, [min(70, n) for n in lens], gpu)


@pytest.mark.parametrize("page", [1, 2, 8, 256])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_page_sizes(D: int, kind: str, page: int, gpu: torch.device) -> None:
    """Pages smaller than the rows that a wave brings at a time."""
    dtype, cache = _wide.kinds(kind)
    c = _wide.widen(_paged.Cache([150, 91], 2, D, page, cache, seed=page))
    q = _wide.queries(2, 4, 90, D, dtype)
    _wide.check(c, q, [150, 91], [90, 2], gpu, 60, 5)
    _wide.check(c, q, [150, 91], None, gpu)


@pytest.mark.parametrize("layout", ["nhd", "both"])
@pytest.mark.parametrize("kind", ["fp16", "bf16-e4m3"])
def test_layouts_and_strides(kind: str, layout: str, gpu: torch.device) -> None:
    dtype, cache = _wide.kinds(kind)
    dt = _wide.Q_DTYPES[dtype]
    c = _wide.widen(_paged.Cache([140, 75], 2, 128, 16, cache, seed=2))
    q = _wide.queries(2, 8, 70, 128, dtype)
    wide = torch.zeros((2, 70, 8, 136), dtype=dt, device=gpu)
    wide[..., 8:] = q.to(gpu).permute(0, 2, 1, 3)
    room = torch.full((2, 8, 70, 160), 3.0, dtype=dt, device=gpu)
    _wide.check(c, q, [140, 75], None, gpu, 50, 3, layout=layout,
                qview=wide[..., 8:].permute(0, 2, 1, 3), out=room[..., 8:136])
    assert bool((room[..., :8] == 3.0).all()) and bool((room[..., 136:] == 3.0).all())


@pytest.mark.parametrize("kind", KINDS)
def test_lengths_at_the_edges(kind: str, gpu: torch.device) -> None:
    dtype, cache = _wide.kinds(kind)
    c = _wide.widen(_paged.Cache([64, 64, 64, 64, 64], 2, 64, 16, cache, seed=3))
    lens = [0, 1, -4, 64, 64]
    q = _wide.queries(5, 4, 80, 64, dtype)
    _wide.check(c, q, lens, [80, 80, 80, 1 << 30, -3], gpu)
    _wide.check(c, q, [0, 1, 5, 70, 64], None, gpu, 12, 3)
    _wide.check(c, q, [2 ** 31 - 1, 64, 5000, 2048, 64], [80, 1, 80, 3, 0], gpu, 2000, 64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [None, 100])
def test_missing_pages(window: int | None, kind: str, gpu: torch.device) -> None:
    """Entries that are no page, among the keys that are seen."""
    dtype, cache = _wide.kinds(kind)
    n, page = 500, 16
    c = _wide.widen(_paged.Cache([n], 2, 64, page, cache, seed=5))
    q = _wide.queries(1, 4, 90, 64, dtype)
    table, out = c.table.clone(), [2, 3, 27, 28, 29]
    for i, e in enumerate(out):
        c.table[0, e] = (-1, c.P, 2 ** 31 - 1)[i % 3]
    got = _wide.call(c, q, [n], None, gpu, window=window, sinks=40 if window else 0)
    c.table = table
    gone = tuple(j for e in out for j in range(page * e, page * e + page))
    _wide.compare(got, _wide.definition(q, _wide.held(c, [n]), [n], [90], window,
                                        40 if window else 0, 1 / 8, _drafts.HALF[q.dtype], gone))


@pytest.mark.parametrize("kind", KINDS)
def test_given_away_pages(kind: str, gpu: torch.device) -> None:
    """Pages between the sinks and the window: -1, another's, or NaN rows."""
    dtype, cache = _wide.kinds(kind)
    n, S, window, sinks, page = 700, 130, 50, 20, 16
    c = _wide.widen(_paged.Cache([n], 1, 64, page, cache, seed=4))
    q = _wide.queries(1, 2, S, 64, dtype)
    want, _ = _wide.check(c, q, [n], None, gpu, window, sinks)
    for i in range(2, (n - S - window + 1) // page):
        pg = int(c.table[0, i])
        for x in (c.k, c.v):
            raw = x.view(torch.uint8) if cache == "e4m3" else x
            raw[pg] = 0x7F if cache == "e4m3" else float("nan")
        if cache == "e4m3":
            c.ks[pg] = c.vs[pg] = float("nan")
        if i % 2:
            c.table[0, i] = -1 if i % 4 == 1 else c.P + 5
    out, _ = _wide.call(c, q, [n], None, gpu, window=window, sinks=sinks)
    assert torch.equal(out, want)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,window", [(32, None), (64, 40), (128, 40), (128, None), (256, 40)])
def test_infinite_values(D: int, window: int | None, kind: str, value: float,
                         gpu: torch.device) -> None:
    """An infinity or NaN in V reaches the tokens that see its row, in its
    column, and no others; so does a NaN scale of a row, in every column."""
    dtype, cache = _wide.kinds(kind)
    lens, S = [130, 300], 90
    c = _wide.widen(_paged.Cache(lens, 2, D, 16, cache, seed=6))
    q = _wide.queries(2, 4, S, D, dtype, std=0.3)
    for b, j, d in ((0, 128, 7), (0, 20, 30), (0, 1, 13), (1, 290, 5), (1, 171, 6), (1, 2, 9)):
        pg = int(c.table[b, j // 16])
        if cache != "e4m3":
            c.v[pg, 1, j % 16, d] = value
        elif value != value:
            c.v.view(torch.uint8)[pg, 1, j % 16, d] = 0x7F
        elif j in (20, 171):
            c.vs[pg, 1, j % 16] = float("nan")
    _wide.check(c, q, lens, None, gpu, window, 3 if window else 0, exact=_drafts.window_attention)


@pytest.mark.parametrize("kind", KINDS)
def test_infinite_keys_and_queries(kind: str, gpu: torch.device) -> None:
    """A NaN in K or q spoils the tokens that see it only; scores of -inf weigh
    nothing, and nothing else gives zeros and -inf."""
    dtype, cache = _wide.kinds(kind)
    n, H, S, D = 100, 2, 80, 64
    c = _wide.widen(_paged.Cache([n], 1, D, 16, cache, seed=7))
    q = _wide.queries(1, H, S, D, dtype).abs()
    pg, at = int(c.table[0, (n - 3) // 16]), (n - 3) % 16
    if cache == "e4m3":
        c.ks[pg, 0, at] = float("nan")
    else:
        c.k[pg, 0, at, 5] = float("nan")
    q[0, 1, 0, 3] = float("nan")
    bad = _wide.call(c, q, [n], None, gpu)[0].cpu().isnan()
    want = torch.zeros_like(bad)
    want[0, :, S - 3:] = True
    want[0, 1, 0] = True
    assert torch.equal(bad, want)
    q[0, 1, 0, 3] = 1.0
    if cache == "e4m3":
        c.k = torch.full_like(c.k.float(), -1.0).to(c.k.dtype)
        c.ks[...] = float("inf")
    else:
        c.k[...] = float("-inf")
    out, lse = _wide.call(c, q, [n], None, gpu)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("window", [None, 64])
def test_largest_values(window: int | None, kind: str, gpu: torch.device) -> None:
    n, D = 300, 64
    c = _wide.widen(_paged.Cache([n], 1, D, 16, kind, seed=8))
    big = float(torch.finfo(_wide.Q_DTYPES[kind]).max)
    c.v = torch.where(c.v.isnan(), c.v, torch.full_like(c.v, big))
    out = _wide.call(c, _wide.queries(1, 2, 150, D, kind), [n], None, gpu, window=window)[0]
    # weights that add up to 1 but for the 16-bit rounding of each
    assert bool((out.cpu().double() >= big * (1 - 2 * _drafts.HALF[_wide.Q_DTYPES[kind]])).all())


def test_many_small_weights(gpu: torch.device) -> None:
    """8000 weights of 2^-19 of the largest each add 2^-6 of it in all: none is
    lost in fp16, in any part."""
    n, D, S = 8064, 64, 150
    c = _paged.Cache([n], 1, D, 64, "fp16", seed=9)
    c.k = torch.where(c.k.isnan(), c.k, torch.zeros_like(c.k))
    c.v = torch.where(c.v.isnan(), c.v, torch.ones_like(c.v))
    q = torch.zeros((1, 1, S, D), dtype=torch.float16)
    q[..., 0] = 19 * math.log(2.0)
    c.k[int(c.table[0, 0]), 0, 0, 0] = 1.0
    c.v[int(c.table[0, 0]), 0, 0] = 0.0
    _wide.check(c, q, [n], None, gpu, scale=1.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 2.0])
def test_scales_and_steep_scores(scale: float, kind: str, gpu: torch.device) -> None:
    """Scores far apart move a row's base in one tile after the other."""
    dtype, cache = _wide.kinds(kind)
    c = _wide.widen(_paged.Cache([390], 2, 64, 16, cache, seed=10))
    q = _wide.queries(1, 4, 80, 64, dtype)
    for window in (None, 200):
        _wide.check(c, q, [390], None, gpu, window, scale=scale)


def test_hint_changes_the_split_only(gpu: torch.device) -> None:
    """In one part (a hint of fewer places takes four waves), in some, in many."""
    lens, m = [5000, 40, 2600], [150, 40, 1]
    c = _paged.Cache(lens, 1, 64, 64, "bf16", seed=11)
    q = _wide.queries(3, 2, 150, 64, "bf16")
    for hint in (None, 1, 2047, 2048, 4000, 2 ** 40):
        _wide.check(c, q, lens, m, gpu, max_seq_len=hint)
    _wide.check(c, q, lens, m, gpu, 3000, 70)


@pytest.mark.parametrize("kind", KINDS)
def test_other_stream_and_graph(kind: str, gpu: torch.device) -> None:
    """Several replays, each against the eager result, lengths changed between."""
    dtype, cache = _wide.kinds(kind)
    for window in (None, 300):
        c = _wide.widen(_paged.Cache([900, 500], 2, 64, 16, cache, seed=14))
        f = c.to(gpu)
        q = _wide.queries(2, 4, 120, 64, dtype).to(gpu)
        lens = torch.tensor([900, 500], dtype=torch.int32, device=gpu)
        call = (lambda: ops.paged_attention(q, seq_lens=lens, window=window, sinks=4, **f))
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


@pytest.mark.parametrize("places", [64, 2048])
@pytest.mark.parametrize("S", [3, 90])
def test_not_finite_values_at_the_largest_lengths(S: int, places: int, gpu: torch.device) -> None:
    """A NaN that is seen, beside rows of padding behind a sequence whose length
    is the largest (their positions pass 32 bits), and tokens before a
    sequence's first row."""
    c = _wide.widen(_paged.Cache([64, 64, 64], 2, 64, 16, "bf16", seed=5), places)
    for b in range(3):
        c.v[int(c.table[b, 1]), 1, 3, 40] = float("nan")
    _wide.check(c, _wide.queries(3, 4, S, 64, "bf16"), [2 ** 31 - 1, 30, 2 ** 31 - 1], [1, S, S],
                gpu, exact=_drafts.window_attention)


@pytest.mark.parametrize("S", [3, 90])
def test_windows_and_sinks_past_64_bits(S: int, gpu: torch.device) -> None:
    c = _paged.Cache([200], 2, 64, 16, "bf16", seed=6)
    q = _wide.queries(1, 4, S, 64, "bf16")
    for window, sinks in ((2 ** 64 + 3, 0), (5, 2 ** 64), (2 ** 63, 2 ** 63)):
        _wide.check(c, q, [200], None, gpu, window, sinks, max_seq_len=2 ** 64 + 16)


@pytest.mark.parametrize("places", [64, 2048, 1 << 20])
@pytest.mark.parametrize("kind,power", [("bf16", -116), ("bf16", -122), ("bf16-e4m3", -90),
                                        ("bf16-e4m3", -110), ("fp16-e4m3", -12)])
@pytest.mark.parametrize("S", [1, 3, 90])
def test_small_values(S: int, kind: str, power: int, places: int, gpu: torch.device) -> None:
    """Values next to the type's smallest, under tables of any size."""
    dtype, cache = _wide.kinds(kind)
    c = _paged.Cache([200], 2, 64, 16, cache, seed=3)
    if cache == "e4m3":
        c.vs *= 2.0 ** power
    else:
        c.v = (c.v.double() * 2.0 ** power).to(c.v.dtype)
    _wide.check(_wide.widen(c, places), _wide.queries(1, 4, S, 64, dtype), [200], None, gpu)
