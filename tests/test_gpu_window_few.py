"""Attention of few new tokens over a paged cache on the GPU: how precise its
weights are, and very wide tables."""

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

# A weight is taken as two 16-bit numbers.  bf16: the first is cut to 8 bits, what
# is left lies below 2^-7 of the weight's power of two, and is rounded to 8 bits
# itself: off by 2^-16 of the weight at most.  fp16: 2^-22 of it, and 2^-32 of the
# row's largest weight, which is taken as 2^7 at least, where the second part is
# subnormal (half a step of those is 2^-25).
TWO_PARTS = 2.0 ** -16

CASES = [  # B, H, Hkv, D, S, lens, qlens, window, sinks, page
    (2, 4, 2, 32, 1, [65, 1], None, None, 0, 16),
    (2, 8, 2, 64, 4, [300, 129], [4, 2], 100, 4, 16),
    (1, 8, 1, 128, 4, [513], None, None, 0, 32),
    (1, 5, 1, 128, 8, [200], None, 64, 65, 16),
    (1, 8, 1, 64, 8, [700], [7], None, 0, 64),
    (2, 4, 2, 256, 3, [150, 33], None, 40, 8, 16),
    (1, 4, 1, 256, 16, [150], None, None, 0, 16),
    (2, 4, 2, 64, 3, [150, 91], None, None, 0, 4),
]


@pytest.mark.parametrize("places", [0, 4096])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_weights_of_two_parts(case: tuple, kind: str, places: int, gpu: torch.device) -> None:
    """In one part of the keys and in several."""
    B, H, Hkv, D, S, lens, qlens, window, sinks, page = case
    dtype, cache = _wide.kinds(kind)
    c = _wide.widen(_paged.Cache(lens, Hkv, D, page, cache, seed=S), places)
    _wide.check(c, _wide.queries(B, H, S, D, dtype, seed=H), lens, qlens, gpu, window, sinks,
                weight_half=TWO_PARTS)


@pytest.mark.parametrize("page", [1, 4, 8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("S,G", [(2, 4), (5, 7)])
def test_pages_of_few_rows(S: int, G: int, D: int, kind: str, page: int, gpu: torch.device) -> None:
    """In one part and in several, with pages that are none among them, infinities
    and NaNs in V."""
    dtype, cache = _wide.kinds(kind)
    lens = [150, 91]
    c = _paged.Cache(lens, 2, D, page, cache, seed=page)
    q = _wide.queries(2, 2 * G, S, D, dtype)
    _wide.check(c, q, lens, [S, 1], gpu, 60, 5, weight_half=TWO_PARTS)
    _wide.check(_wide.widen(c, 4096), q, lens, None, gpu, weight_half=TWO_PARTS)
    for b, j, value in ((0, 147, float("nan")), (0, 74, float("inf")), (1, 3, float("-inf"))):
        at = (int(c.table[b, j // page]), 1, j % page, 11 + b)
        if cache == "e4m3":
            c.v.view(torch.uint8)[at] = 0x7F
        else:
            c.v[at] = value
    _wide.check(c, q, lens, None, gpu, 75, 4, weight_half=TWO_PARTS, exact=_drafts.window_attention)
    gone = c.table[0, 8 // page:64 // page].clone()          # seen by none: given away
    c.table[0, 8 // page:64 // page] = -1
    got = _wide.call(c, q, lens, None, gpu, window=75, sinks=4)
    c.table[0, 8 // page:64 // page] = gone
    _wide.compare(got, _drafts.window_attention(q, _wide.held(c, lens), lens, [S, S], 75, 4,
                                                1 / math.sqrt(D), TWO_PARTS))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("S,G", [(1, 1), (3, 4), (8, 4), (8, 8)])
def test_weights_that_nearly_cancel(S: int, G: int, D: int, kind: str, gpu: torch.device) -> None:
    """Half the keys weigh 1 and have values of 1, the others weigh half a step of
    16 bits less and have values of -1: of one 16-bit number a weight nothing would
    be left of the sum, or twice as much."""
    dtype, cache = _wide.kinds(kind)
    n, window = 80, 48                                  # each token sees as many of both
    part = torch.float16 if cache == "fp16" else torch.bfloat16
    less = math.log1p(-_drafts.HALF[part] / 2)
    weight_half = 2.0 ** -22 + 2.0 ** -32 if cache == "fp16" else TWO_PARTS
    c = _paged.Cache([n], 1, D, 16, cache, seed=1)
    odd = torch.arange(16) % 2 == 1
    k, v = (torch.zeros((c.P, 1, 16, D)) for _ in range(2))
    v[...] = 1.0
    v[:, :, odd] = -1.0
    if cache == "e4m3":
        k[:, :, odd, 0] = -1.0
        c.ks[...], c.vs[...] = -less, 1.0
    else:
        k[:, :, odd, 0] = less
    c.k, c.v = k.to(c.k.dtype), v.to(c.v.dtype)
    q = torch.zeros((1, G, S, D), dtype=_wide.Q_DTYPES[dtype])
    q[..., 0] = 1.0
    want, _, eo, _ = _wide.definition(q, _wide.held(c, [n]), [n], [S], window, 0, 1.0, weight_half)
    assert bool((want.abs() > 4 * _drafts.rounded(want, eo, q.dtype)).all())
    _wide.check(c, q, [n], None, gpu, window, scale=1.0, weight_half=weight_half)


def rows_past_the_caches(B: int, Hkv: int, D: int, cache: str) -> int:
    """Places of a table whose sequences, if they were as long, would have more
    than 256 MiB of rows: V is read past the caches."""
    row = 2 * (D + 4 if cache == "e4m3" else 2 * D)
    return (256 << 20) // (B * Hkv * row) + 64


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("S,G", [(1, 4), (3, 8)])
def test_very_wide_tables(S: int, G: int, D: int, kind: str, gpu: torch.device) -> None:
    dtype, cache = _wide.kinds(kind)
    lens = [700, 33, 5]
    c = _paged.Cache(lens, 2, D, 64, cache, seed=D)
    _wide.widen(c, rows_past_the_caches(3, 2, D, cache))
    q = _wide.queries(3, 2 * G, S, D, dtype)
    _wide.check(c, q, lens, [S, 1, S], gpu, weight_half=TWO_PARTS)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
def test_very_wide_tables_in_one_part(D: int, kind: str, gpu: torch.device) -> None:
    """512 workgroups, too many to be split; with infinities and NaNs in V."""
    dtype, cache = _wide.kinds(kind)
    lens = [1 + 3 * i for i in range(64)]
    c = _paged.Cache(lens, 8, D, 64, cache, seed=D)
    _wide.widen(c, rows_past_the_caches(64, 8, D, cache))
    q = _wide.queries(64, 32, 3, D, dtype)
    qlens = [min(n, 1 + n % 3) for n in lens]
    _wide.check(c, q, lens, qlens, gpu, weight_half=TWO_PARTS)
    for b, value in ((9, float("nan")), (33, float("inf")), (63, float("-inf"))):
        j = lens[b] - 2
        at = (int(c.table[b, j // 64]), 3, j % 64, 11)
        if cache == "e4m3":
            c.v.view(torch.uint8)[at] = 0x7F
        else:
            c.v[at] = value
    _wide.check(c, q, lens, qlens, gpu, weight_half=TWO_PARTS, exact=_drafts.window_attention)


@pytest.mark.parametrize("kind", ["bf16", "fp16-e4m3"])
@pytest.mark.parametrize("S", [3, 90, 200])
def test_rows_far_apart(S: int, kind: str, gpu: torch.device) -> None:
    """Pages, heads and rows whose offsets pass 32 bits, in elements or in bytes."""
    dtype, cache = _wide.kinds(kind)
    n, D, page = 90, 64, 16
    c = _wide.widen(_paged.Cache([n], 2, D, page, cache, seed=3, spare=0), 2048)
    q = _wide.queries(1, 4, S, D, dtype)
    f = c.to(gpu)
    eb = c.k.element_size()
    for strides in ((1 << 30, 1 << 29, 1 << 10), (1 << 7, 1 << 6, 1 << 25), (1 << 15, 1 << 31, 1 << 8)):
        size = sum((m - 1) * st for m, st in zip(c.k.shape, strides)) + D
        room = torch.empty(2 * size * eb, dtype=torch.uint8, device=gpu).view(c.k.dtype)
        for name, at in (("k_cache", 0), ("v_cache", size)):
            far = room[at:].as_strided(c.k.shape, (*strides, 1))
            x = getattr(c, name[0]).to(gpu)
            if eb == 1:
                far.view(torch.uint8).copy_(x.view(torch.uint8))
            else:
                far.copy_(x)
            f[name] = far
        got = ops.paged_attention(q.to(gpu), seq_lens=torch.tensor([n], dtype=torch.int32, device=gpu),
                                  return_lse=True, **f)
        _wide.compare(got, _wide.definition(q, _wide.held(c, [n]), [n], [S], None, 0, 1 / 8,
                                            _drafts.HALF[q.dtype]))
        del room, f["k_cache"], f["v_cache"], far
