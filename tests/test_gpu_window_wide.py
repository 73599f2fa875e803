"""Attention of long prompts over a paged cache, eight waves a workgroup, on the
GPU against 64 bits."""

from __future__ import annotations

import pytest
import torch

import _drafts
import _paged
import _wide

pytestmark = pytest.mark.gpu


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
