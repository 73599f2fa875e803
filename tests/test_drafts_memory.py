"""A drafted step's operators on the CPU: outputs that share memory with another
array of the call are refused before any launch."""

from __future__ import annotations

import struct

import pytest

import test_drafts
import test_paged
from repercep_runtime_amd import _capi

A = test_drafts.FAKE                    # never read
MB = 1 << 20


def rope(**kw) -> int:
    """2 sequences of 5 tokens, 4 + 2 heads of 128, each array in a MiB of its own."""
    a = dict(q=A, k=A + MB, qo=A + 2 * MB, ko=A + 3 * MB, pos=A + 4 * MB, freq=A + 5 * MB,
             qw=A + 6 * MB, kw=A + 7 * MB)
    return test_drafts.rope(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    dict(ko=A + 2 * MB),                                    # one place for both
    dict(ko=A + 2 * MB + 256),                              # a row further
    dict(qo=A + MB),                                        # the other's input
    dict(ko=A),
    dict(qo=A, qob=4 * 640, qoh=128, qos=512),              # its input in another order
    dict(qo=A + 256),                                       # its input a row further
    dict(qo=A + 16),                                        # half a row
    dict(ko=A + MB - 240),                                  # into its input's first row
    dict(q=A + 2 * MB + 4 * 640, qsb=0, qsh=0, qss=0),      # one row for all, among the outputs
    dict(qo=A + 4 * MB), dict(ko=A + 5 * MB - 256), dict(qo=A + 6 * MB), dict(ko=A + 7 * MB),
    dict(pos=A + 2 * MB + 252, psb=0, pss=0),               # the end of an output's first row
    # slices of a projection with a row in common: q's heads 0 to 3, k's 3 and 4
    dict(qsb=5 * 768, qsh=128, qss=768, k=A + 3 * 256, ksb=5 * 768, ksh=128, kss=768, qo=A,
         qob=5 * 768, qoh=128, qos=768, ko=A + 3 * 256, kob=5 * 768, koh=128, kos=768),
])
def test_rotation(kw: dict) -> None:
    assert rope(**kw) == 1
    assert "shares memory" in _capi.lib().rp_last_error().decode()


def test_rotation_of_several_axes() -> None:
    """Positions of an axis that reach into an output."""
    kw = dict(axes=2, sections=struct.pack("2q", 30, 34), psa=MB // 4)
    assert rope(**kw, pos=A + MB + 2048) == 1
    assert "shares memory" in _capi.lib().rp_last_error().decode()


def window(**kw) -> int:
    """2 sequences of 3 tokens, 4 heads of 128, each array in a MiB of its own."""
    c = test_paged.cache(k=A + MB, v=A + 2 * MB, block_table=A + 3 * MB)
    a = dict(q=A, out=A + 4 * MB, lse=A + 5 * MB, lens=A + 6 * MB, qlens=A + 7 * MB, ws=A + 8 * MB)
    return test_drafts.window(c, **{**a, **kw})


@pytest.mark.parametrize("kw", [
    dict(out=A, osb=4 * 3 * 128, osh=128, oss=512),         # q in another order
    dict(out=A + 256), dict(out=A + 8),                     # a row further, a part of one
    dict(out=A + MB), dict(out=A + 2 * MB + 1024),          # the cache's rows
    dict(out=A + 3 * MB - 64), dict(out=A + 6 * MB), dict(out=A + 7 * MB - 8),
    dict(lse=A), dict(lse=A + 4 * MB), dict(lse=A + MB), dict(lse=A + 6 * MB),
    dict(q=A + 4 * MB + 2560, qsb=0, qsh=0, qss=0),         # one row for all, among out's
])
def test_attention(kw: dict) -> None:
    assert window(**kw) == 1
    assert "shares memory" in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("V", [100, 50000])
@pytest.mark.parametrize("kw", [
    dict(out=A), dict(out=A + 40), dict(accepted=A + 16), dict(out=A + MB - 56),
    dict(accepted=A + MB), dict(out=A + 2 * MB + 4), dict(out=A + 3 * MB), dict(accepted=A + 4 * MB),
    dict(out=A + 5 * MB), dict(accepted=A + 5 * MB + 56)])
def test_verdict(V: int, kw: dict) -> None:
    """2 sequences of 3 drafts, each array in a MiB of its own."""
    a = dict(tokens=A, lens=A + MB, u=A + 2 * MB, target=A + 3 * MB, draft=A + 4 * MB,
             out=A + 5 * MB, accepted=A + 6 * MB, V=V, tsn=V, dsn=V, tsb=0, dsb=0)
    a.update(kw)
    if "accepted" not in kw and kw["out"] == A + 5 * MB:
        a["accepted"] = A + 5 * MB + 32
    assert test_drafts.verify(**a) == 1
    assert "shares memory" in _capi.lib().rp_last_error().decode()
