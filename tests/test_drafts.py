"""A drafted step's operators on the CPU: which calls are refused, before any launch."""

from __future__ import annotations

import struct

import pytest
import torch

import test_paged
from repercep_runtime_amd import _capi, ops

FAKE = test_paged.FAKE
BF16, F16 = _capi.RP_DTYPE_BF16, _capi.RP_DTYPE_F16


def window(c: _capi.PagedCache, **kw) -> int:
    a = dict(q=FAKE, dt=BF16, B=2, H=4, S=3, qsb=4 * 3 * 128, qsh=3 * 128, qss=128, cache=c,
             lens=FAKE, qlens=None, window=0, sinks=0, scale=0.1, out=FAKE, osb=4 * 3 * 128,
             osh=3 * 128, oss=128, lse=None, hint=0, ws=FAKE, nbytes=1 << 40, stream=None)
    a.update(kw)
    return _capi.lib().rp_paged_attn_window(*a.values())


def verify(**kw) -> int:
    a = dict(tokens=FAKE, lens=None, B=2, N=3, target=FAKE, tsb=4 * 100, tsn=100, draft=FAKE,
             dsb=300, dsn=100, dt=_capi.RP_OUT_F32, V=100, u=FAKE, out=FAKE, accepted=FAKE,
             ws=FAKE, nbytes=1 << 30, stream=None)
    a.update(kw)
    return _capi.lib().rp_verify_drafts(*a.values())


def rope(**kw) -> int:
    a = dict(q=FAKE, k=FAKE, dt=BF16, B=2, S=5, H=4, Hkv=2, D=128, qsb=4 * 640, qsh=640, qss=128,
             ksb=2 * 640, ksh=640, kss=128, qw=None, kw=None, norm=1, eps=1e-6, pos=FAKE, psa=0,
             psb=5, pss=1, freq=FAKE, f64=0, rot=128, sections=struct.pack("q", 64), axes=1,
             mode=_capi.RP_ROPE_HALF, qo=FAKE, qob=4 * 640, qoh=640, qos=128, ko=FAKE, kob=2 * 640,
             koh=640, kos=128, stream=None)
    a.update(kw)
    return _capi.lib().rp_qk_norm_rope(*a.values())


@pytest.mark.parametrize("kw,status,msg", test_paged.CACHE_REFUSALS)
def test_cache_refusals(kw: dict, status: int, msg: str) -> None:
    assert window(test_paged.cache(**kw)) == status
    assert msg in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("call,kw,status,msg", [
    (window, dict(q=None), 1, "null"),
    (window, dict(lens=None), 1, "null"),
    (window, dict(dt=2), 1, "q dtype"),
    (window, dict(dt=F16), 1, "q's dtype"),
    (window, dict(B=0), 1, "needs"),
    (window, dict(S=0), 1, "needs"),
    (window, dict(H=3), 1, "multiple"),
    (window, dict(window=-1), 1, "window"),
    (window, dict(sinks=-1), 1, "sinks"),
    (window, dict(hint=-1), 1, "max_seq_len"),
    (window, dict(scale=float("nan")), 1, "finite"),
    (window, dict(scale=3e38), 1, "finite"),
    (window, dict(B=1 << 16), 2, "too many"),
    (window, dict(S=1 << 31), 2, "too many"),
    (window, dict(q=FAKE + 8), 2, "aligned"),
    (window, dict(qss=132), 2, "aligned"),
    (window, dict(out=FAKE + 4), 2, "aligned"),
    (window, dict(oss=64), 1, "overlap"),
    (window, dict(osh=128), 1, "overlap"),
    (verify, dict(tokens=None), 1, "null"),
    (verify, dict(target=None), 1, "null"),
    (verify, dict(u=None), 1, "null"),
    (verify, dict(accepted=None), 1, "null"),
    (verify, dict(dt=5), 1, "dtype"),
    (verify, dict(B=0), 1, "sizes"),
    (verify, dict(N=-1), 1, "sizes"),
    (verify, dict(V=0), 1, "sizes"),
    (verify, dict(tsn=-100), 1, "strides"),
    (verify, dict(V=(1 << 22) + 1), 2, "too many"),
    (verify, dict(B=1 << 16), 2, "too many"),
    (verify, dict(target=FAKE + 2), 1, "aligned"),
    (verify, dict(V=50000, ws=None), 3, "workspace"),
    (verify, dict(V=50000, nbytes=16), 3, "workspace"),
    (verify, dict(V=50000, ws=FAKE + 16), 3, "workspace"),
    (rope, dict(q=None), 1, "null"),
    (rope, dict(ko=None), 1, "null"),
    (rope, dict(pos=None), 1, "null"),
    (rope, dict(dt=2), 1, "dtype"),
    (rope, dict(S=0), 1, "non-positive"),
    (rope, dict(D=96), 2, "head dim"),
    (rope, dict(mode=0), 1, "rope mode"),
    (rope, dict(rot=24), 2, "rotated dims"),
    (rope, dict(rot=144), 2, "rotated dims"),
    (rope, dict(axes=0), 1, "axes"),
    (rope, dict(axes=5), 1, "axes"),
    (rope, dict(sections=struct.pack("q", 63)), 1, "sections"),
    (rope, dict(axes=2, sections=struct.pack("2q", -1, 65)), 1, "section"),
    (rope, dict(eps=-1.0), 1, "eps"),
    (rope, dict(eps=float("inf")), 1, "eps"),
    (rope, dict(norm=0, qw=FAKE), 1, "without a norm"),
    (rope, dict(q=FAKE + 8), 2, "aligned"),
    (rope, dict(kss=132), 2, "aligned"),
    (rope, dict(qw=FAKE + 2), 2, "aligned"),
    (rope, dict(freq=FAKE + 4, f64=1), 1, "aligned"),
    (rope, dict(qos=64), 1, "overlap"),
    (rope, dict(koh=128), 1, "overlap"),
    (rope, dict(B=1 << 20, S=1 << 20), 2, "too many"),
])
def test_call_refusals(call, kw: dict, status: int, msg: str) -> None:
    """Refused before any launch: the pointers are never read."""
    c = (test_paged.cache(),) if call is window else ()
    assert call(*c, **kw) == status
    assert msg in _capi.lib().rp_last_error().decode()


def test_split_calls_ask_for_a_workspace() -> None:
    L = _capi.lib()
    c = test_paged.cache(max_pages=4096, num_pages=4096, table_stride=4096)
    for S in (1, 200):
        n = L.rp_paged_window_workspace_bytes(1, 4, S, c, 0, 0, 0)
        assert n > 0
        kw = dict(B=1, S=S, qsb=4 * S * 128, qsh=S * 128, osb=4 * S * 128, osh=S * 128)
        for bad in (dict(ws=None), dict(nbytes=n - 1), dict(ws=FAKE + 128)):
            assert window(c, **kw, **bad) == 3
            assert "workspace" in L.rp_last_error().decode()
    # none for sizes that are refused, nor where one part takes all keys
    assert L.rp_paged_window_workspace_bytes(0, 4, 1, c, 0, 0, 0) == 0
    assert L.rp_paged_window_workspace_bytes(1, 4, 1, c, -1, 0, 0) == 0
    assert L.rp_paged_window_workspace_bytes(1, 4, 1, c, 0, 0, 100) == 0
    assert L.rp_verify_drafts_workspace_bytes(4, 32768) == 0
    assert L.rp_verify_drafts_workspace_bytes(4, 32769) == 4 * 9 * 16
    assert L.rp_verify_drafts_workspace_bytes(4, (1 << 22) + 1) == 0


def test_windows_and_sinks_past_every_length() -> None:
    """Sizes that 32 or 64 bits do not add up: the window takes all keys."""
    L = _capi.lib()
    c = test_paged.cache(max_pages=4096, num_pages=4096, table_stride=4096)
    for S in (1, 200):
        n = L.rp_paged_window_workspace_bytes(1, 4, S, c, 0, 0, 0)
        for window, sinks in ((2 ** 63 - 1, 2 ** 63 - 1), (2 ** 32, 0), (16, 2 ** 32)):
            assert L.rp_paged_window_workspace_bytes(1, 4, S, c, window, sinks, 0) == n


def _step() -> dict:
    return {"q": torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16),
            "k_cache": torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16),
            "v_cache": torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16),
            "block_table": torch.zeros(2, 4, dtype=torch.int32),
            "seq_lens": torch.zeros(2, dtype=torch.int32)}


@pytest.mark.parametrize("kw,error,msg", [
    (dict(), ValueError, "GPU tensor"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), ValueError, "B, H, S, D"),
    (dict(q=torch.zeros(2, 3, 3, 64, dtype=torch.bfloat16)), ValueError, "does not fit"),
    (dict(q=torch.zeros(2, 4, 3, 64)), TypeError, "bfloat16 or float16"),
    (dict(q=torch.zeros(2, 4, 3, 64, dtype=torch.float16)), TypeError, "not read"),
    (dict(window=0), ValueError, "window"),
    (dict(sinks=-1), ValueError, "sinks"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), ValueError, "seq_lens"),
    (dict(q_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "q_lens"),
    (dict(out=torch.zeros(2, 4, 3, 64)), ValueError, "out"),
    (dict(k_scale=torch.zeros(8, 2, 16)), ValueError, "scales"),
])
def test_attention_arguments(kw: dict, error: type, msg: str) -> None:
    with pytest.raises(error, match=msg):
        ops.paged_attention(**{**_step(), **kw})


@pytest.mark.parametrize("kw,error,msg", [
    (dict(), ValueError, "GPU tensor"),
    (dict(draft_tokens=torch.zeros(2, dtype=torch.int64)), ValueError, "B, N"),
    (dict(draft_tokens=torch.zeros(2, 3, dtype=torch.int32)), TypeError, "int64"),
    (dict(target_probs=torch.zeros(2, 3, 10)), ValueError, "target_probs"),
    (dict(target_probs=torch.zeros(2, 4, 10, dtype=torch.float64)), TypeError, "target_probs"),
    (dict(draft_probs=torch.zeros(2, 3, 11)), ValueError, "draft_probs"),
    (dict(draft_probs=torch.zeros(2, 3, 10, dtype=torch.bfloat16)), TypeError, "share"),
    (dict(uniforms=torch.zeros(2, 3)), ValueError, "uniforms"),
    (dict(uniforms=torch.zeros(2, 4, dtype=torch.float64)), ValueError, "uniforms"),
    (dict(draft_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "draft_lens"),
    (dict(target_probs=torch.zeros(2, 10, 4).transpose(1, 2)), ValueError, "contiguous"),
])
def test_verdict_arguments(kw: dict, error: type, msg: str) -> None:
    a = {"draft_tokens": torch.zeros(2, 3, dtype=torch.int64),
         "target_probs": torch.zeros(2, 4, 10), "uniforms": torch.zeros(2, 4), **kw}
    with pytest.raises(error, match=msg):
        ops.verify_drafts(**a)


@pytest.mark.parametrize("kw,error,msg", [
    (dict(), ValueError, "GPU tensor"),
    (dict(q=torch.zeros(2, 5, 64, dtype=torch.bfloat16)), ValueError, "B, H, S, D"),
    (dict(q=torch.zeros(2, 4, 5, 64)), TypeError, "bfloat16 or float16"),
    (dict(q=torch.zeros(2, 4, 5, 48, dtype=torch.bfloat16)), ValueError, "head_dim"),
    (dict(k=torch.zeros(2, 4, 6, 64, dtype=torch.bfloat16)), ValueError, "k "),
    (dict(k=torch.zeros(2, 4, 5, 64, dtype=torch.float16)), TypeError, "k is"),
    (dict(positions=torch.zeros(2, 5, dtype=torch.int64)), ValueError, "positions"),
    (dict(positions=torch.zeros(3, 2, 5, dtype=torch.int32)), ValueError, "positions"),
    (dict(inv_freq=torch.zeros(32, dtype=torch.bfloat16)), ValueError, "inv_freq"),
    (dict(inv_freq=torch.zeros(12)), ValueError, "multiple of 8"),
    (dict(inv_freq=torch.zeros(40)), ValueError, "multiple of 8"),
    (dict(sections=[16, 15], positions=torch.zeros(2, 2, 5, dtype=torch.int32)), ValueError,
     "sections"),
    (dict(sections=[], positions=torch.zeros(0, 2, 5, dtype=torch.int32)), ValueError, "sections"),
    (dict(eps=None, norm_q_weight=torch.ones(64, dtype=torch.bfloat16)), ValueError, "without"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(norm_k_weight=torch.ones(64)), ValueError, "norm_k_weight"),
    (dict(rope_layout="pairs"), ValueError, "rope_layout"),
    (dict(out_q=torch.zeros(2, 4, 5, 32, dtype=torch.bfloat16)), ValueError, "out_q"),
    (dict(k=None, out_k=torch.zeros(2, 4, 5, 64, dtype=torch.bfloat16)), ValueError, "come with k"),
])
def test_rotation_arguments(kw: dict, error: type, msg: str) -> None:
    a = {"q": torch.zeros(2, 4, 5, 64, dtype=torch.bfloat16),
         "k": torch.zeros(2, 2, 5, 64, dtype=torch.bfloat16),
         "positions": torch.zeros(2, 5, dtype=torch.int32), "inv_freq": torch.zeros(32), **kw}
    with pytest.raises(error, match=msg):
        ops.qk_norm_rope(**a)
