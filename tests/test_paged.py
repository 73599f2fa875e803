"""The paged cache's and the token scores' host side, on the CPU: which calls
are refused, and where the kernels look for a row, pages that are none among them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from repercep_runtime_amd import _capi, ops

FAKE = 1 << 20           # 256-byte aligned non-null address; never dereferenced
BF16, F16 = _capi.RP_DTYPE_BF16, _capi.RP_DTYPE_F16


def cache(**kw) -> _capi.PagedCache:
    a = dict(k=FAKE, v=FAKE, k_scale=None, v_scale=None, block_table=FAKE, num_pages=8, heads=2,
             page_size=16, head_dim=128, stride_page=2 * 16 * 128, stride_head=16 * 128,
             stride_row=128, table_stride=4, max_pages=4, dtype=_capi.RP_CACHE_BF16)
    a.update(kw)
    return _capi.PagedCache(*a.values())


CACHE_REFUSALS = [
    (dict(k=None), 1, "null pointer"),
    (dict(block_table=None), 1, "null pointer"),
    (dict(dtype=3), 1, "cache dtype"),
    (dict(dtype=_capi.RP_CACHE_E4M3), 1, "k_scale"),
    (dict(k_scale=FAKE, v_scale=FAKE), 1, "16-bit one takes none"),
    (dict(num_pages=0), 1, "non-positive"),
    (dict(max_pages=0), 1, "non-positive"),
    (dict(head_dim=96), 2, "head dim"),
    (dict(page_size=48), 2, "power of two"),
    (dict(page_size=1 << 17), 2, "power of two"),
    (dict(max_pages=1 << 28), 2, "too many"),
    (dict(num_pages=1 << 31), 2, "too many"),
    (dict(stride_row=64), 1, "strides"),
    (dict(stride_page=-4096), 1, "strides"),
    (dict(stride_head=16 * 128 + 4), 2, "aligned"),
    (dict(v=FAKE + 8), 2, "aligned"),
]


def append(c: _capi.PagedCache, **kw) -> int:
    a = dict(k=FAKE, v=FAKE, dt=BF16, B=2, S=4, ksb=4 * 256, ksh=128, kss=256, vsb=4 * 256,
             vsh=128, vss=256, cache=c, start=FAKE, lengths=None, stream=None)
    a.update(kw)
    return _capi.lib().rp_paged_kv_append(*a.values())


def decode(c: _capi.PagedCache, **kw) -> int:
    a = dict(q=FAKE, dt=BF16, B=2, H=4, qsb=512, qsh=128, cache=c, lens=FAKE, scale=0.1, out=FAKE,
             osb=512, osh=128, lse=None, w=None, wsb=0, wsh=0, hint=0, ws=FAKE, nbytes=1 << 30,
             stream=None)
    a.update(kw)
    return _capi.lib().rp_paged_attn_decode(*a.values())


def evict(c: _capi.PagedCache, **kw) -> int:
    a = dict(cache=c, lens=FAKE, B=2, w=FAKE, wsb=128, wsh=64, budget=32, recent=8, new=2 * FAKE,
             kept=2 * FAKE, W=64, ws=FAKE, nbytes=1 << 20, stream=None)
    a.update(kw)
    return _capi.lib().rp_paged_kv_evict(*a.values())


@pytest.mark.parametrize("kw,status,msg", CACHE_REFUSALS)
def test_cache_refusals(kw: dict, status: int, msg: str) -> None:
    """Every entry point refuses a bad descriptor before any launch."""
    for call in (append, decode, evict):
        assert call(cache(**kw)) == status
        assert msg in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("call,kw,status,msg", [
    (append, dict(k=None), 1, "null"),
    (append, dict(start=None), 1, "null"),
    (append, dict(dt=2), 1, "input dtype"),
    (append, dict(dt=F16), 1, "own dtype"),
    (append, dict(B=0), 1, "non-positive"),
    (append, dict(S=1 << 31), 2, "too many"),
    (append, dict(B=1 << 16), 2, "too many"),
    (append, dict(ksh=100), 2, "aligned"),
    (append, dict(v=FAKE + 8), 2, "aligned"),
    (decode, dict(q=None), 1, "null"),
    (decode, dict(dt=5), 1, "q dtype"),
    (decode, dict(dt=F16), 1, "q's dtype"),
    (decode, dict(H=3), 1, "multiple"),
    (decode, dict(B=0), 1, "B > 0"),
    (decode, dict(hint=-1), 1, "max_seq_len"),
    (decode, dict(scale=float("nan")), 1, "sm_scale"),
    (decode, dict(scale=float("inf")), 1, "sm_scale"),
    (decode, dict(B=1 << 16), 2, "too many"),
    (decode, dict(qsh=132), 2, "aligned"),
    (decode, dict(out=FAKE + 2), 2, "aligned"),
    (decode, dict(w=FAKE, wsb=-1), 1, "key_weights"),
    (decode, dict(w=FAKE, wsb=128, wsh=63), 1, "key_weights"),
    (decode, dict(w=FAKE, wsb=0, wsh=64), 1, "key_weights"),
    (decode, dict(osb=0), 1, "overlap"),
    (decode, dict(osh=64), 1, "overlap"),
    (decode, dict(w=FAKE, ws=None, nbytes=0), 3, "workspace"),
    (evict, dict(lens=None), 1, "null"),
    (evict, dict(new=FAKE), 1, "not the inputs"),
    (evict, dict(kept=FAKE), 1, "not the inputs"),
    (evict, dict(budget=0), 1, "budget"),
    (evict, dict(recent=33), 1, "recent"),
    (evict, dict(recent=-1), 1, "recent"),
    (evict, dict(B=1 << 16), 2, "too many"),
    (evict, dict(W=63), 1, "64 positions"),
    (evict, dict(ws=None), 3, "workspace"),
    (evict, dict(ws=FAKE + 16), 3, "workspace"),
    (evict, dict(nbytes=255), 3, "workspace"),
])
def test_call_refusals(call, kw: dict, status: int, msg: str) -> None:
    assert call(cache(), **kw) == status
    assert msg in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("call", [append, evict])
@pytest.mark.parametrize("kw", [dict(stride_page=0), dict(stride_head=0), dict(stride_head=64)])
def test_writers_refuse_rows_that_overlap(call, kw: dict) -> None:
    """A cache expanded over its pages or heads can be read, not written."""
    assert call(cache(**kw)) == 1
    assert "overlap" in _capi.lib().rp_last_error().decode()


BIG = (0, 1, -1, 1 << 16, 1 << 31, 1 << 32, 1 << 47, 1 << 62, -(1 << 62))


def test_workspace_sizes_of_any_arguments() -> None:
    """Sizes that the calls refuse need no workspace, and none divides by zero."""
    L = _capi.lib()
    for x in BIG:
        for y in BIG:
            L.rp_token_logprobs_workspace_bytes(x, y, 0, 5)
            L.rp_paged_attn_workspace_bytes(x, y, cache(), 0, 1)
            L.rp_paged_attn_workspace_bytes(2, 4, cache(heads=x, page_size=y), 0, 1)
            L.rp_paged_attn_workspace_bytes(2, 4, cache(max_pages=x, head_dim=y), x, 1)
            L.rp_paged_evict_workspace_bytes(x, cache(), y)
            L.rp_paged_evict_workspace_bytes(2, cache(heads=x, max_pages=y), 5)
    assert L.rp_token_logprobs_workspace_bytes(4, 1 << 62, 0, 5) == 0
    assert L.rp_paged_attn_workspace_bytes(1 << 62, 4, cache(), 0, 1) == 0
    assert L.rp_paged_attn_workspace_bytes(2, 1, cache(), 0, 1) == 0        # H below the heads
    assert L.rp_paged_evict_workspace_bytes(2, cache(), 1 << 62) == \
        L.rp_paged_evict_workspace_bytes(2, cache(), 64) == 256 + 2 * 2 * 64 * 4


@pytest.mark.parametrize("B,H,heads,keys,weights,parts", [
    (1, 32, 32, 640, 0, 1),          # 320 KB of keys: one launch
    (16, 32, 32, 640, 0, 1),         # a round of workgroups without a split
    (1, 40, 8, 131072, 0, 64),       # 512 workgroups
    (12, 32, 8, 4096, 0, 5),         # 480: no second round
    (33, 32, 8, 4096, 0, 3),         # 264 would leave most CUs one, some two
    (52, 32, 8, 4096, 0, 1),
    (65, 32, 8, 4096, 0, 8),         # 520: 8 in a second round
    (65, 32, 8, 900, 0, 1),          # parts of less than 256 KB
    (75, 32, 8, 4096, 0, 2),
    (1, 8, 1, 131072, 0, 512),
    (8, 32, 8, 4096, 1, 16),         # with key weights: 1024 workgroups
    (1, 1, 1, 100, 1, 1),            # no more than a workgroup's keys
    (1, 1, 1, 1 << 30, 1, 1024),
    (1, 32, 1, 131072, 0, 256),      # 32 query heads of a kv head: two tiles of 16
])
def test_attention_splits(B: int, H: int, heads: int, keys: int, weights: int,
                          parts: int) -> None:
    """The parts a call's keys are split into, read from the workspace they need."""
    c = cache(heads=heads, page_size=16, max_pages=-(-keys // 16))
    pad = lambda n: (n + 255) // 256 * 256  # noqa: E731
    want = pad(B * H * parts * 8) if parts > 1 or weights else 0
    want += pad(B * H * parts * 128 * 4) if parts > 1 else 0
    want += pad(B * H * (-(-keys // 32) * 32) * 4) if weights else 0
    assert _capi.lib().rp_paged_attn_workspace_bytes(B, H, c, keys, weights) == want


@pytest.mark.parametrize("kw,status,msg", [
    (dict(logits=None), 1, "null"),
    (dict(tokens=None), 1, "null"),
    (dict(top_ids=None), 1, "null"),
    (dict(dt=3), 1, "logits dtype"),
    (dict(N=0), 1, "bad sizes"),
    (dict(ld=99), 1, "bad sizes"),
    (dict(top=33), 1, "top 33"),
    (dict(V=4, top=5), 1, "top 5"),
    (dict(top=-1), 1, "top -1"),
    (dict(temperature=0.0), 1, "temperature"),
    (dict(temperature=float("nan")), 1, "temperature"),
    (dict(temperature=float("inf")), 1, "temperature"),
    (dict(V=1 << 31, ld=1 << 31), 2, "too many"),
    (dict(V=(1 << 21) + 1, ld=1 << 22), 2, "too many"),
    (dict(N=1 << 31), 2, "too many"),
    (dict(temperature=1e-45), 1, "temperature"),
    (dict(logits=FAKE + 1), 1, "aligned"),
    (dict(V=40000, ld=40000, ws=None), 3, "workspace"),
    (dict(V=40000, ld=40000, ws=FAKE + 16), 3, "workspace"),
])
def test_logprob_refusals(kw: dict, status: int, msg: str) -> None:
    a = dict(logits=FAKE, dt=0, N=4, V=100, ld=100, tokens=FAKE, temperature=1.0, top=5, lp=FAKE,
             ent=FAKE, top_lp=FAKE, top_ids=FAKE, ws=FAKE, nbytes=1 << 30, stream=None)
    a.update(kw)
    assert _capi.lib().rp_token_logprobs(*a.values()) == status
    assert msg in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("page", [1, 16, 128])
def test_rows_are_where_the_table_says(page: int) -> None:
    """Position j is row j % page of page table[j / page]; past the table, and
    in a page that is none, there is no row."""
    entries = [3, -1, 0, 7, 8, 2 ** 31 - 1, -2 ** 31, 5]
    table = (ctypes.c_int32 * len(entries))(*entries)
    sp, sh, sr = 2 * page * 128 + 64, page * 128 + 32, 128
    c = cache(block_table=ctypes.cast(table, ctypes.c_void_p), page_size=page, stride_page=sp,
              stride_head=sh, stride_row=sr, max_pages=len(entries))
    at = _capi.lib().rp_selftest_paged_row
    for head in range(2):
        for j in range(len(entries) * page):
            id = entries[j // page]
            want = id * sp + head * sh + j % page * sr if 0 <= id < 8 else -1
            assert at(c, head, j) == want
        for j in (-1, -page, len(entries) * page, 2 ** 31, 2 ** 40):
            assert at(c, head, j) == -1


def test_row_offsets_pass_32_bits() -> None:
    table = (ctypes.c_int32 * 1)(1_000_000)
    c = cache(block_table=ctypes.cast(table, ctypes.c_void_p), num_pages=1_000_001, max_pages=1,
              stride_page=65536 * 128, stride_head=16 * 128, page_size=16)
    assert _capi.lib().rp_selftest_paged_row(c, 1, 15) == 1_000_000 * 65536 * 128 + 16 * 128 + 15 * 128


# ------------------------------------------------------------ torch entry points

def _t(*shape: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    return torch.zeros(shape, dtype=dtype)


def _step(**kw) -> dict:
    """A valid call's tensors (on the CPU: the last check refuses those)."""
    a = dict(k_cache=_t(8, 2, 16, 128), v_cache=_t(8, 2, 16, 128),
             block_table=_t(3, 4, dtype=torch.int32))
    a.update(kw)
    return a


E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("kw,err,msg", [
    ({}, ValueError, "GPU tensor"),
    (dict(v_cache=_t(8, 2, 16, 64)), ValueError, "share one"),
    (dict(k_cache=_t(8, 2, 24, 128), v_cache=_t(8, 2, 24, 128)), ValueError, "page_size"),
    (dict(k_cache=_t(0, 2, 16, 128), v_cache=_t(0, 2, 16, 128)), ValueError, "needs pages"),
    (dict(block_table=_t(3, 0, dtype=torch.int32)), ValueError, "needs pages"),
    (dict(v_cache=_t(8, 2, 16, 128, dtype=torch.float16)), TypeError, "both"),
    (dict(k_cache=_t(8, 2, 16, 256)[..., ::2], v_cache=_t(8, 2, 16, 256)[..., ::2]), ValueError,
     "unit stride"),
    (dict(v_cache=_t(8, 16, 2, 128).permute(0, 2, 1, 3)), ValueError, "share their strides"),
    (dict(block_table=_t(3, 4, dtype=torch.int64)), ValueError, "block_table"),
    (dict(block_table=_t(2, 4, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=_t(3, 8, dtype=torch.int32)[:, ::2]), ValueError, "block_table"),
    (dict(k_scale=_t(8, 2, 16, dtype=torch.float32)), ValueError, "only an e4m3fn"),
    (dict(k_cache=_t(8, 2, 16, 128, dtype=E4M3), v_cache=_t(8, 2, 16, 128, dtype=E4M3)),
     ValueError, "needs k_scale"),
    (dict(k_cache=_t(8, 2, 16, 128, dtype=E4M3), v_cache=_t(8, 2, 16, 128, dtype=E4M3),
          k_scale=_t(8, 2, 8, dtype=torch.float32), v_scale=_t(8, 2, 16, dtype=torch.float32)),
     ValueError, "k_scale must be"),
])
def test_torch_cache_refusals(kw: dict, err: type, msg: str) -> None:
    step = _step(**kw)
    lens = _t(3, dtype=torch.int32)
    with pytest.raises(err, match=msg):
        ops.paged_attention_decode(_t(3, 4, 1, 128), seq_lens=lens, **step)
    with pytest.raises(err, match=msg):
        ops.paged_kv_append(_t(3, 2, 5, 128), _t(3, 2, 5, 128), start=lens, **step)
    with pytest.raises(err, match=msg):
        ops.paged_kv_evict(seq_lens=lens, key_weights=_t(3, 2, 200, dtype=torch.float32), budget=4,
                           recent=1, **step)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(q=_t(3, 4, 128)), ValueError, "q must be"),
    (dict(q=_t(3, 4, 2, 128)), ValueError, "q must be"),
    (dict(q=_t(3, 3, 1, 128)), ValueError, "does not fit"),
    (dict(q=_t(3, 4, 1, 64)), ValueError, "does not fit"),
    (dict(q=_t(3, 4, 1, 128, dtype=torch.float32)), TypeError, "q must be"),
    (dict(q=_t(3, 4, 1, 128, dtype=torch.float16)), TypeError, "not read with"),
    (dict(q=_t(3, 4, 1, 256)[..., ::2]), ValueError, "contiguous"),
    (dict(seq_lens=_t(3, dtype=torch.int64)), ValueError, "seq_lens"),
    (dict(seq_lens=_t(2, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(out=_t(3, 4, 1, 128, dtype=torch.float32)), ValueError, "out must be"),
    (dict(key_weights=_t(3, 2, 63, dtype=torch.float32)), ValueError, "key_weights"),
    (dict(key_weights=_t(3, 4, 64, dtype=torch.float32)), ValueError, "key_weights"),
    (dict(key_weights=_t(3, 2, 64)), ValueError, "key_weights"),
])
def test_torch_decode_refusals(kw: dict, err: type, msg: str) -> None:
    a = dict(q=_t(3, 4, 1, 128), seq_lens=_t(3, dtype=torch.int32), **_step())
    a.update(kw)
    with pytest.raises(err, match=msg):
        ops.paged_attention_decode(**a)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(v=_t(3, 2, 5, 64)), ValueError, "share one"),
    (dict(k=_t(3, 4, 5, 128), v=_t(3, 4, 5, 128)), ValueError, "does not hold"),
    (dict(k=_t(3, 2, 5, 128, dtype=torch.float16), v=_t(3, 2, 5, 128, dtype=torch.float16)),
     TypeError, "takes no"),
    (dict(k=_t(3, 2, 5, 128, dtype=torch.float32)), TypeError, "both"),
    (dict(start=_t(3, dtype=torch.int64)), ValueError, "start"),
    (dict(lengths=_t(4, dtype=torch.int32)), ValueError, "lengths"),
])
def test_torch_append_refusals(kw: dict, err: type, msg: str) -> None:
    a = dict(k=_t(3, 2, 5, 128), v=_t(3, 2, 5, 128), start=_t(3, dtype=torch.int32), **_step())
    a.update(kw)
    with pytest.raises(err, match=msg):
        ops.paged_kv_append(**a)


@pytest.mark.parametrize("kw,msg", [
    (dict(budget=0, recent=0), "recent"),
    (dict(budget=4, recent=5), "recent"),
    (dict(recent=-1), "recent"),
    (dict(seq_lens=_t(3, 1, dtype=torch.int32)), "vector"),
    (dict(key_weights=_t(3, 2, 63, dtype=torch.float32)), "key_weights"),
    (dict(k_cache=_t(8, 2, 16, 96), v_cache=_t(8, 2, 16, 96)), "head_dim"),
])
def test_torch_evict_refusals(kw: dict, msg: str) -> None:
    a = dict(seq_lens=_t(3, dtype=torch.int32), key_weights=_t(3, 2, 64, dtype=torch.float32),
             budget=8, recent=2, **_step())
    a.update(kw)
    with pytest.raises(ValueError, match=msg):
        ops.paged_kv_evict(**a)


@pytest.mark.parametrize("args,kw,err,msg", [
    ((_t(4, 10), _t(4, dtype=torch.int64)), {}, ValueError, "GPU tensor"),
    ((_t(4, 10), _t(5, dtype=torch.int64)), {}, ValueError, "leading shape"),
    ((_t(4, 10), _t(4, dtype=torch.int32)), {}, TypeError, "int64"),
    ((_t(4, 10, dtype=torch.float64), _t(4, dtype=torch.int64)), {}, TypeError, "logits"),
    ((_t(4, 20)[:, ::2], _t(4, dtype=torch.int64)), {}, ValueError, "contiguous"),
    ((_t(4, 10), _t(4, dtype=torch.int64)), dict(top=11), ValueError, "top"),
    ((_t(4, 100), _t(4, dtype=torch.int64)), dict(top=33), ValueError, "top"),
    ((_t(4, 10), _t(4, dtype=torch.int64)), dict(temperature=0.0), ValueError, "temperature"),
    ((_t(4, 10), _t(4, dtype=torch.int64)), dict(temperature=float("inf")), ValueError,
     "temperature"),
])
def test_torch_logprob_refusals(args: tuple, kw: dict, err: type, msg: str) -> None:
    with pytest.raises(err, match=msg):
        ops.token_logprobs(*args, **kw)


# rows of 64 x 2 and 3 elements apart: each stride is as long as a row, and some rows are the same
@pytest.mark.parametrize("call", [append, evict])
@pytest.mark.parametrize("kw", [
    dict(stride_page=16 * 128, stride_head=16 * 128),
    dict(stride_page=128, stride_head=128),
    dict(stride_page=4 * 128, stride_head=16 * 128),
    dict(stride_page=16 * 128, stride_head=8 * 16 * 128 - 128),
    dict(v=FAKE),                                   # K's memory
    dict(v=FAKE + 2 * 128),                         # K's second row
    dict(v=FAKE + 2 * 16 * 128),                    # K's second head
    dict(v=FAKE + 2 * 7 * 2 * 16 * 128),            # K's last page
    dict(v=FAKE - 2 * 2 * 16 * 128),                # a page early: K begins inside V
    dict(stride_row=192, v=FAKE + 2 * 96),          # not past K's columns
])
def test_writers_refuse_rows_that_share_memory(call, kw: dict) -> None:
    """Strides and places under which two rows of K, of V or of both overlap."""
    a = dict(v=3 * FAKE)
    if "v" in kw and "stride_row" in kw:
        a |= dict(stride_head=16 * 192, stride_page=2 * 16 * 192)
    a.update(kw)
    assert call(cache(**a)) == 1
    assert "overlap" in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("kw", [
    dict(w=FAKE, wsb=64, wsh=64),                   # both strides a row: sequence 1 is head 1
    dict(w=FAKE, wsb=64, wsh=127),
    dict(w=FAKE, wsb=100, wsh=64),
    dict(osb=128, osh=128),
    dict(osb=384, osh=128),                         # four heads of 128
    dict(osb=128, osh=252),
])
def test_attention_refuses_outputs_that_share_memory(kw: dict) -> None:
    assert decode(cache(), **kw) == 1
    assert "overlap" in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.4e38])
def test_a_scale_that_leaves_the_range_is_refused(scale: float) -> None:
    """Scores are taken in powers of two: scale * log2(e) has to be finite too."""
    assert decode(cache(), scale=scale) == 1
    assert "sm_scale" in _capi.lib().rp_last_error().decode()


@pytest.mark.parametrize("dim", [0, 1, 2])
def test_strides_of_single_dimensions_do_not_count(dim: int) -> None:
    """K and V of one page, head or row a page: that dimension's stride means
    nothing, and may differ between them."""
    shape = [8, 2, 16, 128]
    shape[dim] = 1
    k, v = _t(*shape), _t(*shape)
    strides = list(v.stride())
    strides[dim] += 8
    step = _step(k_cache=k, v_cache=v.as_strided(shape, strides))
    lens = _t(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):          # the last check
        ops.paged_attention_decode(_t(3, 2 * shape[1], 1, 128), seq_lens=lens, **step)


def test_calls_past_the_launch_limit_are_refused() -> None:
    """2^32 threads along the grid, which the runtime does not launch: refused
    before any kernel has run."""
    L = _capi.lib()
    wide = (FAKE, 0, 1 << 24, 100, 0, FAKE, 1.0, 0, FAKE, None, None, None, None, 0, None)
    assert L.rp_token_logprobs(*wide) == 2
    assert "too many" in L.rp_last_error().decode()
    # sixteen rows of 256 a workgroup, 2^28 of them
    big = cache(v=3 * FAKE, head_dim=256, stride_row=256, stride_head=16 * 256,
                stride_page=2 * 16 * 256)
    assert append(big, S=1 << 27, ksb=0, ksh=0, kss=0, vsb=0, vsh=0, vss=0, B=1) == 2
    assert "too many" in L.rp_last_error().decode()
    # key weights of 2^30 positions and 16 heads: 2^24 workgroups of the second launch
    long = cache(heads=16, max_pages=1 << 26, stride_page=16 * 16 * 128)
    assert decode(long, H=16, w=FAKE, wsb=1 << 34, wsh=1 << 30, nbytes=1 << 62, qsb=2048,
                  osb=2048) == 2
    assert "too many" in L.rp_last_error().decode()


def test_wide_tables_without_key_weights_are_taken() -> None:
    """The key weights' launch limits only the calls that have them: this one
    gets as far as its workspace."""
    long = cache(heads=16, max_pages=1 << 26, stride_page=16 * 16 * 128)
    assert decode(long, H=16, qsb=2048, osb=2048, ws=None, nbytes=0) == 3
