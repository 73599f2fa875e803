"""The paged key-value cache on the GPU against plain 64-bit forms: the writer,
one new token's attention, eviction, and a decoder's loop of all of them."""

from __future__ import annotations

import math

import pytest
import torch

from repercep_runtime_amd import ops
from tests._paged import CACHE_DTYPES, Cache, decode, keep

pytestmark = pytest.mark.gpu

Q_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def bits(x: torch.Tensor) -> torch.Tensor:
    """The raw bits of a tensor, on the CPU (NaNs compare equal)."""
    return x.contiguous().view(torch.uint8).cpu()


def i32(x: list[int], dev: torch.device) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------- writing

@pytest.mark.parametrize("kind,qt", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16"),
                                     ("e4m3", "fp16")])
@pytest.mark.parametrize("D,page,Hkv,layout", [(128, 16, 2, "hnd"), (64, 1, 3, "nhd"),
                                               (32, 64, 1, "both"), (256, 4, 2, "nhd"),
                                               (128, 128, 5, "both")])
def test_append_writes_its_rows_and_no_others(gpu, kind, qt, D, page, Hkv, layout) -> None:
    """Ragged new rows behind ragged contexts, one sequence without any: each
    written row and scale is bit for bit the row (or ``rowwise_quantize``'s
    codes), and everything else keeps its bits, NaNs included."""
    ctx, new = [0, 5, 3 * page, 17], [7, 0, 1, 2 * page + 3]
    S = max(new)
    c = Cache(ctx, Hkv, D, page, kind, seed=D + page, room=S)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(4, S, Hkv, D, generator=g).to(Q_DTYPES[qt]) for _ in range(2))
    k[0, 0], v[0, 1] = 0.0, 1e-8                      # rows under the quantizer's floor
    dev = c.to(gpu, layout)
    kn, vn = (x.to(gpu).permute(0, 2, 1, 3) for x in (k, v))
    ops.paged_kv_append(kn, vn, dev["k_cache"], dev["v_cache"], dev["block_table"], i32(ctx, gpu),
                        i32(new, gpu), k_scale=dev["k_scale"], v_scale=dev["v_scale"])
    for name, x, scale, got, gs in (("k", k, c.ks, dev["k_cache"], dev["k_scale"]),
                                    ("v", v, c.vs, dev["v_cache"], dev["v_scale"])):
        want = getattr(c, name).clone()
        raw = want.view(torch.uint8) if kind == "e4m3" else want
        rows = x
        if kind == "e4m3":
            dq, codes = ops.rowwise_quantize(x.to(gpu))
            rows, dq = codes.view(torch.uint8).cpu(), dq.cpu()
        for b in range(4):
            for i in range(new[b]):
                j = ctx[b] + i
                pg = c.table[b, j // page]
                raw[pg, :, j % page] = rows[b, i]
                if scale is not None:
                    scale[pg, :, j % page] = dq[b, i]
        assert torch.equal(bits(got), bits(want)), name
        if scale is not None:
            assert torch.equal(bits(gs), bits(scale)), name


@pytest.mark.parametrize("kind", ["fp16", "e4m3"])
@pytest.mark.parametrize("D,Hkv", [(256, 2), (128, 5)])
def test_append_of_many_rows(gpu, kind, D, Hkv) -> None:
    """Prompts of thousands of rows, ragged, one shorter than its padding by all but one."""
    new, page = [7001, 1, 6900], 32
    S = max(new)
    P = sum(-(-n // page) for n in new)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    table = torch.full((3, -(-S // page)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(new):
        table[b, :-(-n // page)] = order[at:at + -(-n // page)]
        at += -(-n // page)
    g = torch.Generator(device=gpu).manual_seed(3)
    k, v = (torch.randn(3, Hkv, S, D, generator=g, device=gpu).to(torch.float16) for _ in range(2))
    dt = CACHE_DTYPES[kind]
    kc, vc = (torch.zeros((P, Hkv, page, D), dtype=torch.uint8 if kind == "e4m3" else dt,
                          device=gpu).view(dt) for _ in range(2))
    ks, vs = (torch.zeros((P, Hkv, page), device=gpu) if kind == "e4m3" else None
              for _ in range(2))
    ops.paged_kv_append(k, v, kc, vc, table.to(gpu), i32([0, 0, 0], gpu), i32(new, gpu),
                        k_scale=ks, v_scale=vs)
    for x, got, gs in ((k, kc, ks), (v, vc, vs)):
        want, scale = x, None
        if kind == "e4m3":
            scale, want = ops.rowwise_quantize(x)
        raw = got.view(torch.uint8) if kind == "e4m3" else got
        for b, n in enumerate(new):
            pages = table[b, :-(-n // page)].long().to(gpu)
            rows = raw[pages].transpose(0, 1).reshape(Hkv, -1, D)
            ref = want[b].view(torch.uint8) if kind == "e4m3" else want[b]
            assert torch.equal(rows[:, :n], ref[:, :n])
            assert (rows[:, n:] == 0).all()
            if scale is not None:
                s = gs[pages].transpose(0, 1).reshape(Hkv, -1)
                assert torch.equal(s[:, :n], scale[b, :, :n]) and (s[:, n:] == 0).all()


def test_append_leaves_out_what_has_no_place(gpu) -> None:
    """Rows past the table, before its start, and in pages that are none."""
    c = Cache([64, 64], 2, 64, 16, "bf16", seed=3)
    c.table[0] = torch.tensor([c.table[0, 0], c.P, -1, -7], dtype=torch.int32)
    dev = c.to(gpu)
    x = torch.randn(2, 2, 70, 64).to(torch.bfloat16)
    ops.paged_kv_append(x.to(gpu), x.to(gpu), dev["k_cache"], dev["v_cache"], dev["block_table"],
                        i32([-3, 20], gpu))
    want = c.k.clone()
    for i in range(3, 19):                       # positions 0 .. 15 of sequence 0
        want[c.table[0, 0], :, i - 3] = x[0, :, i]
    for i in range(44):                          # positions 20 .. 63 of sequence 1
        j = 20 + i
        want[c.table[1, j // 16], :, j % 16] = x[1, :, i]
    assert torch.equal(bits(dev["k_cache"]), bits(want))


def test_append_takes_all_rows_without_lengths_and_a_single_token(gpu) -> None:
    c = Cache([40], 3, 128, 16, "bf16", seed=4, room=1)
    dev = c.to(gpu)
    x = torch.randn(1, 3, 1, 128).to(torch.bfloat16)
    ops.paged_kv_append(x.to(gpu), (2 * x).to(gpu), dev["k_cache"], dev["v_cache"],
                        dev["block_table"], i32([40], gpu))
    assert torch.equal(dev["k_cache"][c.table[0, 2], :, 8].cpu(), x[0, :, 0])
    assert torch.equal(dev["v_cache"][c.table[0, 2], :, 8].cpu(), 2 * x[0, :, 0])


# ----------------------------------------------------------------- attention

def check_decode(gpu, c: Cache, lens: list[int], H: int, qt: str, layout: str = "hnd",
                 weights: bool = False, scale: float | None = None, hint: int | None = None,
                 seed: int = 0, q: torch.Tensor | None = None, columns: int = 0) -> None:
    if columns:                            # a table wider than any sequence
        wide = torch.full((len(lens), columns), -1, dtype=torch.int32)
        wide[:, :c.table.shape[1]] = c.table
        c.table = wide
    g = torch.Generator().manual_seed(100 + seed)
    if q is None:
        q = torch.randn(len(lens), H, c.D, generator=g).to(Q_DTYPES[qt])
    sc = 1.0 / math.sqrt(c.D) if scale is None else scale
    out, lse, ws, eo, el = decode(q, c, lens, sc)
    dev = c.to(gpu, layout)
    kw = None
    if weights:
        kw = torch.rand(len(lens), c.Hkv, c.table.shape[1] * c.page + 3, generator=g)
        before = kw.clone()
        kw = kw.to(gpu)
    got, got_lse = ops.paged_attention_decode(
        q.unsqueeze(2).to(gpu), dev["k_cache"], dev["v_cache"], dev["block_table"],
        i32(lens, gpu), scale=scale, k_scale=dev["k_scale"], v_scale=dev["v_scale"],
        key_weights=kw, return_lse=True, max_seq_len=hint)
    half = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * half       # a subnormal's half step
    err = (got.squeeze(2).double().cpu() - out).abs()
    assert (err <= eo + half * (out.abs() + eo) + tiny).all(), \
        float((err / (eo + half * out.abs() + tiny)).max())
    fin = torch.isfinite(lse)
    assert torch.equal(torch.isfinite(got_lse.cpu()), fin)
    assert torch.equal(got_lse.cpu()[~fin].double(), lse[~fin])
    assert ((got_lse.cpu().double() - lse).abs()[fin] <= el[fin]).all()
    if weights:
        G = H // c.Hkv
        for b, n in enumerate(lens):
            want = before[b].double()
            add = ws[b].reshape(c.Hkv, G, n)
            # each head's weight is off by its own bound, their sum by G roundings and the total's
            tol = (add * (2 * el[b].reshape(c.Hkv, G, 1) + 8 * 2.0 ** -24)).sum(1)
            want[:, :n] += add.sum(1)
            d = (kw[b].cpu().double() - want).abs()
            assert (d[:, :n] <= tol + (G + 2) * 2.0 ** -24 * want[:, :n]).all()
            assert torch.equal(kw[b, :, n:].cpu(), before[b, :, n:])


@pytest.mark.parametrize("kind,qt", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16"),
                                     ("e4m3", "fp16")])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("H,Hkv,page,layout,weights", [
    (4, 4, 16, "hnd", False),
    (8, 2, 1, "nhd", True),
    (5, 1, 64, "both", False),
    (32, 2, 32, "hnd", True),
    (40, 2, 16, "nhd", True),
])
def test_decode_over_ragged_lengths(gpu, kind, qt, D, H, Hkv, page, layout, weights) -> None:
    """Lengths of zero and one, at and beside the ends of tiles and pages, in one batch."""
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 63, 65, 255, 256, 257, 300, 700]
    c = Cache(lens, Hkv, D, page, kind, seed=D + H)
    check_decode(gpu, c, lens, H, qt, layout, weights)


@pytest.mark.parametrize("kind,qt", [("bf16", "bf16"), ("e4m3", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("n,weights", [(5000, False), (8192, True), (9001, True)])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (8, 1)])
def test_decode_over_long_caches(gpu, kind, qt, n, weights, H, Hkv) -> None:
    """Few rows and many keys: the keys are split and the parts joined."""
    c = Cache([n], Hkv, 128, 16, kind, seed=n)
    check_decode(gpu, c, [n], H, qt, weights=weights, hint=n)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("weights", [False, True])
def test_decode_with_room_for_long_sequences(gpu, kind, D, weights) -> None:
    """Tables of a million positions, so the call is planned for a cache of
    gigabytes: its V rows read past the last-level cache, a sequence's chunks
    shared by few workgroups or ending in the first one."""
    lens = [9000, 0, 130]
    c = Cache(lens, 2, D, 16, kind, seed=D)
    check_decode(gpu, c, lens, 4, "fp16" if kind == "fp16" else "bf16", weights=weights,
                 columns=1 << 16)


@pytest.mark.parametrize("B,Hkv", [(35, 8), (65, 8), (20, 32)])
def test_decode_of_many_heads(gpu, B, Hkv) -> None:
    """More workgroups than a round: 280, 520 and 640 heads, split and not."""
    g = torch.Generator(device=gpu).manual_seed(B)
    n, page, D = 1300, 64, 64
    P = -(-n // page)
    k, v = (torch.randn(P * 4, Hkv, page, D, generator=g, device=gpu).to(torch.bfloat16)
            for _ in range(2))
    table = torch.stack([torch.randperm(P * 4, generator=g, device=gpu)[:P] for _ in range(B)])
    q = torch.randn(B, Hkv, 1, D, generator=g, device=gpu).to(torch.bfloat16)
    lens = torch.randint(1, n + 1, (B,), generator=g, device=gpu)
    out, lse = ops.paged_attention_decode(q, k, v, table.to(torch.int32), lens.to(torch.int32),
                                          return_lse=True)
    for b in range(0, B, 7):
        rows = [x[table[b]].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :lens[b]].double().cpu()
                for x in (k, v)]
        s = (rows[0] @ q[b, :, 0].double().cpu().unsqueeze(-1)).squeeze(-1) / 8.0
        p = torch.softmax(s, -1).unsqueeze(1)
        want, size = (p @ rows[1]).squeeze(1), (p @ rows[1].abs()).squeeze(1)
        # the output's rounding; the fp32 sums and the weights' 16 bits within 2^-13 of sum p|v|
        assert ((out[b, :, 0].double().cpu() - want).abs()
                <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * size).all()
        # scores below 16 off by (64 + 8) 2^-24 of sum |q k| / 8 < 16, and 1300 roundings of a sum
        assert ((lse[b].double().cpu() - torch.logsumexp(s, -1)).abs()
                <= (72 * 16 + 2600 + 200) * 2.0 ** -24).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [2, 4, 8, 1024])
def test_decode_of_small_and_large_pages(gpu, kind, page) -> None:
    lens = [1, 7, 500, 1100]
    c = Cache(lens, 2, 128, page, kind, seed=page)
    check_decode(gpu, c, lens, 6, "bf16", weights=True)


def test_decode_reads_an_expanded_cache(gpu) -> None:
    """One head's rows seen as several heads': equal to copies of them."""
    lens = [90, 33]
    c = Cache(lens, 1, 64, 16, "bf16", seed=7)
    dev = c.to(gpu)
    q = torch.randn(2, 6, 1, 64).to(torch.bfloat16).to(gpu)
    kx, vx = (dev[n].expand(-1, 3, -1, -1) for n in ("k_cache", "v_cache"))
    got = ops.paged_attention_decode(q, kx, vx, dev["block_table"], i32(lens, gpu))
    want = ops.paged_attention_decode(q, kx.contiguous(), vx.contiguous(), dev["block_table"],
                                      i32(lens, gpu))
    assert torch.equal(got, want)


@pytest.mark.parametrize("hint", [None, 1, 64, 3000, 10 ** 9])
@pytest.mark.parametrize("weights", [False, True])
def test_decode_does_not_depend_on_the_expected_length(gpu, hint, weights) -> None:
    lens = [3000, 1, 900]
    c = Cache(lens, 2, 64, 16, "bf16", seed=8)
    check_decode(gpu, c, lens, 4, "bf16", hint=hint, weights=weights)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_decode_scales(gpu, scale) -> None:
    """No scale, a negative one and one that leaves a single key."""
    lens = [200, 33]
    c = Cache(lens, 2, 64, 16, "bf16", seed=9)
    check_decode(gpu, c, lens, 4, "bf16", scale=scale, weights=True)


def test_decode_of_scores_that_rise_and_fall(gpu) -> None:
    """Scores of hundreds, rising then falling along the keys: the running
    maximum moves at every tile, and early parts weigh nothing."""
    n, D = 2000, 64
    c = Cache([n], 1, D, 16, "bf16", seed=10)
    q = torch.zeros(1, 2, D, dtype=torch.bfloat16)
    q[0, 0, 0], q[0, 1, 0] = 64.0, -64.0
    ramp = torch.arange(n, dtype=torch.float32) / 20 - 50
    for j in range(n):
        c.k[c.table[0, j // 16], 0, j % 16, 0] = ramp[j].to(torch.bfloat16)
    check_decode(gpu, c, [n], 2, "bf16", q=q, weights=True)


def test_decode_views_and_given_output(gpu) -> None:
    """Queries and output as views of wider buffers; what lies around the output stays."""
    lens, H, D = [77, 5], 4, 128
    c = Cache(lens, 2, D, 16, "bf16", seed=11)
    dev = c.to(gpu)
    q = torch.randn(2, 1, H + 2, D).to(torch.bfloat16)
    wide = torch.full((2, 1, H + 3, 2 * D), 7.0, dtype=torch.bfloat16, device=gpu)
    out = wide[:, :, 1:1 + H, D:].transpose(1, 2)
    view = q.to(gpu)[:, :, 2:].transpose(1, 2)
    got = ops.paged_attention_decode(view, dev["k_cache"], dev["v_cache"], dev["block_table"],
                                     i32(lens, gpu), out=out)
    assert got is out
    want = ops.paged_attention_decode(view.contiguous(), dev["k_cache"], dev["v_cache"],
                                      dev["block_table"], i32(lens, gpu))
    assert torch.equal(out, want)
    rest = wide.clone()
    rest[:, :, 1:1 + H, D:] = 7.0
    assert (rest == 7.0).all()


def test_decode_of_pages_that_are_none(gpu) -> None:
    """Entries outside the cache hold no keys, lengths past the table end at
    it, and a sequence of such pages only sees nothing."""
    c = Cache([64, 48, 40], 2, 64, 16, "bf16", seed=12)
    c.table[0, 1], c.table[0, 3] = -1, c.P + 5
    c.table[1, :] = torch.tensor([2 ** 31 - 1, -2 ** 31, c.P, -1], dtype=torch.int32)
    dev = c.to(gpu)
    q = torch.randn(3, 4, 1, 64).to(torch.bfloat16)
    w = torch.zeros(3, 2, 64, device=gpu)
    out, lse = ops.paged_attention_decode(q.to(gpu), dev["k_cache"], dev["v_cache"],
                                          dev["block_table"], i32([64, 48, -4], gpu),
                                          return_lse=True, key_weights=w)
    assert (out[1:] == 0).all() and torch.isneginf(lse[1:]).all() and (w[1:] == 0).all()
    # sequence 0 is that of its pages 0 and 2 alone
    c2 = Cache([32], 2, 64, 16, "bf16", seed=12)
    c2.k, c2.v, c2.P = c.k, c.v, c.P
    c2.table = c.table[:1, [0, 2]].contiguous()
    want, wlse, ws, eo, el = decode(q[:1, :, 0], c2, [32], 0.125)
    err = (out[0, :, 0].double().cpu() - want[0]).abs()
    assert (err <= eo[0] + 2.0 ** -8 * (want[0].abs() + eo[0])).all()
    assert ((lse[0].cpu().double() - wlse[0]).abs() <= el[0]).all()
    assert (w[0, :, 16:32] == 0).all() and (w[0, :, 48:] == 0).all()
    assert abs(float(w[0].sum()) - 4.0) < 1e-4
    # past the table: its 4 pages are all there is
    a = ops.paged_attention_decode(q.to(gpu), dev["k_cache"], dev["v_cache"], dev["block_table"],
                                   i32([10 ** 6, 48, 0], gpu))
    assert torch.equal(a[0], out[0])


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_decode_passes_on_what_its_rows_hold(gpu, bad) -> None:
    """A non-finite value in an attended row of V reaches its column of that
    sequence's output and nothing else; -inf scores weigh nothing."""
    lens = [40, 40]
    c = Cache(lens, 1, 64, 16, "bf16", seed=13)
    c.v[c.table[0, 1], 0, 3, 7] = bad
    dev = c.to(gpu)
    q = torch.randn(2, 2, 1, 64).to(torch.bfloat16).to(gpu)
    out = ops.paged_attention_decode(q, dev["k_cache"], dev["v_cache"], dev["block_table"],
                                     i32(lens, gpu))
    good = torch.isfinite(out)
    assert not good[0, :, 0, 7].any()
    good[0, :, 0, 7] = True
    assert good.all()


def test_decode_of_one_finite_score(gpu) -> None:
    """Keys whose scores are all -inf but one: that one's value; none: zeros."""
    c = Cache([20, 20], 1, 32, 16, "fp16", seed=14)
    c.k[..., 0] = -float("inf")
    c.k[c.table[0, 1], 0, 2] = 0.25
    dev = c.to(gpu)
    q = torch.zeros(2, 1, 1, 32, dtype=torch.float16, device=gpu)
    q[..., 0] = 1.0
    c.k[..., 1:] = 0
    out, lse = ops.paged_attention_decode(q, dev["k_cache"], dev["v_cache"], dev["block_table"],
                                          i32([20, 20], gpu), return_lse=True)
    assert torch.equal(out[0, 0, 0].cpu(), c.v[c.table[0, 1], 0, 2])
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()


def test_decode_past_32_bit_offsets(gpu) -> None:
    """Pages whose elements lie past 2^32 of the cache."""
    P, page, D = (1 << 32) // (16 * 128) + 40, 16, 128
    free, _ = torch.cuda.mem_get_info(gpu)
    if free < 24 << 30:
        pytest.skip("needs 24 GB of GPU memory")
    c = Cache([37], 1, D, page, "bf16", seed=15)
    ids = torch.tensor([[P - 1, P - 30, 2]], dtype=torch.int32)
    k, v = (torch.empty((P, 1, page, D), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    x = torch.randn(1, 1, 37, D).to(torch.bfloat16).to(gpu)
    ops.paged_kv_append(x, -x, k, v, ids.to(gpu), i32([0], gpu))
    assert torch.equal(k[P - 1, 0], x[0, 0, :16]) and torch.equal(v[2, 0, :5], -x[0, 0, 32:])
    q = torch.randn(1, 1, 1, D).to(torch.bfloat16).to(gpu)
    got = ops.paged_attention_decode(q, k, v, ids.to(gpu), i32([37], gpu))
    kp = torch.stack([k[i] for i in ids[0].tolist()])
    vp = torch.stack([v[i] for i in ids[0].tolist()])
    want = ops.paged_attention_decode(q, kp, vp, i32([0, 1, 2], gpu).view(1, 3), i32([37], gpu))
    assert torch.equal(got, want)
    w = torch.rand(1, 1, 48, device=gpu)
    ops.paged_kv_evict(k, v, ids.to(gpu), i32([37], gpu), w, budget=20, recent=5)
    ops.paged_kv_evict(kp, vp, i32([0, 1, 2], gpu).view(1, 3), i32([37], gpu), w, budget=20,
                       recent=5)
    for i, id in enumerate(ids[0, :2].tolist()):
        assert torch.equal(k[id, 0, :20 - 16 * i], kp[i, 0, :20 - 16 * i])
        assert torch.equal(v[id, 0, :20 - 16 * i], vp[i, 0, :20 - 16 * i])


# ------------------------------------------------------------------ eviction

def check_evict(gpu, c: Cache, lens: list[int], w: torch.Tensor, budget: int, recent: int,
                layout: str = "hnd") -> None:
    dev = c.to(gpu, layout)
    new, kept = ops.paged_kv_evict(dev["k_cache"], dev["v_cache"], dev["block_table"],
                                   i32(lens, gpu), w.to(gpu), budget=budget, recent=recent,
                                   k_scale=dev["k_scale"], v_scale=dev["v_scale"])
    assert new.tolist() == [min(n, budget) for n in lens]
    want_w = torch.zeros_like(w)
    want = {n: t.clone() for n, t in (("k_cache", c.k), ("v_cache", c.v))}
    if c.ks is not None:
        want |= {"k_scale": c.ks.clone(), "v_scale": c.vs.clone()}
    for b, n in enumerate(lens):
        for h in range(c.Hkv):
            rows = keep(w[b, h], n, budget, recent)
            want_w[b, h, :len(rows)] = w[b, h, rows]
            src = torch.tensor(rows, dtype=torch.long)
            dst = torch.arange(len(rows))
            sp, dp = c.table[b, src // c.page].long(), c.table[b, dst // c.page].long()
            for t in want.values():
                t = t.view(torch.uint8) if t.element_size() == 1 else t
                t[dp, h, dst % c.page] = t[sp, h, src % c.page].clone()
    assert torch.equal(bits(kept), bits(want_w))
    for name, t in want.items():
        assert torch.equal(bits(dev[name]), bits(t)), name


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D,page,Hkv,layout", [(128, 16, 2, "hnd"), (32, 1, 1, "nhd"),
                                               (64, 64, 3, "both"), (256, 16, 1, "nhd")])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (100, 0), (100, 100), (300, 64),
                                           (1100, 3), (5000, 17)])
def test_evict_keeps_the_heavy_and_the_recent(gpu, kind, D, page, Hkv, layout, budget,
                                              recent) -> None:
    lens = [1500, 0, 1, 99, 100, 101, 301, 2049]
    c = Cache(lens, Hkv, D, page, kind, seed=D)
    g = torch.Generator().manual_seed(budget)
    w = torch.exp(torch.randn(len(lens), Hkv, c.table.shape[1] * page + 5, generator=g))
    check_evict(gpu, c, lens, w, budget, recent, layout)


@pytest.mark.parametrize("values", [[0.0], [0.0, -0.0], [1.0, 2.0], [0.5, 0.5 + 2.0 ** -24, 0.75],
                                    [float("nan"), 1.0, float("inf"), -1.0, -2.0, -0.0, 0.0],
                                    [1e-45, 0.0, 2e-45, -1e-45]])
def test_evict_ties_go_to_the_lower_position(gpu, values) -> None:
    """Few distinct weights, so most of the border is ties; special values in order."""
    lens = [1200, 5000]
    c = Cache(lens, 2, 64, 16, "bf16", seed=21)
    g = torch.Generator().manual_seed(22)
    pick = torch.randint(0, len(values), (2, 2, c.table.shape[1] * 16), generator=g)
    check_evict(gpu, c, lens, torch.tensor(values)[pick], 700, 50)


@pytest.mark.parametrize("lens,odd", [([40000], 0), ([20000, 9000, 70], 0), ([20000, 8200], 3),
                                      ([40001], 1)])
def test_evict_of_a_long_cache(gpu, lens, odd) -> None:
    """Weights that do not fit the short tables' registers, on and off 16-byte borders."""
    c = Cache(lens, 1, 32, 64, "bf16", seed=23)
    w = torch.rand(len(lens), 1, c.table.shape[1] * 64 + odd,
                   generator=torch.Generator().manual_seed(5))
    check_evict(gpu, c, lens, w, max(lens) // 2, 1000)


def test_evict_writes_every_head_of_many_caches(gpu) -> None:
    """Caches enough for whole-line column slices: 24 x 6 heads of 256-byte rows."""
    lens = [40 + 9 * b for b in range(24)]
    c = Cache(lens, 6, 128, 16, "fp16", seed=25)
    w = torch.rand(24, 6, c.table.shape[1] * 16, generator=torch.Generator().manual_seed(6))
    check_evict(gpu, c, lens, w, 100, 10)


def test_evict_weight_views_and_lengths_past_the_table(gpu) -> None:
    """Strided weights; a length past the table ends at it; a budget past it cuts nothing."""
    c = Cache([64, 30], 2, 64, 16, "bf16", seed=24)
    w = torch.rand(2, 4, 64)
    dev = c.to(gpu)
    args = (dev["k_cache"], dev["v_cache"], dev["block_table"])
    new, kept = ops.paged_kv_evict(*args, i32([10 ** 6, -2], gpu), w.to(gpu)[:, ::2], budget=10 ** 8,
                                   recent=10 ** 7)
    assert new.tolist() == [64, 0]
    assert torch.equal(kept[0].cpu(), w[0, ::2]) and (kept[1] == 0).all()
    assert torch.equal(bits(dev["k_cache"]), bits(c.k))
    new, kept = ops.paged_kv_evict(*args, i32([10 ** 6, 30], gpu), w.to(gpu)[:, ::2], budget=40,
                                   recent=8)
    rows = [keep(w[0, h], 64, 40, 8) for h in (0, 2)]
    assert new.tolist() == [40, 30]
    for h in range(2):
        assert torch.equal(kept[0, h, :40].cpu(), w[0, 2 * h, rows[h]])


# ------------------------------------------------------------- run together

@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_decoder_loop_of_all_operators(gpu, kind) -> None:
    """A prompt appended, then steps of append, attention with its weights
    totalled, the next token's score, and an eviction on the way; each step
    against a 64-bit decoder over the rows that are kept."""
    B, H, Hkv, D, page, V = 3, 4, 2, 64, 16, 1000
    prompt, steps, budget, recent = [50, 1, 33], 12, 40, 8
    g = torch.Generator().manual_seed(31)
    c = Cache([0] * B, Hkv, D, page, kind, seed=31, room=80)
    c.ks = c.vs = None if kind != "e4m3" else torch.zeros(c.P, Hkv, page)
    dev = c.to(gpu)
    args = {n: dev[n] for n in ("k_cache", "v_cache", "block_table", "k_scale", "v_scale")}
    total = torch.zeros(B, Hkv, c.table.shape[1] * page, device=gpu)
    lens = i32([0] * B, gpu)
    rows = [[([], []) for _ in range(Hkv)] for _ in range(B)]       # kept (k, v) rows, 64 bits
    sums = [[[] for _ in range(Hkv)] for _ in range(B)]
    evicted = False
    for step in range(steps):
        S = max(prompt) if step == 0 else 1
        k, v = (torch.randn(B, Hkv, S, D, generator=g).to(torch.bfloat16) for _ in range(2))
        count = prompt if step == 0 else [1] * B
        ops.paged_kv_append(k.to(gpu), v.to(gpu), start=lens, lengths=i32(count, gpu), **args)
        lens = lens + i32(count, gpu)
        if kind == "e4m3":
            k, v = ((lambda dq, x8: x8.cpu().double() * dq.cpu().double().unsqueeze(-1))(
                *ops.rowwise_quantize(x.to(gpu))) for x in (k, v))
        for b in range(B):
            for h in range(Hkv):
                for i in range(count[b]):
                    rows[b][h][0].append(k[b, h, i].double())
                    rows[b][h][1].append(v[b, h, i].double())
                    sums[b][h].append(0.0)
        q = torch.randn(B, H, 1, D, generator=g).to(torch.bfloat16)
        out = ops.paged_attention_decode(q.to(gpu), seq_lens=lens, key_weights=total, **args)
        for b in range(B):
            for h in range(H):
                kk, vv = (torch.stack(x) for x in rows[b][h // 2])
                s = kk @ q[b, h, 0].double() / 8.0
                p = torch.softmax(s, 0)
                for j, x in enumerate(p.tolist()):
                    sums[b][h // 2][j] += x
                # one rounding to bf16; the rest is far below it (2^-14 of sum p|v|)
                tol = 2.0 ** -8 * (p @ vv).abs() + 2.0 ** -13 * (p @ vv.abs())
                assert ((out[b, h, 0].double().cpu() - p @ vv).abs() <= tol).all()
        logits = (out.float().sum(dim=(1, 2)) @ torch.randn(D, V, generator=g).to(gpu)).to(
            torch.bfloat16)
        best = logits.argmax(dim=-1)
        r = ops.token_logprobs(logits, best, top=3)
        assert torch.equal(r.logprobs, r.top_logprobs[:, 0])
        assert (logits.gather(1, r.top_ids[:, :1]) == logits.amax(dim=1, keepdim=True)).all()
        if int(lens.max()) > budget + 6 and not evicted:
            evicted = True
            before = total.cpu()
            want = [[keep(before[b, h], int(lens[b]), budget, recent) for h in range(Hkv)]
                    for b in range(B)]
            lens, total = ops.paged_kv_evict(args["k_cache"], args["v_cache"],
                                             args["block_table"], lens, total, budget=budget,
                                             recent=recent, k_scale=args["k_scale"],
                                             v_scale=args["v_scale"])
            for b in range(B):
                for h in range(Hkv):
                    rows[b][h] = tuple([x[j] for j in want[b][h]] for x in rows[b][h])
                    sums[b][h] = [sums[b][h][j] for j in want[b][h]]
        for b in range(B):
            for h in range(Hkv):
                t = torch.tensor(sums[b][h], dtype=torch.float64)
                # a weight is off by 2^-14 of itself at most, each sum by a rounding a step
                assert ((total[b, h, :len(t)].cpu().double() - t).abs() <= 2.0 ** -13 * t).all()
                assert (total[b, h, len(t):] == 0).all()
    assert evicted


def test_candidates_share_the_pages_of_their_prefix(gpu) -> None:
    """16 candidates name one prefix's pages and own the rest: equal to 16
    sequences with copies of it."""
    B, H, D, page, prefix = 16, 8, 128, 16, 512
    lens = [prefix + 1 + b for b in range(B)]
    c = Cache(lens, H, D, page, "bf16", seed=41)
    k, v = c.k, c.v
    for b in range(1, B):
        for x in (k, v):
            x[c.table[b, :prefix // page].long()] = x[c.table[0, :prefix // page].long()]
    shared = c.table.clone()
    shared[:, :prefix // page] = c.table[0, :prefix // page]
    dev = c.to(gpu)
    q = torch.randn(B, H, 1, D).to(torch.bfloat16).to(gpu)
    a = ops.paged_attention_decode(q, dev["k_cache"], dev["v_cache"], dev["block_table"],
                                   i32(lens, gpu))
    b = ops.paged_attention_decode(q, dev["k_cache"], dev["v_cache"], shared.to(gpu),
                                   i32(lens, gpu))
    assert torch.equal(a, b)
    check_decode(gpu, c, lens, H, "bf16")


def test_equal_calls_give_equal_bits(gpu) -> None:
    lens = [3000, 700, 33]
    c = Cache(lens, 2, 128, 16, "e4m3", seed=51)
    dev = c.to(gpu)
    q = torch.randn(3, 16, 1, 128).to(torch.bfloat16).to(gpu)
    first = None
    for _ in range(4):
        w = torch.zeros(3, 2, c.table.shape[1] * 16, device=gpu)
        got = (*ops.paged_attention_decode(q, dev["k_cache"], dev["v_cache"], dev["block_table"],
                                           i32(lens, gpu), k_scale=dev["k_scale"],
                                           v_scale=dev["v_scale"], key_weights=w,
                                           return_lse=True), w)
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))


def _step(dev: dict, q: torch.Tensor, x: torch.Tensor, lens: torch.Tensor, w: torch.Tensor,
          logits: torch.Tensor, tokens: torch.Tensor) -> tuple:
    """One decoder step on given buffers; the eviction works on copies of the cache."""
    args = {n: dev[n] for n in ("k_cache", "v_cache", "block_table", "k_scale", "v_scale")}
    ops.paged_kv_append(x, -x, start=lens - 1, **args)
    total = w.clone()
    out, lse = ops.paged_attention_decode(q, seq_lens=lens, key_weights=total, return_lse=True,
                                          **args)
    k, v = dev["k_cache"].clone(), dev["v_cache"].clone()
    ks, vs = dev["k_scale"].clone(), dev["v_scale"].clone()
    new, kept = ops.paged_kv_evict(k, v, dev["block_table"], lens, total, budget=200, recent=20,
                                   k_scale=ks, v_scale=vs)
    r = ops.token_logprobs(logits, tokens, top=4)
    return out, lse, total, new, kept, k.view(torch.uint8), ks, vs, *r


def test_captured_steps_replay_as_eager_ones(gpu) -> None:
    """Two graphs of a whole step, replayed in turn with new inputs and eager
    work between them, equal eager steps bit for bit."""
    lens = [1000, 300, 90]
    c = Cache(lens, 2, 128, 16, "e4m3", seed=61)
    c.k.view(torch.uint8)[c.k.isnan()], c.v.view(torch.uint8)[c.v.isnan()] = 0, 0
    g = torch.Generator(device=gpu).manual_seed(62)

    def inputs(i: int) -> dict:
        B, L, V = len(lens), c.table.shape[1] * 16, 5000
        rnd = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
        return {"q": rnd(B, 8, 1, 128).to(torch.bfloat16), "x": rnd(B, 2, 1, 128).to(torch.bfloat16),
                "lens": i32([n - 7 * i for n in lens], gpu), "w": rnd(B, 2, L).abs(),
                "logits": rnd(B, V).to(torch.bfloat16),
                "tokens": torch.randint(0, V, (B,), generator=g, device=gpu)}

    sides = []
    for _ in range(2):
        dev, buf = c.to(gpu), inputs(0)
        _step(dev, **buf)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _step(dev, **buf)
        sides.append((dev, buf, graph, got))
    for rep in range(3):
        for i, (dev, buf, graph, got) in enumerate(sides):
            for name, t in inputs(rep + i).items():
                buf[name].copy_(t)
        for dev, buf, graph, got in sides:
            graph.replay()
        _ = torch.randn(1024, device=gpu).sum().item()
        for dev, buf, graph, got in sides:
            fresh = {n: t.clone() if t is not None else None for n, t in dev.items()}
            for x, y in zip(got, _step(fresh, **{n: t.clone() for n, t in buf.items()})):
                assert torch.equal(bits(x), bits(y)), f"replay {rep}"


def test_calls_on_two_streams(gpu) -> None:
    """Calls on two streams at once, and on a stream other than the current
    one's tensors, give what one stream gives."""
    lens = [4000, 100]
    cs = [Cache(lens, 2, 128, 16, "bf16", seed=70 + i) for i in range(2)]
    devs = [c.to(gpu) for c in cs]
    q = torch.randn(2, 8, 1, 128).to(torch.bfloat16).to(gpu)
    n = i32(lens, gpu)
    ws = [torch.zeros(2, 2, c.table.shape[1] * 16, device=gpu) for c in cs]

    def call(i: int, w: torch.Tensor) -> torch.Tensor:
        d = devs[i]
        return ops.paged_attention_decode(q, d["k_cache"], d["v_cache"], d["block_table"], n,
                                          key_weights=w)

    want = [(call(i, w), w) for i, w in enumerate(torch.zeros_like(w) for w in ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got[i] = call(i, ws[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i][0]) and torch.equal(ws[i], want[i][1])


def test_batches_of_none(gpu) -> None:
    c = Cache([5], 2, 64, 16, "bf16")
    dev = c.to(gpu)
    none = torch.empty((0, 1), dtype=torch.int32, device=gpu)
    q = torch.empty((0, 4, 1, 64), dtype=torch.bfloat16, device=gpu)
    out, lse = ops.paged_attention_decode(q, dev["k_cache"], dev["v_cache"], none, i32([], gpu),
                                          return_lse=True)
    assert out.shape == (0, 4, 1, 64) and lse.shape == (0, 4)
    x = torch.empty((0, 2, 3, 64), dtype=torch.bfloat16, device=gpu)
    ops.paged_kv_append(x, x, dev["k_cache"], dev["v_cache"], none, i32([], gpu))
    x = torch.empty((1, 2, 0, 64), dtype=torch.bfloat16, device=gpu)
    ops.paged_kv_append(x, x, dev["k_cache"], dev["v_cache"], dev["block_table"], i32([0], gpu))
    new, kept = ops.paged_kv_evict(dev["k_cache"], dev["v_cache"], none, i32([], gpu),
                                   torch.empty((0, 2, 16), device=gpu), budget=4, recent=1)
    assert new.shape == (0,) and kept.shape == (0, 2, 16)
    assert torch.equal(bits(dev["k_cache"]), bits(c.k))


# ------------------------------------------- weights and values of all sizes

def _rows_of(c: Cache, n: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The pages and offsets of the first n rows of sequence 0."""
    j = torch.arange(n)
    return c.table[0, j // c.page].long(), j % c.page


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("n,page", [(700, 16), (700, 4), (20000, 16)])
@pytest.mark.parametrize("gap", [14, 18, 22, 26, 30, 36])
def test_decode_of_a_heavy_key_without_value(gpu, kind, n, page, gap) -> None:
    """One key takes nearly all the weight and its value is 0; the others, 2^-gap
    of it to half that each, are the output: they keep 16 bits as any weight
    does."""
    D = 64
    c = Cache([n], 1, D, page, kind, seed=gap)
    pg, at = _rows_of(c, n)
    g = torch.Generator().manual_seed(n + gap)
    c.k[pg, 0, at] = 0
    c.k[pg, 0, at, 0] = -torch.rand(n, generator=g).to(c.k.dtype)
    c.v[pg, 0, at] = (torch.rand(n, D, generator=g) * 4e4 + 2e4).to(c.v.dtype)
    heavy = n // 3
    c.k[pg[heavy], 0, at[heavy], 0] = gap
    c.v[pg[heavy], 0, at[heavy]] = 0
    q = torch.zeros(1, 2, D, dtype=Q_DTYPES[kind])
    q[0, :, 0] = 1.0
    check_decode(gpu, c, [n], 2, kind, q=q, scale=math.log(2.0), weights=True, hint=n)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,page", [(1, 16), (2, 4), (40, 16), (700, 16), (300, 4), (6000, 16)])
def test_decode_of_infinite_values(gpu, kind, n, page) -> None:
    """Infinities in attended rows of V come out as the sum's: of one sign
    infinite, of both or with a NaN NaN, in their columns only."""
    D, H = 64, 3
    c = Cache([n], 1, D, page, kind, seed=n)
    pg, at = _rows_of(c, n)
    inf = float("inf")
    for column, values in ((3, [inf]), (5, [-inf]), (7, [inf, -inf]), (9, [float("nan")]),
                           (11, [inf, inf, inf]), (D - 1, [-inf, -inf])):
        for i, x in enumerate(values):
            j = (n // 2 + 17 * i) % n if n > 2 else i % n
            c.v[pg[j], 0, at[j], column] = x
    q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(n)).to(Q_DTYPES[kind])
    want, lse, _, eo, el = decode(q, c, [n], 0.125)
    dev = c.to(gpu)
    got, got_lse = ops.paged_attention_decode(q.unsqueeze(2).to(gpu), dev["k_cache"],
                                              dev["v_cache"], dev["block_table"], i32([n], gpu),
                                              return_lse=True, max_seq_len=n)
    got = got.squeeze(2).double().cpu()
    fin = torch.isfinite(want)
    assert int((~fin).sum()) == 6 * H
    assert torch.equal(got[~fin].nan_to_num(nan=7.0), want[~fin].nan_to_num(nan=7.0))
    half = torch.finfo(q.dtype).eps / 2
    assert ((got - want).abs()[fin] <= (eo + half * (want.abs() + eo))[fin]).all()
    assert ((got_lse.cpu().double() - lse).abs() <= el).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("n,page", [(1, 16), (33, 16), (700, 16), (700, 4), (9000, 16)])
def test_decode_of_very_large_and_small_values(gpu, kind, n, page) -> None:
    """Values up to the type's largest: sums of weights about a base may leave
    fp32's range where the weighted mean does not.  And values near its
    smallest, which a scale against that would lose."""
    D = 64
    c = Cache([n], 1, D, page, kind, seed=n)
    pg, at = _rows_of(c, n)
    if kind == "e4m3":
        c.vs[pg[::2], 0, at[::2]] = 7e35
        raw = c.v.view(torch.uint8)
        raw[pg, 0, at, 3] = 0x7E                              # 448
        raw[pg, 0, at, 5] = 0x7E + (torch.arange(n) % 2 * 128).to(torch.uint8)
    else:
        top = torch.finfo(c.v.dtype).max
        c.v[pg, 0, at, 3] = top
        c.v[pg, 0, at, 5] = (top * (-1.0) ** torch.arange(n)).to(c.v.dtype)
        c.v[pg, 0, at, 7] = top / 2 ** 14
        c.v[pg, 0, at, 9] = -top
        c.v[pg, 0, at, 11] *= 1e-30 if kind == "bf16" else 1e-6
    g = torch.Generator().manual_seed(n)
    qt = "fp16" if kind == "fp16" else "bf16"
    q = torch.randn(1, 2, D, generator=g).to(Q_DTYPES[qt])
    check_decode(gpu, c, [n], 2, qt, q=q, weights=True, hint=n)
    if kind != "e4m3":                                        # small values alone
        small = 1e-33 if kind == "bf16" else 1e-6
        c.v[pg, 0, at] = (torch.randn(n, D, generator=g) * small).to(c.v.dtype)
        check_decode(gpu, c, [n], 2, qt, q=q, hint=n)


def _halves(layout: str, P: int, Hkv: int, page: int, D: int, dev: torch.device
            ) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V as two halves of one buffer, none of their rows shared."""
    def buf(*s: int) -> torch.Tensor:
        return torch.zeros(s, dtype=torch.bfloat16, device=dev)

    if layout == "columns":
        x = buf(P, Hkv, page, 2 * D)
        return x[..., :D], x[..., D:]
    if layout == "heads":
        x = buf(P, 2 * Hkv, page, D)
        return x[:, Hkv:], x[:, :Hkv]
    if layout == "every other head":
        x = buf(P, page, 2 * Hkv, D).permute(0, 2, 1, 3)
        return x[:, ::2], x[:, 1::2]
    if layout == "every other page":
        x = buf(2 * P, page, Hkv, D).permute(0, 2, 1, 3)
        return x[::2], x[1::2]
    x = buf(2 * P, Hkv, page, D)
    return x[P:], x[:P]


@pytest.mark.parametrize("layout", ["columns", "heads", "every other head", "every other page",
                                    "pages"])
def test_caches_that_are_halves_of_one_buffer(gpu, layout) -> None:
    """Written, read and cut as two separate caches are."""
    P, Hkv, page, D, lens = 12, 3, 16, 64, [70, 33, 40]
    g = torch.Generator(device=gpu).manual_seed(1)
    table = torch.randperm(P, generator=g, device=gpu)[:12].view(3, 4).to(torch.int32)
    table = torch.cat([table, torch.full_like(table[:, :1], -1)], 1)
    x, y = (torch.randn(3, Hkv, 70, D, generator=g, device=gpu).to(torch.bfloat16)
            for _ in range(2))
    q = torch.randn(3, 6, 1, D, generator=g, device=gpu).to(torch.bfloat16)
    n, got = i32(lens, gpu), []
    separate = [torch.zeros(P, Hkv, page, D, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    for k, v in (_halves(layout, P, Hkv, page, D, gpu), separate):
        ops.paged_kv_append(x, y, k, v, table, i32([0, 0, 0], gpu), n)
        # totals and output with the heads outermost
        w = torch.zeros(Hkv, 3, 5 * page, device=gpu).transpose(0, 1)
        out = torch.empty(6, 1, 3, D, dtype=torch.bfloat16, device=gpu).permute(2, 0, 1, 3)
        ops.paged_attention_decode(q, k, v, table, n, key_weights=w, out=out)
        got.append([w, out, *ops.paged_kv_evict(k, v, table, n, w, budget=36, recent=4), k, v])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_shared_memory_is_refused(gpu) -> None:
    """One tensor as K and V, totals that two heads share, an expanded output."""
    c = Cache([20, 20], 2, 64, 16, "bf16")
    d = c.to(gpu)
    n = i32([20, 20], gpu)
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16, device=gpu)
    k, table = d["k_cache"], d["block_table"]
    w = torch.zeros(2, 2, table.shape[1] * 16, device=gpu)
    with pytest.raises(ops.C.HipLibraryError, match="overlap"):
        ops.paged_kv_append(x, x, k, k, table, n)
    with pytest.raises(ops.C.HipLibraryError, match="overlap"):
        ops.paged_kv_evict(k, k, table, n, w, budget=4, recent=1)
    both = torch.zeros(3, table.shape[1] * 16, device=gpu)
    both = both.as_strided((2, 2, both.shape[1]), (both.shape[1], both.shape[1], 1))
    with pytest.raises(ops.C.HipLibraryError, match="overlap"):
        ops.paged_attention_decode(x, k, k, table, n, key_weights=both)
    with pytest.raises(ops.C.HipLibraryError, match="overlap"):
        ops.paged_attention_decode(x, k, k, table, n, out=x[:1].expand(2, -1, -1, -1))
    want = ops.paged_attention_decode(x, k, k.clone(), table, n)
    assert torch.equal(ops.paged_attention_decode(x, k, k, table, n), want)     # reading may


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("page", [16, 4])
def test_decode_weights_have_32_bits(gpu, kind, page) -> None:
    """Two keys whose weighted values nearly cancel leave what the weights lost.

    Scores are single products below 1 in size: rounded three times on the way
    to the exponential's argument (8 u with its own 2 u in a weight), the sum
    and its reciprocal as often again, at both keys, and the mean's up to twelve
    partial sums one u each: 40 u sum p|v| beside the output's rounding.  A
    weight of 16 bits would be off by up to 2^-16 = 256 u."""
    B, H, D, u = 64, 4, 64, 2.0 ** -24
    lens = [2] * B
    c = Cache(lens, 1, D, page, kind, seed=page)
    g = torch.Generator().manual_seed(5)
    qt = "fp16" if kind == "fp16" else "bf16"
    q = torch.zeros(B, H, D, dtype=Q_DTYPES[qt])
    q[:, :, 0] = (torch.rand(B, H, generator=g) * 2 - 1).to(q.dtype)
    pg = c.table[:, 0].long()
    for j in (0, 1):
        c.k[pg, 0, j] = torch.zeros(B, D).to(c.k.dtype)
        c.k[pg, 0, j, 0] = (torch.rand(B, generator=g) * 2 - 1).to(c.k.dtype)
    if kind == "e4m3":
        c.ks[pg] = 0.875
    p = torch.stack([w[0] for w in decode(q, c, lens, 1.0)[2]])         # head 0's weights
    ratio = p[:, :1] / p[:, 1:]
    if kind == "e4m3":
        ratio = ratio * (c.vs[pg, 0, 0] / c.vs[pg, 0, 1]).double().unsqueeze(1)
    c.v[pg, 0, 1] = (c.v[pg, 0, 0].double() * -ratio).clamp(-448.0, 448.0).to(c.v.dtype)
    out = decode(q, c, lens, 1.0)[0]
    assert torch.isfinite(out).all()
    size = torch.stack([(w.unsqueeze(-1) * c.rows(c.v, c.vs, b, 2).abs()).sum(1)
                        for b, w in enumerate(decode(q, c, lens, 1.0)[2])])
    dev = c.to(gpu)
    got = ops.paged_attention_decode(q.unsqueeze(2).to(gpu), dev["k_cache"], dev["v_cache"],
                                     dev["block_table"], i32(lens, gpu), scale=1.0,
                                     k_scale=dev["k_scale"], v_scale=dev["v_scale"])
    half = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * half
    err = (got.squeeze(2).double().cpu() - out).abs()
    assert (err <= 40 * u * size * (1 + half) + half * out.abs() + tiny).all(), \
        float(((err - half * out.abs()) / (u * size)).max())
