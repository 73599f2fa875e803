"""QK norm and rotation in 16 bits on the GPU against 64 bits."""

from __future__ import annotations

import pytest
import torch

import _drafts
from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(B: int, H: int, Hkv: int, S: int, D: int, pairs: int, dtype: str,
         sections: list[int] | None = None, far: int = 100000, weights: bool = True,
         seed: int = 0, std: float = 1.0) -> dict:
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    axes = 1 if sections is None else len(sections)
    pos = torch.randint(0, far, (axes, B, S), generator=g, dtype=torch.int32)
    return {"q": (torch.randn((B, H, S, D), generator=g) * std).to(dt),
            "k": (torch.randn((B, Hkv, S, D), generator=g) * std).to(dt),
            "wq": (1 + 0.3 * torch.randn(D, generator=g)).to(dt) if weights else None,
            "wk": (1 + 0.3 * torch.randn(D, generator=g)).to(dt) if weights else None,
            "pos": pos if sections is not None else pos[0],
            "freq": 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs),
            "sections": sections}


def call(c: dict, dev: torch.device, layout: str, eps: float | None, **views: torch.Tensor
         ) -> tuple[torch.Tensor, torch.Tensor | None]:
    f = {k: (v.to(dev) if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    f.update(views)
    return ops.qk_norm_rope(f["q"], f["k"], f["pos"], f["freq"], sections=f["sections"],
                            norm_q_weight=f["wq"], norm_k_weight=f["wk"], eps=eps,
                            rope_layout=layout, out_q=f.get("out_q"), out_k=f.get("out_k"))


def check(c: dict, got: tuple, layout: str, eps: float | None) -> None:
    for x, w, y in ((c["q"], c["wq"], got[0]), (c["k"], c["wk"], got[1])):
        if x is None:
            assert y is None
            continue
        want, err = _drafts.norm_rope(x, w, eps, c["pos"], c["freq"], c["sections"], layout)
        bound = _drafts.rounded(want, err, x.dtype)
        off = (y.cpu().double() - want).abs()
        assert y.dtype == x.dtype and y.shape == x.shape
        assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,H,Hkv,S,D,pairs", [
    (1, 1, 1, 1, 32, 16), (1, 4, 2, 1, 128, 64), (3, 5, 1, 7, 64, 32), (2, 3, 3, 33, 128, 64),
    (2, 8, 2, 5, 256, 128), (1, 2, 1, 9, 128, 32), (2, 2, 2, 3, 64, 8), (1, 40, 8, 65, 128, 40),
    (1, 3, 2, 4, 256, 8)])
def test_matches_definition(B: int, H: int, Hkv: int, S: int, D: int, pairs: int, layout: str,
                            dtype: str, gpu: torch.device) -> None:
    for eps, weights in ((1e-6, True), (1e-5, False), (None, False)):
        c = make(B, H, Hkv, S, D, pairs, dtype, weights=weights, seed=H + S)
        check(c, call(c, gpu, layout, eps), layout, eps)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("sections", [[22, 21, 21], [64, 0], [0, 0, 64], [16, 16, 16, 16], [1, 63]])
def test_axes(sections: list[int], layout: str, gpu: torch.device) -> None:
    c = make(2, 3, 2, 19, 128, 64, "bf16", sections=sections, seed=len(sections))
    check(c, call(c, gpu, layout, 1e-6), layout, 1e-6)


def test_grid_expanded_over_the_batch(gpu: torch.device) -> None:
    """A frames x rows x columns grid, its positions expanded over the batch and
    laid out token by token; fp32 frequencies."""
    t, h, w = torch.meshgrid(torch.arange(2), torch.arange(5), torch.arange(7), indexing="ij")
    grid = torch.stack([t, h, w], -1).reshape(-1, 3).to(torch.int32)          # (S, axes)
    c = make(3, 4, 4, 70, 64, 32, "fp16", sections=[12, 10, 10])
    c["pos"] = grid.t()[:, None].expand(3, 3, 70)
    c["freq"] = c["freq"].float()
    pos = grid.to(gpu).t()[:, None].expand(3, 3, 70)
    check(c, call(c, gpu, "interleaved", 1e-6, pos=pos), "interleaved", 1e-6)


def test_far_and_negative_positions(gpu: torch.device) -> None:
    """Angles of up to 2^31 radians and below zero keep their fraction of a turn."""
    c = make(1, 2, 1, 6, 128, 64, "fp16", weights=False)
    c["pos"] = torch.tensor([[0, 1, -5, 2 ** 31 - 1, -2 ** 31, 16777217]], dtype=torch.int32)
    check(c, call(c, gpu, "half", 1e-6), "half", 1e-6)


def test_slices_of_a_projection(gpu: torch.device) -> None:
    """Rows where a fused projection left them; outputs into views, or in place."""
    B, H, Hkv, S, D = 2, 6, 2, 37, 64
    c = make(B, H, Hkv, S, D, 32, "bf16")
    x = torch.randn(B, S, (H + 2 * Hkv) * D).to(torch.bfloat16).to(gpu)
    q = x[..., :H * D].view(B, S, H, D).permute(0, 2, 1, 3)
    k = x[..., H * D:(H + Hkv) * D].view(B, S, Hkv, D).permute(0, 2, 1, 3)
    c["q"], c["k"] = q.cpu(), k.cpu()
    check(c, call(c, gpu, "half", 1e-6, q=q, k=k), "half", 1e-6)
    room = torch.full((B, H + Hkv, S, 2 * D), 7.0, dtype=torch.bfloat16, device=gpu)
    got = call(c, gpu, "half", 1e-6, q=q, k=k, out_q=room[:, :H, :, D:], out_k=room[:, H:, :, D:])
    check(c, got, "half", 1e-6)
    assert bool((room[..., :D] == 7.0).all())
    v = x[..., (H + Hkv) * D:].clone()
    got = call(c, gpu, "half", 1e-6, q=q, k=k, out_q=q, out_k=k)
    check(c, got, "half", 1e-6)
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(x[..., (H + Hkv) * D:], v)


def test_without_k(gpu: torch.device) -> None:
    c = make(2, 3, 1, 11, 32, 16, "fp16")
    c["k"] = c["wk"] = None
    check(c, call(c, gpu, "half", 1e-6), "half", 1e-6)


def test_sizes_of_values(gpu: torch.device) -> None:
    """Squares past fp32's range on either side, rows of zeros, an eps of 0; an
    infinity or a NaN stays in its row, and among unrotated dims in its place."""
    c = make(1, 2, 1, 8, 64, 16, "bf16", weights=False)
    for i, s in enumerate((1e38, 3e19, 1e-18, 1e-30, 1e-38, 0.0)):
        c["q"][:, :, i] *= s
    c["q"][:, :, 0].clamp_(-3e38, 3e38)
    check(c, call(c, gpu, "half", 1e-6), "half", 1e-6)
    c["q"][:, :, 5] = 1.0
    check(c, call(c, gpu, "half", 0.0), "half", 0.0)
    c["q"][0, 1, 3, 40] = float("nan")
    y, _ = call(c, gpu, "half", 1e-6)
    bad = y.isnan()
    assert bool(bad[0, 1, 3].all()) and int(bad.sum()) == 64
    c["q"][0, 1, 3, 40] = float("inf")
    y, _ = call(c, gpu, "half", None)
    assert torch.isinf(y[0, 1, 3, 40]) and int((~y.isfinite()).sum()) == 1


def test_empty(gpu: torch.device) -> None:
    for B, S in ((0, 3), (2, 0)):
        c = make(B, 2, 1, S, 64, 32, "bf16")
        y, z = call(c, gpu, "half", 1e-6)
        assert y.shape == (B, 2, S, 64) and z.shape == (B, 1, S, 64)


def test_no_key_heads_and_one_row_for_all_tokens(gpu: torch.device) -> None:
    """A k of no heads, whose strides mean nothing; q rows that share memory."""
    c = make(2, 3, 1, 6, 64, 32, "bf16")
    c["q"] = c["q"][:, :, :1].expand(2, 3, 6, 64)
    q = c["q"][:, :, :1].to(gpu).expand(2, 3, 6, 64)
    k = torch.empty((2, 0, 6, 67), dtype=torch.bfloat16, device=gpu)[..., 1:65]
    y, z = call(c, gpu, "half", 1e-6, q=q, k=k)
    assert z.shape == (2, 0, 6, 64)
    c["k"] = c["wk"] = None
    check(c, (y, None), "half", 1e-6)
    with pytest.raises(RuntimeError, match="overlap"):
        call(c, gpu, "half", 1e-6, q=q, out_q=q)


def test_many_tokens(gpu: torch.device) -> None:
    """More row groups than one round of workgroups; checked at the ends."""
    c = make(1, 2, 1, 40001, 128, 64, "bf16")
    y, z = call(c, gpu, "interleaved", 1e-6)
    for part in (slice(0, 9), slice(20000, 20009), slice(39992, 40001)):
        d = {**c, "q": c["q"][:, :, part], "k": c["k"][:, :, part], "pos": c["pos"][:, part]}
        check(d, (y[:, :, part], z[:, :, part]), "interleaved", 1e-6)


def test_other_stream_and_graph(gpu: torch.device) -> None:
    c = {k: (v.to(gpu) if isinstance(v, torch.Tensor) else v)
         for k, v in make(2, 4, 2, 50, 128, 64, "bf16").items()}
    run = (lambda: call(c, gpu, "half", 1e-6))
    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for step in range(3):
        c["pos"].add_(step)
        c["q"].mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
