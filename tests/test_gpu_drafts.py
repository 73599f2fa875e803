"""Drafted tokens' verdict on the GPU against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

import _drafts
from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def make(B: int, N: int, V: int, dtype: str, drafts: bool, seed: int) -> dict:
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B, N + 1, V), generator=g) * 2
    p = torch.softmax(x, -1).to(DTYPES[dtype])
    q = torch.softmax(x[:, :N] + torch.randn((B, N, V), generator=g), -1).to(DTYPES[dtype])
    if drafts and N:
        t = torch.multinomial(q.float().reshape(B * N, V), 1, generator=g).view(B, N)
    else:
        t = p[:, :N].float().argmax(-1).view(B, N)
    lens = torch.randint(0, N + 1, (B,), generator=g)
    lens[0] = N
    return {"tokens": t, "target": p, "draft": q if drafts else None, "lens": lens.int(),
            "u": torch.rand((B, N + 1), generator=g)}


def check(c: dict, dev: torch.device, **views: torch.Tensor) -> ops.DraftVerdict:
    f = {k: (None if v is None else v.to(dev)) for k, v in c.items()}
    f.update(views)
    r = ops.verify_drafts(f["tokens"], f["target"], f["u"], draft_probs=f["draft"],
                          draft_lens=f["lens"])
    lens = c["lens"].tolist() if c["lens"] is not None else [c["tokens"].shape[1]] * len(c["u"])
    want, counts = _drafts.verify(c["tokens"].tolist(), c["target"], c["draft"], c["u"], lens)
    assert r.accepted.tolist() == counts
    assert r.tokens.tolist() == want
    return r


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("B,N,V", [(1, 1, 1), (1, 4, 5), (3, 7, 1000), (5, 3, 4095), (4, 2, 4097),
                                   (2, 70, 257), (2, 5, 128256), (9, 0, 4100)])
def test_matches_definition(B: int, N: int, V: int, dtype: str, drafts: bool,
                            gpu: torch.device) -> None:
    check(make(B, N, V, dtype, drafts, seed=B * 31 + V), gpu)


def test_all_tokens_drafted(gpu: torch.device) -> None:
    c = make(6, 5, 300, "fp32", True, 3)
    c["lens"] = None
    check(c, gpu)


def test_strided_and_unaligned_rows(gpu: torch.device) -> None:
    """Rows that begin at any multiple of the type, views of a larger tensor."""
    for dtype in DTYPES:
        c = make(3, 4, 4103, dtype, True, 5)
        p = torch.full((3, 2, 5, 4110), float("nan"), dtype=DTYPES[dtype], device=gpu)
        q = torch.full((4, 3, 4107), float("nan"), dtype=DTYPES[dtype], device=gpu)
        p[:, 1, :, 3:4106] = c["target"].to(gpu)
        q[:, :, 1:4104] = c["draft"].to(gpu).transpose(0, 1)
        check(c, gpu, target=p[:, 1, :, 3:4106], draft=q[:, :, 1:4104].transpose(0, 1))


def test_one_row_for_all(gpu: torch.device) -> None:
    """Expanded probabilities: the same row at every position."""
    c = make(4, 3, 500, "fp32", True, 7)
    row = c["target"][:1, :1].to(gpu).contiguous()
    c["target"] = c["target"][:1, :1].expand(4, 4, 500)
    check(c, gpu, target=row.expand(4, 4, 500))


def test_borders(gpu: torch.device) -> None:
    """u q = p is no acceptance; u = 0 draws the first token of any weight;
    u >= 1 the last one; a draft outside the vocabulary is rejected."""
    p = torch.tensor([0.0, 0.25, 0.0, 0.5, 0.25, 0.0])
    q = torch.tensor([0.0, 0.5, 0.5, 0.0, 0.0, 0.0])
    cases = [([1], [0.5, 0.0]), ([1], [0.499, 0.5]), ([2], [0.0, 0.3]), ([0], [0.0, 0.9]),
             ([-1], [0.0, 0.0]), ([6], [0.0, 1.0]), ([1 << 40], [0.0, 0.25]),
             ([1], [0.0, 0.25]), ([1], [0.0, 1.0]), ([1], [0.0, 0.2499999])]
    B = len(cases)
    c = {"tokens": torch.tensor([t for t, _ in cases]), "u": torch.tensor([u for _, u in cases]),
         "target": p.expand(B, 2, 6).contiguous(), "draft": q.expand(B, 1, 6).contiguous(),
         "lens": torch.ones(B, dtype=torch.int32)}
    r = check(c, gpu)
    assert r.accepted.tolist() == [0, 1, 0, 0, 0, 0, 0, 1, 1, 1]
    check({**c, "draft": None}, gpu)


def test_nothing_left(gpu: torch.device) -> None:
    """p = q with a rejected draft draws from p; a p of zeros and NaNs gives -1."""
    p = torch.zeros((3, 2, 4200))
    p[0, :, 4150] = 0.5
    p[0, :, 17] = 0.5
    p[2] = float("nan")
    p[2, 0, 4199] = 1e-30
    c = {"tokens": torch.tensor([[3], [3], [3]]), "u": torch.tensor([[0.0, 0.6]] * 3), "target": p,
         "draft": p[:, :1].clone(), "lens": torch.ones(3, dtype=torch.int32)}
    c["draft"][2] = 0.0
    r = check(c, gpu)
    assert r.tokens[:, 0].tolist() == [4150, -1, 4199]


def test_lens_out_of_range(gpu: torch.device) -> None:
    c = make(4, 5, 64, "fp32", True, 11)
    c["lens"] = torch.tensor([-7, 99, 0, 2 ** 31 - 1], dtype=torch.int32)
    check(c, gpu)


def test_draws_from_the_target(gpu: torch.device) -> None:
    """Over a grid of random numbers the first token comes out as p has it: a
    token's share of a 128 x 128 grid is off by its two borders' cells in each
    direction, here at most (V + 2) / 128 / 2."""
    g = torch.Generator().manual_seed(1)
    V, n = 7, 128
    p, q = (torch.softmax(torch.randn(V, generator=g), 0) for _ in range(2))
    at = (torch.arange(n) + 0.5) / n
    share = torch.zeros(V, dtype=torch.float64)
    for t in range(V):                  # the draft is t with probability q(t)
        u = torch.stack([at.repeat_interleave(n), at.repeat(n)], 1).to(gpu)
        B = n * n
        r = ops.verify_drafts(torch.full((B, 1), t, device=gpu),
                              p.to(gpu).expand(B, 2, V), u,
                              draft_probs=q.to(gpu).expand(B, 1, V))
        share += float(q[t]) * torch.bincount(r.tokens[:, 0].cpu(), minlength=V).double() / B
    assert float((share - p.double()).abs().max()) < (V + 2) / n / 2


def test_other_stream_and_graph(gpu: torch.device) -> None:
    c = {k: (None if v is None else v.to(gpu)) for k, v in make(5, 4, 9000, "bf16", True, 13).items()}
    call = (lambda: ops.verify_drafts(c["tokens"], c["target"], c["u"], draft_probs=c["draft"],
                                      draft_lens=c["lens"]))
    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got.tokens, want.tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in range(3):
        c["u"].copy_(torch.rand(c["u"].shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.accepted, want.accepted)
