"""Drafted tokens' verdict on the GPU over vocabularies on both sides of 32768
tokens, up to which one launch takes a row; longer ones are taken in parts of 4096,
128 parts at a time."""

from __future__ import annotations

import pytest
import torch

import test_gpu_drafts as drafts
from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu
ONE, BATCH = 32768, 128 * 4096


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("B,N,V", [(3, 3, 4103), (2, 2, ONE), (2, 2, ONE + 1), (3, 4, 36871),
                                   (2, 0, 40960), (1, 70, 33000), (2, 1, BATCH), (2, 1, BATCH + 77)])
def test_matches_definition(B: int, N: int, V: int, with_draft: bool, dtype: str,
                            gpu: torch.device) -> None:
    drafts.check(drafts.make(B, N, V, dtype, with_draft, seed=B + V), gpu)


@pytest.mark.parametrize("V", [4103, 36871])
def test_strided_and_unaligned_rows(V: int, gpu: torch.device) -> None:
    for dtype in drafts.DTYPES:
        c = drafts.make(3, 4, V, dtype, True, 5)
        dt = drafts.DTYPES[dtype]
        p = torch.full((3, 2, 5, V + 7), float("nan"), dtype=dt, device=gpu)
        q = torch.full((4, 3, V + 4), float("nan"), dtype=dt, device=gpu)
        p[:, 1, :, 3:V + 3] = c["target"].to(gpu)
        q[:, :, 1:V + 1] = c["draft"].to(gpu).transpose(0, 1)
        drafts.check(c, gpu, target=p[:, 1, :, 3:V + 3], draft=q[:, :, 1:V + 1].transpose(0, 1))
        row = c["target"][:1, :1].to(gpu).contiguous()
        c["target"] = c["target"][:1, :1].expand(3, 5, V)
        drafts.check(c, gpu, target=row.expand(3, 5, V))


@pytest.mark.parametrize("V", [6, 4200, ONE, ONE + 1, 36871, BATCH + 4097])
def test_borders(V: int, gpu: torch.device) -> None:
    """Weights that add up without rounding, at the row's ends and on both sides of
    the borders of parts: u q = p is no acceptance; u = 0 draws the first token of any
    weight; u >= 1 draws the last one; a draft outside the vocabulary is rejected."""
    spots = sorted({1, 3, 4, V - 1, *(t for edge in (4096, ONE, BATCH) for t in (edge - 1, edge)
                                      if t < V)})
    p, q = torch.zeros(V), torch.zeros(V)
    p[spots] = 1.0 / 64
    p[1], q[1], q[2] = 0.25, 0.5, 0.5
    total = 0.25 + (len(spots) - 1) / 64                     # of p; p - q leaves all but token 1
    cases = [([1], [0.5, 0.0]), ([1], [0.499, 0.5]), ([2], [0.0, 0.3]), ([0], [0.0, 0.9]),
             ([-1], [0.0, 0.0]), ([V], [0.0, 1.0]), ([1 << 40], [0.0, 0.25]), ([1], [0.0, 1.0])]
    for i in range(len(spots)):                              # the goal within each token's weight
        cases += [([1], [0.0, (0.25 + (i - 0.5) / 64) / total]), ([2], [0.0, (i + 0.5) / (len(spots) - 1)])]
    B = len(cases)
    c = {"tokens": torch.tensor([t for t, _ in cases]), "u": torch.tensor([u for _, u in cases]),
         "target": p.expand(B, 2, V), "draft": q.expand(B, 1, V),
         "lens": torch.ones(B, dtype=torch.int32)}
    place = dict(target=p.to(gpu).expand(B, 2, V))
    r = drafts.check(c, gpu, draft=q.to(gpu).expand(B, 1, V), **place)
    assert r.accepted.tolist()[:8] == [0, 1, 0, 0, 0, 0, 0, 1]
    assert set(spots) <= set(r.tokens.flatten().tolist())
    drafts.check({**c, "draft": None}, gpu, **place)


@pytest.mark.parametrize("V", [4200, 36871, BATCH + 5000])
def test_nothing_left(V: int, gpu: torch.device) -> None:
    """p = q with a rejected draft draws from p; a p of zeros and NaNs gives -1;
    infinities leave the last token of any weight."""
    p = torch.zeros((5, 2, V))
    p[0, :, V - 50] = 0.5
    p[0, :, 17] = 0.5
    p[2] = float("nan")
    p[2, 0, V - 1] = 1e-30
    p[3, :, [5, V - 9]] = float("inf")
    p[4] = -1.0
    c = {"tokens": torch.full((5, 1), 3), "u": torch.tensor([[0.0, 0.6]] * 5), "target": p,
         "draft": p[:, :1].clone(), "lens": torch.ones(5, dtype=torch.int32)}
    c["draft"][2:] = 0.0
    r = drafts.check({**c, "target": p[:3], "tokens": c["tokens"][:3], "u": c["u"][:3],
                      "draft": c["draft"][:3], "lens": c["lens"][:3]}, gpu)
    assert r.tokens[:, 0].tolist() == [V - 50, -1, V - 1]
    f = {k: v.to(gpu) for k, v in c.items()}
    r = ops.verify_drafts(f["tokens"], f["target"], f["u"], draft_probs=f["draft"],
                          draft_lens=f["lens"])
    assert r.tokens[:, 0].tolist() == [V - 50, -1, V - 1, V - 9, -1]
    assert r.accepted.tolist() == [0] * 5


@pytest.mark.parametrize("V", [64, 36871])
def test_lens_out_of_range(V: int, gpu: torch.device) -> None:
    c = drafts.make(4, 5, V, "fp32", True, 11)
    c["lens"] = torch.tensor([-7, 99, 0, 2 ** 31 - 1], dtype=torch.int32)
    drafts.check(c, gpu)
    c["lens"] = None
    drafts.check(c, gpu)


@pytest.mark.parametrize("V", [4103, 36871, BATCH + 77])
def test_other_stream_and_graph(V: int, gpu: torch.device) -> None:
    c = {k: (None if v is None else v.to(gpu))
         for k, v in drafts.make(3, 3, V, "bf16", True, 13).items()}
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
    for seed in range(4):
        c["u"].copy_(torch.rand(c["u"].shape, generator=torch.Generator().manual_seed(seed)))
        c["lens"].fill_(seed)
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.accepted, want.accepted)
