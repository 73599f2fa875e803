"""A decoder's drafted steps as a program runs them: a prompt, then drafts that
are verified, the cache cut back to the accepted tokens."""

from __future__ import annotations

import math

import pytest
import torch

import _drafts
import _paged
from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu


class Decoder:
    """One attention layer between random projections, on a paged cache; the
    same in 64 bits beside it, from the rows that the cache holds."""

    def __init__(self, kind: str, B: int, seed: int, dev: torch.device) -> None:
        self.H, self.Hkv, self.D, self.V, self.page, self.dev = 4, 2, 64, 50, 16, dev
        self.window, self.sinks, self.B, self.kind = 40, 4, B, kind
        g = torch.Generator().manual_seed(seed)
        E = 96
        r = (lambda *s: torch.randn(s, generator=g))
        self.embed = r(self.V, E)
        self.proj = r(E, (self.H + 2 * self.Hkv) * self.D) / math.sqrt(E)
        self.head = r(self.H * self.D, self.V) * 0.2
        self.wq, self.wk = (1 + 0.2 * r(self.D) for _ in range(2))
        self.freq = 10000.0 ** (-torch.arange(self.D // 2, dtype=torch.float64) / (self.D // 2))
        n = 12
        dt = _paged.CACHE_DTYPES[kind]
        shape = (B * n, self.Hkv, self.page, self.D)
        self.k, self.v = (torch.zeros(shape, dtype=dt, device=dev) for _ in range(2))
        self.ks = self.vs = None
        if kind == "e4m3":
            self.ks, self.vs = (torch.zeros(shape[:3], device=dev) for _ in range(2))
        self.table = torch.randperm(B * n, generator=g).view(B, n).to(torch.int32).to(dev)
        self.lens = torch.zeros(B, dtype=torch.int32, device=dev)

    def step(self, tokens: torch.Tensor, m: torch.Tensor) -> torch.Tensor:
        """Logits of ``tokens`` (B, S), of which sequence b has m[b]; checks the attention."""
        B, S = tokens.shape
        x = (self.embed[tokens.cpu()] @ self.proj).to(torch.bfloat16).to(self.dev)
        H, Hkv, D = self.H, self.Hkv, self.D
        q, k, v = (x[..., a * D:b * D].view(B, S, b - a, D).permute(0, 2, 1, 3)
                   for a, b in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv)))
        pos = (self.lens[:, None] + torch.arange(S, device=self.dev)).to(torch.int32)
        bf = (lambda w: w.to(torch.bfloat16).to(self.dev))
        qr, kr = ops.qk_norm_rope(q, k, pos, self.freq.to(self.dev), norm_q_weight=bf(self.wq),
                                  norm_k_weight=bf(self.wk))
        cache = dict(k_cache=self.k, v_cache=self.v, block_table=self.table, k_scale=self.ks,
                     v_scale=self.vs)
        ops.paged_kv_append(kr, v, start=self.lens, lengths=m, **cache)
        self.lens += m
        out, lse = ops.paged_attention(qr, seq_lens=self.lens, q_lens=m, window=self.window,
                                       sinks=self.sinks, return_lse=True, **cache)
        for a, w, y in ((q, self.wq, qr), (k, self.wk, kr)):
            want, err = _drafts.norm_rope(a.cpu(), w.to(torch.bfloat16), 1e-6, pos.cpu(), self.freq,
                                          None, "half")
            assert bool(((y.cpu().double() - want).abs()
                         <= _drafts.rounded(want, err, torch.bfloat16)).all())
        rows = []
        for b, n in enumerate(self.lens.tolist()):
            j = torch.arange(n)
            pg = self.table[b].cpu()[j // self.page].long()
            got = []
            for t, s in ((self.k, self.ks), (self.v, self.vs)):
                r = t.cpu().double()[pg, :, j % self.page]
                got.append((r if s is None else r * s.cpu().double()[pg, :, j % self.page, None])
                           .transpose(0, 1))
            rows.append(tuple(got))
        want, wlse, eo, el = _drafts.window_attention(
            qr.cpu(), rows, self.lens.tolist(), m.tolist(), self.window, self.sinks,
            1 / math.sqrt(D), _drafts.HALF[torch.bfloat16])
        assert bool(((out.cpu().double() - want).abs()
                     <= _drafts.rounded(want, eo, torch.bfloat16)).all())
        return out.permute(0, 2, 1, 3).reshape(B, S, H * D).float() @ self.head.to(self.dev)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_drafted_steps(kind: str, gpu: torch.device) -> None:
    """A ragged prompt, then four verified drafts at a time; the accepted tokens
    stay, the cache's length is cut back, and the definition gives the same."""
    B, N, V = 3, 4, 50
    d = Decoder(kind, B, 3, gpu)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, V, (B, 70), generator=g)
    m = torch.tensor([70, 33, 1], dtype=torch.int32, device=gpu)
    logits = d.step(prompt, m)
    last = torch.stack([logits[b, int(m[b]) - 1].argmax() for b in range(B)])
    for _ in range(4):
        q = torch.softmax(2 * torch.randn((B, N, V), generator=g), -1).to(gpu)
        drafts = torch.multinomial(q.view(B * N, V).cpu(), 1, generator=g).view(B, N).to(gpu)
        n = torch.randint(1, N + 1, (B,), generator=g).to(torch.int32).to(gpu)
        before = d.lens.clone()
        p = torch.softmax(d.step(torch.cat([last[:, None], drafts], 1), n + 1), -1)
        u = torch.rand((B, N + 1), generator=g).to(gpu)
        r = ops.verify_drafts(drafts, p, u, draft_probs=q, draft_lens=n)
        want, counts = _drafts.verify(drafts.tolist(), p.cpu(), q.cpu(), u.cpu(), n.tolist())
        assert r.tokens.tolist() == want and r.accepted.tolist() == counts
        d.lens = before + 1 + r.accepted
        last = r.tokens.gather(1, r.accepted.long()[:, None])[:, 0]
        scored = ops.token_logprobs(p.log().gather(1, r.accepted.long()[:, None, None]
                                                   .expand(B, 1, V))[:, 0], last)
        assert bool((scored.logprobs < 0).all())
