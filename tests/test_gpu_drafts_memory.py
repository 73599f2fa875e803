"""A drafted step's operators on the GPU: outputs that share memory with another
array of the call are refused, those that lie between its rows are not."""

from __future__ import annotations

import pytest
import torch

import _paged
import _wide
import test_gpu_rope as rope
from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu


def test_rotation(gpu: torch.device) -> None:
    """Slices of one projection, in place and as outputs."""
    B, H, Hkv, S, D = 2, 4, 2, 9, 64
    c = rope.make(B, H, Hkv, S, D, 32, "bf16")
    x = torch.zeros((B, S, (H + Hkv) * D), dtype=torch.bfloat16, device=gpu)
    q = x[..., :H * D].view(B, S, H, D).permute(0, 2, 1, 3)
    k = x[..., H * D:].view(B, S, Hkv, D).permute(0, 2, 1, 3)
    late = x.view(B, S, H + Hkv, D).permute(0, 2, 1, 3)[:, 2:]      # q's last heads, then k's
    for kw in (dict(out_q=late), dict(out_k=q[:, 1:3]), dict(out_q=q, out_k=q[:, 2:]),
               dict(out_k=late[:, 1:3])):
        with pytest.raises(RuntimeError, match="shares memory"):
            rope.call(c, gpu, "half", 1e-6, q=q, k=k, **kw)
    y = torch.empty((B, S, H + Hkv, D), dtype=torch.bfloat16, device=gpu).permute(0, 2, 1, 3)
    for kw in (dict(out_q=y[:, Hkv:], out_k=y[:, :Hkv]), dict(out_q=q, out_k=k)):
        q.copy_(c["q"])
        k.copy_(c["k"])
        rope.check(c, rope.call(c, gpu, "half", 1e-6, q=q, k=k, **kw), "half", 1e-6)


@pytest.mark.parametrize("S,places", [(1, 64), (3, 64), (3, 4096), (90, 64), (90, 2048), (90, 150000)])
def test_attention(S: int, places: int, gpu: torch.device) -> None:
    """The queries' own place, in one part and in several; slices of a projection."""
    B, H, Hkv, D = 2, 4, 2, 64
    c = _wide.widen(_paged.Cache([190, 90], Hkv, D, 16, "bf16", seed=3), places)
    x = torch.zeros((B, S, (H + Hkv) * D), dtype=torch.bfloat16, device=gpu)
    heads = x.view(B, S, H + Hkv, D).permute(0, 2, 1, 3)
    q = _wide.queries(B, H, S, D, "bf16")
    heads[:, :H].copy_(q)
    for out in (heads[:, 1:1 + H], heads[:, 2:]):
        with pytest.raises(RuntimeError, match="shares memory"):
            _wide.call(c, q, [190, 90], None, gpu, qview=heads[:, :H], out=out)
    _wide.check(c, q, [190, 90], [S, 1], gpu, 70, 3, qview=heads[:, :H], out=heads[:, :H])
    assert bool((heads[:, H:] == 0).all())
    # between the rows of another tensor
    y = torch.zeros((B, S, 2 * H, D), dtype=torch.bfloat16, device=gpu).permute(0, 2, 1, 3)
    y[:, ::2].copy_(q)
    _wide.check(c, q, [190, 90], None, gpu, qview=y[:, ::2], out=y[:, 1::2])
    assert torch.equal(y[:, ::2].cpu(), q)


def test_attention_into_the_cache(gpu: torch.device) -> None:
    c = _paged.Cache([20], 4, 64, 16, "bf16")
    f = c.to(gpu)
    q = torch.zeros((1, 4, 16, 64), dtype=torch.bfloat16, device=gpu)
    lens = torch.tensor([20], dtype=torch.int32, device=gpu)
    for name in ("k_cache", "v_cache"):
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.paged_attention(q, seq_lens=lens, out=f[name][1:2], **f)
