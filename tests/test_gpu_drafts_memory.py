"""A drafted step's operators on the GPU: outputs that share memory with another
array of the call are refused, those that lie between its rows are not."""

from __future__ import annotations

import pytest
import torch

import test_gpu_rope as rope

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
