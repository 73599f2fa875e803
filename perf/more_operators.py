"""A decoder's drafted step, and the rotary prologue in 16 bits, as measurable cases.

``listed()`` holds the calls with which a decoder takes several tokens at once
into a paged cache: its queries and keys normed and rotated, attention of the
new tokens over the cache within a window, and the verdict on drafted tokens;
a video transformer makes the first of them on its whole latent grid.
``draw(rng)`` gives more cases of the same ranges.  For one case,
``prepare(case, seed)`` makes what the program holds before the call,
``run(state)`` is one call, ``work(case)`` the bytes and operations it cannot
do without, ``exact(case, seed)`` its result in 64 bits.  ``run`` computes
plain torch operations, or, where ``own`` is true, calls the package's public
entry point.

Kinds of case:

* ``rope``: ``ops.qk_norm_rope``, each head's RMSNorm of queries and keys and
  the rotation by their positions, along one axis or along time, height and
  width.
* ``attend``: ``ops.paged_attention``, the last tokens of each sequence (one,
  a few drafted ones, a prompt) over a paged cache, each seeing the keys of a
  window before it and a few first ones.
* ``verify``: ``ops.verify_drafts``, drafted tokens accepted or rejected by
  given random numbers, and one more token drawn.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


def listed() -> list[dict]:
    return [
        # one decoder's step of 16 sequences: launches and host work
        {"name": "rope_token", "kind": "rope", "B": 16, "H": 32, "Hkv": 8, "S": 1, "D": 128,
         "rot": 128, "sections": "", "norm": True, "layout": "half", "dtype": "bf16",
         "far": 131072},
        # prompts of 4 sequences, half of each head rotated, without a norm
        {"name": "rope_prompts", "kind": "rope", "B": 4, "H": 32, "Hkv": 8, "S": 2047, "D": 64,
         "rot": 32, "sections": "", "norm": False, "layout": "half", "dtype": "fp16", "far": 8192},
        # queries and keys of the 21 x 45 x 80 latent grid, rotated along its three axes
        {"name": "rope_video", "kind": "rope", "B": 1, "H": 40, "Hkv": 40, "S": 75600, "D": 128,
         "rot": 128, "sections": "22,21,21", "norm": True, "layout": "interleaved",
         "dtype": "bf16", "far": 1024},
        # the next token of a batch within a window, two pages of sinks kept
        {"name": "attend_window", "kind": "attend", "B": 32, "H": 32, "Hkv": 8, "D": 128, "S": 1,
         "slo": 1, "L": 16384, "lo": 100, "window": 1024, "sinks": 32, "page": 16,
         "dtype": "bf16", "cache": "bf16"},
        # drafts of 1 to 6 tokens of 16 sequences over e4m3fn caches of ragged lengths
        {"name": "attend_drafts", "kind": "attend", "B": 16, "H": 32, "Hkv": 8, "D": 128, "S": 6,
         "slo": 1, "L": 8000, "lo": 640, "window": 0, "sinks": 0, "page": 16, "dtype": "bf16",
         "cache": "e4m3"},
        # eight drafted tokens of one sequence after a very long context
        {"name": "attend_drafts_long", "kind": "attend", "B": 1, "H": 40, "Hkv": 8, "D": 128,
         "S": 8, "slo": 8, "L": 131071, "lo": 131071, "window": 0, "sinks": 0, "page": 64,
         "dtype": "fp16", "cache": "fp16"},
        # a chunk of two prompts after what came before, within a window, four sinks
        {"name": "attend_chunk", "kind": "attend", "B": 2, "H": 32, "Hkv": 8, "D": 128, "S": 4000,
         "slo": 1800, "L": 32768, "lo": 12345, "window": 4096, "sinks": 4, "page": 32,
         "dtype": "fp16", "cache": "fp16"},
        # the largest: a whole prompt, every key before a token seen
        {"name": "attend_prompt", "kind": "attend", "B": 1, "H": 32, "Hkv": 8, "D": 128,
         "S": 16384, "slo": 16384, "L": 16384, "lo": 16384, "window": 0, "sinks": 0, "page": 16,
         "dtype": "bf16", "cache": "bf16"},
        # four drafted tokens of one sequence
        {"name": "verify_one", "kind": "verify", "B": 1, "N": 4, "V": 32000, "drafts": True,
         "dtype": "fp32"},
        # drafts looked up in the prompt, without probabilities of their own
        {"name": "verify_lookup", "kind": "verify", "B": 16, "N": 10, "V": 32064, "drafts": False,
         "dtype": "fp32"},
        # a full batch under a large vocabulary
        {"name": "verify_batch", "kind": "verify", "B": 256, "N": 5, "V": 128256, "drafts": True,
         "dtype": "fp32"},
    ]


def _between(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("rope", "attend", "attend", "attend", "attend", "verify"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    D = rng.choice((64, 128, 128, 128, 256))
    Hkv = rng.choice((1, 2, 4, 8, 8, 32))
    G = rng.choice((1, 2, 4, 4, 5, 8))
    if kind == "verify":
        N = _between(rng, 1, 16)
        V = _between(rng, 1000, 160000)
        return {"kind": kind, "B": _between(rng, 1, min(256, 400_000_000 // (V * (2 * N + 1)))),
                "N": N, "V": V, "drafts": rng.random() < 0.7,
                "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16"))}
    if kind == "rope":
        S = rng.choice((1, _between(rng, 2, 75600)))
        H = Hkv * G if Hkv * G <= 64 else Hkv
        B = _between(rng, 1, max(1, min(64, 380_000_000 // (S * H * D))))
        rot = rng.choice((D, D, D // 2))
        third = rot // 6
        return {"kind": kind, "B": B, "H": H, "Hkv": Hkv, "S": S, "D": D, "rot": rot,
                "sections": rng.choice(("", f"{rot // 2 - 2 * third},{third},{third}")),
                "norm": rng.random() < 0.7, "layout": rng.choice(("half", "interleaved")),
                "dtype": dtype, "far": _between(rng, 64, 1 << 20)}
    H = Hkv * G if Hkv * G <= 64 else Hkv
    S = rng.choice((1, _between(rng, 2, 16), _between(rng, 17, 8192)))
    L = _between(rng, S, max(S, min(131072, 3_000_000_000_000 // (4 * S * H * D))))
    window = rng.choice((0, _between(rng, 16, 8192)))
    # the caches' room, and the pairs that are looked at
    B = _between(rng, 1, max(1, min(64, 600_000_000 // (L * Hkv * D),
                                    3_000_000_000_000 // (8 * S * L * H * D))))
    return {"kind": kind, "B": B, "H": H, "Hkv": Hkv, "D": D, "S": S, "slo": rng.randint(1, S),
            "L": L, "lo": rng.randint(1, L), "window": window,
            "sinks": rng.choice((0, 1, 4, 64)) if window else 0,
            "page": rng.choice((16, 16, 32, 64, 128)), "dtype": dtype,
            "cache": rng.choice((dtype, dtype, "e4m3"))}


def _steps(B: int, lo: int, hi: int) -> list[int]:
    """Even steps from ``lo`` to ``hi``, both among them."""
    return [hi] if B == 1 else [lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _lens(c: dict) -> list[tuple[int, int]]:
    """(rows in the cache, new tokens among them) of each sequence."""
    return [(n, min(n, s)) for n, s in zip(_steps(c["B"], c["lo"], c["L"]),
                                           _steps(c["B"], c["slo"], c["S"]))]


def _sections(c: dict) -> list[int]:
    return [int(x) for x in c["sections"].split(",")] if c["sections"] else [c["rot"] // 2]


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "verify":
        # one row of each is drawn from; a test takes two of its values
        rows = 2 if c["drafts"] else 1
        return {"bytes": c["B"] * (rows * c["V"] * SIZES[c["dtype"]] + c["N"] * 20 + 24),
                "flops": 3 * c["B"] * c["V"]}
    if c["kind"] == "rope":
        rows = c["B"] * c["S"] * (c["H"] + c["Hkv"])
        axes = len(_sections(c))
        return {"bytes": rows * 4 * c["D"] + 4 * axes * c["B"] * c["S"] + 4 * c["rot"],
                "flops": rows * (3 * c["rot"] + (4 * c["D"] if c["norm"] else 0))}
    row = 2 * (c["D"] * SIZES[c["cache"]] + (4 if c["cache"] == "e4m3" else 0))
    pairs = keys = 0
    for n, s in _lens(c):
        w = c["window"] or n
        first = n - s                                   # the first new token's position
        lo = max(0, first - w + 1)
        keys += n - lo + min(c["sinks"], lo)
        for p in ((first, n - 1) if s > 1 else (first,)):   # linear between, nearly
            pairs += (min(p + 1, w) + min(c["sinks"], max(0, p + 1 - w))) * (s / 2 if s > 1 else 1)
    io = sum(s for _, s in _lens(c)) * c["H"] * (4 * c["D"] + 4)
    return {"bytes": int(keys * c["Hkv"] * row + io + 4 * keys // c["page"]),
            "flops": int(4 * pairs * c["H"] * c["D"])}


# ------------------------------------------------------------------ inputs

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _fill(g: torch.Generator, shape: tuple[int, ...], dtype: torch.dtype,
          std: float = 1.0) -> torch.Tensor:
    """N(0, std) in ``dtype``, a slice at a time (the whole in fp32 may be large)."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    flat = x.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        y = torch.randn(n, generator=g, device="cuda").mul_(std)
        flat[i:i + n] = (y.clamp_(-448.0, 448.0) if x.element_size() == 1 else y).to(dtype)
    return x


def _prepare_rope(c: dict, g: torch.Generator) -> dict:
    B, S, D, H, Hkv = c["B"], c["S"], c["D"], c["H"], c["Hkv"]
    # a fused projection's output, its queries and keys seen as (B, heads, S, D)
    x = _fill(g, (B, S, (H + 2 * Hkv) * D), DTYPES[c["dtype"]], 1.7)
    q = x[..., :H * D].view(B, S, H, D).permute(0, 2, 1, 3)
    k = x[..., H * D:(H + Hkv) * D].view(B, S, Hkv, D).permute(0, 2, 1, 3)
    sections = _sections(c)
    if len(sections) == 1:      # a sequence's tokens follow a context of their own length
        start = torch.randint(0, max(1, c["far"] - S), (B, 1), generator=g, device="cuda")
        pos = (start + torch.arange(S, device="cuda")).to(torch.int32)
    else:                       # a grid of frames, rows and columns, the batch's own first frame
        w = max(1, min(80, S))
        h = max(1, min(45, S // w))
        i = torch.arange(S, device="cuda")
        t0 = torch.randint(0, c["far"], (B, 1), generator=g, device="cuda")
        pos = torch.stack([t0 + i // (h * w), (i // w % h).expand(B, S),
                           (i % w).expand(B, S)]).to(torch.int32)
    # each axis has its own frequencies, from 1 down to nearly 1 / 10000
    freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in sections])
    weight = [(1.0 + _fill(g, (D,), torch.float32, 0.2)).to(DTYPES[c["dtype"]]) for _ in range(2)]
    return {"case": c, "q": q, "k": k, "pos": pos, "freq": freq.float().cuda(),
            "sections": sections if len(sections) > 1 else None,
            "wq": weight[0] if c["norm"] else None, "wk": weight[1] if c["norm"] else None}


def _prepare_attend(c: dict, g: torch.Generator) -> dict:
    B, page = c["B"], c["page"]
    lens = _lens(c)
    order = torch.randperm(B, generator=g, device="cuda").cpu().tolist()
    lens = [lens[i] for i in order]
    need = [-(-n // page) for n, _ in lens]
    deal = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):       # pages in a random order, -1 behind the last
        table[b, :n] = deal[at:at + n]
        at += n
    shape = (sum(need) + 3, c["Hkv"], page, c["D"])
    st = {"case": c, "table": table.cuda(), "ks": None, "vs": None,
          "lens": torch.tensor([n for n, _ in lens], dtype=torch.int32, device="cuda"),
          "qlens": torch.tensor([s for _, s in lens], dtype=torch.int32, device="cuda"),
          "max": c["L"], "q": _fill(g, (B, c["S"], c["H"], c["D"]), DTYPES[c["dtype"]])
          .permute(0, 2, 1, 3)}
    if c["cache"] == "e4m3":
        st["ks"], st["vs"] = (torch.rand(shape[:3], generator=g, device="cuda") * 0.004 + 0.004
                              for _ in range(2))
        st["k"], st["v"] = (_fill(g, shape, torch.float8_e4m3fn, 130.0) for _ in range(2))
    else:
        st["k"], st["v"] = (_fill(g, shape, DTYPES[c["cache"]]) for _ in range(2))
    return st


def _prepare_verify(c: dict, g: torch.Generator) -> dict:
    B, N, V = c["B"], c["N"], c["V"]
    # a few tokens stand out; the draft model's logits lie near the target's
    target = torch.empty((B, N + 1, V), dtype=DTYPES[c["dtype"]], device="cuda")
    draft = torch.empty((B, N, V), dtype=DTYPES[c["dtype"]], device="cuda") if c["drafts"] else None
    tokens = torch.empty((B, N), dtype=torch.int64, device="cuda")
    rows = max(1, (1 << 26) // ((N + 1) * V))
    for b in range(0, B, rows):
        x = torch.randn((min(rows, B - b), N + 1, V), generator=g, device="cuda").mul_(2.0)
        best = torch.randint(0, V, (*x.shape[:2], 6), generator=g, device="cuda")
        x.scatter_(2, best, 11.0 + 2.0 * torch.randn(best.shape, generator=g, device="cuda"))
        p = torch.softmax(x, dim=2)
        target[b:b + rows] = p.to(target.dtype)
        if draft is None:
            tokens[b:b + rows] = p[:, :N].argmax(dim=2)
            continue
        x = x[:, :N] + 0.5 * torch.randn((x.shape[0], N, V), generator=g, device="cuda")
        p = torch.softmax(x, dim=2)
        draft[b:b + rows] = p.to(draft.dtype)
        tokens[b:b + rows] = torch.multinomial(p.view(-1, V), 1, generator=g).view(-1, N)
    # the number of tokens that were drafted differs between the sequences
    n = torch.randint((N + 1) // 2, N + 1, (B,), generator=g, device="cuda").to(torch.int32)
    return {"case": c, "tokens": tokens, "target": target, "draft": draft, "n": n,
            "u": torch.rand((B, N + 1), generator=g, device="cuda")}


def prepare(case: dict, seed: int) -> dict:
    return {"rope": _prepare_rope, "attend": _prepare_attend,
            "verify": _prepare_verify}[case["kind"]](case, _gen(seed))


# -------------------------------------------------------------- plain forms

def _angles(s: dict) -> torch.Tensor:
    """Each token's rotation of each pair, (B, S, rot / 2), in 64 bits: a far
    position's angle is thousands of turns."""
    pos = s["pos"] if s["sections"] else s["pos"].unsqueeze(0)
    axis = torch.repeat_interleave(torch.arange(pos.shape[0]),
                                   torch.tensor(_sections(s["case"]))).cuda()
    return pos.double()[axis].permute(1, 2, 0) * s["freq"].double()


def _plain_rope(s: dict) -> list:
    c, rot = s["case"], s["case"]["rot"]
    a = _angles(s)
    cos, sin = a.cos().float().unsqueeze(1), a.sin().float().unsqueeze(1)
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.float()
        if c["norm"]:
            y = y * torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + 1e-6) * w.float()
        if c["layout"] == "half":
            a0, a1 = y[..., :rot // 2], y[..., rot // 2:rot]
            parts = [a0 * cos - a1 * sin, a1 * cos + a0 * sin]
        else:
            a0, a1 = y[..., 0:rot:2], y[..., 1:rot:2]
            parts = [torch.stack([a0 * cos - a1 * sin, a1 * cos + a0 * sin], dim=-1).flatten(-2)]
        out.append(torch.cat(parts + [y[..., rot:]], dim=-1).to(x.dtype))
    return out


def _rows(s: dict, name: str, b: int, heads: slice, dtype: torch.dtype) -> torch.Tensor:
    """The rows of the sequence ``b`` in its pages, (heads, slots, D)."""
    t = s["table"][b].clamp(min=0).long()
    x = s[name][:, heads]
    x = x.view(torch.uint8)[t].view(x.dtype) if x.element_size() == 1 else x[t]
    x = x.to(dtype)
    if s[name + "s"] is not None:
        x = x * s[name + "s"][:, heads][t].to(dtype).unsqueeze(-1)
    return x.transpose(0, 1).flatten(1, 2)


def _plain_attend(s: dict) -> list:
    c, q = s["case"], s["q"]
    B, H, S, D = q.shape
    G = H // c["Hkv"]
    out = torch.zeros((B, H, S, D), dtype=q.dtype, device="cuda")
    lse = torch.full((B, H, S), -math.inf, device="cuda")
    L = s["table"].shape[1] * c["page"]
    j = torch.arange(L, device="cuda")
    i = torch.arange(S, device="cuda").unsqueeze(1)
    step = max(1, min(c["Hkv"], (1 << 29) // (G * S * L)))       # kv heads at a time
    for b in range(B):
        p = s["lens"][b] - s["qlens"][b] + i
        seen = (j <= p) & (i < s["qlens"][b])
        if c["window"]:
            seen &= (p - j < c["window"]) | (j < c["sinks"])
        for h in range(0, c["Hkv"], step):
            k = _rows(s, "k", b, slice(h, h + step), torch.float32)
            v = _rows(s, "v", b, slice(h, h + step), torch.float32)
            n = k.shape[0]
            qh = q[b, h * G:(h + n) * G].float().reshape(n, G * S, D)
            x = torch.matmul(qh, k.transpose(1, 2).contiguous()).view(n, G, S, L) / math.sqrt(D)
            x = x.masked_fill_(~seen, -math.inf)
            m = x.amax(dim=-1, keepdim=True).clamp_(min=-3e38)
            e = torch.exp(x.sub_(m))
            l = e.sum(dim=-1, keepdim=True)
            o = torch.matmul(e.view(n, G * S, L), v).view(n, G, S, D)
            out[b, h * G:(h + n) * G] = torch.where(l > 0, o / l, 0.0).reshape(-1, S, D).to(q.dtype)
            lse[b, h * G:(h + n) * G] = (m + torch.log(l)).reshape(-1, S)
    return [out, lse]


def _plain_verify(s: dict) -> list:
    """In 64 bits: a draw lies next to the border of two tokens now and then."""
    c, tokens, u = s["case"], s["tokens"], s["u"]
    B, N, V = c["B"], c["N"], c["V"]
    b = torch.arange(B, device="cuda")
    p = s["target"][:, :N].gather(2, tokens.unsqueeze(2)).squeeze(2).double()
    q = torch.ones_like(p)
    if s["draft"] is not None:
        q = s["draft"].gather(2, tokens.unsqueeze(2)).squeeze(2).double()
    at = torch.arange(N, device="cuda")
    ok = (u[:, :N].double() * q < p) & (at < s["n"].unsqueeze(1))
    n = ok.to(torch.int64).cumprod(dim=1).sum(dim=1)
    w = s["target"][b, n].double()
    last = (n - 1 + (n < N)).clamp(min=0)              # the draft at n, where there is one
    left = w.clone()
    if s["draft"] is not None:
        left -= s["draft"][b, last].double()
    else:
        left[b, tokens[b, last]] -= 1.0
    left.clamp_(min=0.0)
    rejected = (n < s["n"]) & (left.sum(dim=1) > 0)
    w = torch.where(rejected.unsqueeze(1), left, w)
    total = w.cumsum(dim=1)
    drawn = (total > u[:, N:].double() * total[:, -1:]).to(torch.int8).argmax(dim=1)
    out = torch.where(at < n.unsqueeze(1), tokens, -1)
    out = torch.cat([out, torch.full((B, 1), -1, dtype=torch.int64, device="cuda")], dim=1)
    out[b, n] = drawn
    return [out, n.to(torch.int32)]


def run(state: dict):
    s, c = state, state["case"]
    if own:
        from repercep_runtime_amd import ops

        if c["kind"] == "rope":
            return list(ops.qk_norm_rope(s["q"], s["k"], s["pos"], s["freq"],
                                         sections=s["sections"], norm_q_weight=s["wq"],
                                         norm_k_weight=s["wk"], eps=1e-6 if c["norm"] else None,
                                         rope_layout=c["layout"]))
        if c["kind"] == "attend":
            return list(ops.paged_attention(
                s["q"], s["k"], s["v"], s["table"], s["lens"], s["qlens"],
                window=c["window"] or None, sinks=c["sinks"], k_scale=s["ks"], v_scale=s["vs"],
                max_seq_len=s["max"], return_lse=True))
        r = ops.verify_drafts(s["tokens"], s["target"], s["u"], draft_probs=s["draft"],
                              draft_lens=s["n"])
        return [r.tokens, r.accepted]
    return {"rope": _plain_rope, "attend": _plain_attend, "verify": _plain_verify}[c["kind"]](s)


# ------------------------------------------------------------------- 64 bits

def _exact_rope(s: dict) -> list:
    """Pairs as complex numbers, turned by a unit one."""
    c, rot = s["case"], s["case"]["rot"]
    pos = s["pos"] if s["pos"].dim() == 3 else s["pos"][None]
    turn, at = [], 0
    for axis, n in enumerate(_sections(c)):
        turn.append(torch.einsum("bs,f->bsf", pos[axis].double(),
                                 s["freq"][at:at + n].double()))
        at += n
    turn = torch.cat(turn, dim=2)
    turn = torch.polar(torch.ones_like(turn), turn)[:, None]
    outs = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        res = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        for h in range(x.shape[1]):                     # a head at a time: 64 bits take room
            y = x[:, h:h + 1].double()
            if w is not None:
                y = y / (y.square().sum(dim=-1, keepdim=True) / c["D"] + 1e-6).sqrt() * w.double()
            z = y[..., :rot]
            z = z.unflatten(-1, (2, -1)).transpose(-1, -2) if c["layout"] == "half" \
                else z.unflatten(-1, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = z.transpose(-1, -2) if c["layout"] == "half" else z
            res[:, h:h + 1, :, :rot] = z.flatten(-2)
            res[:, h:h + 1, :, rot:] = y[..., rot:]
        outs.append(res)
    return outs


def _exact_attend(s: dict) -> list:
    c, q = s["case"], s["q"]
    B, H, S, D = q.shape
    G = H // c["Hkv"]
    out = torch.zeros((B, H, S, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64, device="cuda")
    lens, qlens = s["lens"].tolist(), s["qlens"].tolist()
    for b in range(B):
        for h in range(c["Hkv"]):
            k = _rows(s, "k", b, slice(h, h + 1), torch.float64)[0, :lens[b]]
            v = _rows(s, "v", b, slice(h, h + 1), torch.float64)[0, :lens[b]]
            kt = k.t().contiguous()
            for i0 in range(0, qlens[b], 2048):         # some tokens at a time
                i = torch.arange(i0, min(i0 + 2048, qlens[b]), device="cuda")
                p = (lens[b] - qlens[b] + i)[:, None]
                j = torch.arange(lens[b], device="cuda")[None]
                hide = j > p
                if c["window"]:
                    hide |= (j <= p - c["window"]) & (j >= c["sinks"])
                rows = q[b, h * G:(h + 1) * G, i].double()                 # (G, tokens, D)
                x = torch.stack([torch.mm(r, kt) for r in rows]) * D ** -0.5
                x = torch.where(hide, -math.inf, x)
                z = torch.logsumexp(x, dim=-1)
                e = torch.exp(x - z[..., None])
                out[b, h * G:(h + 1) * G, i] = torch.stack([torch.mm(r, v) for r in e])
                lse[b, h * G:(h + 1) * G, i] = z
    return [out, lse]


def _exact_verify(s: dict) -> list:
    """A sequence and a test at a time."""
    tokens, u, n = s["tokens"].tolist(), s["u"].double().tolist(), s["n"].tolist()
    N = s["case"]["N"]
    out, counts = torch.full((len(n), N + 1), -1, dtype=torch.int64), []
    for b, drafted in enumerate(n):
        got, weights = 0, None
        ids = s["tokens"][b].unsqueeze(1)
        ps = s["target"][b, :N].gather(1, ids).squeeze(1).tolist()
        qs = [1.0] * N if s["draft"] is None else s["draft"][b].gather(1, ids).squeeze(1).tolist()
        while got < drafted and u[b][got] * qs[got] < ps[got]:
            out[b, got] = tokens[b][got]
            got += 1
        weights = s["target"][b, got].double()
        if got < drafted:
            rest = weights - s["draft"][b, got].double() if s["draft"] is not None else weights.clone()
            if s["draft"] is None:
                rest[tokens[b][got]] -= 1.0
            rest = torch.where(rest > 0, rest, 0.0)
            weights = rest if bool((rest > 0).any()) else weights
        total = torch.cumsum(weights, dim=0)
        out[b, got] = int(torch.searchsorted(total, u[b][N] * total[-1:], right=True).item())
        counts.append(got)
    return [out, torch.tensor(counts, dtype=torch.int32)]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attend": _exact_attend,
            "verify": _exact_verify}[case["kind"]](s)
