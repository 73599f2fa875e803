"""A decoder's step on a paged key-value cache as measurable cases.

``listed()`` holds the calls that a token-VLA decoder, or any decoder served
from this package, makes for each new token, from one robot's single step to
a full batch over long contexts; ``draw(rng)`` gives more cases of the same
ranges.  For one case, ``prepare(case, seed)`` makes what the program holds
before the call, ``run(state)`` is one call, ``work(case)`` the bytes and
operations it cannot do without, ``exact(case, seed)`` its result in 64 bits.
``run`` computes plain torch operations, or, where ``own`` is true, calls the
package's public entry point.

Kinds of case:

* ``append``: ``ops.paged_kv_append``, new keys and values written into the
  pages of a cache, in 16 bits or as e4m3fn codes with one scale per row.
* ``decode``: ``ops.paged_attention_decode``, one new token's attention over
  the pages, optionally adding each key's attention weight to a running total.
* ``evict``: ``ops.paged_kv_evict``, a cache cut to a budget of rows by those
  totals.
* ``logprob``: ``ops.token_logprobs``, chosen tokens' log probabilities with
  the entropy and the best alternatives.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
FP8_TARGET = 425.6        # 0.95 * 448, what a row's largest element maps to


def listed() -> list[dict]:
    return [
        # 16 candidates' next token into an e4m3fn cache: launches and host work
        {"name": "append_token", "kind": "append", "B": 16, "Hkv": 32, "D": 128, "S": 1,
         "lo": 1, "ctx": 640, "page": 16, "dtype": "bf16", "cache": "e4m3"},
        # the prompts of a batch, ragged, quantized into the cache's pages
        {"name": "append_prompts", "kind": "append", "B": 16, "Hkv": 8, "D": 128, "S": 4000,
         "lo": 37, "ctx": 0, "page": 32, "dtype": "bf16", "cache": "e4m3"},
        # one sequence's next token after 512 prompt tokens and its own 128
        {"name": "decode_one", "kind": "decode", "B": 1, "H": 32, "Hkv": 32, "D": 128, "S": 640,
         "lo": 640, "shared": 0, "page": 16, "dtype": "bf16", "cache": "bf16", "weights": False},
        # 16 candidates that share the pages of a prefix of 512
        {"name": "decode_candidates", "kind": "decode", "B": 16, "H": 32, "Hkv": 32, "D": 128,
         "S": 640, "lo": 520, "shared": 512, "page": 16, "dtype": "bf16", "cache": "bf16",
         "weights": False},
        # a batch of mixed lengths with grouped heads, its keys' weights totalled for eviction
        {"name": "decode_weights", "kind": "decode", "B": 8, "H": 32, "Hkv": 8, "D": 128,
         "S": 4100, "lo": 1, "shared": 0, "page": 16, "dtype": "fp16", "cache": "fp16",
         "weights": True},
        # one very long context, few heads: the work has to be split over the keys
        {"name": "decode_long", "kind": "decode", "B": 1, "H": 40, "Hkv": 8, "D": 128,
         "S": 131071, "lo": 131071, "shared": 0, "page": 64, "dtype": "bf16", "cache": "e4m3",
         "weights": False},
        # the largest: a full batch over long caches
        {"name": "decode_batch", "kind": "decode", "B": 64, "H": 32, "Hkv": 8, "D": 128,
         "S": 16384, "lo": 2048, "shared": 0, "page": 16, "dtype": "bf16", "cache": "bf16",
         "weights": False},
        # one sequence's cache cut back after a few hundred new tokens
        {"name": "evict_one", "kind": "evict", "B": 1, "Hkv": 8, "D": 128, "S": 1100, "lo": 1100,
         "budget": 768, "recent": 128, "page": 16, "cache": "bf16"},
        # a batch of e4m3fn caches halved
        {"name": "evict_batch", "kind": "evict", "B": 32, "Hkv": 8, "D": 128, "S": 8192,
         "lo": 1000, "budget": 2048, "recent": 512, "page": 16, "cache": "e4m3"},
        # one sequence's next token chosen from its logits
        {"name": "logprob_one", "kind": "logprob", "N": 1, "V": 32000, "top": 20,
         "dtype": "bf16"},
        # 16 candidates x 8 tokens scored, the logits left in 32 bits
        {"name": "logprob_candidates", "kind": "logprob", "N": 128, "V": 32064, "top": 5,
         "dtype": "fp32"},
        # the answers of a batch scored under a large vocabulary
        {"name": "logprob_batch", "kind": "logprob", "N": 4096, "V": 128256, "top": 20,
         "dtype": "bf16"},
    ]


def _between(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("append", "decode", "decode", "decode", "evict", "logprob"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    cache = rng.choice((dtype, "e4m3"))
    page = rng.choice((16, 16, 32, 64, 128))
    D = rng.choice((64, 128, 128, 128, 256))
    Hkv = rng.choice((1, 2, 4, 8, 8, 32))
    if kind == "logprob":
        V = _between(rng, 1000, 160000)
        return {"kind": kind, "N": _between(rng, 1, min(4096, 500_000_000 // V)), "V": V,
                "top": rng.choice((0, 1, 5, 20, 32)), "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    if kind == "append":
        S = rng.choice((1, _between(rng, 2, 4000)))
        B = _between(rng, 1, max(1, min(64, 60_000_000 // (S * Hkv * D))))
        return {"kind": kind, "B": B, "Hkv": Hkv, "D": D, "S": S, "lo": rng.randint(1, S),
                "ctx": rng.choice((0, rng.randint(1, 700))), "page": page, "dtype": dtype,
                "cache": cache}
    S = _between(rng, 1 if kind == "decode" else 300, 131071 if kind == "decode" else 16384)
    B = _between(rng, 1, max(1, min(64, 600_000_000 // (S * Hkv * D))))
    lo = rng.randint(1, S)
    if kind == "evict":
        budget = _between(rng, 64, S)
        return {"kind": kind, "B": B, "Hkv": Hkv, "D": D, "S": S, "lo": lo, "budget": budget,
                "recent": rng.randint(0, budget), "page": page, "cache": cache}
    G = rng.choice((1, 2, 4, 5, 8, 16))
    weights = rng.random() < 0.3
    shared = 0 if weights or rng.random() < 0.7 else lo // page * page
    return {"kind": kind, "B": B, "H": Hkv * G, "Hkv": Hkv, "D": D, "S": S, "lo": lo,
            "shared": shared, "page": page, "dtype": dtype, "cache": cache, "weights": weights}


def _lens(c: dict) -> list[int]:
    """The lengths of a batch: even steps from ``lo`` to ``S``, both among them."""
    B, lo, hi = c["B"], c["lo"], c["S"]
    return [hi] if B == 1 else [lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _row_bytes(c: dict) -> int:
    """A key's and its value's bytes in the cache, scales included."""
    return 2 * (c["D"] * SIZES[c["cache"]] + (4 if c["cache"] == "e4m3" else 0))


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "logprob":
        N, V = c["N"], c["V"]
        return {"bytes": N * V * SIZES[c["dtype"]] + N * (16 + 12 * c["top"]), "flops": 6 * N * V}
    lens = _lens(c)
    table = sum(-(-n // c["page"]) for n in lens) * 4
    rows = sum(lens) * c["Hkv"]
    if c["kind"] == "append":
        return {"bytes": rows * (4 * c["D"] + _row_bytes(c)) + 4 * sum(lens) // c["page"],
                "flops": 6 * rows * c["D"]}
    if c["kind"] == "evict":
        # the totals are read, those kept are written, and a kept row is read and
        # written if an earlier one goes: all but the first few of them
        kept = sum(min(n, c["budget"]) for n in lens) * c["Hkv"]
        moved = sum(c["budget"] for n in lens if n > c["budget"]) * c["Hkv"]
        return {"bytes": 4 * rows + 4 * kept + 2 * moved * _row_bytes(c) + table, "flops": 0}
    seen = rows
    if c["shared"]:    # the pages of a shared prefix are read once
        seen = (sum(lens) - (c["B"] - 1) * c["shared"]) * c["Hkv"]
    io = c["B"] * c["H"] * (2 * c["D"] * SIZES[c["dtype"]] + 4)
    return {"bytes": seen * _row_bytes(c) + io + table + (8 * rows if c["weights"] else 0),
            "flops": 4 * sum(lens) * c["H"] * c["D"]}


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


def _tables(c: dict, lens: list[int], extra: int, g: torch.Generator) -> tuple[torch.Tensor, int]:
    """A block table whose sequences own pages in a random order (the first
    ``shared`` tokens' pages are one sequence's, named by all), -1 behind
    each one's last page; and the number of pages."""
    page = c["page"]
    need = [-(-(n + extra) // page) for n in lens]
    common = c.get("shared", 0) // page
    total = common + sum(n - common for n in need)
    order = torch.randperm(total + 3, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((c["B"], max(need)), -1, dtype=torch.int32)
    at = common
    for b, n in enumerate(need):
        table[b, :common] = order[:common]
        table[b, common:n] = order[at:at + n - common]
        at += n - common
    return table.cuda(), total + 3


def _caches(c: dict, pages: int, g: torch.Generator) -> dict:
    shape = (pages, c["Hkv"], c["page"], c["D"])
    if c["cache"] != "e4m3":
        return {"k": _fill(g, shape, DTYPES[c["cache"]]), "v": _fill(g, shape, DTYPES[c["cache"]]),
                "ks": None, "vs": None}
    # codes of rows whose largest element is near 400, and their scales
    ks, vs = (torch.rand(shape[:3], generator=g, device="cuda") * 0.004 + 0.004 for _ in range(2))
    return {"k": _fill(g, shape, torch.float8_e4m3fn, 130.0), "ks": ks,
            "v": _fill(g, shape, torch.float8_e4m3fn, 130.0), "vs": vs}


def prepare(case: dict, seed: int) -> dict:
    c, g = case, _gen(seed)
    if c["kind"] == "logprob":
        # a few tokens stand out, as in a decoder's logits
        x = _fill(g, (c["N"], c["V"]), DTYPES[c["dtype"]], 2.5)
        best = torch.randint(0, c["V"], (c["N"], 8), generator=g, device="cuda")
        x.scatter_(1, best, (12.0 + 3.0 * torch.randn(best.shape, generator=g, device="cuda"))
                   .to(x.dtype))
        return {"case": c, "logits": x, "tokens": best[:, 0].contiguous()}
    lens = _lens(c)
    order = torch.randperm(c["B"], generator=g, device="cuda").cpu().tolist()
    lens = [lens[i] for i in order]
    extra = c["ctx"] if c["kind"] == "append" else 0
    table, pages = _tables(c, lens, extra, g)
    st = {"case": c, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
          **_caches(c, pages, g)}
    if c["kind"] == "append":
        # a projection's output: (B, S, Hkv, D) seen as (B, Hkv, S, D)
        shape = (c["B"], c["S"], c["Hkv"], c["D"])
        st["new_k"] = _fill(g, shape, DTYPES[c["dtype"]]).permute(0, 2, 1, 3)
        st["new_v"] = _fill(g, shape, DTYPES[c["dtype"]]).permute(0, 2, 1, 3)
        st["start"] = torch.full((c["B"],), c["ctx"], dtype=torch.int32, device="cuda")
    else:
        slots = table.shape[1] * c["page"]
        if c["kind"] == "evict" or c["weights"]:
            st["weights"] = torch.exp(_fill(g, (c["B"], c["Hkv"], slots), torch.float32, 1.5))
        if c["kind"] == "decode":
            st["q"] = _fill(g, (c["B"], c["H"], 1, c["D"]), DTYPES[c["dtype"]])
            st["max"] = max(lens)
    return st


# -------------------------------------------------------------- plain forms

def _dense(cache: torch.Tensor, scale: torch.Tensor | None, table: torch.Tensor,
           dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The rows that each sequence's table names, (B, Hkv, slots, D)."""
    t = table.clamp(min=0).long()
    x = cache.view(torch.uint8)[t].view(cache.dtype) if cache.element_size() == 1 else cache[t]
    x = x.to(dtype)
    if scale is not None:
        x = x * scale[t].to(dtype).unsqueeze(-1)
    B, N, Hkv, page, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * page, D)


def _row_scales(amax: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """(multiplier, dequant scale) of rows from their largest magnitudes: each
    step rounded to the input's type, as the row-wise quantizer defines them."""
    a = torch.maximum(amax, torch.tensor(1e-6, dtype=dtype, device="cuda")).float()
    r = (1.0 / a).to(dtype).float()
    target = torch.tensor(FP8_TARGET, dtype=torch.float32, device="cuda")
    dq = a * (1.0 / target) if dtype == torch.float16 else a / target
    return (r * target).to(dtype).float(), dq.to(dtype).float()


def _plain_append(s: dict) -> list:
    c, table, start, lens = s["case"], s["table"], s["start"], s["lens"]
    i = torch.arange(c["S"], device="cuda").unsqueeze(0)
    b, i = (i < lens.unsqueeze(1)).nonzero(as_tuple=True)
    pos = start[b].long() + i
    page, off = table[b, pos // c["page"]].long(), pos % c["page"]
    for name, x in (("k", s["new_k"]), ("v", s["new_v"])):
        rows = x[b, :, i]                                        # (tokens, Hkv, D)
        if s[name + "s"] is None:
            s[name][page, :, off] = rows
            continue
        mul, dq = _row_scales(rows.abs().amax(dim=-1), rows.dtype)
        codes = (rows.float() * mul.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        s[name].view(torch.uint8)[page, :, off] = codes.view(torch.uint8)
        s[name + "s"][page, :, off] = dq
    return [s["k"], s["v"], s["ks"], s["vs"]]


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor
            ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Attention of q (B, H, 1, D) over the first ``lens`` rows of k and v (B,
    Hkv, slots, D), in their type: the output, the log of the sum of
    exponentials and the weights (B, Hkv, H / Hkv, slots)."""
    B, Hkv, L, D = k.shape
    qg = q.to(k.dtype).reshape(B, Hkv, -1, D)
    sc = torch.matmul(qg, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    seen = torch.arange(L, device="cuda") < lens.view(B, 1, 1, 1)
    sc = torch.where(seen, sc, torch.full_like(sc[:1, :1, :1, :1], -math.inf))
    m = sc.amax(dim=-1, keepdim=True)
    e = torch.exp(sc - m)
    l = e.sum(dim=-1, keepdim=True)
    p = e / l
    return torch.matmul(p, v).reshape(q.shape), (m + torch.log(l)).reshape(q.shape[:2]), p


def _plain_decode(s: dict) -> list:
    k, v = _dense(s["k"], s["ks"], s["table"]), _dense(s["v"], s["vs"], s["table"])
    out, lse, p = _attend(s["q"], k, v, s["lens"])
    if s["case"]["weights"]:
        s["weights"] += p.sum(dim=2)
    return [out.to(s["q"].dtype), lse, s.get("weights")]


def _keep(w: torch.Tensor, lens: torch.Tensor, budget: int, recent: int
          ) -> tuple[torch.Tensor, torch.Tensor]:
    """(slots (B, Hkv, min(budget, slots)) to keep in rising order, the new
    lengths): a sequence longer than the budget keeps its last ``recent`` rows
    and the heaviest of the others, the lower slot where weights are equal."""
    B, Hkv, L = w.shape
    i = torch.arange(L, device="cuda").view(1, 1, L)
    n = lens.view(B, 1, 1)
    last = (i >= n - recent) | (n <= budget)
    w = torch.where(last, math.inf, w)
    w = torch.where(i < n, w, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
    return torch.sort(order, dim=-1).values, lens.clamp(max=budget)


def _plain_evict(s: dict) -> list:
    c, w, table = s["case"], s["weights"], s["table"]
    keep, new = _keep(w, s["lens"], c["budget"], c["recent"])
    B, Hkv, n = keep.shape
    at = torch.arange(n, device="cuda").view(1, 1, n)
    b, h, j = (at < new.view(B, 1, 1)).expand(B, Hkv, n).nonzero(as_tuple=True)
    src = keep[b, h, j]
    moved = src != j
    b, h, j, src = b[moved], h[moved], j[moved], src[moved]
    pages = table.long()
    sp, so = pages[b, src // c["page"]], src % c["page"]
    dp, do = pages[b, j // c["page"]], j % c["page"]
    for name in ("k", "v"):
        x = s[name].view(torch.uint8) if s[name].element_size() == 1 else s[name]
        x[dp, h, do] = x[sp, h, so]
        if s[name + "s"] is not None:
            s[name + "s"][dp, h, do] = s[name + "s"][sp, h, so]
    kept = torch.zeros_like(w)
    kept[..., :n] = torch.where(at < new.view(B, 1, 1), w.gather(2, keep), 0.0)
    return [new, kept, s["k"], s["v"], s["ks"], s["vs"]]


def _scores(x: torch.Tensor, tokens: torch.Tensor, top: int) -> list:
    """Log probabilities of ``tokens``, entropies, the ``top`` best log
    probabilities and their tokens (the lower one first where they are equal)
    of rows of logits, in the logits' type."""
    m = x.amax(dim=1, keepdim=True)
    z = x - m
    e = torch.exp(z)
    l = e.sum(dim=1, keepdim=True)
    lg = torch.log(l)
    chosen = (z.gather(1, tokens.unsqueeze(1)) - lg).squeeze(1)
    entropy = (lg - (e * z).sum(dim=1, keepdim=True) / l).squeeze(1)
    del e
    if not top:
        return [chosen, entropy]
    # ties to the lowest token: of the values at the border the first ones count
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return [chosen, entropy, z.gather(1, ids) - lg, ids]


def _plain_logprob(s: dict) -> list:
    rows = max(1, (1 << 28) // s["logits"].shape[1])     # a sort's room
    parts = [_scores(x.float(), t, s["case"]["top"])
             for x, t in zip(s["logits"].split(rows), s["tokens"].split(rows))]
    return [torch.cat(p) for p in zip(*parts)]


def run(state: dict):
    s, c = state, state["case"]
    if own:
        from repercep_runtime_amd import ops

        if c["kind"] == "append":
            ops.paged_kv_append(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["start"],
                                s["lens"], k_scale=s["ks"], v_scale=s["vs"])
            return [s["k"], s["v"], s["ks"], s["vs"]]
        if c["kind"] == "decode":
            out, lse = ops.paged_attention_decode(
                s["q"], s["k"], s["v"], s["table"], s["lens"], k_scale=s["ks"], v_scale=s["vs"],
                max_seq_len=s["max"], key_weights=s.get("weights"), return_lse=True)
            return [out, lse, s.get("weights")]
        if c["kind"] == "evict":
            new, kept = ops.paged_kv_evict(s["k"], s["v"], s["table"], s["lens"], s["weights"],
                                           budget=c["budget"], recent=c["recent"],
                                           k_scale=s["ks"], v_scale=s["vs"])
            return [new, kept, s["k"], s["v"], s["ks"], s["vs"]]
        r = ops.token_logprobs(s["logits"], s["tokens"], top=c["top"])
        return [r.logprobs, r.entropy] + ([r.top_logprobs, r.top_ids] if c["top"] else [])
    return {"append": _plain_append, "decode": _plain_decode, "evict": _plain_evict,
            "logprob": _plain_logprob}[c["kind"]](s)


# ------------------------------------------------------------------- 64 bits

def _near_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The e4m3fn number nearest to x (even on ties), |x| <= 448, in 64 bits."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_append(s: dict) -> list:
    c, outs = s["case"], []
    values = {n: s[n].double() for n in ("k", "v")}
    scales = {n: None if s[n + "s"] is None else s[n + "s"].double() for n in ("k", "v")}
    lens, start, table = s["lens"].tolist(), s["start"].tolist(), s["table"].cpu()
    for b, n in enumerate(lens):
        pos = torch.arange(start[b], start[b] + n)
        pg, off = table[b, pos // c["page"]].long().cuda(), (pos % c["page"]).cuda()
        for name in ("k", "v"):
            x = s["new_" + name][b, :, :n].transpose(0, 1)                 # (n, Hkv, D)
            y = x.double()
            if scales[name] is not None:
                big = y.abs().amax(dim=-1)
                big = torch.maximum(big, torch.tensor(1e-6, dtype=x.dtype).double().cuda())
                mul = ((1.0 / big).to(x.dtype).double() * FP8_TARGET).to(x.dtype).double()
                scales[name][pg, :, off] = (big / FP8_TARGET).to(x.dtype).double()
                y = _near_e4m3((y * mul.unsqueeze(-1)).clamp(-448.0, 448.0))
            values[name][pg, :, off] = y
    outs = [values["k"], values["v"], scales["k"], scales["v"]]
    return outs


def _exact_decode(s: dict) -> list:
    c = s["case"]
    outs, lses, tot = [], [], []
    for b, n in enumerate(s["lens"].tolist()):      # a sequence at a time: 64 bits take room
        t = s["table"][b:b + 1, :-(-n // c["page"])]
        k = _dense(s["k"], s["ks"], t, torch.float64)[:, :, :n]
        v = _dense(s["v"], s["vs"], t, torch.float64)[:, :, :n]
        q = s["q"][b:b + 1].double().reshape(1, c["Hkv"], -1, c["D"])
        x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(c["D"])
        lse = torch.logsumexp(x, dim=-1)
        p = torch.exp(x - lse.unsqueeze(-1))
        outs.append(torch.matmul(p, v).reshape(1, c["H"], 1, c["D"]))
        lses.append(lse.reshape(1, c["H"]))
        if c["weights"]:
            w = s["weights"][b:b + 1].double()
            w[..., :n] += p.sum(dim=2)
            tot.append(w)
    return [torch.cat(outs), torch.cat(lses), torch.cat(tot) if c["weights"] else None]


def _exact_evict(s: dict) -> list:
    c = s["case"]
    k, v = s["k"].double(), s["v"].double()
    ks, vs = (None if s[n] is None else s[n].double() for n in ("ks", "vs"))
    kept = torch.zeros_like(s["weights"], dtype=torch.float64)
    lens, new = s["lens"].tolist(), []
    for b, n in enumerate(lens):
        pages = s["table"][b].long()
        new.append(min(n, c["budget"]))
        if n <= c["budget"]:
            kept[b, :, :n] = s["weights"][b, :, :n].double()
            continue
        old = n - c["recent"]
        for h in range(c["Hkv"]):
            w = s["weights"][b, h, :old].double()
            heavy = torch.argsort(w, descending=True, stable=True)[:c["budget"] - c["recent"]]
            rows = torch.cat([heavy.sort().values, torch.arange(old, n, device="cuda")])
            to = torch.arange(c["budget"], device="cuda")
            kept[b, h, :c["budget"]] = s["weights"][b, h, rows].double()
            for x in (k, v, ks, vs):
                if x is not None:
                    x[pages[to // c["page"]], h, to % c["page"]] = \
                        x[pages[rows // c["page"]], h, rows % c["page"]]
    return [torch.tensor(new, dtype=torch.int32), kept, k, v, ks, vs]


def _exact_logprob(s: dict) -> list:
    top, got = s["case"]["top"], []
    for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
        lp = torch.log_softmax(x.double(), dim=1)
        p = torch.exp(lp)
        one = [lp.gather(1, t.unsqueeze(1)).squeeze(1), -(p * lp).sum(dim=1)]
        if top:
            best = torch.argsort(x.double(), dim=1, descending=True, stable=True)[:, :top]
            one += [lp.gather(1, best), best]
        got.append(one)
    return [torch.cat(p) for p in zip(*got)]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "evict": _exact_evict,
            "logprob": _exact_logprob}[case["kind"]](s)
