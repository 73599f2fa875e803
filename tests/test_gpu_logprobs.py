"""Token log probabilities, entropy and best alternatives on the GPU against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from repercep_runtime_amd import ops

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -24
NAN, INF = float("nan"), float("inf")


def reference(x: torch.Tensor, tokens: torch.Tensor, top: int, T: float) -> tuple:
    """(logprobs, entropy, top values, top ids) in 64 bits; ids by (value, lower id)."""
    z = x.double() / T
    lp = torch.log_softmax(z, dim=-1)
    p = torch.exp(lp)
    plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    ids = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    return lp.gather(1, tokens.unsqueeze(1)).squeeze(1), -plogp.sum(-1), lp.gather(1, ids), ids


def check(gpu, x: torch.Tensor, top: int, T: float = 1.0, seed: int = 0) -> None:
    """A shifted logit z = x / T - m is off by two roundings at |x| / T and one
    at |z| (R below); an exponential by R |z|'s share plus its own 2 u, a sum
    of V of them by V u more, its logarithm by that and 2 u; the entropy's
    second sum by as much of sum p |z|."""
    N, V = x.shape
    tokens = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(seed))
    lp, ent, tv, ti = reference(x, tokens, top, T)
    r = ops.token_logprobs(x.to(gpu), tokens.to(gpu), top=top, temperature=T)
    z = x.double() / T
    big = torch.where(torch.isfinite(z), z.abs(), torch.zeros_like(z)).amax(-1)
    R = 6 * U * big + 4 * U
    tol = 2 * R + (min(V, 4096) + 16) * U        # sums of up to 4096 terms in a row, then trees
    zz = torch.where(torch.isfinite(z), z - z.amax(-1, keepdim=True), torch.zeros_like(z))
    spread = (torch.softmax(z, -1) * zz.abs()).sum(-1)
    got = r.logprobs.cpu().double()
    fin = torch.isfinite(lp)
    assert torch.equal(torch.isfinite(got), fin) and torch.equal(got[~fin], lp[~fin])
    assert ((got - lp).abs()[fin] <= (tol + 2 * U * lp.abs())[fin]).all()
    assert ((r.entropy.cpu().double() - ent).abs() <= 2 * tol * (1 + spread)).all()
    if not top:
        assert r.top_ids is None and r.top_logprobs is None
        return
    assert torch.equal(r.top_ids.cpu(), ti)
    fin = torch.isfinite(tv)
    got = r.top_logprobs.cpu().double()
    assert torch.equal(torch.isfinite(got), fin) and torch.equal(got[~fin], tv[~fin])
    assert ((got - tv).abs()[fin] <= (tol.unsqueeze(1) + 2 * U * tv.abs())[fin]).all()


def logits(N: int, V: int, dt: str, seed: int, std: float = 2.5) -> torch.Tensor:
    return (torch.randn(N, V, generator=torch.Generator().manual_seed(seed)) * std).to(DTYPES[dt])


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V", [(1, 1), (3, 2), (1, 7), (5, 63), (4, 64), (2, 65), (3, 1000),
                                 (2, 1023), (1, 4097), (7, 8192), (1, 8193), (2, 16385),
                                 (1, 32000), (3, 32769), (1, 65537), (2, 100003), (1, 152064)])
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_scores(gpu, dt, N, V, top) -> None:
    check(gpu, logits(N, V, dt, N * V), min(top, V), seed=V)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("N", [130, 600, 1500])
def test_many_rows(gpu, dt, N) -> None:
    check(gpu, logits(N, 4100, dt, N), 5)


@pytest.mark.parametrize("T", [0.25, 0.7, 3.0])
def test_temperature(gpu, T) -> None:
    check(gpu, logits(4, 5000, "bf16", 1), 8, T)


@pytest.mark.parametrize("T", [1e-7, 1e-20, 1e20])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_extreme_temperatures(gpu, dt, T) -> None:
    """All weight on the best tokens, or the same on every one.  The logits are
    whole, so their differences are 0 or at least 1 / T."""
    x = torch.randint(-9, 10, (3, 3000), generator=torch.Generator().manual_seed(3)).to(DTYPES[dt])
    r = ops.token_logprobs(x.to(gpu), torch.zeros(3, dtype=torch.int64, device=gpu), top=4,
                           temperature=T)
    z = x.double() / T
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    # log p of the best is -log of their number; of the others about -1 / T: both to 2^-20
    assert ((r.entropy.cpu().double() - ent).abs() <= 2.0 ** -20 * (1 + ent)).all()
    got, want = r.logprobs.cpu().double(), lp[:, 0]
    assert ((got - want).abs() <= 2.0 ** -20 * (1 + want.abs())).all()
    assert ((r.top_logprobs.cpu().double() - lp.gather(1, r.top_ids.cpu())).abs() <= 2.0 ** -20
            * 10).all()


@pytest.mark.parametrize("shift", [-3e4, 1e3, 3e4])
def test_large_logits(gpu, shift) -> None:
    """Logits far from zero: only their differences count."""
    check(gpu, (logits(3, 3001, "fp32", 2) + shift).float(), 8)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [60, 5001, 33000, 100000])
@pytest.mark.parametrize("gap", [12.0, 25.0, 60.0])
def test_nearly_certain_rows(gpu, dt, V, gap) -> None:
    """One logit far above the others: the small entropy and the small log
    probability of its token keep their relative precision.  With r the others'
    weight, log(1 + r) and sum p |z| are sums of positive terms, each off by
    the rounding of its power's argument (at most 90: 90 u, a few u more), a
    sum's V u at most (trees: far less) and a handful of operations."""
    x = logits(3, V, dt, V, std=1.0)
    best = torch.tensor([0, V // 2, V - 1])
    x[torch.arange(3), best] = x.amax(-1) + torch.tensor(gap).to(x.dtype)
    lp, ent, _, _ = reference(x, best, 1, 1.0)
    z = x.double() - x.double().amax(-1, keepdim=True)
    rest = torch.exp(z)
    rest[torch.arange(3), best] = 0.0
    # in 64 bits from the others alone: logsumexp's own 1 + r loses r below 2^-53
    r = rest.sum(-1)
    lp = -torch.log1p(r)
    ent = torch.log1p(r) - (rest * z).sum(-1) / (1 + r)
    got = ops.token_logprobs(x.to(gpu), best.to(gpu), top=1)
    tol = (2 * 100 + min(V, 4096) + 32) * U
    assert torch.equal(got.top_ids[:, 0].cpu(), best)
    assert ((got.logprobs.cpu().double() - lp).abs() <= tol * lp.abs()).all()
    assert ((got.top_logprobs[:, 0].cpu().double() - lp).abs() <= tol * lp.abs()).all()
    assert ((got.entropy.cpu().double() - ent).abs() <= tol * ent).all()


def test_wide_spread(gpu) -> None:
    """One token takes all; the others' probabilities leave the type's range."""
    check(gpu, logits(3, 5000, "fp32", 3, std=200.0), 32)
    x = torch.full((2, 3000), -1e4)
    x[:, 1234] = 1e4
    check(gpu, x, 4)


@pytest.mark.parametrize("V", [50, 3000, 40000, 140000])
def test_ties_go_to_the_lower_token(gpu, V) -> None:
    """All equal, two values, few values, zeros of both signs: ids by (value, lower id)."""
    g = torch.Generator().manual_seed(V)
    few = torch.tensor([0.0, 1.0, 2.0])[torch.randint(0, 3, (V,), generator=g)]
    signs = torch.tensor([0.0, -0.0])[torch.randint(0, 2, (V,), generator=g)]
    one = torch.zeros(V)
    one[V // 2] = 1.0
    check(gpu, torch.stack([torch.full((V,), 1.5), few, signs, one]).to(torch.bfloat16), 32)


@pytest.mark.parametrize("V", [300, 9000, 140000])
def test_sorted_rows(gpu, V) -> None:
    """The best logits next to each other, at either end or in the middle."""
    up = torch.arange(V, dtype=torch.float32) * 1e-3
    check(gpu, torch.stack([up, -up, up.roll(V // 3), -(up - up[V // 2]).abs()]), 32)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [100, 33000])
def test_masked_logits(gpu, dt, V) -> None:
    """-inf at most places (fewer left than asked for among them), the type's
    lowest value at most places, and a single one left."""
    x = logits(4, V, dt, V)
    g = torch.Generator().manual_seed(1)
    x[0][torch.rand(V, generator=g) < 0.7] = -INF
    x[1, 10:] = -INF
    x[2, :V - 3] = torch.finfo(x.dtype).min
    x[3, :] = -INF
    x[3, V // 2] = 0.5
    check(gpu, x, 32)


@pytest.mark.parametrize("V", [70, 50000])
def test_rows_without_a_distribution(gpu, V) -> None:
    """Nothing but -inf: -inf and 0; a NaN or +inf anywhere: NaN, in that row only."""
    x = logits(4, V, "bf16", 4)
    x[0] = -INF
    x[1, V - 1] = NAN
    x[2, 3] = INF
    tokens = torch.tensor([1, 2, 3, 4])
    r = ops.token_logprobs(x.to(gpu), tokens.to(gpu), top=3)
    assert r.logprobs[0] == -INF and r.entropy[0] == 0
    assert torch.isneginf(r.top_logprobs[0]).all() and r.top_ids[0].tolist() == [0, 1, 2]
    for i in (1, 2):
        assert r.logprobs[i].isnan() and r.entropy[i].isnan() and r.top_logprobs[i].isnan().all()
    assert int(r.top_ids[1, 0]) == V - 1 and int(r.top_ids[2, 0]) == 3
    # row 3 alone lies at another offset from a 16-byte border, so its sums run
    # in another order: both sides are within check()'s bound of 64 bits, |x| < 12
    want = ops.token_logprobs(x[3:].to(gpu), tokens[3:].to(gpu), top=3)
    tol = 2 * (6 * 12 + 4) * U + (min(V, 4096) + 16) * U + 2 * U * 24
    assert float(x[3].abs().max()) < 12
    assert abs(float(r.logprobs[3] - want.logprobs[0])) <= 2 * tol
    assert torch.equal(r.top_ids[3:], want.top_ids)


def test_padding_and_foreign_tokens(gpu) -> None:
    x = logits(4, 50, "bf16", 5).to(gpu)
    r = ops.token_logprobs(x, torch.tensor([-100, 50, 49, -1], device=gpu))
    assert r.logprobs[0] == 0 and r.logprobs[3] == 0 and r.logprobs[1].isnan()
    assert torch.isfinite(r.logprobs[2]) and torch.isfinite(r.entropy).all()
    assert r.top_ids is None


def test_views_and_leading_shapes(gpu) -> None:
    """(B, S, V) logits, rows at an odd stride and address, one row, none."""
    x = logits(12, 5003, "bf16", 6)
    wide = torch.full((12, 5010), 99.0, dtype=torch.bfloat16, device=gpu)
    wide[:, 3:5006] = x.to(gpu)
    t = torch.arange(12, device=gpu)
    want = ops.token_logprobs(x.to(gpu), t, top=4)
    got = ops.token_logprobs(wide[:, 3:5006], t, top=4)
    for a, b in zip(want[:3], got[:3]):
        assert torch.allclose(a, b, rtol=0, atol=64 * U * 8)
    assert torch.equal(want.top_ids, got.top_ids)
    r = ops.token_logprobs(x.to(gpu).view(3, 4, 5003), t.view(3, 4), top=4)
    assert r.logprobs.shape == (3, 4) and r.top_ids.shape == (3, 4, 4)
    assert torch.equal(r.top_ids.view(12, 4), want.top_ids)
    one = ops.token_logprobs(x[2].to(gpu), t[2], top=4)
    assert one.logprobs.shape == () and torch.equal(one.top_ids, want.top_ids[2])
    none = ops.token_logprobs(x[:0].to(gpu), t[:0], top=4)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 4)


def test_rows_past_32_bit_offsets(gpu) -> None:
    V, N = 1 << 20, (1 << 12) + 3
    free, _ = torch.cuda.mem_get_info(gpu)
    if free < 12 << 30:
        pytest.skip("needs 12 GB of GPU memory")
    x = torch.zeros((N, V), dtype=torch.bfloat16, device=gpu)
    x[N - 1, 777] = 20.0
    t = torch.full((N,), 777, device=gpu)
    r = ops.token_logprobs(x, t, top=1)
    # the other V - 1 weigh e^-20 each: V e^-20 = 0.00216
    assert abs(float(r.logprobs[N - 1]) + math.log1p((V - 1) * math.exp(-20))) < 1e-5
    assert int(r.top_ids[N - 1, 0]) == 777 and int(r.top_ids[N - 2, 0]) == 0
    assert abs(float(r.logprobs[0]) + math.log(V)) < 1e-4


def test_equal_calls_give_equal_bits(gpu) -> None:
    for N, V in ((1, 32000), (300, 32000), (2, 150000)):
        x = logits(N, V, "bf16", 9).to(gpu)
        t = torch.zeros(N, dtype=torch.int64, device=gpu)
        a = ops.token_logprobs(x, t, top=20)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(a, ops.token_logprobs(x, t, top=20)))


def _rows_below_zero(V: int, dt: str, top: int) -> torch.Tensor:
    """Rows whose logits lie wholly or mostly below zero: shifted by their
    maximum; log probabilities of nearly certain rows, the best at -0 in one;
    N(-9, 2.5) and N(-30, 2.5); a negative bulk with 1, top - 1, top and 40
    logits at or above zero; zeros of both signs among negatives; sorted rows
    that cross zero, either way."""
    g = torch.Generator().manual_seed(V + top)
    rnd = torch.randn(10, V, generator=g, dtype=torch.float64) * 2.5
    shifted = rnd[0] - rnd[0].max()
    sure = rnd[1].clone()
    sure[V // 3] += 40.0
    sure = torch.log_softmax(sure, 0)
    best = sure.clone()
    best[V // 3] = -0.0
    few = []
    for i, n in enumerate((1, top - 1, top, 40)):
        x = rnd[4 + i] - 14.0
        at = torch.randperm(V, generator=g)[:n]
        x[at] = torch.rand(len(at), generator=g, dtype=torch.float64) * 6.0
        few.append(x)
    zeros = torch.tensor([0.0, -0.0, -1.0, -2.0, -3.0], dtype=torch.float64)
    mixed = zeros[torch.randint(2, 5, (V,), generator=g)]
    at = torch.randperm(V, generator=g)[:max(2, min(V // 4, 2 * top))]
    mixed[at] = zeros[torch.randint(0, 2, (len(at),), generator=g)]
    lowest = zeros[torch.randint(2, 5, (V,), generator=g)]
    lowest[at] = -0.0
    up = torch.linspace(-6.0, 3.0, V, dtype=torch.float64)
    rows = [shifted, sure, best, rnd[8] - 9.0, rnd[9] - 30.0, *few, mixed, lowest, up, up.flip(0)]
    return torch.stack(rows).to(DTYPES[dt])


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("V", [60, 1000, 2047, 8192, 32000, 40001, 128256])
@pytest.mark.parametrize("top", [1, 5, 16, 20, 32])
def test_best_of_rows_below_zero(gpu, dt, V, top) -> None:
    """16-bit logits at or below zero: the best and their order, one part a
    row and several, rows on and off 16-byte borders."""
    check(gpu, _rows_below_zero(V, dt, top), top, seed=top)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [50, 40000])
def test_one_row_of_logits_for_many_tokens(gpu, dt, V) -> None:
    """An expanded row is read as it lies: what copies of it give."""
    x = logits(1, V, dt, V).to(gpu)
    t = torch.tensor([0, V - 1, -1, V // 2, 3, V], device=gpu)
    got = ops.token_logprobs(x.expand(6, V), t, top=7)
    want = ops.token_logprobs(x, t[:1], top=7)
    assert got.logprobs[2] == 0 and got.logprobs[5].isnan()
    for i in range(6):
        assert torch.equal(got.entropy[i], want.entropy[0])
        assert torch.equal(got.top_ids[i], want.top_ids[0])
        assert torch.equal(got.top_logprobs[i], want.top_logprobs[0])
    for i in (0, 1, 3, 4):
        one = ops.token_logprobs(x, t[i:i + 1])
        assert torch.equal(got.logprobs[i], one.logprobs[0])


def test_logits_that_do_not_flatten(gpu) -> None:
    """Leading dimensions of no one row stride: copied first, the same answers."""
    x = logits(12, 300, "fp32", 3).to(gpu).view(3, 4, 300)
    t = torch.arange(12, device=gpu).view(4, 3)
    got = ops.token_logprobs(x.transpose(0, 1), t, top=3)
    want = ops.token_logprobs(x.transpose(0, 1).contiguous(), t, top=3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
