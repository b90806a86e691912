"""``token_logprobs`` of finite logits far from zero and at small temperatures, where a logit times
log2(e) / T is large: rows filled whole or in part with one large value, as a finite mask leaves them, and
rows whose logits lie close together a long way from zero.

The formulas in float64, from the differences to each row's largest logit (which a difference of stored
values keeps to one rounding). Tolerances as for ordinary logits, u = 2^-24 (2^-53 for float64 logits) and
x the exponents (z - max) / T: a log-probability (16 + 4 |x| + vocab / 64) u, an entropy that at |x| = 40 times
1 + log(vocab), a probability relatively (32 + 8 |x| + vocab / 64) u, a gradient one more rounding to its type."""

from __future__ import annotations

import math

import pytest
import torch

from torchisotonic_amd import token_logprobs

pytestmark = pytest.mark.gpu

# Rows by a few lanes, by a wave, by a workgroup, by several workgroups (few rows of 65536 logits or more).
VOCABS = [4, 300, 5000, 40_000, 70_001]
# From ones whose product with log2(e) keeps its fraction to ones near the end of the range.
FAR = {
    torch.float32: [1e7, 2.0**24, 1e8, 1e9, 3e9, 1e10, 1e12, 1e20, 1e30, 3e36, 6.9e36, 7.2e36, 1e38],
    torch.bfloat16: [1e7, 1e9, 3e9, 1e10, 1e20, 1e30, 6.9e36],
    torch.float16: [2.0**15, 65_504.0],
    torch.float64: [1e10, 4.0e15, 1e16, 1e18, 1e19, 1e20, 1e30, 1e100, 1e306, 1e308],
}
UNIT = {t: torch.finfo(t).eps / 2 for t in FAR}


def say(*a: object) -> None:
    print(*a, flush=True)


def check(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0) -> None:
    acc = torch.float64 if logits.dtype == torch.float64 else torch.float32
    u, dtype, vocab = UNIT[acc], logits.dtype, logits.shape[-1]
    gen = torch.Generator().manual_seed(vocab)
    g, ge = (torch.randn(targets.shape, generator=gen, dtype=torch.float64).to(acc) for _ in range(2))
    z = logits.clone().requires_grad_()
    logp, h = token_logprobs(z, targets, temperature=temperature, entropy=True)
    (grad,) = torch.autograd.grad([logp, h], [z], [g.cuda(), ge.cuda()])
    only = token_logprobs(z, targets, temperature=temperature)
    (only_grad,) = torch.autograd.grad([only], [z], [g.cuda()])

    zd, at = logits.cpu().double(), targets.cpu()[:, None]
    x = (zd - zd.amax(-1, keepdim=True)) / temperature
    e = x.exp()
    logs = e.sum(-1).log()
    p = e / e.sum(-1, keepdim=True)
    far = torch.where(e > 0, x, 0.0)
    want = x.gather(-1, at)[:, 0] - logs
    entropy = logs - (p * far).sum(-1)
    hit = torch.zeros_like(p).scatter_(-1, at, 1.0)
    gd, hd = g.double()[:, None], ge.double()[:, None]
    want_only = gd * (hit - p) / temperature
    want_grad = want_only - hd * p * (far - logs[:, None] + entropy[:, None]) / temperature

    def close(got: torch.Tensor, want: torch.Tensor, tol, what: str) -> None:
        got, want = got.detach().cpu().double(), want.to(got.dtype).double() if what == "logp" else want
        same = got == want  # (infinities among them)
        assert bool(((got - want).abs() <= tol)[~same].all()), f"{what}: {got[~same][:4]} for {want[~same][:4]}"

    # (a float32 logit or difference past the type's range is infinite: x too)
    close(logp, want, (16 + 4 * (want.abs() + math.log(vocab)) + vocab / 64) * u, "logp")
    close(only, want, (16 + 4 * (want.abs() + math.log(vocab)) + vocab / 64) * u, "logp")
    close(h, entropy, (16 + 160 + vocab / 64) * u * (1 + math.log(vocab)), "entropy")
    scale = gd.abs() + hd.abs() * (1 + far.abs() + math.log(vocab))
    least = {torch.float16: 2.0**-25}.get(dtype, 2.0**-126)
    for got, exact in ((grad, want_grad), (only_grad, want_only)):
        tol = (p * scale * (32 + 8 * far.abs() + vocab / 64) * u + 8 * u * exact.abs() + 2.0**-126 * scale) / temperature
        close(got, exact, tol + UNIT[dtype] * exact.abs() + least, "gradient")


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", FAR)
def test_rows_of_one_large_value(dtype: torch.dtype, vocab: int) -> None:
    for sign in (-1.0, 1.0):
        values = torch.tensor([sign * v for v in FAR[dtype]], dtype=torch.float64).to(dtype).cuda()
        say(f"rows of {sign:+} large values, {vocab} {dtype}")
        logits = values[:, None].expand(-1, vocab).contiguous()
        check(logits, torch.arange(len(values), device="cuda") % vocab)


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", FAR)
def test_rows_masked_in_part(dtype: torch.dtype, vocab: int) -> None:
    # ordinary logits in the first half, in the second, in one place; the large value everywhere else
    gen = torch.Generator().manual_seed(vocab)
    for sign in (-1.0, 1.0):
        say(f"rows masked in part by {sign:+} large values, {vocab} {dtype}")
        values = torch.tensor([sign * v for v in FAR[dtype]], dtype=torch.float64).to(dtype).cuda()
        for keep in (slice(0, vocab // 2), slice(vocab // 2, vocab), slice(vocab // 3, vocab // 3 + 1)):
            logits = torch.randn(len(values), vocab, generator=gen).to(dtype).cuda()
            masked = values[:, None].expand(-1, vocab).contiguous()
            masked[:, keep] = logits[:, keep]
            targets = torch.arange(len(values), device="cuda") % vocab
            targets[::2] = keep.start
            check(masked, targets)


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize(("dtype", "bases"), [
    (torch.float32, [2.0**20, 2.0**22, 2.0**23 - 4, 11_629_076.0, 11_629_080.0, 2.0**24 - 9]),
    (torch.float64, [2.0**30, 2.0**51, 2.0**52 - 4, 6_243_314_768_165_355.0, 6_243_314_768_165_359.0, 2.0**53 - 9]),
])
def test_close_logits_far_from_zero(dtype: torch.dtype, bases: list[float], vocab: int) -> None:
    # whole numbers that the type still tells apart, in a distribution that counts all of them; around 11629080
    # (6.24e15) a logit times log2(e) passes 2^24 (2^53), the last where it is a whole number
    gen = torch.Generator().manual_seed(vocab)
    for sign in (-1.0, 1.0):
        base = torch.tensor([b * sign for b in bases], dtype=torch.float64)[:, None]
        steps = torch.randint(0, 9, (len(bases), vocab), generator=gen)
        rising = torch.linspace(0, 8, vocab).round().expand(len(bases), -1)
        for name, step in (("mixed", steps), ("rising", rising), ("falling", rising.flip(-1))):
            say(f"close logits {sign:+}, {name}, {vocab} {dtype}")
            logits = (base + step.double()).to(dtype).cuda()
            assert torch.equal(logits.cpu().double(), base + step.double())
            check(logits, torch.arange(len(bases), device="cuda") * (vocab - 1) // (len(bases) - 1))


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("temperature", [1e-3, 1e-5, 1e-9, 1e-12, 1e-20, 1e-30, 1e-37])
def test_small_temperatures(dtype: torch.dtype, vocab: int, temperature: float) -> None:
    say(f"temperature {temperature}, {vocab} {dtype}")
    gen = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(5, vocab, generator=gen) * 3).to(dtype)
    logits[1, :2] = 20.0  # two largest
    logits[2] = 1.5  # all of them
    logits[3, ::2] = -20.0
    logits[4] = 0.0
    if dtype == torch.float16:
        logits[3, :2] = 65_504.0
    targets = torch.tensor([3, 1, 2, 0, 1], device="cuda")
    check_small(logits.cuda(), targets, temperature)


def check_small(logits: torch.Tensor, targets: torch.Tensor, temperature: float) -> None:
    """As ``check``, with gradients whose 1 / T the type of the gradient may not hold."""
    if logits.dtype != torch.float16 and temperature > 1e-36:
        check(logits, targets, temperature)
        return
    z = logits.clone().requires_grad_()
    logp, h = token_logprobs(z, targets, temperature=temperature, entropy=True)
    (grad,) = torch.autograd.grad(logp.sum() + h.sum(), z)
    x = (logits.cpu().double() - logits.cpu().double().amax(-1, keepdim=True)) / temperature
    want = torch.log_softmax(x, -1)
    logw = want.gather(-1, targets.cpu()[:, None])[:, 0]
    vocab = logits.shape[-1]
    tol = (16 + 4 * (logw.abs() + math.log(vocab)) + vocab / 64) * 2.0**-24
    got = logp.detach().cpu().double()
    # (past float32's range: minus infinity, or a value near the end of the range)
    out = logw < -3.4e38
    assert bool(((got - logw).abs() <= tol)[~out].all()) and bool((got[out] < -1e36).all())
    p = want.exp()
    entropy = -(p * torch.where(p > 0, want, 0.0)).sum(-1)
    bound = (16 + 160 + vocab / 64) * 2.0**-24 * (1 + math.log(vocab))
    assert float((h.detach().cpu().double() - entropy).abs().max()) <= bound
    assert not bool(grad.isnan().any())


def test_temperatures_below_the_types_range() -> None:
    # 1 / T past float32: what is not the row's largest has probability zero
    logits = torch.tensor([[1.0, 3.0, 3.0, -5.0], [0.0, 0.0, 0.0, 0.0], [-7.0, -8.0, -9.0, -7.0]]).cuda()
    for dtype in (torch.float32, torch.bfloat16):
        for vocab in (4, 5000, 70_000):
            z = torch.full((3, vocab), -40.0, dtype=dtype, device="cuda")
            z[:, :4] = logits.to(dtype)
            logp, h = token_logprobs(z, torch.tensor([1, 3, 0]).cuda(), temperature=1e-40, entropy=True)
            ties = torch.tensor([2.0, 4.0, 2.0])
            torch.testing.assert_close(logp.cpu(), -ties.log(), rtol=1e-6, atol=0)
            torch.testing.assert_close(h.cpu(), ties.log(), rtol=1e-6, atol=0)
