"""Offsets on the GPU that are not what they have to be: nothing waits for the GPU to refuse them, so the loss
and the gradient of every token that counts are NaN, for one workgroup's tokens and for many."""

from __future__ import annotations

import pytest
import torch

from torchisotonic_amd import policy_loss, preference_loss

pytestmark = pytest.mark.gpu


def say(*a: object) -> None:
    print(*a, flush=True)


def wrong(total: int, count: int) -> dict[str, list[int]]:
    """Offsets of ``count`` sequences (four at least) over ``total`` tokens, each wrong in one way."""
    even = [i * total // count for i in range(count + 1)]
    middle = count // 2
    return {
        "short of the end": [*even[:-1], total - 1],
        "past the end": [*even[:-1], total + 5],
        "not from the start": [1, *even[1:]],
        "below the start": [-3, *even[1:]],
        "decreasing in the middle": [*even[:middle], even[middle + 1] + 1, *even[middle + 1:]],
        "decreasing after an empty one": [0, 0, total, total - 3, *[total] * (count - 3)],
        "backwards": even[::-1],
        "far outside": [0, *[1 << 40] * (count - 1), total],
    }


SIZES = [(10, 4), (4096, 64), (5000, 4), (5000, 90), (300_000, 2000), (1_200_000, 40), (1_300_001, 60_000)]


@pytest.mark.parametrize(("total", "count"), SIZES)
@pytest.mark.parametrize("masked", [False, True])
def test_policy_gradients(total: int, count: int, masked: bool) -> None:
    gen = torch.Generator().manual_seed(total)
    x, old, adv = (torch.randn(n, generator=gen).cuda() for n in (total, total, count))
    mask = (torch.rand(total, generator=gen) < 0.6).cuda() if masked else None
    for name, offsets in wrong(total, count).items():
        for reduction in ("token_mean", "sequence_mean", "sum"):
            for advantages in (adv, old):
                say(f"policy of {count} sequences, {total} tokens, {masked=}, {name}, {reduction}")
                z = x.clone().requires_grad_()
                out = policy_loss(z, old, advantages, offsets=torch.tensor(offsets).cuda(), mask=mask, reduction=reduction)
                assert bool(out.loss.isnan())
                for _ in range(2):  # (the second backward computes its gradient again)
                    (grad,) = torch.autograd.grad(out.loss, z, retain_graph=True)
                    check(grad, mask)
                (grad,) = torch.autograd.grad(out.loss * 0.25, z)
                check(grad, mask)


def check(grad: torch.Tensor, mask: torch.Tensor | None) -> None:
    if mask is None:
        assert bool(grad.isnan().all())
    else:
        assert bool(grad[mask].isnan().all()) and not bool(grad[~mask].any())


@pytest.mark.parametrize(("total", "count"), SIZES)
@pytest.mark.parametrize("masked", [False, True])
def test_preference_gradients(total: int, count: int, masked: bool) -> None:
    gen = torch.Generator().manual_seed(total)
    x, ref = (torch.randn(total, generator=gen).cuda() for _ in range(2))
    mask = (torch.rand(total, generator=gen) < 0.6).cuda() if masked else None
    for name, offsets in wrong(total, count).items():
        for reduction in ("mean", "sum"):
            for loss in ("logistic", "hinge"):
                say(f"preference of {count} sequences, {total} tokens, {masked=}, {name}, {reduction}, {loss}")
                z = x.clone().requires_grad_()
                out = preference_loss(z, ref, offsets=torch.tensor(offsets).cuda(), mask=mask, reduction=reduction, loss=loss)
                assert bool(out.loss.isnan())
                (grad,) = torch.autograd.grad(out.loss, z, torch.tensor(0.5).cuda())
                check(grad, mask)
        # single losses: the pairs' whose own they are
        off = torch.tensor(offsets)
        a, b = off[:-1], off[1:]
        bad = (a > b) | (a < 0) | (b > total)
        bad[0] |= a[0] != 0
        bad[-1] |= b[-1] != total
        out = preference_loss(x, ref, offsets=off.cuda(), mask=mask, reduction="none")
        pairs = bad[:count // 2] | bad[count // 2:]
        assert bool(out.loss.cpu()[pairs].isnan().all())


def test_sound_offsets_have_gradients() -> None:
    for total, count in SIZES:
        gen = torch.Generator().manual_seed(total)
        z, old, adv = (torch.randn(n, generator=gen).cuda() for n in (total, total, count))
        off = torch.tensor([i * total // count for i in range(count + 1)]).cuda()
        z.requires_grad_()
        for loss in (policy_loss(z, old, adv, offsets=off).loss, preference_loss(z, old, offsets=off).loss):
            (grad,) = torch.autograd.grad(loss, z)
            assert bool(loss.isfinite()) and bool(grad.isfinite().all())


def test_values_that_are_nan_leave_other_gradients() -> None:
    """A NaN among the tokens is no wrong offset: what does not depend on it has its gradient."""
    for total, count in SIZES:
        x = torch.zeros(total, device="cuda")
        x[total - 1] = float("nan")
        off = torch.tensor([i * total // count for i in range(count + 1)]).cuda()
        z = x.clone().requires_grad_()
        out = policy_loss(z, torch.zeros_like(x), torch.ones(count, device="cuda"), offsets=off)
        (grad,) = torch.autograd.grad(out.loss, z)
        assert bool(out.loss.isnan()) and bool(grad[:-1].isfinite().all()) and bool(grad[-1].isnan())
        z = x.clone().requires_grad_()
        out = preference_loss(z, offsets=off)
        (grad,) = torch.autograd.grad(out.loss, z)
        assert bool(out.loss.isnan())
        last = int(off[-2])
        lo, hi = int(off[count // 2 - 1]), int(off[count // 2])
        own = torch.zeros(total, dtype=torch.bool, device="cuda")
        own[last:] = own[lo:hi] = True
        assert bool(grad[own].isnan().all()) and bool(grad[~own].isfinite().all())


@pytest.mark.parametrize("kind", ["offsets", "lengths"])
@pytest.mark.parametrize("place", ["cpu", "cuda"])
def test_tokens_of_no_sequence_are_refused(kind: str, place: str) -> None:
    """What the number of offsets alone says is wrong needs no waiting."""
    x = torch.zeros(10, device="cuda", requires_grad=True)
    none = torch.zeros(1 if kind == "offsets" else 0, dtype=torch.int64, device=place)
    for call in (lambda: preference_loss(x, **{kind: none}), lambda: policy_loss(x, x.detach(), x.detach(), **{kind: none}),
                 lambda: policy_loss(x, x.detach(), x.detach()[:0], **{kind: none}, reduction="sequence_mean")):
        with pytest.raises(ValueError, match="offsets must run from 0"):
            call()
    empty = x[:0]
    assert float(preference_loss(empty, **{kind: none}).loss) == 0.0
    assert float(policy_loss(empty, empty.detach(), empty.detach(), **{kind: none}).loss) == 0.0
