"""``token_logprobs`` and the losses among autograd's other means: hooks that keep saved tensors elsewhere and
give them back in another layout."""

from __future__ import annotations

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

from torchisotonic_amd import policy_loss, preference_loss, token_logprobs

pytestmark = pytest.mark.gpu


def say(*a: object) -> None:
    print(*a, flush=True)


def transposed(t: torch.Tensor) -> torch.Tensor:
    """A copy whose last two dimensions lie the other way round in memory."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.ndim > 1 else t.clone()


LAYOUTS = {
    "on the CPU": save_on_cpu,
    "a contiguous copy": lambda: saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
    "a transposed copy": lambda: saved_tensors_hooks(lambda t: t, transposed),
    "every other element": lambda: saved_tensors_hooks(
        lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0] if t.ndim else t.clone()),
}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("vocab", [40, 1003, 9001])
def test_saved_logits_in_another_layout(layout: str, vocab: int) -> None:
    gen = torch.Generator().manual_seed(vocab)
    base = torch.randn(4, 33, vocab, generator=gen).cuda()
    targets = torch.randint(0, vocab - 3, (4, 33), generator=gen).cuda()
    targets[1, ::3] = -100
    cases = {
        "contiguous": (base, targets),
        "all but each text's last place": (base[:, :-1], targets[:, :-1]),
        "a window of the vocabulary": (base[:, :, 1:vocab - 1], targets),
        "every other place": (base[:, ::2], targets[:, ::2]),
        "texts transposed": (base.transpose(0, 1), targets.t()),
        "one row for all": (base[0, :1].expand(6, vocab), targets[0, :6]),
        "no rows": (base[:0], targets[:0]),
    }
    for name, (logits, t) in cases.items():
        say(f"saved {layout}: {name}, {vocab}")

        def grad() -> torch.Tensor:
            z = logits.detach().requires_grad_()
            logp, h = token_logprobs(z, t, entropy=True)
            return torch.autograd.grad(logp.sum() + 0.5 * h.sum(), z)[0]

        want = grad()
        with LAYOUTS[layout]():
            got = grad()
        assert torch.equal(got, want)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_saved_losses_in_another_layout(layout: str) -> None:
    gen = torch.Generator().manual_seed(1)
    x, old, ref = (torch.randn(6, 300, generator=gen).cuda() for _ in range(3))
    mask = (torch.rand(6, 300, generator=gen) < 0.7).cuda()
    adv = torch.randn(6, generator=gen).cuda()
    offsets = torch.tensor([0, 100, 100, 901, 1500, 1700, 1800]).cuda()
    calls = {
        "preference": lambda z: preference_loss(z, ref, mask=mask).loss,
        "preference, packed": lambda z: preference_loss(z.flatten(), ref.flatten(), offsets=offsets).loss,
        "policy": lambda z: policy_loss(z, old, adv, reference_logps=ref, mask=mask, kl_coef=0.1).loss,
        "policy, an advantage a token": lambda z: policy_loss(z, old, ref, mask=mask, reduction="sequence_mean").loss,
        "policy, packed": lambda z: policy_loss(z.flatten(), old.flatten(), adv, offsets=offsets).loss,
    }
    for name, call in calls.items():
        say(f"saved {layout}: {name}")

        def grads() -> list[torch.Tensor]:
            z = x.clone().requires_grad_()
            loss = call(z)
            # (the second backward of a policy loss computes its gradient again, from what was saved)
            return [torch.autograd.grad(loss, z, retain_graph=True)[0].clone() for _ in range(2)]

        want = grads()
        with LAYOUTS[layout]():
            got = grads()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_of_another_size_are_refused() -> None:
    logits, t = torch.randn(6, 50).cuda(), torch.zeros(6, dtype=torch.int64, device="cuda")
    x, adv = torch.randn(4, 30).cuda(), torch.ones(4).cuda()
    mask = torch.ones(4, 30, dtype=torch.bool, device="cuda")
    calls = {
        "logprobs": (logits, lambda z: token_logprobs(z, t).sum()),
        "preference": (x, lambda z: preference_loss(z, mask=mask).loss),
        "policy": (x, lambda z: policy_loss(z, x, adv, mask=mask).loss),
    }
    changes = {"shorter": lambda t: t[:2], "on the host": lambda t: t.cpu(),
               "in another type": lambda t: t.double() if t.is_floating_point() else t.int()}
    for what, change in changes.items():
        for name, (value, call) in calls.items():
            say(f"saved {what}: {name}")
            z = value.clone().requires_grad_()
            with saved_tensors_hooks(lambda t: t, change):
                loss = call(z)
            if name == "policy":  # (the first backward reads nothing that was saved)
                torch.autograd.grad(loss, z, retain_graph=True)
            with pytest.raises(RuntimeError, match="came back|must match|must be"):
                torch.autograd.grad(loss, z, retain_graph=True)


def test_forward_mode_is_refused() -> None:
    """Without a forward derivative, a call on a dual tensor raises: a result without a tangent would read as a
    derivative of zero."""
    from torch.autograd import forward_ad

    gen = torch.Generator().manual_seed(2)
    logits, t = torch.randn(5, 40, generator=gen).cuda(), torch.zeros(5, dtype=torch.int64, device="cuda")
    x, old, adv = torch.randn(4, 30, generator=gen).cuda(), torch.randn(4, 30, generator=gen).cuda(), torch.ones(4).cuda()
    calls = {
        "logprobs": lambda d: token_logprobs(d(logits), t),
        "logprobs with entropy": lambda d: token_logprobs(d(logits), t, entropy=True),
        "preference": lambda d: preference_loss(d(x), old),
        "preference, none": lambda d: preference_loss(d(x), reduction="none"),
        "preference, the reference's": lambda d: preference_loss(x, d(old)),
        "preference, half": lambda d: preference_loss(d(x.half())),
        "policy": lambda d: policy_loss(d(x), old, adv),
        "policy, the old ones'": lambda d: policy_loss(x, d(old), adv),
        "policy, advantages": lambda d: policy_loss(x, old, d(adv)),
        "policy, the reference's": lambda d: policy_loss(x, old, adv, reference_logps=d(old), kl_coef=0.1),
    }
    constants = {n for n in calls if "'" in n or "advantages" in n}
    for name, call in calls.items():
        # (tensors that get no gradient may not require one)
        for tracked in (False,) if name in constants else (False, True):
            for no_grad in (False, True):
                say(f"forward mode: {name}, {tracked=}, {no_grad=}")
                with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
                    with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                        call(lambda v: forward_ad.make_dual(v.clone().requires_grad_(tracked), torch.ones_like(v)))
        call(lambda v: v)  # (and none of it outside)


def test_function_transforms() -> None:
    gen = torch.Generator().manual_seed(3)
    logits, t = torch.randn(5, 40, generator=gen).cuda(), torch.zeros(5, dtype=torch.int64, device="cuda")
    x, adv = torch.randn(4, 30, generator=gen).cuda(), torch.ones(4).cuda()
    calls = {
        "logprobs": (lambda z: token_logprobs(z, t).sum(), logits),
        "preference": (lambda z: preference_loss(z).loss, x),
        "policy": (lambda z: policy_loss(z, x, adv).loss, x),
    }
    for name, (call, value) in calls.items():
        say(f"transforms: {name}")
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (value,), (torch.ones_like(value),))
        with pytest.raises(RuntimeError):
            torch.func.grad(call)(value)
        # (a map over a batch: one call after another, with their gradients)
        z = torch.stack([value, 0.5 * value]).requires_grad_()
        out = torch.func.vmap(call)(z)
        (grad,) = torch.autograd.grad(out.sum(), z)
        for i in range(2):
            one = z[i].detach().requires_grad_()
            want = call(one)
            assert torch.equal(out[i], want) and torch.equal(grad[i], torch.autograd.grad(want, one)[0])
