"""The losses over more than 2^20 places, where a wave takes tiles of 512: sequences that end with a tile,
one place before it and one after, and tiles of other lengths beside them.

Tolerances as for the losses' other tests (u = 2^-24, 2^-53 in float64), but that among a million tokens some
ratios lie within their own rounding, (|x| + 8) u, of a bound of the clip: such a token may count as clipped or
not. Its loss is the same to that rounding; it is left out of the share of clipped tokens and of the gradient."""

from __future__ import annotations

import pytest
import torch
from test_gpu_losses import UNIT, check_preference, cpu, offsets_of, sequence_of, tokens, want_policy

from torchisotonic_amd import policy_loss

pytestmark = pytest.mark.gpu

LENGTHS = {
    "of a tile each": [512] * 2200,
    "one place less": [511] * 2200,
    "one place more": [513] * 2200,
    "of half a tile": [256] * 4200,
    "of a tile and a half": [768] * 1400,
    "of two tiles": [1024] * 1100,
    "tiles and single places": [512, 1] * 1100 + [512, 0, 511, 1] * 500,
    "a long one, then tiles": [600_000, *[512] * 900, 1, 0, *[511] * 50, 3, 512, 2],
    "just over a million, not whole tiles": [2**20 - 5, 7],
}


def check_policy(lengths, dtype, *, use_mask, advantages="sequence", reduction="token_mean", dense=None):
    (x, old, ref), mask, gen = tokens(lengths, dtype)
    n, of, lo, hi, k, u = len(lengths), sequence_of(lengths), 0.2, 0.28, 0.05, UNIT[dtype]
    mask = mask if use_mask else None
    adv = torch.randn(x.numel() if advantages == "token" else n, generator=gen, dtype=torch.float64).to(dtype).cuda()
    each = adv if advantages == "token" else adv[of.cuda()]
    g = torch.randn((), generator=gen, dtype=torch.float64).to(dtype).cuda()
    rows = (lambda t: t) if dense is None else (lambda t: None if t is None else t.view(n, dense))
    z = rows(x.clone()).requires_grad_()
    kw = {"offsets": offsets_of(lengths).cuda()} if dense is None else {}
    out = policy_loss(z, rows(old), rows(adv) if advantages == "token" else adv, reference_logps=rows(ref), mask=rows(mask),
                      clip=lo, clip_high=hi, kl_coef=k, reduction=reduction, **kw)
    (grad,) = torch.autograd.grad(out.loss, z, g)
    wl, wk, wc, wg, bound, kl = want_policy(x, old, each, ref, mask, of, n, lo, hi, k, reduction, g)
    d = cpu(x) - cpu(old)
    r = d.exp()
    near = ((r - (1 - lo)).abs() <= (d.abs() + 8) * u * r) | ((r - (1 + hi)).abs() <= (d.abs() + 8) * u * r)
    doubt = near & cpu(mask).bool() if use_mask else near
    assert int(doubt.sum()) <= 1e-4 * x.numel()
    share = float(doubt.sum()) / (int(mask.sum()) if use_mask else x.numel())
    slack = 8 * u * float(bound.sum()) + 1e-300
    torch.testing.assert_close(float(out.loss.detach()), float(wl), rtol=4 * u, atol=slack)
    torch.testing.assert_close(float(out.kl), float(wk), rtol=64 * u, atol=64 * u * float(kl.sum() / x.numel()))
    assert abs(float(out.clip_fraction) - float(wc)) <= 4 * u * float(wc) + share * (1 + 1e-6)
    off = (cpu(grad) - wg).abs() - (8 * u * bound * abs(float(g)) + 8 * u * wg.abs())
    assert float(off[~doubt].max()) <= 0, f"gradient over its bound by {float(off[~doubt].max())}"


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_lengths_around_tiles_of_512(name: str, dtype: torch.dtype) -> None:
    lengths = LENGTHS[name]
    assert sum(lengths) > 2**20 and len(lengths) % 2 == 0
    for mask in (False, True):
        print(f"tiles of 512: {name}, {dtype}, mask={mask}", flush=True)
        check_preference(lengths, dtype, use_mask=mask, average=mask)
        check_policy(lengths, dtype, use_mask=mask, reduction="sequence_mean")
        check_policy(lengths, dtype, use_mask=mask, advantages="token")


@pytest.mark.parametrize("dense", [511, 512, 513])
def test_rows_around_tiles_of_512(dense: int) -> None:
    for mask in (False, True):
        print(f"rows of {dense}, mask={mask}", flush=True)
        check_preference([dense] * 2200, torch.float32, dense=dense, use_mask=mask)
        check_policy([dense] * 2200, torch.float32, dense=dense, use_mask=mask, reduction="sequence_mean")
