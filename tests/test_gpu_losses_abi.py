"""The losses' C ABI called directly on the GPU with arrays of no tokens, whose pointers a caller may leave set."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from torchisotonic_amd import _ext

pytestmark = pytest.mark.gpu


def workspace(size_of, total: int, sequences: int) -> torch.Tensor:
    size = ctypes.c_size_t(0)
    assert size_of(total, sequences, ctypes.byref(size)) == 0
    return torch.empty(max(size.value, 1), dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("sequences", [2, 64, 66, 100, 5000])
@pytest.mark.parametrize("by_offsets", [True, False])
@pytest.mark.parametrize("masked", [True, False])
def test_no_tokens(sequences: int, by_offsets: bool, masked: bool) -> None:
    lib, stream = _ext.load(), torch.cuda.current_stream().cuda_stream
    tokens = torch.zeros(16, device="cuda")
    marks = torch.ones(16, dtype=torch.bool, device="cuda")
    offsets = torch.zeros(sequences + 1, dtype=torch.int64, device="cuda")
    mask, off = marks.data_ptr() if masked else None, offsets.data_ptr() if by_offsets else None
    adv = torch.ones(sequences, device="cuda")
    for reduction in (1, 2, 3):  # the tokens' mean, sum, the sequences' mean
        print(f"policy of no tokens: {sequences} sequences, {by_offsets=}, {masked=}, reduction {reduction}", flush=True)
        out = torch.full((3,), float("nan"), device="cuda")
        ws = workspace(lib.ti_policy_workspace, 0, sequences)
        t, o = tokens.data_ptr(), out.data_ptr()
        rc = lib.ti_policy(t, t, adv.data_ptr(), 0, t, mask, off, 0, sequences, 0, 0.2, 0.2, 0.1, reduction, o, o + 4, o + 8,
                           t, _ext.F32, ws.data_ptr(), ws.numel(), stream)
        assert rc == 0, lib.ti_last_error().decode()
        assert out.tolist() == [0.0, 0.0, 0.0]
        assert lib.ti_policy_bwd(t, 0, o, _ext.F32, stream) == 0
    pairs = sequences // 2
    for reduction, want in ((0, math.log(2)), (1, math.log(2)), (2, pairs * math.log(2))):
        print(f"preference of no tokens: {sequences} sequences, {by_offsets=}, {masked=}, reduction {reduction}", flush=True)
        loss, rewards, slopes = (torch.full((n,), float("nan"), device="cuda")
                                 for n in (pairs if reduction == 0 else 1, sequences, sequences))
        ws = workspace(lib.ti_preference_workspace, 0, sequences)
        t, r = tokens.data_ptr(), rewards.data_ptr()
        rc = lib.ti_preference(t, t, mask, off, 0, sequences, 0, 0, 0.1, 0.0, 0, reduction, loss.data_ptr(), r, r + 4 * pairs,
                               slopes.data_ptr(), _ext.F32, ws.data_ptr(), ws.numel(), stream)
        assert rc == 0, lib.ti_last_error().decode()
        torch.testing.assert_close(loss.cpu(), torch.full_like(loss.cpu(), want), rtol=1e-6, atol=0)
        assert not bool(rewards.any()) and bool(slopes.isfinite().all())
        assert lib.ti_preference_bwd(mask, off, 0, sequences, 0, slopes.data_ptr(), loss.data_ptr(), int(reduction == 0), t,
                                     _ext.F32, stream) == 0
    assert not bool(tokens.any())
