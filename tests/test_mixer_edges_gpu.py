"""Operators around a recurrent mixer at the edges of their definitions: 8-bit outputs against
IEEE division, decays of long chunks, infinities at the ends of sequences and chunks and beside
padded states, calls without a sequence, and calls whose stream decides their values."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mixer_oracle as orc

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _n64(t):
    return None if t is None else t.detach().cpu().double().numpy()


# --------------------------------------------------------------------------- norm ----
@pytest.mark.parametrize("group", [None, 32, 64, 128])
@pytest.mark.parametrize("dtype,D", [(F32, 4096), (BF16, 8192), (F16, 1032), (F32, 5003), (BF16, 301),
                                     (F32, 9000), (F16, 8191)])
def test_norm_scales_and_codes_are_ieee_quotients(dtype, D, group):
    """Rows of +-1 have the sum of squares D whatever its order, so the values before the 8-bit
    form are those of the 32-bit call, bit by bit, and scale = amax / 448 and y / scale are
    quotients rounded once: no tolerance."""
    from pto_fuser import add_rms_norm
    for seed in range(6):
        g = _gen(seed)
        w = torch.randn(D, generator=g) * torch.exp(2 * torch.randn(D, generator=g))
        x = torch.randint(0, 2, (3, D), generator=g).mul(2).sub(1).float()
        y = add_rms_norm(x.cuda(), w.cuda())[0].cpu()
        q, _, s = add_rms_norm(x.to(dtype).cuda(), w.cuda(), out_dtype=F8, group_size=group)
        size = group or D
        parts = torch.nn.functional.pad(y, (0, -D % size)).view(3, -1, size)
        scale = torch.clamp(parts.abs().amax(-1) / 448.0, min=2.0 ** -126)
        want = (parts / scale[..., None]).view(3, -1)[:, :D].to(F8)
        assert torch.equal(s.cpu(), scale)
        assert torch.equal(q.cpu().float(), want.float())


def test_norm_to_8_bits_of_values_beyond_the_type():
    """An infinite value has an infinite scale: the others of its group are 0, itself NaN."""
    from pto_fuser import add_rms_norm
    for D in (256, 301):
        w = torch.ones(D)
        w[3] = 3e38
        x = torch.full((2, D), 1.0)
        x[:, 3] = 4.0               # normed to 3.9 and more, so 3e38 times it is infinite
        for group in (None, 128):
            y, _, s = add_rms_norm(x.cuda(), w.cuda(), out_dtype=F8, group_size=group)
            y, s = y.float().cpu(), s.cpu()
            assert torch.isinf(s[:, 0]).all() and torch.isnan(y[:, 3]).all()
            rest = torch.ones(D, dtype=torch.bool)
            rest[3] = False
            assert (y[:, rest][:, :100] == 0).all()
