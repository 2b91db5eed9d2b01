"""Clipping where a factor of 32 bits would not do: far from 1, and next to the last bit.

Bounds. The factor max_norm / (norm + 1e-6) is formed in 64 bits from the norm (a given one: as it is given), and its product with an
element too, so that the element takes its rounding to 32 bits, half a step (2^-24 of itself; of a subnormal number 2^-150), and
a bf16 one then another (2^-8; 2^-134). What 64 bits lose, a few 2^-53, is within the hundredth that is added."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def make(gpu, dtype, scale, n=20011):
    import torch
    g = torch.Generator(device=gpu).manual_seed(n)
    return (torch.randn(n, device=gpu, dtype=torch.float64, generator=g).clamp(-3, 3) * scale).to(dtype)


def close(got, want, dtype):
    import torch
    off = np.abs(got.double().cpu().numpy() - want)
    tol = np.abs(want) * 2.0 ** -24 + 2.0 ** -150
    if dtype is torch.bfloat16:
        tol = tol + (np.abs(want) + tol) * 2.0 ** -8 + 2.0 ** -134
    assert np.all(off <= 1.01 * tol), float(np.max(off / tol))


@pytest.mark.parametrize("norm,max_norm", [(10.0, 5.0), (3.0, 2.9999), (3e38, 1e-3), (1e25, 1e-30), (2e38, 1.0), (1e-3, 1e-38), (3e20, 1e-25)])
@pytest.mark.parametrize("in_place", [False, True])
def test_known_norms(gpu, norm, max_norm, in_place):
    """Factors down to 1e-55, whose products are ordinary numbers."""
    import torch
    import ds41_gfx950 as G
    for dtype in (torch.float32, torch.bfloat16):
        x = make(gpu, dtype, min(norm, 1e38))
        b = x.double().cpu().numpy()
        out = None if in_place else [torch.full_like(x, 7)]
        G.grad_clip([x], max_norm, out=out, norm=torch.tensor([norm], device=gpu), known=True)
        factor = float(np.float32(max_norm)) / (float(np.float32(norm)) + 1e-6)
        assert factor < 1
        close(x if in_place else out[0], b * factor, dtype)
