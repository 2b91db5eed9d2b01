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


@pytest.mark.parametrize("scale", [1e-3, 1.0, 1e38])
@pytest.mark.parametrize("in_place", [False, True])
def test_own_norms(gpu, scale, in_place):
    """The norm of the call itself is not rounded on its way to the factor, and may be beyond the largest number of 32 bits."""
    import torch
    import ds41_gfx950 as G
    for seed in range(3):
        grads = [make(gpu, torch.float32, scale, 30001 + seed), make(gpu, torch.bfloat16, scale, 7), make(gpu, torch.float32, scale, 1)]
        b = [t.double().cpu().numpy() for t in grads]
        norm = math.sqrt(math.fsum(float(np.dot(t / scale, t / scale)) for t in b)) * scale
        out = None if in_place else [torch.full_like(t, 7) for t in grads]
        got = float(G.grad_clip(grads, scale * 2.0, out=out))
        with np.errstate(over="ignore"):
            assert got == np.float32(norm) or abs(got - norm) <= norm * 1.01 * 2.0 ** -24
        factor = float(np.float32(scale * 2.0)) / (norm + 1e-6)
        for t, v in zip(out or grads, b):
            close(t, v * factor, t.dtype)


def test_norm_and_clipping_in_one_call(gpu):
    """As the two calls one after the other where 32 bits hold the norm exactly; captured, and with no workspace of its own."""
    import torch
    import ds41_gfx950 as G
    a = torch.tensor([3.0, -4.0, 12.0, 84.0], device=gpu)
    square, norm, out = torch.empty(1, dtype=torch.float64, device=gpu), torch.empty(1, device=gpu), torch.empty_like(a)
    ws = torch.empty(G.lib().ds41_grad_workspace_bytes(1), dtype=torch.uint8, device=gpu)
    G.grad_clip([a], 8.5, out=[out], norm=norm, square_sum=square, workspace=ws)
    two = torch.empty_like(a)
    G.grad_clip([a], 8.5, out=[two], norm=norm, known=True)
    assert float(norm) == 85.0 and float(square) == 7225.0 and torch.equal(out, two)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        G.grad_clip([a], 8.5, out=[out], norm=norm, square_sum=square, workspace=ws)
    for i in range(3):
        for t in (out, norm, square, ws):
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert float(norm) == 85.0 and float(square) == 7225.0 and torch.equal(out, two)
        a.sum().item()
