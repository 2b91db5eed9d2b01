"""ds41_dense_bf16 against the product in 64 bits.

Bound: products of two bf16 are exact in fp32; adding K of them (and the bias) in any order loses at most
(K + 2) eps of the sum of their magnitudes, eps = 2^-23 for an adder that truncates. The activations have slope
at most 1.13, and their own evaluation (exp, erf, divide, two products) is off by at most 16 eps of |pre| + |act|.
Then the residual's add (eps of either term) and the one rounding of the output, half a step: 2^-8 or 2^-24."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _act(y, act):
    import torch
    return {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "silu": lambda v: v * torch.special.expit(v),
            "gelu": lambda v: v * torch.special.ndtr(v)}[act](y)


def _rand(gpu, seed, *shape, std=1.0):
    import torch
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.empty(shape, device=gpu).normal_(0, std, generator=g)


def check(y, x, w, bias, residual, act):
    import torch
    xd, wd = x.double(), w.double()
    pre, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        pre, mag = pre + bias.double(), mag + bias.double().abs()
    out = _act(pre, act)
    eps = 2.0 ** -23
    tol = 1.13 * (x.shape[1] + 2) * eps * mag
    if act in ("silu", "gelu"):
        tol = tol + 16 * eps * (pre.abs() + out.abs())
    if residual is not None:
        out = out + residual.double()
        tol = tol + eps * out.abs()
    tol = tol * 1.01 + (out.abs() + tol) * (2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24) + 1e-37
    off = (y.double() - out).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


SHAPES = [  # M, N, K: tiny, GEMV rows, whole tiles, ragged, tall, wide
    (1, 1, 1), (1, 7, 3), (2, 16, 8), (1, 5120, 2304), (3, 129, 513), (4, 4096, 4096), (5, 1000, 2880), (8, 257, 96), (9, 640, 1024),
    (16, 384, 4096), (17, 512, 512), (31, 96, 160), (32, 2304, 5120), (33, 100, 72), (64, 64, 64), (65, 2881, 1007), (100, 4096, 512),
    (128, 128, 32), (129, 384, 136), (200, 5120, 256), (256, 256, 1024), (257, 511, 1032), (300, 33, 8), (512, 2880, 4096), (1000, 96, 2304),
    (5, 70000, 64), (700, 1030, 40), (1, 64, 20000), (48, 64, 16384),
]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_shapes(gpu, M, N, K):
    import torch
    import ds41_gfx950 as G
    x, w = _rand(gpu, M + N, M, K).bfloat16(), _rand(gpu, K, N, K, std=1 / math.sqrt(K)).bfloat16()
    bias, ws = _rand(gpu, 3, N), torch.empty(max(G.dense_bf16_workspace_bytes(M, N, K), 1), dtype=torch.uint8, device=gpu)
    for dt in (torch.bfloat16, torch.float32):
        res = _rand(gpu, 4, M, N).to(dt)
        y = torch.full((M, N), float("nan"), dtype=dt, device=gpu)
        G.dense_bf16(x, w, out=y)
        check(y, x, w, None, None, "none")
        a = G.dense_bf16(x, w, bias=bias, residual=res, act="silu", out_dtype=dt, workspace=ws)
        check(a, x, w, bias, res, "silu")
        assert torch.equal(a, G.dense_bf16(x, w, bias=bias, residual=res, act="silu", out_dtype=dt, workspace=ws))  # same bits again


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("M", [3, 40, 300])
def test_epilogues(gpu, act, M):
    import torch
    import ds41_gfx950 as G
    N, K = 320, 256
    x, w = _rand(gpu, 1, M, K).bfloat16(), _rand(gpu, 2, N, K, std=0.2).bfloat16()
    bias = _rand(gpu, 3, N, std=4.0)
    for dt in (torch.bfloat16, torch.float32):
        for b in (None, bias):
            res = _rand(gpu, 5, M, N).to(dt)
            check(G.dense_bf16(x, w, bias=b, act=act, out_dtype=dt), x, w, b, None, act)
            y = res.clone()
            G.dense_bf16(x, w, bias=b, residual=y, act=act, out=y)  # the residual in place
            check(y, x, w, b, res, act)


@pytest.mark.parametrize("M", [2, 20, 150])
def test_strides_and_alignment(gpu, M):
    """Rows apart by odd and even strides, bases off by one element; what lies between the rows stays."""
    import torch
    import ds41_gfx950 as G
    N, K = 130, 192
    for ldx, ldw, ldy, ox, ow, oy in ((K, K, N, 0, 0, 0), (K + 8, K + 64, N + 6, 8, 16, 2), (K + 1, K + 3, N + 5, 1, 3, 1), (K + 8, K, N + 1, 4, 0, 0)):
        xb, wb = _rand(gpu, 7, M * ldx + ox).bfloat16(), _rand(gpu, 8, N * ldw + ow, std=0.1).bfloat16()
        x, w = xb[ox:].as_strided((M, K), (ldx, 1)), wb[ow:].as_strided((N, K), (ldw, 1))
        for dt in (torch.bfloat16, torch.float32):
            yb = torch.full((M * ldy + oy + 3,), 77.0, dtype=dt, device=gpu)
            y = yb[oy:].as_strided((M, N), (ldy, 1))
            res = _rand(gpu, 9, M, N + 3).to(dt)[:, 1:N + 1]
            G.dense_bf16(x, w, residual=res, out=y)
            check(y, x, w, None, res, "none")
            touched = torch.zeros_like(yb, dtype=torch.bool)
            touched[oy:].as_strided((M, N), (ldy, 1))[:] = True
            assert bool((yb[~touched] == 77).all())


def test_infinities_and_nan_stay_in_their_rows(gpu):
    import torch
    import ds41_gfx950 as G
    for M in (4, 70, 300):
        x, w = _rand(gpu, 1, M, 512).bfloat16(), _rand(gpu, 2, 300, 512).bfloat16()
        x[1, 5], w[17, 511], w[18, 0] = float("nan"), float("inf"), float("nan")
        y, ref = G.dense_bf16(x, w, out_dtype=torch.float32), x.double().cpu() @ w.double().cpu().t()
        fine = torch.isfinite(ref)
        assert bool((torch.isnan(y).cpu() == torch.isnan(ref)).all()) and bool((torch.isinf(y).cpu() == torch.isinf(ref)).all())
        assert bool(((y.cpu().double() - ref)[fine].abs() < 1e-2).all())


def test_other_stream_and_graph(gpu):
    """A captured call replayed on new inputs, with eager work of the same shapes between the replays."""
    import torch
    import ds41_gfx950 as G
    for M, N, K in ((4, 512, 4096), (96, 512, 2048), (512, 1024, 512)):
        x, w = _rand(gpu, 1, M, K).bfloat16(), _rand(gpu, 2, N, K, std=0.02).bfloat16()
        y, ws = torch.empty(M, N, device=gpu), torch.empty(max(1, G.dense_bf16_workspace_bytes(M, N, K)), dtype=torch.uint8, device=gpu)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            G.dense_bf16(x, w, out=y, workspace=ws)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                G.dense_bf16(x, w, out=y, workspace=ws)
        torch.cuda.synchronize()
        for i in range(4):
            x.copy_(_rand(gpu, 10 + i, M, K))
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, G.dense_bf16(x, w, out_dtype=torch.float32, workspace=ws))
