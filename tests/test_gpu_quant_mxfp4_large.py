"""ds41_quantize_mxfp4 from 2^20 pieces of eight entries on, where a thread takes four: the same bits as slices of few rows, which are
held to the rule in 64 bits (test_gpu_quant_mxfp4.py) and take one; nothing behind the outputs is written."""
import numpy as np
import pytest

import ds41_gfx950 as G
import test_gpu_quant_mxfp4 as Q

pytestmark = pytest.mark.gpu


def outputs(gpu, rows, cols):
    """Tensors at the start of buffers whose rest holds a mark."""
    import torch
    made = []
    for width, dtype in ((cols // 2, torch.uint8), (cols // 32, torch.uint8), (cols, torch.bfloat16)):
        b = torch.full((rows * width + 4096,), 77, dtype=dtype, device=gpu)
        made.append((b, b[:rows * width].view(rows, width)))
    return [b for b, _ in made], [t for _, t in made]


def check(gpu, x, slices, ruled):
    import torch
    rows, cols = x.shape
    (buffers, (codes, scales, values)) = outputs(gpu, rows, cols)
    G.quantize_mxfp4(x, codes=codes, scales=scales, values=values)
    for b, t in zip(buffers, (codes, scales, values)):
        assert (b[t.numel():] == 77).all()
    q, s, _ = G.quantize_mxfp4(x)  # nothing else written where no values are asked for
    assert torch.equal(q, codes) and torch.equal(s, scales)
    bits = values.view(torch.int16)
    for rs, cs in slices:
        part = x[rs, cs]
        assert part.numel() // 8 < 1 << 20
        a, b, v = G.quantize_mxfp4(part, values=True)
        c0 = (cs.start or 0)
        c1 = cols if cs.stop is None else min(cs.stop, cols)
        assert torch.equal(codes[rs, c0 // 2:c1 // 2], a) and torch.equal(scales[rs, c0 // 32:c1 // 32], b)
        assert torch.equal(bits[rs, c0:c1], v.view(torch.int16))
    if ruled.stop == ruled.start:
        return
    wq, ws, wv = Q.rule(x[ruled].float().cpu().numpy().reshape(1, -1))
    assert np.array_equal(scales[ruled].cpu().numpy().reshape(1, -1), ws) and np.array_equal(codes[ruled].cpu().numpy().reshape(1, -1), wq)
    got = values[ruled].float().cpu().numpy().astype(np.float64).reshape(1, -1)
    assert np.array_equal(np.isnan(got), np.isnan(wv)) and np.array_equal(np.nan_to_num(got), np.nan_to_num(wv))


def make(gpu, rows, cols, ld, dtype):
    """Rows of sizes far apart; a few groups with infinities or NaN, of zeros, and of subnormal numbers."""
    import torch
    g = torch.Generator(device=gpu).manual_seed(rows + cols)
    b = torch.full((rows, ld), float("nan"), dtype=dtype, device=gpu)
    x = b[:, :cols]
    v = torch.empty((rows, cols), device=gpu).normal_(0, 1, generator=g)
    v *= torch.exp2(torch.randint(-60, 60, (rows, cols // 32, 1), device=gpu, generator=g).float()).expand(-1, -1, 32).reshape(rows, cols)
    x.copy_(v)
    if rows > 8:
        x[3, :32], x[5, 64], x[7, 40], x[rows - 1, cols - 1], x[rows - 2, -32:] = 0.0, float("inf"), float("nan"), -float("inf"), 1e-40
    return x


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,cols,pad", [(2311, 3680, 0), (2311, 3680, 5), (2304, 5120, 0), (70001, 160, 0), (70001, 160, 32)])
def test_rows(gpu, rows, cols, pad, dtype):
    """Whole and partial last workgroups, with rows side by side and apart."""
    import torch
    x = make(gpu, rows, cols, cols + pad, getattr(torch, dtype))
    assert rows * cols // 8 >= 1 << 20
    step = min(rows, (1 << 19) // (cols // 8))
    check(gpu, x, [(slice(i, min(i + step, rows)), slice(None)) for i in range(0, rows, step)], slice(rows - 3, rows))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("groups", [(1 << 18) - 1, 1 << 18, (1 << 18) + 1, (1 << 18) + 255])
def test_one_row_around_the_change(gpu, groups, dtype):
    """2^20 pieces but one group, exactly, and with a last workgroup of four pieces."""
    import torch
    x = make(gpu, 1, 32 * groups, 32 * groups, getattr(torch, dtype))
    step = 32 << 17
    check(gpu, x, [(slice(0, 1), slice(i, min(i + step, 32 * groups))) for i in range(0, 32 * groups, step)], slice(0, 0))
