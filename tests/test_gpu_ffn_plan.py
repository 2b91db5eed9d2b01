"""Every way in which the feed-forward block's products are put into tiles gives the formulas' results.

A product is formed in tiles of 128 or 256, all of them whole, all in parts of the sum that a second launch adds up, or some of each;
its last step of 64 may be full or not. The plan decides by the sizes. What the lists here and in test_gpu_ffn.py reach is checked on
the CPU against a scan of sizes, so that another plan cannot leave a way untested. Bounds: see test_gpu_ffn.py."""
import random

import pytest

import ds41_gfx950 as G
import test_gpu_ffn as F

SIZES = [(405, 4096, 2880), (4125, 4096, 2880), (1152, 1120, 32), (6784, 512, 3712), (1283, 7664, 2200), (768, 3384, 5080), (2941, 6448, 1360),
         (2368, 1280, 6848), (3732, 2240, 2816), (4977, 872, 3336), (3264, 3648, 1152), (5429, 3256, 1032), (7342, 1320, 2248), (1, 8, 32)]


def ways(M, H, I):
    """{(product, side of a tile, whole or split or mixed, a last step that is not full)}."""
    K = dict(gate_up=H, y=I, dh=H, grad_x=2 * I, grad_gate_up=M, grad_one=M, grad_down=M)
    return {(p, side, "whole" if whole == tiles else "mixed" if whole else "split", K[p] % 64 != 0)
            for p, (side, tiles, whole, parts) in G.ffn_plan(M, H, I).items() if side}


def test_the_lists_reach_every_way():
    rng, seen = random.Random(1), set()
    for _ in range(40000):
        M, H, I = int(2 ** rng.uniform(0, 13)), 8 * int(2 ** rng.uniform(0, 10)), 8 * int(2 ** rng.uniform(0, 10))
        if rng.random() < 0.4:
            H, I = max(64, H // 64 * 64), max(64, I // 64 * 64)
        if rng.random() < 0.3:
            M = max(64, M // 64 * 64)
        seen |= ways(M, H, I)
    reached = set().union(*(ways(*s) for s in SIZES + F.sizes()))
    assert len(seen) > 40 and not seen - reached, sorted(seen - reached, key=str)


def test_plans_stay_within_their_workspace():
    """Parts and their sums: at most one round of them, each with steps of its own, in the workspace that the call asks for."""
    rng = random.Random(2)
    sizes = SIZES + F.sizes() + [(int(2 ** rng.uniform(0, 14)), 8 * int(2 ** rng.uniform(0, 10)), 8 * int(2 ** rng.uniform(0, 10))) for _ in range(5000)]
    for M, H, I in sizes:
        K = dict(gate_up=H, y=I, dh=H, grad_x=2 * I, grad_gate_up=M, grad_one=M, grad_down=M)
        held = 6 * ((M * I + 127) // 128 * 128)  # h, dg and du
        for p, (side, tiles, whole, parts) in G.ffn_plan(M, H, I).items():
            if not side:
                continue
            rest = tiles - whole
            assert 0 <= whole <= tiles and parts >= 1 and (rest == 0 or parts >= 2), (M, H, I, p)
            if rest:
                steps = -(-K[p] // 64)
                assert parts * 4 <= steps and rest * parts <= (256 if side == 256 else 512), (M, H, I, p)
                assert held + rest * parts * side * side * 4 <= G.ffn_workspace_bytes(M, H, I), (M, H, I, p)


def test_plan_refusals():
    P = 1 << 20
    for bad in ((0, 64, 64, P), (3, 60, 64, P), (3, 64, 60, P), ((1 << 20) + 1, 64, 64, P), (3, 64, 65544, P), (3, 64, 64, None)):
        assert G.lib().ds41_ffn_plan(*bad) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("M,H,I", SIZES)
def test_sizes(gpu, M, H, I):
    """Forward and backward; the weights' gradients as new ones in bf16, and added in fp32 and in bf16 to what is there; those of the gate
    and of the up projection each alone; what lies behind the outputs stays."""
    import torch
    x, wg, wu, wd, dy = F.make(gpu, M, H, I)
    w = x, wg, wu, wd
    saved = torch.full((M, 2 * I), float("nan"), device=gpu)
    rows = [torch.full((M + 1, H + 8), 7.0, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    y = G.ffn_forward(*w, limit=1.5, out=rows[0][:M, :H], saved=saved)
    F.check_forward(*w, y, saved, 1.5)
    want = F.backward(*w, saved, dy, 1.5)

    def check(got, before=(None,) * 4):
        for (v, tol), t, b in zip(want, got, before):
            if t is None:
                continue
            half = F.B if t.dtype == torch.bfloat16 else F.F
            v = v if b is None else v + b.double()
            tol = tol + half * (v.abs() + tol) + 1e-38
            if b is not None:
                tol = tol + F.F * (v.abs() + b.double().abs() + tol)
            off = (t.double() - v).abs()
            assert (off <= tol).all(), float((off / tol).max())
    check(G.ffn_backward(*w, saved, dy, limit=1.5, grad_x=rows[1][:M, :H]))
    for b in rows:
        assert (b[M] == 7).all() and (b[:, H:] == 7).all()
    for dtype in (torch.float32, torch.bfloat16):
        before = [None] + [torch.randn(s, device=gpu).to(dtype) for s in ((I, H), (I, H), (H, I))]
        behind = [torch.full((t.numel() + 64,), 5.0, dtype=dtype, device=gpu) for t in before[1:]]
        more = [b[:t.numel()].view(t.shape).copy_(t) for b, t in zip(behind, before[1:])]
        check(G.ffn_backward(*w, saved, dy, limit=1.5, grad_x=False, grad_gate=more[0], grad_up=more[1], grad_down=more[2], accumulate=True), before)
        assert all((b[-64:] == 5).all() for b in behind)
    none = dict(grad_x=False, grad_down=False)
    check((None, G.ffn_backward(*w, saved, dy, limit=1.5, grad_up=False, **none)[1], None, None))
    check((None, None, G.ffn_backward(*w, saved, dy, limit=1.5, grad_gate=False, **none)[2], None))


@pytest.mark.gpu
@pytest.mark.parametrize("M,H,I", [(1, 8, 8), (3, 64, 40), (33, 128, 4104), (65, 72, 1000), (300, 1000, 1352), (1152, 1120, 32)])
def test_bf16_gradients_added_to_what_is_there(gpu, M, H, I):
    import torch
    x, wg, wu, wd, dy = F.make(gpu, M, H, I)
    w = x, wg, wu, wd
    saved = torch.empty((M, 2 * I), device=gpu)
    G.ffn_forward(*w, saved=saved)
    before = [None] + [torch.randn(s, device=gpu).bfloat16() for s in ((I, H), (I, H), (H, I))]
    more = [t.clone() for t in before[1:]]
    got = G.ffn_backward(*w, saved, dy, grad_gate=more[0], grad_up=more[1], grad_down=more[2], accumulate=True)
    assert all(a is b for a, b in zip(got[1:], more))
    F.check_backward(w, saved, dy, 0.0, got, before)
