"""One workspace serves every smaller call: the sizes that the dense, top-logits and distillation entries ask for never
fall as a call grows, on the CPU; and on the GPU, calls of every smaller size take the largest one's workspace and give
what they give with their own."""
import itertools

import pytest

import ds41_gfx950 as G

VOCABS = (1, 100, 4096, 4097, 16384, 16385, 50257, 129280, 151936, 1 << 20)
ROWS = sorted({*range(1, 70), 99, 100, 127, 128, 255, 256, 257, 400, 512, 1023, 1024, 1025, 2048, 65535})


def rising(sizes):
    return all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_top_logits_sizes_rise():
    f = G.lib().ds41_top_logits_workspace_bytes
    for V, k in itertools.product(VOCABS, (1, 20, 24, 25, 64, 128)):
        if k <= V:
            assert rising([f(n, V, k) for n in ROWS]), (V, k)
    for V, n in itertools.product(VOCABS, (1, 4, 33, 300)):
        assert rising([f(n, V, k) for k in range(1, min(V, 128) + 1)]), (V, n)
    for n, k in itertools.product((1, 8, 33, 300), (1, 24, 25)):
        assert rising([f(n, V, k) for V in range(k, 140000, 511)]), (n, k)


def test_distill_sizes_rise():
    f = G.lib().ds41_distill_workspace_bytes
    for V in VOCABS:
        assert rising([f(n, V) for n in ROWS]), V
    for n in (1, 8, 33, 300):
        assert rising([f(n, V) for V in range(1, 140000, 511)]), n


def test_dense_sizes_rise_with_rows():
    f = G.lib().ds41_dense_bf16_workspace_bytes
    some = 0
    for N, K in itertools.product((64, 130, 1000, 2880, 4096, 5120, 20001, 129280), (512, 1024, 2304, 4096, 16384, 1 << 20)):
        sizes = [f(M, N, K) for M in (*range(1, 600), *range(600, 5000, 37))]
        assert rising(sizes), (N, K)
        some += sizes[-1] > 0
    assert some > 20  # and most of these products are split at some number of rows


@pytest.mark.gpu
def test_smaller_calls_in_the_largest_ones_workspace(gpu):
    import torch

    def room(size):
        return torch.full((size,), 0xFF, dtype=torch.uint8, device=gpu)
    L, V, most, k = G.lib(), 50257, 90, 33
    x = torch.randn(most, V, device=gpu) * 2.5
    ws = room(L.ds41_top_logits_workspace_bytes(most, V, k))
    dws = room(L.ds41_distill_workspace_bytes(most, V))
    one = torch.ones(most, device=gpu)
    for n, kk in ((1, 1), (1, 33), (78, 20), (79, 20), (80, 24), (78, 25), (90, 33)):  # 13 short chunks a row: 78 rows of them at most
        ids, values, lse, _ = G.top_logits(x[:n], kk, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip((ids, values, lse), G.top_logits(x[:n], kk)[:3])), (n, kk)
        a = G.distill_step(x[:n], ids, values, one[:n], teacher_lse=lse, workspace=dws)
        assert all(torch.equal(p, q) for p, q in zip(a, G.distill_step(x[:n], ids, values, one[:n], teacher_lse=lse))), n
    M, N, K = 600, 4096, 4096
    h, w = torch.randn(M, K, device=gpu).bfloat16(), torch.randn(N, K, device=gpu).bfloat16()
    ws = room(L.ds41_dense_bf16_workspace_bytes(M, N, K))
    big = torch.empty(256 << 20, dtype=torch.uint8, device=gpu)
    for m in (1, 33, 64, 65, 100, 128, 129, 190, 256, 300, 511, 600):
        # with room for whatever parts it takes: the same parts, so the same bits
        assert torch.equal(G.dense_bf16(h[:m], w, workspace=ws), G.dense_bf16(h[:m], w, workspace=big)), m


@pytest.mark.gpu
def test_a_product_without_a_workspace_makes_its_own(gpu):
    """The same parts, so the same bits, as with a workspace, on the current stream, on another and in a graph."""
    import torch
    K = 4096
    s = torch.cuda.Stream()
    for M, N in ((1, 4096), (33, 4096), (64, 4096), (100, 2881), (128, 5120), (200, 640), (512, 4096)):
        x, w = torch.randn(M, K, device=gpu).bfloat16(), torch.randn(N, K, device=gpu).bfloat16() * 0.02
        ws = torch.empty(max(1, G.dense_bf16_workspace_bytes(M, N, K)), dtype=torch.uint8, device=gpu)
        want = G.dense_bf16(x, w, out_dtype=torch.float32, workspace=ws)
        assert torch.equal(G.dense_bf16(x, w, out_dtype=torch.float32), want)
        torch.cuda.synchronize()
        got = G.dense_bf16(x, w, out_dtype=torch.float32, stream=s)
        s.synchronize()
        assert torch.equal(got, want)
        y, g = torch.empty_like(want), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            G.dense_bf16(x, w, out=y)
        for i in range(3):
            x.copy_(torch.randn(M, K, device=gpu))
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, G.dense_bf16(x, w, out_dtype=torch.float32, workspace=ws))
