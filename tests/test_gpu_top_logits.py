"""ds41_top_logits: ids and values equal a stable sort; the sums against 64 bits.

Bound of lse: a term's exponent (|a| <= 2^-24 relative, weighted mean of |a| at most log2 V + 2) and its exp2
(two steps) put at most (log2 V + 4) 2^-23 on the sum, the adds (a thread's, the lanes', the waves', the
chunks': at most 32 + 6 + 8 + 70) 2^-24 each; then max / T, the logarithm and one add of up to |lse|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def lse_bound(V, lse):
    return (np.log2(V) + 4) * 2.0 ** -23 + 116 * 2.0 ** -24 + 6 * 2.0 ** -24 * (np.abs(lse) + 1)


def check(gpu, x, k, T=1.0, chosen=None, ws=None):
    """x: fp32 or bf16 tensor with any row stride."""
    import torch
    import ds41_gfx950 as G
    n, V = x.shape
    ids, values, lse, lp = G.top_logits(x, k, temperature=T, chosen=chosen, workspace=ws)
    xd = x.double().cpu().numpy()
    ids, values, lse = ids.cpu().numpy(), values.cpu().numpy(), lse.cpu().numpy().astype(np.float64)
    for r in range(n):
        row = xd[r]
        if np.isnan(row).any() or (row == np.inf).any():
            assert (ids[r] == -1).all() and np.isnan(values[r]).all() and np.isnan(lse[r])
            assert lp is None or bool(torch.isnan(lp[r]))
            continue
        order = np.argsort(-(row + 0.0), kind="stable")[:k]
        assert np.array_equal(ids[r], order), (r, ids[r][:8], order[:8])
        assert np.array_equal(values[r].astype(np.float64), row[order]) and not np.signbit(values[r][values[r] == 0]).any()
        if np.isneginf(row).all():
            assert np.isneginf(lse[r])
            continue
        m = row.max() / T
        want = m + np.log(np.exp(row / T - m).sum())
        assert abs(lse[r] - want) <= lse_bound(V, want), (r, lse[r], want)
        if chosen is not None:
            c = int(chosen[r])
            if not 0 <= c < V:
                assert bool(torch.isnan(lp[r]))
            elif np.isfinite(row[c]):
                assert abs(float(lp[r]) - (row[c] / T - want)) <= lse_bound(V, want) + 4 * 2.0 ** -24 * (abs(row[c] / T) + abs(want))
            else:
                assert float(lp[r]) == -np.inf


def rows(gpu, kind, n, V, dtype, seed=0):
    import torch
    g = torch.Generator(device=gpu).manual_seed(seed + V)
    x = torch.empty((n, V), device=gpu).normal_(0, 2.5, generator=g)
    if kind == "ties":
        x = torch.randint(-2, 3, (n, V), device=gpu, generator=g).float()
    elif kind == "equal":
        x = torch.full((n, V), 1.5, device=gpu)
    elif kind == "ascending":
        x = torch.arange(V, device=gpu).float().repeat(n, 1) * 1e-3
    elif kind == "descending":
        x = -torch.arange(V, device=gpu).float().repeat(n, 1) * 1e-3
    elif kind == "peaks":  # the largest all in one stretch, which few threads of one workgroup hold
        x[:, V // 2:V // 2 + 300] += 50 + torch.arange(min(300, V - V // 2), device=gpu)
    elif kind == "masked":
        x = torch.where(torch.rand((n, V), device=gpu, generator=g) < 0.999, -float("inf"), x)
        x[:, V // 3] = 2.0
    elif kind == "lowest":
        x = torch.where(torch.rand((n, V), device=gpu, generator=g) < 0.9999, torch.finfo(torch.float32).min, x)
        x[:, V // 3] = 2.0
    elif kind == "zeros":
        x = torch.where(torch.rand((n, V), device=gpu, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "periodic":  # every stretch of the row holds the same large values
        x = (torch.arange(V, device=gpu) % 4096).float().repeat(n, 1)
    return x.to(dtype)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 500, 4095, 4097, 16385, 50257, 129280, 129281])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sizes(gpu, V, dtype):
    import torch
    for n in (1, 3):
        x = rows(gpu, "normal", n, V, getattr(torch, dtype))
        for k in sorted({1, min(V, 5), min(V, 64), min(V, 128)}):
            chosen = torch.tensor([V - 1, -1, V][:n], dtype=torch.int32, device=gpu)
            check(gpu, x, k, T=0.7 if k == 5 else 1.0, chosen=chosen)


@pytest.mark.parametrize("kind", ["ties", "equal", "ascending", "descending", "peaks", "masked", "lowest", "zeros", "periodic"])
def test_distributions(gpu, kind):
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        for V in (700, 9000, 129281):
            for k in (1, 20, 128):
                check(gpu, rows(gpu, kind, 2, V, dtype), k)


@pytest.mark.parametrize("n", [70, 300, 1500])
def test_many_rows(gpu, n):
    """Enough rows that the chunks are the long ones."""
    import torch
    for dtype, V, k in ((torch.float32, 20000, 128), (torch.bfloat16, 33001, 33)):
        x = rows(gpu, "normal", n, V, dtype, seed=n)
        x[:: 7] = rows(gpu, "ties", len(x[:: 7]), V, dtype)
        x[3:: 50] = rows(gpu, "equal", len(x[3:: 50]), V, dtype)
        check(gpu, x, k, T=2.0, chosen=(torch.arange(n, device=gpu) * 31 % V).int())


def test_bad_rows_and_strides(gpu):
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        for V, pad in ((1000, 1), (5001, 3), (40000, 8)):
            buf = torch.full((7, V + pad), float("nan"), dtype=dtype, device=gpu)  # what lies between the rows is not read as theirs
            x = buf[:, :V]
            x.copy_(rows(gpu, "normal", 7, V, dtype))
            x[1, V - 1], x[2, 0], x[3], x[4, 5] = float("nan"), float("inf"), -float("inf"), -float("inf")
            check(gpu, x, 10, chosen=torch.tensor([0, 1, 2, 3, 5, 6, 7], dtype=torch.int32, device=gpu))
            flat = torch.zeros(3 * V + 1, dtype=dtype, device=gpu)
            y = flat[1:].view(3, V)  # a base off by one element
            y.copy_(x[4:7])
            check(gpu, y, 10)


def test_small_temperature(gpu):
    """At a temperature of 1e-5 and less one token holds all the mass: lse is max / T, rounded, and its log-probability 0
    to the sum's bound; 1e-37 overflows max * log2(e) / T."""
    import torch
    import ds41_gfx950 as G
    x = torch.randn(4, 5000, device=gpu) * 3
    best = x.max(1)
    for T in (1e-5, 1e-20, 1e-37):
        ids, values, lse, lp = G.top_logits(x, 3, temperature=T, chosen=best.indices.int())
        assert torch.equal(ids[:, 0], best.indices.int()) and torch.equal(values[:, 0], best.values)
        want = best.values.double() / T
        assert bool(((lse.double() - want).abs() <= 2.0 ** -22 * want.abs()).all()) and float(lp.abs().max()) <= lse_bound(5000, 0)


def test_longest_vocabulary(gpu):
    import torch
    V = 1 << 20
    x = rows(gpu, "normal", 2, V, torch.float32)
    x[1] = (torch.arange(V, device=gpu) % 16384).float()
    check(gpu, x, 128)
    check(gpu, x[:1].bfloat16(), 1)


def test_parts_alone(gpu):
    """ids without sums and sums without ids, through the C entry."""
    import torch
    import ds41_gfx950 as G
    n, V, k = 4, 50000, 16
    x = rows(gpu, "normal", n, V, torch.float32)
    ids, values, lse, lp = G.top_logits(x, k, chosen=torch.arange(n, dtype=torch.int32, device=gpu))
    ws = torch.empty(G.lib().ds41_top_logits_workspace_bytes(n, V, k), dtype=torch.uint8, device=gpu)
    i2, v2, l2, p2 = torch.zeros_like(ids), torch.zeros_like(values), torch.zeros_like(lse), torch.zeros_like(lp)
    c = torch.arange(n, dtype=torch.int32, device=gpu)
    args = lambda i, v, s, ch, p: (x.data_ptr(), 0, V, n, V, k, 1.0, i, v, s, ch, p, ws.data_ptr(), ws.numel(), G._stream())  # noqa: E731
    assert G.lib().ds41_top_logits(*args(i2.data_ptr(), v2.data_ptr(), None, None, None)) == 0
    assert torch.equal(i2, ids) and torch.equal(v2, values)
    assert G.lib().ds41_top_logits(*args(None, None, l2.data_ptr(), None, None)) == 0 and torch.equal(l2, lse)
    assert G.lib().ds41_top_logits(*args(None, None, None, c.data_ptr(), p2.data_ptr())) == 0 and torch.equal(p2, lp)


def test_two_streams_and_graph(gpu):
    """Two calls at once on two workspaces, and a captured one replayed on new rows."""
    import torch
    import ds41_gfx950 as G
    a, b = rows(gpu, "normal", 64, 50257, torch.float32, 1), rows(gpu, "normal", 64, 50257, torch.bfloat16, 2)
    want_a, want_b = G.top_logits(a, 32), G.top_logits(b, 32)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            got_a = G.top_logits(a, 32)
        with torch.cuda.stream(s2):
            got_b = G.top_logits(b, 32)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got_a[:3] + got_b[:3], want_a[:3] + want_b[:3]))
    x = a[:4].clone()
    ws = torch.empty(G.lib().ds41_top_logits_workspace_bytes(4, 50257, 20), dtype=torch.uint8, device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = G.top_logits(x, 20, workspace=ws)
    for i in range(4):
        x.copy_(a[4 * i:4 * i + 4])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out[:3], G.top_logits(x, 20)[:3]))


def test_sums_beyond_fp32_and_gaps_beyond_it(gpu):
    """The log-probability is a difference that fp32 holds where max / T lies below its range, and where two logits are
    further apart than its range while T brings them together."""
    import torch
    import ds41_gfx950 as G
    x = torch.randn(3, 50257, device=gpu) - 100
    best = x.max(1)
    for T in (1e-37, 2e-38):
        ids, values, lse, lp = G.top_logits(x, 2, temperature=T, chosen=best.indices.int())
        assert bool((lse == -float("inf")).all()) and torch.equal(ids[:, 0], best.indices.int())
        assert float(lp.abs().max()) <= lse_bound(50257, 0)
        second = G.top_logits(x, 2, temperature=T, chosen=ids[:, 1].contiguous())[3].double()
        want = (values[:, 1].double() - values[:, 0].double()) / float(np.float32(T))
        want = torch.where(want < -torch.finfo(torch.float32).max, -float("inf"), want)
        assert bool(((second == want) | ((second - want).abs() <= 2.0 ** -22 * want.abs())).all())
    for n, V in ((2, 50257), (300, 40000)):  # short and long chunks
        x = torch.full((n, V), -3e38, device=gpu)
        x[:, 30000:30010], x[0, 17], x[1, 20000:20004] = 3e38, 1e38, 2e38
        for T in (1e38, 5e37):
            z = x.double() / float(np.float32(T))
            for c in (0, 17, 30005):
                chosen = torch.full((n,), c, dtype=torch.int32, device=gpu)
                lse, lp = G.top_logits(x, 3, temperature=T, chosen=chosen)[2:]
                want = z.logsumexp(1)
                # exponents of up to 12, each a few roundings
                assert float((lse.double() - want).abs().max()) <= lse_bound(V, 12)
                assert float((lp.double() - (z[:, c] - want)).abs().max()) <= lse_bound(V, 12) + 24 * 2.0 ** -22
