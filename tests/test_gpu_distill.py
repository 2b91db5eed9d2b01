"""ds41_distill_{forward,backward,step} against the formulas in 64 bits, and the gradient against differences of
the loss.

Bounds. S = (log2 V + 4) 2^-23 + 116 2^-24 bounds the relative error of a sum over the vocabulary (see
test_gpu_top_logits.py), so log-sum-exps are off by S plus their rounding. The set's part is 64-bit. loss: the
log q of the set and of the rest shift by at most 2 S each, weighted with probabilities that add up to 1, and
the loss is rounded once. Gradient of an entry outside: exp2 of a rounded argument (|z| + |lse|, three roundings
of 2^-24, two steps of exp2), the saved statistics' rounding, and p_r / q_r off by 2 S; inside: q - P with q's
error. Then the product with g / T (three steps) and the output's half step."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def S(V):
    return (np.log2(V) + 4) * 2.0 ** -23 + 116 * 2.0 ** -24


def reference(x, ids, t, tlse, T):
    """(loss, stats [n][2], derivative d loss / d logit, set mask, p_r / q_r [n][1]) in 64 bits."""
    n, V = x.shape
    z = x.astype(np.float64) / T
    loss, stats, d = np.zeros(n), np.zeros((n, 2)), np.zeros((n, V))
    inset, ratio = np.zeros((n, V), bool), np.zeros((n, 1))
    for r in range(n):
        ok = (ids[r] >= 0) & (ids[r] < V) & ~np.isneginf(t[r])
        if not ok.any():
            continue
        tz = t[r][ok].astype(np.float64) / T
        if tlse is None:
            w = np.exp(tz - tz.max())
            p = w / w.sum()
        else:
            p = np.exp(tz - float(tlse[r]))
        P = np.zeros(V)
        np.add.at(P, ids[r][ok], p)
        inset[r, ids[r][ok]] = True
        i = inset[r]
        m = z[r].max()
        e = np.exp(z[r] - m)
        lse = m + np.log(e.sum())
        q = e / e.sum()
        with np.errstate(divide="ignore", invalid="ignore"):
            logq = z[r] - lse
            pos = i & (P > 0)
            loss[r] = np.sum(P[pos] * (np.log(P[pos]) - logq[pos]))
            d[r] = q - P
            stats[r, 0] = lse
            if tlse is not None:
                inside, outside = e[i].sum(), e[~i].sum()
                logr = -np.log1p(inside / outside) if outside else -np.inf
                pr = max(0.0, 1 - p.sum()) if outside or not i.all() else 0.0
                if pr > 0:
                    loss[r] += pr * (np.log(pr) - logr)
                    ratio[r] = pr / np.exp(logr)
                d[r] = np.where(i, q - P, q * (1 - ratio[r]))
                stats[r, 1] = logr
    return loss, stats, d / T, inset, ratio


def grad_bound(x, stats, d, inset, ratio, g, T, half):
    V = x.shape[1]
    z, lse = np.abs(x.astype(np.float64)) / T, np.abs(stats[:, :1])
    q = np.exp(np.minimum(x.astype(np.float64) / T - stats[:, :1], 0))
    z = np.where(np.isfinite(z), z, 0)
    rel = S(V) + 2.0 ** -23 * (3 * (z + lse) + 4)
    scale = np.where(inset, 1.0, np.abs(1 - ratio))
    logr = np.where(np.isinf(stats[:, 1:]), 0, np.abs(stats[:, 1:]))
    tol = q * scale * rel + np.where(inset, 0.0, q * ratio * (2 * S(V) + 2.0 ** -22 * (logr + 1)))
    gT = np.abs(g)[:, None] / T
    tol = 1.05 * gT * tol + 4 * 2.0 ** -24 * np.abs(d) * np.abs(g)[:, None]
    return tol + half * (np.abs(d) * np.abs(g)[:, None] + tol) + 2e-38


def make(gpu, seed, n, V, k, dtype, T, rest, noise=0.5, pad=0):
    import torch
    g = torch.Generator(device=gpu).manual_seed(seed)
    buf = torch.full((n, V + pad), float("nan"), dtype=dtype, device=gpu)
    x = buf[:, :V]
    base = torch.empty((n, V), device=gpu).normal_(0, 2.5, generator=g)
    base[:, :: max(1, V // 50)] += 8
    x.copy_(base)
    t = x.float() + torch.empty((n, V), device=gpu).normal_(0, noise, generator=g)
    best = t.topk(k, dim=1)
    ids, tl = best.indices.int(), best.values.contiguous()
    tlse = (t.double() / T).logsumexp(1).float() if rest else None
    return x, ids, tl, tlse, 0.5 + torch.rand(n, device=gpu, generator=g)


def check(x, ids, tl, tlse, gl, T, in_place=False):
    import torch
    import ds41_gfx950 as G
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
    xn, n, V = x.double().cpu().numpy(), *x.shape
    want, wstats, d, inset, ratio = reference(xn, ids.cpu().numpy(), tl.cpu().numpy(), None if tlse is None else tlse.cpu().numpy(), T)
    loss, stats = G.distill_forward(x, ids, tl, teacher_lse=tlse, temperature=T)
    ln, sn = loss.double().cpu().numpy(), stats.double().cpu().numpy()
    assert np.all(np.abs(ln - want) <= 4 * S(V) + 2.0 ** -24 * np.abs(want)), np.max(np.abs(ln - want))
    assert np.array_equal(np.isinf(sn), np.isinf(wstats))  # log q_r of a set that is the whole vocabulary
    sn, fin = np.where(np.isinf(wstats), 0, sn), np.where(np.isinf(wstats), 0, wstats)
    assert np.all(np.abs(sn - fin) <= 2 * S(V) + 2.0 ** -23 * np.abs(fin)), np.max(np.abs(sn - fin))
    gn = gl.double().cpu().numpy()
    tol = grad_bound(xn, wstats, d, inset, ratio, gn, T, half)
    outs = [G.distill_backward(x, ids, tl, stats, gl, teacher_lse=tlse, temperature=T)]
    l2, s2, g2 = G.distill_step(x, ids, tl, gl, teacher_lse=tlse, temperature=T)
    outs.append(g2)
    assert np.all(np.abs(l2.double().cpu().numpy() - want) <= 4 * S(V) + 2.0 ** -24 * np.abs(want))
    assert np.all(np.abs(np.where(np.isinf(wstats), 0, s2.double().cpu().numpy()) - fin) <= 2 * S(V) + 2.0 ** -23 * np.abs(fin))
    if in_place:
        y = x.clone() if x.is_contiguous() else x
        G.distill_step(y, ids, tl, gl, teacher_lse=tlse, temperature=T, grad=y)
        outs.append(y)
    for got in outs:
        off = np.abs(got.double().cpu().numpy() - d * gn[:, None])
        assert np.all(off <= tol), (float(np.max(off / tol)), np.unravel_index(np.argmax(off / tol), off.shape))
    again = G.distill_step(x, ids, tl, gl, teacher_lse=tlse, temperature=T) if not in_place else None
    if again:
        assert torch.equal(again[0], l2) and torch.equal(again[2], g2)  # the same bits again


@pytest.mark.parametrize("V", [1, 2, 7, 64, 500, 16384, 16385, 50257, 129281])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sizes(gpu, V, dtype):
    import torch
    for n, k, T, rest in ((1, 1, 1.0, False), (3, 20, 1.0, True), (2, 128, 2.0, True), (5, 33, 1.5, False)):
        x, ids, tl, tlse, gl = make(gpu, V + k, n, V, min(k, V), getattr(torch, dtype), T, rest)
        check(x, ids, tl, tlse, gl, T)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_rows_and_strides(gpu, dtype):
    import torch
    dt = getattr(torch, dtype)
    for n, V, k, T, rest, pad in ((600, 3001, 64, 1.0, True, 0), (300, 33000, 20, 2.0, False, 0), (40, 5000, 16, 1.0, True, 1), (40, 5000, 16, 1.0, False, 8),
                                  (3500, 3001, 10, 1.0, True, 1), (800, 16384, 100, 1.0, True, 0), (700, 16385, 5, 1.5, False, 3), (450, 30001, 33, 1.0, True, 0),
                                  (110, 100003, 64, 1.0, True, 1), (90, 129281, 128, 2.0, False, 0)):
        x, ids, tl, tlse, gl = make(gpu, n, n, V, k, dt, T, rest, pad=pad)
        check(x, ids, tl, tlse, gl, T)
        check(x, ids, tl, tlse, gl, T, in_place=True)


@pytest.mark.parametrize("rest", [False, True])
def test_left_out_and_repeated_entries(gpu, rest):
    """Padding ids, ids outside, logits of -infinity, the same id twice, rows with nothing in their set."""
    import torch
    import ds41_gfx950 as G
    n, V, k = 8, 4000, 12
    for dt in (torch.float32, torch.bfloat16):
        x, ids, tl, tlse, gl = make(gpu, 3, n, V, k, dt, 1.0, rest)
        ids[0, 5:], ids[1, 0], ids[1, 1] = -1, V, -7
        tl[2, 3:] = -float("inf")
        ids[3, 4], tl[3, 4] = ids[3, 0], tl[3, 0] - 1
        ids[4, :] = ids[4, 0]
        if rest:
            tlse[4] += 5
        ids[5] = -1
        tl[6] = -float("inf")
        tl[0, 7] = float("nan")  # an entry left out by its id: its logit is not looked at
        clean = tl.clone()
        clean[0, 7] = 0
        check(x, ids, clean, tlse, gl, 1.0)
        x[5], x[6, 0] = float("nan"), float("inf")  # padding rows hold anything
        for got in (G.distill_step(x, ids, tl, gl, teacher_lse=tlse),
                    (*(f := G.distill_forward(x, ids, tl, teacher_lse=tlse)), G.distill_backward(x, ids, tl, f[1], gl, teacher_lse=tlse))):
            assert not bool(got[0][5:7].any()) and not bool(got[1][5:7].any()) and not bool(got[2][5:7].any())
            assert bool(torch.isfinite(got[0]).all()) and bool(torch.isfinite(got[2]).all())


def test_masked_student_entries_and_bad_rows(gpu):
    import torch
    import ds41_gfx950 as G
    n, V, k = 6, 9000, 10
    for rest in (False, True):
        for low in (-float("inf"), torch.finfo(torch.float32).min):
            x, ids, tl, tlse, gl = make(gpu, 5, n, V, k, torch.float32, 1.0, rest)
            keep = torch.zeros_like(x, dtype=torch.bool)
            keep.scatter_(1, ids.long(), True)
            keep[:, :: 7] = True
            x = torch.where(keep, x, low)  # a grammar's mask outside the set
            check(x, ids, tl, tlse, gl, 1.0)
        x[1, 17], x[2, int(ids[2, 0])] = float("nan"), float("nan")
        x[3, int(ids[3, 0])] = -float("inf")  # the student rules out what the teacher wants
        tl[4, 2] = float("nan")
        loss, stats, grad = G.distill_step(x, ids, tl, gl, teacher_lse=tlse)
        assert bool(torch.isnan(loss[[1, 2, 4]]).all()) and bool(loss[3] == float("inf"))
        assert bool(torch.isnan(grad[1]).any()) and bool(torch.isnan(grad[2]).any()) and bool(torch.isnan(grad[4]).any())
        assert bool(torch.isfinite(loss[[0, 5]]).all()) and bool(torch.isfinite(grad[[0, 3, 5]]).all())


@pytest.mark.parametrize("rest", [False, True])
def test_gradient_against_differences(gpu, rest):
    """(loss(x + h v) - loss(x - h v)) / 2h along v with entries in [-1, 1]. The loss is off by 4 S (2e-5) and its
    third derivative along v is a third cumulant of a variable in [-1, 1] (below 1) for the log-sum-exp, and another
    for the rest: h^2 / 6 * 2 + 2 * 4 S / 2h, with h = 1 / 16."""
    import torch
    import ds41_gfx950 as G
    n, V, k, h = 16, 3000, 24, 1 / 16
    x, ids, tl, tlse, _ = make(gpu, 11, n, V, k, torch.float32, 1.0, rest, noise=1.5)
    one = torch.ones(n, device=gpu)
    loss, stats, grad = G.distill_step(x, ids, tl, one, teacher_lse=tlse)
    for seed in range(4):
        g = torch.Generator(device=gpu).manual_seed(seed)
        v = torch.rand((n, V), device=gpu, generator=g) * 2 - 1
        if seed % 2:  # along the set alone
            v = torch.zeros_like(v).scatter_(1, ids.long(), v[:, :k])
        up, down = (G.distill_forward(x + s * h * v, ids, tl, teacher_lse=tlse)[0].double() for s in (1, -1))
        off = (up - down) / (2 * h) - (grad.double() * v.double()).sum(1)
        assert float(off.abs().max()) <= h * h / 3 + 4 * S(V) / h + 1e-4, float(off.abs().max())


@pytest.mark.parametrize("rest", [False, True])
def test_rows_held_whole_hold_what_chunks_give(gpu, rest):
    """Enough bytes that a step keeps its rows in registers: padding, repeated ids, masked, NaN and infinite entries as in
    few rows, which go in chunks."""
    import torch
    import ds41_gfx950 as G
    for dt, n, V in ((torch.bfloat16, 1200, 9000), (torch.float32, 600, 9001)):
        x, ids, tl, tlse, gl = make(gpu, 9, n, V, 20, dt, 1.0, rest)
        keep = torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids.long(), True)
        keep[:, ::5] = True
        x[::3] = torch.where(keep[::3], x[::3], torch.finfo(torch.float32).min if dt == torch.float32 else -float("inf"))
        ids[1, 3:] = -1
        tl[2, 4:] = -float("inf")
        ids[4, 6], ids[7], x[10, 77], x[11, int(ids[11, 0])] = ids[4, 0], -1, float("nan"), float("nan")
        x[12, 5], x[13, int(ids[13, 3])], x[14] = float("inf"), -float("inf"), torch.finfo(torch.float32).min
        x[15] = -float("inf")
        x[16, int(ids[16, 1])] = 90.0  # far above what lies outside the set
        whole = G.distill_step(x, ids, tl, gl, teacher_lse=tlse)
        for a in range(0, 40, 8):
            b = a + 8
            few = G.distill_step(x[a:b], ids[a:b], tl[a:b], gl[a:b], teacher_lse=None if tlse is None else tlse[a:b])
            for u, v, tol in zip(whole, few, (4 * S(V), 4 * S(V), 2.0 ** -7 if dt == torch.bfloat16 else 1e-4)):
                u, v = u[a:b].double(), v.double()
                assert bool((torch.isnan(u) == torch.isnan(v)).all()) and bool((torch.isinf(u) == torch.isinf(v)).all())
                fin = torch.isfinite(v)
                # both within the bound of the formula, so within twice that of each other; gradients by their half step
                assert bool(((u - v).abs()[fin] <= 2 * tol * (1 + v.abs()[fin])).all()), float(((u - v).abs()[fin] / (1 + v.abs()[fin])).max())


def test_teacher_is_student(gpu):
    """The student's own top logits with its own log-sum-exp: loss and gradient vanish."""
    import torch
    import ds41_gfx950 as G
    x = torch.randn(5, 20000, device=gpu) * 2.5
    ids, values, lse, _ = G.top_logits(x, 50)
    loss, stats, grad = G.distill_step(x, ids, values, torch.ones(5, device=gpu), teacher_lse=lse)
    assert float(loss.abs().max()) <= 4 * S(20000) and float(grad.abs().max()) <= 1e-5


def test_streams_and_graph(gpu):
    import torch
    import ds41_gfx950 as G
    n, V, k = 6, 50257, 20
    x, ids, tl, tlse, gl = make(gpu, 1, n, V, k, torch.bfloat16, 1.0, True)
    ws = torch.empty(G.lib().ds41_distill_workspace_bytes(n, V), dtype=torch.uint8, device=gpu)
    loss, stats, grad = torch.empty(n, device=gpu), torch.empty(n, 2, device=gpu), torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        G.distill_step(x, ids, tl, gl, teacher_lse=tlse, loss=loss, stats=stats, grad=grad, workspace=ws)
    for i in range(4):
        y, ids2, tl2, tlse2, gl2 = make(gpu, 20 + i, n, V, k, torch.bfloat16, 1.0, True)
        for a, b in ((x, y), (ids, ids2), (tl, tl2), (tlse, tlse2), (gl, gl2)):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        want = G.distill_step(y, ids2, tl2, gl2, teacher_lse=tlse2)
        assert torch.equal(loss, want[0]) and torch.equal(stats, want[1]) and torch.equal(grad, want[2])
