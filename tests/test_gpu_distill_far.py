"""ds41_distill_* where the student's set and the rest of its row lie far apart, at temperatures from one end of the
range to the other, and for masked rows, against the formulas in 64 bits with every log-sum-exp kept as a maximum and
a logarithm (added up, a masked row's would lose the logarithm).

Bounds. S as in test_gpu_distill.py, for a sum over the vocabulary. With t = |x - max| / T, an entry outside is
weight * exp(-t) / sum: the exponent is off by at most four roundings of t (scale, product, difference), exp2 by two
steps, the product by four more; the weight q_r - p_r by S q_r. Of the saved statistics, 32 bits each, the second holds
what rounding left of the first, and is rounded itself, which counts up to 8,192: from there on the backward call forms
them again. With a rest class, a backward call in place or of bf16 rows takes the first as it is. The rest is 64-bit, and
the output rounds once."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
REACH = 8192.0
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}
KINDS = 10


def S(V):
    return (np.log2(V) + 4) * 2.0 ** -23 + 116 * 2.0 ** -24


def make(gpu, seed, n, V, k, dtype, T, rest):
    """Row r of kind r % KINDS: ordinary; the set 50, 100 and 1,000 (of z) above the rest; the rest all -100, -1e4 and the
    type's lowest; the set 200 below the rest; everything the type's lowest; half the rest the type's lowest."""
    import torch
    g = torch.Generator(device=gpu).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device=gpu).normal_(0, std, generator=g)
    dt = getattr(torch, dtype)
    ids = torch.rand((n, V), device=gpu, generator=g).topk(k, 1).indices
    low = torch.finfo(dt).min
    x = normal(n, V, std=2.5)
    inside = torch.zeros((n, V), dtype=torch.bool, device=gpu).scatter_(1, ids, True)
    kind = torch.arange(n, device=gpu) % KINDS
    x[kind == 0] += 8.0 * inside[kind == 0]
    for i, gap in ((1, 50.0), (2, 100.0), (3, 1000.0), (7, -200.0)):
        x[kind == i] = T * (x[kind == i] + gap * inside[kind == i])
    for i, value in ((4, -100.0), (5, -1e4), (6, low)):
        x[kind == i] = torch.where(inside[kind == i], x[kind == i], value)
    x[kind == 8] = low
    x[kind == 9] = torch.where(inside[kind == 9] | (torch.rand((int((kind == 9).sum()), V), device=gpu, generator=g) < 0.5), x[kind == 9], low)
    tl = normal(n, k, std=2.5) * min(T, 1.0)
    full = (tl.double() / T).logsumexp(1)
    # the rest: a twentieth, or what rounding leaves
    tlse = (full - torch.where(torch.arange(n, device=gpu) % 3 == 1, 0.0, np.log(0.95))).float() if rest else None
    return x.to(dt), ids.int(), tl, tlse, 0.5 + torch.rand(n, device=gpu, generator=g)


def reference(x, ids, tl, tlse, gl, T, half):
    """(loss, stats, gradient, bounds of the loss, of the statistics, of a step's gradient, of a pair's, of a pair's in place).
    Entries left out, repeated ids and rows without a set as the header defines them."""
    import torch
    n, V = x.shape
    x, T = x.double(), float(np.float32(T))
    inf = float("inf")
    ok = (ids >= 0) & (ids < V) & (tl != -inf)
    at, t = torch.where(ok, ids.long(), 0), torch.where(ok, tl.double() / T, -inf)
    some = ok.any(1, keepdim=True)
    inset = torch.zeros((n, V), device=x.device).scatter_add_(1, at, ok.float()) > 0
    p = (t - (torch.where(some, t, 0.0).logsumexp(1, keepdim=True) if tlse is None else tlse.double()[:, None])).exp()
    P = torch.zeros_like(x).scatter_add_(1, at, torch.where(ok, p, 0.0))

    def part(mask):
        m = x.masked_fill(~mask, -inf).amax(1, keepdim=True)
        e = torch.where(mask, ((x - m) / T).exp(), 0.0)
        return m, e, e.sum(1, keepdim=True)
    s, gT, zero = S(V), gl.double()[:, None] / T, torch.zeros((n, 1), dtype=torch.float64, device=x.device)

    def exponent(m):  # relative error of exp(-t) as computed
        t = (x - m).abs() / T
        return s + 2.0 ** -24 * (4 * torch.where(t < 200, t, 0.0) + 16)
    if tlse is None:
        m, e, total = part(torch.ones_like(inset))
        q, logq = e / total, (x - m) / T - total.log()
        lse, logr, rest = m / T + total.log(), zero, zero
        d = q - P
        tol = q * exponent(m)
        tol_pair = tol_place = tol
    else:
        mi, ei, si = part(inset)
        mo, eo, so = part(~inset)
        dist = (mi - mo) / T + si.log() - so.log()
        logr, logi = -torch.logaddexp(zero, dist), -torch.logaddexp(zero, -dist)
        logq = (x - mi) / T - si.log() + logi
        rest = (1 - P.sum(1, keepdim=True)).clamp(min=0)
        lse = torch.where(dist > 0, mi / T + (si.log() - logi), mo / T + (so.log() - logr))
        q, weight = ei / si * logi.exp(), logr.exp() - rest
        d = torch.where(inset, q - P, weight * (eo / so))
        tol = torch.where(inset, q * s, (weight.abs() * exponent(mo) + logr.exp() * s + 1e-14) * (eo / so))
        second, first = 2.0 ** -24 * logr.abs().clamp(max=REACH), 2.0 ** -24 * lse.abs().clamp(max=REACH)
        tol_pair = tol + torch.where(inset, q, (weight.abs() + logr.exp()) * (eo / so)) * second
        tol_place = tol_pair + torch.where(inset, q, logr.exp() * (eo / so)) * first
    loss = torch.where(inset & (P > 0), P * (P.log() - logq), 0.0).sum(1) + torch.where(rest > 0, rest * (rest.log() - logr), zero).squeeze(1)
    grad, stats = d * gT, torch.cat((lse, logr), 1)
    done = []
    for t in (tol, tol_pair, tol_place):
        t = 1.05 * gT * (t + 2e-38) + 8 * 2.0 ** -24 * grad.abs()
        done.append(t + half * (grad.abs() + t) + 2e-38)
    tol_s = 2 * s + 2.0 ** -23 * stats.abs()
    tol_s[:, 1] += 2.0 ** -24 * torch.where(lse.abs() <= REACH, lse.abs(), 0.0).squeeze(1)
    # what the set leaves of 1 is off by 128 terms' 2^-53 (1.4e-14) either way, times log q_r, which a mask makes 1e38
    tol_l = 2 * s + 2.0 ** -23 * loss.abs() + torch.where(rest > 0, 2 * 1.4e-14 * logr.abs(), zero).squeeze(1)
    got = [loss, stats, grad, tol_l, tol_s, *done]
    none = ~some.squeeze(1)
    for g in got:
        g[none] = 0
    if half > 2.0 ** -24:
        got[-2] = got[-1]
    return got


def near(got, want, tol, what):
    """Within tol; beyond fp32 the same infinity."""
    import torch
    got, top = got.double(), torch.finfo(got.dtype).max
    over = want.abs() > top
    assert bool((got[over] == torch.sign(want[over]) * float("inf")).all()), what
    off = torch.where(over, 0.0, (got - want).abs())
    assert not bool(torch.isnan(got).any()), (what, "NaN in rows", torch.isnan(got.flatten(1) if got.dim() > 1 else got[:, None]).any(1).nonzero()[:12, 0].tolist())
    bad = off > tol
    assert not bool(bad.any()), (what, float((off / tol).nan_to_num(0).max()), bad.nonzero()[:4].tolist())


# rows of 20,000: a few (short chunks), long chunks, and enough bytes that a step holds its rows
ROWS = {"few": {"float32": 10, "bfloat16": 10}, "chunks": {"float32": 230, "bfloat16": 230}, "held": {"float32": 300, "bfloat16": 600}}


def check(x, ids, tl, tlse, gl, T, dtype):
    import ds41_gfx950 as G
    loss, stats, grad, tol_l, tol_s, tol_g, tol_p, tol_i = reference(x, ids, tl, tlse, gl, T, HALF[dtype])
    kw = dict(teacher_lse=tlse, temperature=T)
    l1, s1 = G.distill_forward(x, ids, tl, **kw)
    got = [("forward", l1, s1, None, None), ("backward", l1, s1, G.distill_backward(x, ids, tl, s1, gl, **kw), tol_p)]
    y = x.clone()
    G.distill_backward(y, ids, tl, s1, gl, grad=y, **kw)
    got.append(("backward in place", l1, s1, y, tol_i))
    got.append(("step", *G.distill_step(x, ids, tl, gl, **kw), tol_g))
    y = x.clone()
    got.append(("step in place", *G.distill_step(y, ids, tl, gl, grad=y, **kw), tol_g))
    for what, l, s, g, tol in got:
        near(l, loss, tol_l, what + " loss")
        near(s, stats, tol_s, what + " statistics")
        if g is not None:
            near(g, grad, tol, what + " gradient")


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("path", list(ROWS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [0.01, 0.1, 1.0, 100.0])
def test_sets_far_from_the_rest(gpu, T, dtype, path, rest):
    n, V, k = ROWS[path][dtype], 20000, 20 if path == "few" else 100
    check(*make(gpu, int(T * 100) + n, n, V, k, dtype, T, rest), T, dtype)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("path", list(ROWS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_left_out_and_repeated_entries_of_such_rows(gpu, dtype, path, rest):
    """Ids outside the vocabulary, teacher's logits of -infinity, an id twice, the same id throughout, nothing in the set."""
    n, V, k = ROWS[path][dtype], 20000, 70
    x, ids, tl, tlse, gl = make(gpu, n, n, V, k, dtype, 1.0, rest)
    for r in range(0, 20 if n > 20 else 10):
        what = r // 2 % 5
        if what == 0:
            ids[r, 3:] = -1
        elif what == 1:
            tl[r, 66:], ids[r, 1] = -float("inf"), V
        elif what == 2:
            ids[r, 65], ids[r, 9] = ids[r, 0], ids[r, 64]
        elif what == 3:
            ids[r] = ids[r, 0]
        else:
            ids[r] = -3
    check(x, ids, tl, tlse, gl, 1.0, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_nothing_outside_the_set(gpu, dtype):
    """Every entry outside masked with -infinity: log q_r is -infinity, the loss +infinity where the teacher leaves a rest
    (0 times log q_r is 0 where it leaves none), the gradient outside 0 and inside q - P. A set of 128 in a row of 129 too."""
    import torch
    import ds41_gfx950 as G
    for n, V, k in ((9, 20000, 20), (700, 20000, 20), (5, 129, 128)):
        x, ids, tl, tlse, gl = make(gpu, V, n, V, k, dtype, 1.0, True)
        inset = torch.zeros((n, V), dtype=torch.bool, device=gpu).scatter_(1, ids.long(), True)
        x = torch.where(inset, torch.randn(n, V, device=gpu).to(x.dtype), float("-inf"))
        tlse[::2] -= 1.0  # the set's probabilities add up to more than 1: nothing is left
        P = (tl.double() - tlse.double()[:, None]).exp()
        logq = x.double().log_softmax(1).gather(1, ids.long())
        pr = (1 - P.sum(1)).clamp(min=0)
        loss = torch.where(pr > 0, float("inf"), (P * (P.log() - logq)).sum(1))
        want = (logq.exp() - P) * gl.double()[:, None]
        assert bool((pr[::2] == 0).all()) and bool((pr[1::2] > 0).any())
        l1, s1 = G.distill_forward(x, ids, tl, teacher_lse=tlse)
        y = x.clone()
        for l, s, g in ((l1, s1, G.distill_backward(x, ids, tl, s1, gl, teacher_lse=tlse)), G.distill_step(x, ids, tl, gl, teacher_lse=tlse),
                        G.distill_step(y, ids, tl, gl, teacher_lse=tlse, grad=y)):
            near(l, loss, S(V) * 4 + 2.0 ** -23 * loss.abs().nan_to_num(0, 0), "loss")
            assert bool((s[:, 1] == -float("inf")).all())
            assert bool((g[~inset] == 0).all())
            at = g.double().gather(1, ids.long())
            assert bool(((at - want).abs() <= 2 * S(V) + 2 * HALF[dtype] * want.abs()).all())
