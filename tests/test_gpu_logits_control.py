"""The token table and ds41_logits_control against numpy.

Bound of a touched entry: divide or multiply, two products and subtractions, an add: each rounds to half a step
(2^-24) of a value no larger than |x1| + |frequency c| + |presence| + |bias|, at most six of them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
LOWEST = np.float32(-3.4028234663852886e38)


def table_of(rng, S, V, length, generated_share=0.5):
    counts, seen = np.zeros((S, V), np.int32), np.zeros((S, V), bool)
    for s in range(S):
        for v in rng.integers(0, V, length) if length else ():
            seen[s, v] = True
            counts[s, v] += rng.random() < generated_share
    return counts, seen


def pack(flags):
    """[..., V] truth values as int32 words."""
    pad = -flags.shape[-1] % 32
    f = np.concatenate([flags, np.zeros(flags.shape[:-1] + (pad,), bool)], -1)
    return np.packbits(f, axis=-1, bitorder="little").view(np.int32)


def reference(x, rows, counts, seen, index, drafts, pen, bias, mask, mask_index, masked):
    """(values in 64 bits, bound) of every entry; untouched and masked ones with bound 0."""
    n, V = x.shape
    y, tol = x.astype(np.float64), np.zeros((n, V))
    floor = float(LOWEST) if masked == -np.inf else float(masked) / 2
    bits = None if mask is None else np.unpackbits(mask.view(np.uint8), axis=-1, bitorder="little")[:, :V].astype(bool)
    empty = 0
    for r in range(n):
        s, j = divmod(r, rows)
        c, m = np.zeros(V, np.int64), np.zeros(V, bool)
        t = s if index is None else index[s]
        if counts is not None and 0 <= t < len(counts):
            c = counts[t].astype(np.int64)
        if seen is not None and 0 <= t < len(seen):
            m = seen[t].copy()
            c = np.where(m, c, 0)
        elif seen is None:
            m = c > 0
        if drafts is not None:
            for d in drafts[s][:j]:
                if 0 <= d < V:
                    c[d] += 1
                    m[d] = True
        rep, freq, pres = (1.0, 0.0, 0.0) if pen is None else pen[s].astype(np.float64)
        b, has = np.zeros(V), np.zeros(V, bool)
        for i, v in bias[s] if bias else ():
            if 0 <= i < V:
                b[i], has[i] = v, True
        touched = m | (c > 0) | has
        with np.errstate(invalid="ignore", over="ignore"):
            x1 = np.where(m, np.where(y[r] > 0, y[r] / rep, y[r] * rep), y[r])
            v = x1 - freq * c - np.where(c > 0, pres, 0.0) + b
            v = np.where(v < floor, floor, v)
            bound = 6 * 2.0 ** -24 * (np.abs(x1) + np.abs(freq * c) + abs(pres) + np.abs(b)) * 1.01 + 1e-44
            y[r] = np.where(touched, v, y[r])
            tol[r] = np.where(touched & np.isfinite(v), np.nan_to_num(bound), 0)
        if mask is not None:
            mi = r if mask_index is None else mask_index[r]
            if mi >= 0:
                ok = bits[mi] if mi < len(bits) else np.zeros(V, bool)
                if not ok.any():
                    y[r], tol[r] = np.nan, 0
                    empty += 1
                else:
                    y[r], tol[r] = np.where(ok, y[r], masked), np.where(ok, tol[r], 0)
    return y, tol, empty


def same(got, want, tol):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    off = np.abs(got[fin] - want[fin])
    assert np.all(off <= tol[fin]), float(np.max(off - tol[fin]))


def dev(a, gpu):
    import torch
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


def run(gpu, rng, S, rows, V, *, history=50, use=("counts", "seen", "drafts", "pen", "bias", "mask"), masked=LOWEST, allowed=0.3, n_bias=20,
        index=None, special=False, mask_index=None, pad=0):
    """In place and out of place, with rows `pad` entries apart beyond V, against the reference."""
    import torch
    import ds41_gfx950 as G
    n = S * rows
    x = (rng.standard_normal((n, V)) * 3).astype(np.float32)
    if special and V > 8:
        for v in (np.nan, np.inf, -np.inf, LOWEST, -LOWEST, -0.0):
            x[rng.integers(0, n, 3), rng.integers(0, V, 3)] = v
    T = S if index is None else max(int(np.max(index)) + 1, 1)
    counts, seen = table_of(rng, T, V, history)
    counts, seen = counts if "counts" in use else None, seen if "seen" in use else None
    drafts = rng.integers(-1, V + 1, (S, max(rows - 1, 1))).astype(np.int32) if "drafts" in use else None
    if drafts is not None and rows > 2:
        drafts[:, 1] = drafts[:, 0]  # the same token twice
    pen = (rng.random((S, 3)) * [1.5, 2, 2] + [0.5, -1, -1]).astype(np.float32) if "pen" in use else None
    bias = ids = vals = offs = None
    if "bias" in use:
        bias = [[(int(rng.integers(-2, V + 2)), float(np.float32(rng.standard_normal() * 5))) for _ in range(n_bias)] for _ in range(S)]
        for b in bias:
            if len(b) > 3:
                b[3] = (b[0][0], 9.5)   # a later entry for the same id
                b[2] = (b[2][0], -np.inf)
        ids = np.array([i for b in bias for i, _ in b] or [0], np.int32)
        vals = np.array([v for b in bias for _, v in b] or [0], np.float32)
        offs = (np.arange(S + 1) * n_bias).astype(np.int32)
    mask = None
    if "mask" in use:
        flags = rng.random((n, V)) < allowed
        flags[np.arange(n), rng.integers(0, V, n)] = True
        if n > 2:
            flags[1] = False       # nothing allowed
            flags[2] = False
            flags[2, V - 1] = True  # the last entry alone
        mask = pack(flags)
        if V % 32:
            mask[:, -1] |= np.int32(-1) << np.int32(V % 32)  # bits past the vocabulary mean nothing
    want, tol, empty = reference(x, rows, counts, seen, index, drafts, pen, bias, mask, mask_index, masked)
    seen_w = None if seen is None else pack(seen)
    kw = dict(rows=rows, counts=dev(counts, gpu), seen=dev(seen_w, gpu), table_index=dev(index, gpu), drafts=dev(drafts, gpu),
              penalties=dev(pen, gpu), bias_ids=dev(ids, gpu), bias_values=dev(vals, gpu), bias_offsets=dev(offs, gpu), mask=dev(mask, gpu),
              mask_index=dev(mask_index, gpu), masked_value=float(masked))
    G.take_status()
    buf = torch.full((n, V + pad), 5.0, device=gpu)
    src = buf[:, :V]
    src.copy_(dev(x, gpu))
    out = torch.full((n, V + 2 * pad), 6.0, device=gpu)
    G.logits_control(src, out=out[:, :V], **kw)
    assert np.array_equal(src.cpu().numpy().view(np.uint32), x.view(np.uint32))  # the input stays
    same(out[:, :V].cpu().numpy(), want, tol)
    assert bool((out[:, V:] == 6).all())
    assert G.take_status() == (8 if empty else 0)
    G.logits_control(src, **kw)
    assert np.array_equal(src.cpu().numpy().view(np.uint32), out[:, :V].cpu().numpy().view(np.uint32))
    assert bool((buf[:, V:] == 5).all())
    assert G.take_status() == (8 if empty else 0)


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 1023, 1025, 4097, 129280, 129281])
def test_control_sizes(gpu, V):
    rng = np.random.default_rng(V)
    for S, rows in ((1, 1), (1, 4), (2, 6)):
        run(gpu, rng, S, rows, V, special=V > 1000, masked=LOWEST if rows == 4 else -np.inf)


@pytest.mark.parametrize("use", [(), ("counts",), ("seen",), ("drafts",), ("bias",), ("mask",), ("pen",), ("counts", "pen"), ("seen", "pen"),
                                 ("drafts", "pen"), ("counts", "drafts", "pen"), ("bias", "mask"), ("counts", "seen", "pen", "mask")])
def test_control_parts(gpu, use):
    rng = np.random.default_rng(len(use) * 7 + sum(map(len, use)))
    run(gpu, rng, 3, 3, 2500, use=use, special=True, history=300)
    run(gpu, rng, 2, 5, 777, use=use, pad=3)


def test_control_rows_index_and_strides(gpu):
    rng = np.random.default_rng(5)
    run(gpu, rng, 5, 2, 1500, index=np.array([3, -1, 3, 99, 0], np.int32), pad=1)   # a row twice, none, outside, another
    run(gpu, rng, 1, 64, 1300, pad=2)
    run(gpu, rng, 40, 1, 3000, allowed=0.001)
    run(gpu, rng, 3, 2, 5000, n_bias=3000)
    run(gpu, rng, 4, 2, 1100, n_bias=0)
    run(gpu, rng, 2, 3, 1100, mask_index=np.array([-1, 4, 4, 1, 0, 6], np.int32))   # none, shared, nothing allowed, outside


def test_allowed_bias_of_minus_infinity_stays_above_the_mask(gpu):
    """The one allowed token with a bias of -infinity is still the row's largest entry, and the samplers take it."""
    import torch
    import ds41_gfx950 as G
    V = 5000
    x = torch.randn(1, V, device=gpu)
    mask = np.zeros((1, V), bool)
    mask[0, 1234] = True
    i32 = dict(dtype=torch.int32, device=gpu)
    G.logits_control(x, bias_ids=torch.tensor([1234], **i32), bias_values=torch.tensor([-np.inf], device=gpu),
                     bias_offsets=torch.tensor([0, 1], **i32), mask=dev(pack(mask), gpu))
    assert int(x.argmax()) == 1234 and bool(torch.isfinite(x).all())
    out = torch.zeros(1, **i32)
    for T, top_p in ((1.0, 1.0), (0.7, 0.9), (0.0, 1.0)):
        G.sample_logits(x, T, top_p, 1, 2, 0, 1, out, G.sample_workspace(1, V, gpu))
        assert int(out) == 1234


def test_token_table(gpu):
    import torch
    import ds41_gfx950 as G
    rng = np.random.default_rng(0)
    for V, T in ((1, 1), (33, 3), (5000, 4), (129281, 2)):
        counts, seen = G.token_counts(T, V, gpu)
        c, m = np.zeros((T, V), np.int64), np.zeros((T, V), bool)
        for generated in (False, True, True):
            n = 6
            index = rng.integers(-1, T + 1, n).astype(np.int32)
            lengths = rng.integers(0, 400, n)
            lengths[1] = 0
            lengths[2] = 1
            offs = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
            toks = rng.integers(-1, V + 1, offs[-1]).astype(np.int32)
            toks[: len(toks) // 2] = toks[0]  # one token many times
            G.token_counts_add(counts, seen, V, dev(toks, gpu), dev(offs, gpu), table_index=dev(index, gpu), generated=generated)
            for i in range(n):
                if 0 <= index[i] < T:
                    for v in toks[offs[i]:offs[i + 1]]:
                        if 0 <= v < V:
                            m[index[i], v] = True
                            c[index[i], v] += generated
        assert np.array_equal(counts.cpu().numpy(), c) and np.array_equal(seen.cpu().numpy(), pack(m))
        res = np.zeros((3, 10), np.int32)  # tokens[6], emitted, ...
        res[:, :6] = rng.integers(0, V, (3, 6))
        res[:, 6] = (4, -1, 6)
        res[2, 1] = V
        index = np.array([0, 0, T - 1], np.int32)
        G.token_counts_commit(counts, seen, V, dev(res, gpu), n=3, table_index=dev(index, gpu))
        for i in range(3):
            for v in res[i, :max(res[i, 6], 0)]:
                if v < V:
                    m[index[i], v] = True
                    c[index[i], v] += 1
        assert np.array_equal(counts.cpu().numpy(), c) and np.array_equal(seen.cpu().numpy(), pack(m))
        G.token_counts_clear(counts, seen, V, table_index=dev(np.array([T - 1, -1, T, T - 1], np.int32), gpu))
        c[T - 1], m[T - 1] = 0, False
        assert np.array_equal(counts.cpu().numpy(), c) and np.array_equal(seen.cpu().numpy(), pack(m))
        G.token_counts_add(counts, seen, V, dev(np.zeros(0, np.int32), gpu), dev(np.zeros(T + 1, np.int32), gpu))  # nothing
        G.token_counts_add(counts, seen, V, dev(np.zeros(5, np.int32), gpu), dev(np.array([-3] + [9] * T, np.int32), gpu))  # clamped
        c[0, 0] += 5
        m[0, 0] = True
        assert np.array_equal(counts.cpu().numpy(), c) and np.array_equal(seen.cpu().numpy(), pack(m))
        G.token_counts_clear(counts, seen, V)
        assert not bool(counts.any()) and not bool(seen.any())


def test_long_history_of_one_sequence(gpu):
    import torch
    import ds41_gfx950 as G
    V, L = 129280, 300001
    toks = (torch.arange(L, device=gpu) ** 2 % V).int()
    counts, seen = G.token_counts(1, V, gpu)
    for generated in (True, False):
        G.token_counts_add(counts, seen, V, toks, torch.tensor([0, L], dtype=torch.int32, device=gpu), generated=generated)
    want = torch.bincount(toks.long(), minlength=V)
    assert torch.equal(counts[0].long(), want)
    assert np.array_equal(seen.cpu().numpy(), pack((want > 0).cpu().numpy()[None]))


def test_control_and_commit_in_a_graph(gpu):
    """Control, greedy pick's result and commit captured together: every replay sees the table the one before left."""
    import torch
    import ds41_gfx950 as G
    V, rows = 3000, 2
    rng = np.random.default_rng(3)
    x0 = dev((rng.standard_normal((rows, V)) * 3).astype(np.float32), gpu)
    pen = dev(np.array([[1.2, 0.5, 1.0]], np.float32), gpu)
    drafts = dev(np.array([[7]], np.int32), gpu)
    res = dev(np.array([[7, 9, 9, 0, 0, 0, 3, 0, 0, 0]], np.int32), gpu)

    def step(table, out):
        G.logits_control(x0, rows=rows, counts=table[0], seen=table[1], drafts=drafts, penalties=pen, out=out)
        G.token_counts_commit(*table, V, res)
    eager, out_e = G.token_counts(1, V, gpu), torch.empty_like(x0)
    table, out_g = G.token_counts(1, V, gpu), torch.empty_like(x0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(table, out_g)
    for _ in range(4):
        step(eager, out_e)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_e, out_g) and torch.equal(eager[0], table[0]) and torch.equal(eager[1], table[1])
    assert int(table[0][0, 9]) == 8


def test_totals_up_to_the_largest(gpu):
    """total bounds the offsets; a buffer may be said to hold up to 2^31 - 1 tokens, whatever the sequences take of it."""
    import torch
    import ds41_gfx950 as G
    V = 100
    tokens, offsets = dev(np.array([5, 5, 7, 99, 1], np.int32), gpu), dev(np.array([0, 3, 5], np.int32), gpu)
    for total in (5, (1 << 31) - 2, (1 << 31) - 1):
        counts, seen = G.token_counts(2, V, gpu)
        rc = G.lib().ds41_token_counts_add(counts.data_ptr(), seen.data_ptr(), 2, V, None, tokens.data_ptr(), offsets.data_ptr(), 2, total, 1,
                                           G._stream())
        assert rc == 0
        want = torch.zeros(2, V, dtype=torch.int32)
        want[0, 5], want[0, 7], want[1, 99], want[1, 1] = 2, 1, 1, 1
        assert torch.equal(counts.cpu(), want)
