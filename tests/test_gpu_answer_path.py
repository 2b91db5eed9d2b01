"""The operators together as a serving loop uses them: hidden states through the head (ds41_dense_bf16, with the
drafter's per-token row as the residual), penalties and a grammar on target and draft rows, drafts drawn and
verified by the samplers, the emitted tokens committed to the table; the target's top logits kept, and the
drafter's rows distilled from them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_answer_path(gpu):
    import torch
    import ds41_gfx950 as G
    V, H, K, steps = 5003, 256, 3, 6
    g = torch.Generator(device=gpu).manual_seed(0)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device=gpu).normal_(0, std, generator=g)
    head, drafter = normal(V, H, std=0.15).bfloat16(), normal(V, H, std=0.15).bfloat16()
    markov = normal(64, V, std=0.3)
    allowed = torch.rand(V, device=gpu, generator=g) < 0.05
    words = np.packbits(np.pad(allowed.cpu().numpy(), (0, -V % 32)), bitorder="little").view(np.int32)
    mask = torch.from_numpy(words).to(gpu)[None]
    prompt = torch.randint(0, V, (40,), device=gpu, generator=g).int()
    pen = torch.tensor([[1.3, 0.4, 0.6]], device=gpu)
    i32 = dict(dtype=torch.int32, device=gpu)
    counts, seen = G.token_counts(1, V, gpu)
    G.token_counts_add(counts, seen, V, prompt, torch.tensor([0, 40], **i32), generated=False)
    result = torch.zeros(40, dtype=torch.uint8, device=gpu)
    sample_ws, accept_ws = G.sample_workspace(1, V, gpu), G.accept_workspace(K, V, gpu)
    answer = []
    for step in range(steps):
        hidden = normal(K + 1, H)
        # drafts one after another: each row sees those before it
        drafts = torch.full((1, K), -1, **i32)
        draft_rows = torch.empty(K, V, device=gpu)
        last = step
        for j in range(K):
            raw = torch.empty(K, V, device=gpu)
            G.dense_bf16(hidden[:K].bfloat16(), drafter, residual=markov[last % 64].expand(K, V).contiguous(), out=raw)
            G.logits_control(raw, rows=K, counts=counts, seen=seen, drafts=drafts, penalties=pen, mask=mask,
                             mask_index=torch.zeros(K, **i32))
            draft_rows[j] = raw[j]
            G.sample_logits(draft_rows[j:j + 1], 1.0, 0.95, 7, step, j, 1, drafts[0, j:j + 1], sample_ws)
            last = int(drafts[0, j])
            assert bool(allowed[last])
        target = G.dense_bf16(hidden.bfloat16(), head, out_dtype=torch.float32)
        ref = hidden.bfloat16().double() @ head.double().t()
        assert float((target.double() - ref).abs().max()) < 1e-4
        ids, values, lse, lp = G.top_logits(target, 32)
        G.logits_control(target, rows=K + 1, counts=counts, seen=seen, drafts=drafts, penalties=pen, mask=mask,
                         mask_index=torch.zeros(K + 1, **i32))
        # the penalised rows, on the host
        c, s = counts[0].double(), torch.zeros(V, dtype=torch.bool, device=gpu)
        s[prompt.long()] = True
        if answer:
            s[torch.tensor(answer, device=gpu)] = True
        for j in range(K + 1):
            if j:
                c[drafts[0, j - 1].long()] += 1
                s[drafts[0, j - 1].long()] = True
            y = torch.where(s, torch.where(ref[j] > 0, ref[j] / pen[0, 0].double(), ref[j] * pen[0, 0].double()), ref[j])
            y = y - pen[0, 1].double() * c - pen[0, 2].double() * (c > 0)
            assert float((target[j].double() - y).abs()[allowed].max()) < 2e-4 and bool((target[j][~allowed] == G.LOWEST).all())
        G.verify_logits(target, draft_rows, drafts[0], 1.0, 0.95, 7, step, result, accept_ws)
        G.token_counts_commit(counts, seen, V, result)
        r = result.view(torch.int32).tolist()
        assert 1 <= r[6] <= K + 1 and all(bool(allowed[t]) for t in r[:r[6]])
        answer += r[:r[6]]
        # the drafter learns from the rows the target just produced
        x = draft_rows.clone()
        loss, stats, grad = G.distill_step(x, ids[:K].contiguous(), values[:K].contiguous(), torch.ones(K, device=gpu),
                                           teacher_lse=lse[:K].contiguous())
        assert bool((grad[:, ~allowed].abs()[:, :] <= 1).all()) and bool(torch.isfinite(grad).all())
    want = np.bincount(answer, minlength=V)
    assert np.array_equal(counts[0].cpu().numpy(), want) and G.take_status() == 0
    marks = np.unpackbits(seen.cpu().numpy().view(np.uint8), bitorder="little")[:V].astype(bool)
    assert np.array_equal(marks, (want > 0) | np.isin(np.arange(V), prompt.cpu().numpy()))


def test_host_tensors_among_device_tensors_are_refused(gpu):
    import torch
    import ds41_gfx950 as G
    x, w = torch.zeros(4, 64, device=gpu).bfloat16(), torch.zeros(32, 64, device=gpu).bfloat16()
    z, pen = torch.zeros(4, 96, device=gpu), torch.ones(12)
    ids, t = torch.zeros(4, 5, dtype=torch.int32, device=gpu), torch.zeros(4, 5, device=gpu)
    for f in (lambda: G.dense_bf16(x, w.cpu()), lambda: G.dense_bf16(x, w, bias=torch.zeros(32)), lambda: G.logits_control(z, penalties=pen),
              lambda: G.top_logits(z, 5, chosen=torch.zeros(4, dtype=torch.int32)), lambda: G.distill_forward(z, ids.cpu(), t),
              lambda: G.distill_step(z, ids, t, torch.zeros(4))):
        with pytest.raises(ValueError, match="tensors on"):
            f()


def test_tensors_made_for_another_stream_are_of_its_memory(gpu):
    """A call on a stream of its own, right after tensors of the sizes it makes were freed with work of the current
    stream still to come on them: its results are not written over, and equal the current stream's."""
    import torch
    import ds41_gfx950 as G
    rng = torch.Generator(device="cpu").manual_seed(5)
    x, w = torch.randn(64, 512, generator=rng).to(gpu).bfloat16(), torch.randn(4096, 512, generator=rng).to(gpu).bfloat16()
    z = torch.randn(64, 4096, generator=rng).to(gpu)
    t, ids = torch.topk(z, 20)
    ids, gl = ids.int(), torch.ones(64, device=gpu)
    want = [G.dense_bf16(x, w), *G.top_logits(z, 20)[:3], *G.distill_step(z, ids, t, gl)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        for o in want:  # written late by the current stream, and free at once
            held = [torch.empty_like(o) for _ in range(4)]
            for h in held:
                for _ in range(20):
                    h.fill_(3)
            del held, h
        got = [G.dense_bf16(x, w, stream=s), *G.top_logits(z, 20, stream=s)[:3], *G.distill_step(z, ids, t, gl, stream=s)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
