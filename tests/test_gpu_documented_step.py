"""The documented training step of an expert as it stands in the integration notes, twice over (two micro-batches whose gradients
add up): fp32 masters quantised, g and u saved in fp32, bf16 logits with their gradient in their place, fp32 gradients accumulated and
clipped in place, and the new masters quantised. Every operator is held against 64 bits at the very inputs that the one before it
left, with its own test's bounds, so that nothing is hidden behind what a chain loses. Rows are clipped on both sides, padding and
tied to a reference; the limit cuts gates and up projections."""
import numpy as np
import pytest

import ds41_gfx950 as G
import test_gpu_ffn as F
import test_gpu_policy as P
import test_gpu_quant_mxfp4 as Q

pytestmark = pytest.mark.gpu


def product(got, a, b):
    """bf16 a b^T: a sum in fp32, rounded once."""
    a, b = a.double(), b.double()
    want, tol = a @ b.t(), 2 * a.shape[1] * F.F * (a.abs() @ b.abs().t())
    assert ((got.double() - want).abs() <= tol + F.B * (want.abs() + tol) + 1e-38).all()


@pytest.mark.parametrize("M,H,I,V", [(24, 256, 320, 3001), (200, 512, 384, 8000), (700, 288, 352, 16001)])
def test_documented_step(gpu, M, H, I, V):
    import torch
    bf16 = torch.bfloat16
    g = torch.Generator(device=gpu).manual_seed(M)
    rng = np.random.default_rng(M)

    def normal(shape, std, dtype=torch.float32):
        return torch.empty(shape, device=gpu).normal_(0, std, generator=g).to(dtype)

    def on(v):
        return torch.from_numpy(np.asarray(v, np.float32)).to(gpu)
    masters = [normal(s, 0.06) for s in ((I, H), (I, H), (H, I))]
    head = normal((V, H), 0.08, bf16)
    head_t = head.t().contiguous()
    limit, kl, low, high, max_norm = 1.0, 0.02, 0.2, 0.28, 0.05

    def quantise():
        out = []
        for w in masters:
            q, s, v = G.quantize_mxfp4(w, values=True)
            wq, ws, wv = Q.rule(w.cpu().numpy())
            assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws) and np.array_equal(v.double().cpu().numpy(), wv)
            out.append(v)
        return out
    values = quantise()
    grads = [torch.full_like(w, float("nan")) for w in masters]
    for batch in range(2):
        x = normal((M, H), 1.0, bf16)
        saved = torch.empty((M, 2 * I), device=gpu)
        y = G.ffn_forward(x, *values, limit=limit, saved=saved)
        F.check_forward(x, *values, y, saved, limit)
        assert (saved[:, :I] > limit).any() and (saved[:, I:].abs() > limit).any()
        logits = G.dense_bf16(y, head)
        product(logits, y, head)
        tok = torch.randint(0, V, (M,), device=gpu, generator=g).int()
        tok[::9] = -1
        z = logits.double()
        lp = torch.log_softmax(z, 1)[torch.arange(M, device=gpu), tok.clamp(min=0).long()].cpu().numpy()
        moved = rng.normal(0, 0.3, M)
        for border in (np.log(1 - low), np.log(1 + high)):  # no ratio where rounding would decide
            moved = np.where(np.abs(moved - border) < 1e-3, border + 2e-3, moved)
        old, A, ref, gl = on(lp - moved), on(rng.normal(0, 1, M)), on(lp + rng.normal(0, 0.3, M)), on(np.full(M, 0.5 / M))
        ratio, sign = np.exp(moved), A.cpu().numpy()
        live = tok.cpu().numpy() >= 0
        assert (live & (sign > 0) & (ratio > 1 + high)).any() and (live & (sign < 0) & (ratio < 1 - low)).any()
        before = logits.clone()
        given = dict(ref_logprob=ref, kl_coef=kl, clip_low=low, clip_high=high)
        loss, logprob, stats, dz = G.policy_step(logits, tok, old, A, gl, grad=logits, **given)
        assert dz is logits
        P.check(before, tok, old, A, ref, gl, 1.0, kl=kl, lo=low, hi=high)  # a step of its own against 64 bits
        apart = G.policy_step(before, tok, old, A, gl, **given)
        assert torch.equal(apart[0], loss) and torch.equal(apart[1], logprob) and torch.equal(apart[3], dz)
        dy = G.dense_bf16(dz, head_t)
        product(dy, dz, head_t)
        was = [t.clone() for t in grads] if batch else [None] * 3
        got = G.ffn_backward(x, *values, saved, dy, limit=limit, grad_gate=grads[0], grad_up=grads[1], grad_down=grads[2], accumulate=bool(batch))
        assert all(a is b for a, b in zip(got[1:], grads))
        F.check_backward((x, *values), saved, dy, limit, got, [None] + was)
    was = [t.double() for t in grads]
    norm64 = torch.stack([t.square().sum() for t in was]).sum().sqrt()
    norm = G.grad_clip(grads, max_norm)
    assert float(norm64) > max_norm and abs(float(norm) - float(norm64)) <= float(norm64) * 1.01 * 2.0 ** -24
    factor = float(np.float32(max_norm)) / (float(norm64) + 1e-6)
    for t, w in zip(grads, was):
        assert ((t.double() - w * factor).abs() <= (w * factor).abs() * 1.01 * 2.0 ** -24 + 2.0 ** -149).all()
    for w, d in zip(masters, grads):
        w.add_(d, alpha=-4.0)
    again = quantise()
    assert not any(torch.equal(a, b) for a, b in zip(again, values))
    # and the new codes are what the library's readers of the format take
    q, s, v = G.quantize_mxfp4(masters[0], values=True)
    assert torch.equal(G.dequant_mxfp4(q, s, I, H), v.float())
