"""The policy loss's sum over the vocabulary keeps what 32 bits can hold of it.

Bounds. The logits lie near each other, N(0, 0.1^2), so that no few entries carry the sum. An entry's exponential is within two steps of
itself (2^-22) and its argument rounded at its own size, below 0.7 (2^-24 of it); a piece of 4 or 8 entries is added up in fp32 in
two or three levels (2^-24 each). These roundings are of thousands of entries and pieces, independent and of either sign: of n of them
the sum keeps 1 / sqrt(n), 1e-9 at the least n here. What has one sign for all of a row is the temperature's factor log2(e) / T,
rounded once: 2^-24 times the mean argument, below 0.7 - 4e-8 times 0.7 ln 2 / 2, 1.5e-8 with the worst of it. All above is 64-bit, and the
result takes one rounding to fp32, 2^-24 at most. Together 2^-24 + 1.5e-8 + 0.1e-8: 1.27 times 2^-24. Sums joined in fp32 are
off by up to 2.5 times 2^-24 in hundreds of rows."""
import numpy as np
import pytest

import ds41_gfx950 as G

pytestmark = pytest.mark.gpu
BOUND = 1.27 * 2.0 ** -24


@pytest.mark.parametrize("dtype,n,V", [
    ("float32", 30, 129280), ("float32", 16, 100500),    # chunks of 4,096
    ("float32", 400, 129280), ("bfloat16", 300, 151936),  # chunks of 16,384, rows too wide to be held
    ("bfloat16", 400, 129280), ("float32", 600, 50257), ("bfloat16", 600, 40000)])  # rows held by a step
def test_sums_of_even_rows(gpu, dtype, n, V):
    import torch
    g = torch.Generator(device=gpu).manual_seed(n + V)
    x = torch.empty((n, V), device=gpu).normal_(0, 0.1, generator=g).to(getattr(torch, dtype))
    tok = torch.randint(0, V, (n,), device=gpu, generator=g).int()
    at = tok.long().unsqueeze(1)
    z = x.double().scatter_(1, at, -float("inf"))
    m = z.max(1, keepdim=True).values
    s = torch.exp(z - m).sum(1)
    d = x.double().gather(1, at).squeeze(1) - m.squeeze(1) - torch.log(s)
    lp = -torch.log1p(torch.exp(-d))
    old, one = lp.float(), torch.ones(n, device=gpu)
    for got in (G.policy_forward(x, tok, old, one), G.policy_step(x, tok, old, one, one)):
        _, logprob, stats = got[:3]
        assert torch.equal(stats[:, 0].double(), m.squeeze(1))
        off = (stats[:, 1].double() / s - 1).abs().cpu().numpy()
        assert off.max() <= BOUND, (off.max() * 2.0 ** 24, np.sqrt((off ** 2).mean()) * 2.0 ** 24)
        # log p, of size 11: the sum's error and half a step of its own
        assert ((logprob.double() - lp).abs() <= BOUND + lp.abs() * 2.0 ** -24).all()


@pytest.mark.parametrize("n,V", [(30, 129280), (400, 129280), (600, 50257)])
def test_a_rows_factor_is_rounded_once(gpu, n, V):
    """The gradient of a row's other tokens is a factor times their exponentials. Logits N(16, 0.1^2), whose exponents are taken from an
    offset of 23 or so that is itself rounded. What an entry's own roundings do averages out over a row (its gradient's half step
    too: 2^-24 / sqrt(V)), so the mean of its entries over the formula's, at the maximum and sum that the call left, is off by the
    factor's one rounding, 2^-24, and by 1.5e-8 of the temperature's as above."""
    import torch
    g = torch.Generator(device=gpu).manual_seed(n + V)
    x = torch.empty((n, V), device=gpu).normal_(16, 0.1, generator=g)
    tok = torch.randint(0, V, (n,), device=gpu, generator=g).int()
    at = tok.long().unsqueeze(1)
    one = torch.ones(n, device=gpu)
    old = torch.log_softmax(x.double(), 1).gather(1, at).squeeze(1).float()
    loss, logprob, stats, grad = G.policy_step(x, tok, old, one, one)
    back = G.policy_backward(x, tok, old, one, stats, one)
    m, s, xa = (stats[:, i].double() for i in range(3))
    assert torch.equal(xa, x.double().gather(1, at).squeeze(1))
    d = xa - m - torch.log(s)
    slope = -torch.exp(-torch.log1p(torch.exp(-d)) - old.double())
    want = -(slope / (1 + torch.exp(d)) / s).unsqueeze(1) * torch.exp(x.double() - m.unsqueeze(1))
    want.scatter_(1, at, float("nan"))
    for t in (grad, back):
        off = ((t.double() / want).nanmean(1) - 1).abs().cpu().numpy()
        assert off.max() <= BOUND, off.max() * 2.0 ** 24
