"""The operators between the last MoE layer and the sampler, and between the sampler and the drafter's next
training step, each as a serving or training program calls it.

Operators (`case["op"]`):
  dense     y = act(x w^T + bias) + residual, bf16 in, bf16 or fp32 out: the head that makes the logits, and
            projections of the model's sizes.
  control   repetition, frequency and presence penalties, token biases and grammar masks on the fp32 rows
            that the samplers read; row j of a verify step sees the j drafts before it.
  history   a batch of sequences entered into the token table that `control` reads.
  top       the k largest logits of every row with ids, the row's log-sum-exp and the chosen token's
            log-probability: what an answer reports and what a drafter is taught with.
  distill   distillation of a drafter's rows from a teacher's top logits: "step" is the loss with its gradient
            in one call, "pair" the forward call and then the backward call.

Activations are N(0, 1), weights N(0, 0.02^2) (a head's logits then spread by about 1.3), logits N(0, 2.5^2)
with 100 tokens of every row raised, so that they hold most of its mass as a language model's do; tokens follow
a Zipf-like law, so that a history repeats its frequent ones.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
LOWEST = -3.4028234663852886e38
ACTS = ("none", "relu", "silu", "gelu")


def _framework():
    pkg = os.path.abspath("deepseek-v4.1-flash-pro6000_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ds41_gfx950
    return ds41_gfx950


def listed():
    return [
        # a drafter's logits for the verify width: the head over the vocabulary, plus the Markov row of the token before
        dict(name="head_4rows", op="dense", M=4, N=129280, K=4096, out="fp32", bias=False, residual=True, act="none"),
        # one token through a projection of the drafter's sizes
        dict(name="projection_1row", op="dense", M=1, N=5120, K=2304, out="bf16", bias=True, residual=False, act="silu"),
        # the head over a prefill chunk (scoring, or a teacher's rows)
        dict(name="head_512rows", op="dense", M=512, N=129280, K=4096, out="bf16", bias=False, residual=False, act="none"),
        # sizes that no tile divides, rows that no 16-byte load aligns with
        dict(name="dense_ragged", op="dense", M=67, N=2881, K=1007, out="bf16", bias=True, residual=True, act="gelu"),
        # the rows of one verify step (1 committed + 3 drafts) of a constrained answer
        dict(name="control_verify", op="control", sequences=1, rows=4, vocab=129280, history=8192, biases=64, masked="lowest", allowed=0.3),
        # verify steps of a batch, some rows with a grammar
        dict(name="control_batch", op="control", sequences=64, rows=4, vocab=129280, history=2048, biases=16, masked="-inf", allowed=0.02),
        # eight prompts arriving
        dict(name="history_prompts", op="history", sequences=8, length=32768, vocab=129280, generated=False),
        # log-probabilities of a verify step's answer
        dict(name="top_verify", op="top", rows=4, vocab=129280, k=20, dtype="fp32", temperature=1.0),
        # a teacher's record over a chunk of rows
        dict(name="top_record", op="top", rows=2048, vocab=129280, k=64, dtype="bf16", temperature=1.0),
        # the drafter learns from one verify step
        dict(name="distill_verify", op="distill", call="step", rows=4, vocab=129280, k=20, dtype="fp32", rest=False, temperature=1.0),
        # a training batch of the drafter, the teacher's remaining mass as one more class
        dict(name="distill_batch", op="distill", call="step", rows=2048, vocab=129280, k=64, dtype="bf16", rest=True, temperature=2.0),
        # forward and backward apart, odd sizes
        dict(name="distill_ragged", op="distill", call="pair", rows=333, vocab=50257, k=33, dtype="fp32", rest=False, temperature=1.0),
    ]


VOCABS = (129280, 129281, 32000, 50257, 151936, 100003)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("dense", "dense", "dense", "control", "control", "history", "top", "top", "distill", "distill"))
    if op == "dense":
        M, N, K = _log(rng, 1, 1024), _log(rng, 64, 129280), _log(rng, 32, 8192)
        if rng.random() < 0.6:  # most models' sizes are multiples of 64
            N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
        while M * N * K > 512 * 129280 * 4096:
            M //= 2
        return dict(op=op, M=M, N=N, K=K, out=rng.choice(("bf16", "fp32")), bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                    act=rng.choice(ACTS))
    vocab = rng.choice(VOCABS)
    if op == "control":
        rows = rng.randint(1, 6)
        return dict(op=op, sequences=_log(rng, 1, 256 // rows), rows=rows, vocab=vocab, history=_log(rng, 1, 32768),
                    biases=rng.choice((0, 1, 16, 300)), masked=rng.choice(("lowest", "-inf")), allowed=rng.choice((1e-4, 0.02, 0.3, 0.99)))
    if op == "history":
        return dict(op=op, sequences=rng.randint(1, 64), length=_log(rng, 1, 32768), vocab=vocab, generated=rng.random() < 0.5)
    rows, k, dtype = _log(rng, 1, 1024), rng.choice((1, 5, 20, 33, 64, 100, 128)), rng.choice(("fp32", "bf16"))
    if op == "top":
        return dict(op=op, rows=rows, vocab=vocab, k=k, dtype=dtype, temperature=rng.choice((1.0, 0.7, 2.0)))
    return dict(op=op, call=rng.choice(("step", "pair")), rows=rows, vocab=vocab, k=k, dtype=dtype, rest=rng.random() < 0.5,
                temperature=rng.choice((1.0, 1.5, 2.0)))


# ---- inputs -----------------------------------------------------------------------


def _tokens(shape, vocab, g):
    """Token ids whose frequency falls with their rank, spread over the vocabulary."""
    u = torch.rand(shape, device=DEV, generator=g, dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab)) - 1).long().clamp_(0, vocab - 1)
    return (rank * 7919 % vocab).int()


def _bits(flags):
    """Truth values [..., vocab] as int32 words, bit b of word w for entry 32 w + b."""
    pad = -flags.shape[-1] % 32
    f = torch.nn.functional.pad(flags, (0, pad)).unflatten(-1, (-1, 32)).long()
    w = (f << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _flags(words, vocab):
    """The truth values of _bits' words."""
    return ((words.unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).flatten(-2)[..., :vocab].bool()


def _table(case, g):
    """A token table as the history calls leave it: counts of generated tokens, and a bit for every token that
    the prompt or the answer holds."""
    S, V, L = case["sequences"], case["vocab"], case["history"]
    toks = _tokens((S, L), V, g).long()
    answer = torch.arange(L, device=DEV).expand(S, L) >= L // 2  # the second half was generated
    counts = torch.zeros(S, V, dtype=torch.int32, device=DEV).scatter_add_(1, toks, answer.int())
    seen = torch.zeros(S, V, dtype=torch.bool, device=DEV).scatter_(1, toks, True)
    return counts, seen


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(shape, std=1.0, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)

    s = dict(case=case)
    if case["op"] == "dense":
        M, N, K = case["M"], case["N"], case["K"]
        dt = torch.float32 if case["out"] == "fp32" else torch.bfloat16
        s["x"], s["w"] = normal((M, K), 1.0, torch.bfloat16), normal((N, K), 0.02, torch.bfloat16)
        s["bias"] = normal((N,), 0.1) if case["bias"] else None
        s["residual"] = normal((M, N), 1.0, dt) if case["residual"] else None
        s["y"] = torch.empty((M, N), dtype=dt, device=DEV)
        s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    elif case["op"] == "control":
        S, R, V = case["sequences"], case["rows"], case["vocab"]
        s["logits"], s["out"] = normal((S * R, V), 2.5), torch.empty((S * R, V), device=DEV)
        s["counts"], seen = _table(case, g)
        s["seen"] = _bits(seen)
        s["drafts"] = _tokens((S, max(R - 1, 1)), V, g)
        s["penalties"] = torch.tensor([[1.1, 0.2, 0.4]], device=DEV).repeat(S, 1) + 0.1 * torch.rand((S, 3), device=DEV, generator=g)
        n = case["biases"]
        s["bias_ids"] = _tokens((S * n,), V, g) if n else None
        s["bias_values"] = normal((S * n,), 4.0) if n else None
        s["bias_offsets"] = torch.arange(S + 1, dtype=torch.int32, device=DEV) * n if n else None
        rows = torch.arange(S * R, device=DEV)
        # a row in four of a batch is unconstrained; every grammar allows something
        s["mask_index"] = torch.where((rows % 4 == 3) & (S > 1), -1, rows).int()
        allowed = torch.rand((S * R, V), device=DEV, generator=g) < case["allowed"]
        allowed[rows, _tokens((S * R,), V, g).long()] = True
        s["mask"] = _bits(allowed)
        s["masked"] = LOWEST if case["masked"] == "lowest" else -math.inf
    elif case["op"] == "history":
        S, L, V = case["sequences"], case["length"], case["vocab"]
        s["tokens"] = _tokens((S * L,), V, g)
        s["offsets"] = torch.arange(S + 1, dtype=torch.int32, device=DEV) * L
        s["counts"] = torch.zeros((S, V), dtype=torch.int32, device=DEV)
        s["seen"] = torch.zeros((S, (V + 31) // 32), dtype=torch.int32, device=DEV)
    else:
        n, V, k = case["rows"], case["vocab"], case["k"]
        dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        s["logits"] = normal((n, V), 2.5, dt)
        likely = torch.randint(0, V, (n, 100), device=DEV, generator=g)
        s["logits"].scatter_(1, likely, (9 + 7 * torch.rand(V, device=DEV, generator=g)).to(dt)[likely])
        s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
        if case["op"] == "top":
            s["chosen"] = _tokens((n,), V, g)
            s["ids"] = torch.empty((n, k), dtype=torch.int32, device=DEV)
            s["values"] = torch.empty((n, k), device=DEV)
            s["lse"], s["logprob"] = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
        else:
            # the teacher's rows are the drafter's with noise, as a verify step leaves them
            part = max(1, (1 << 28) // V)
            top = [(s["logits"][i:i + part].float() + normal((min(part, n - i), V), 0.5)) for i in range(0, n, part)]
            best = [t.topk(k, dim=1) for t in top]
            s["teacher_ids"] = torch.cat([b.indices for b in best]).int()
            s["teacher_logits"] = torch.cat([b.values for b in best])
            s["teacher_lse"] = torch.cat([(t / case["temperature"]).logsumexp(1) for t in top]) if case["rest"] else None
            s["grad_loss"] = 0.5 + torch.rand(n, device=DEV, generator=g)
            s["loss"], s["stats"] = torch.empty(n, device=DEV), torch.empty((n, 2), device=DEV)
            s["grad"] = torch.empty((n, V), dtype=dt, device=DEV)
    return s


# ---- one pass ---------------------------------------------------------------------


def run(s):
    return {"dense": _dense, "control": _control, "history": _history, "top": _top, "distill": _distill}[s["case"]["op"]](s)


def _dense(s):
    if own:
        G = _framework()
        return G.dense_bf16(s["x"], s["w"], bias=s["bias"], residual=s["residual"], act=s["case"]["act"], out=s["y"], workspace=s["workspace"])
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"]
    act = s["case"]["act"]
    if act == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif act == "silu":
        y = y / (1 + torch.exp(-y))
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["y"].dtype)


def _control(s):
    c = s["case"]
    S, R, V = c["sequences"], c["rows"], c["vocab"]
    drafts = s["drafts"] if R > 1 else None
    if own:
        G = _framework()
        return G.logits_control(s["logits"], R, counts=s["counts"], seen=s["seen"], drafts=drafts, penalties=s["penalties"], bias_ids=s["bias_ids"],
                                bias_values=s["bias_values"], bias_offsets=s["bias_offsets"], mask=s["mask"], mask_index=s["mask_index"],
                                masked_value=s["masked"], out=s["out"])
    x = s["logits"].view(S, R, V)
    count = s["counts"].unsqueeze(1).expand(S, R, V)
    seen = _flags(s["seen"], V).unsqueeze(1).expand(S, R, V)
    if drafts is not None:
        before = (torch.arange(R - 1, device=DEV) < torch.arange(R, device=DEV).unsqueeze(1)).int().expand(S, R, R - 1)
        extra = torch.zeros(S, R, V, dtype=torch.int32, device=DEV).scatter_add_(2, drafts.long().unsqueeze(1).expand(S, R, R - 1), before)
        count, seen = count + extra, seen | (extra > 0)
    rep, freq, pres = (p.view(S, 1, 1) for p in s["penalties"].unbind(1))
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * count - pres * (count > 0)
    if s["bias_ids"] is not None:
        at = torch.arange(S * c["biases"], device=DEV).view(S, -1)
        last = torch.full((S, V), -1, device=DEV).scatter_reduce_(1, s["bias_ids"].view(S, -1).long(), at, "amax")
        x = x + torch.where(last >= 0, s["bias_values"][last.clamp(min=0)], 0.0).unsqueeze(1)
    x = x.reshape(S * R, V)
    # the masks here allow something, and no bias or penalty reaches the lower bound of what they allow
    banned = ~_flags(s["mask"], V)[s["mask_index"].clamp(min=0).long()] & (s["mask_index"] >= 0).unsqueeze(1)
    return torch.where(banned, s["masked"], x)


def _history(s):
    c = s["case"]
    if own:
        G = _framework()
        G.token_counts_clear(s["counts"], s["seen"], c["vocab"])
        G.token_counts_add(s["counts"], s["seen"], c["vocab"], s["tokens"], s["offsets"], generated=c["generated"])
        return s["counts"], s["seen"]
    toks = s["tokens"].view(c["sequences"], c["length"]).long()
    n = torch.zeros_like(s["counts"]).scatter_add_(1, toks, torch.ones_like(toks, dtype=torch.int32))
    return n * int(c["generated"]), _bits(n > 0)


def _top(s):
    c = s["case"]
    if own:
        G = _framework()
        return G.top_logits(s["logits"], c["k"], temperature=c["temperature"], chosen=s["chosen"], ids=s["ids"], values=s["values"], lse=s["lse"],
                            logprob=s["logprob"], workspace=s["workspace"])
    x = s["logits"].float() + 0.0
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits) << 32  # the order of the values, then the lowest index
    best = (key | (0xffffffff - torch.arange(c["vocab"], device=DEV))).topk(c["k"], dim=1).values
    ids = 0xffffffff - (best & 0xffffffff)
    del key, bits
    z = x / c["temperature"]
    m = z.amax(1, keepdim=True)
    lse = m.squeeze(1) + torch.log(torch.exp(z - m).sum(1))
    return ids.int(), x.gather(1, ids), lse, z.gather(1, s["chosen"].long().unsqueeze(1)).squeeze(1) - lse


def _distill(s):
    c, T = s["case"], s["case"]["temperature"]
    if own:
        G = _framework()
        given = dict(teacher_lse=s["teacher_lse"], temperature=T, workspace=s["workspace"])
        if c["call"] == "step":
            G.distill_step(s["logits"], s["teacher_ids"], s["teacher_logits"], s["grad_loss"], loss=s["loss"], stats=s["stats"], grad=s["grad"], **given)
        else:
            G.distill_forward(s["logits"], s["teacher_ids"], s["teacher_logits"], loss=s["loss"], stats=s["stats"], **given)
            G.distill_backward(s["logits"], s["teacher_ids"], s["teacher_logits"], s["stats"], s["grad_loss"], grad=s["grad"],
                               teacher_lse=s["teacher_lse"], temperature=T)
        return s["loss"], s["stats"], s["grad"]
    ids = s["teacher_ids"].long()
    t = s["teacher_logits"].double() / T
    logp = t - (s["teacher_lse"].double().unsqueeze(1) if c["rest"] else t.logsumexp(1, keepdim=True))
    p = logp.exp()
    z = s["logits"].float() / T
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    # long sums, and differences of near values (of log-sums, of what the k leave of 1), in 64 bits
    inside, total = e.gather(1, ids).double().sum(1, keepdim=True), e.sum(1, keepdim=True, dtype=torch.float64)
    lse = m.double() + torch.log(total)
    at = (z.gather(1, ids) - lse).exp() - p
    loss = (p * (logp - (z.gather(1, ids) - lse))).sum(1)
    scale, logr = torch.ones_like(lse), torch.zeros_like(lse)
    if c["rest"]:
        outside = e.scatter(1, ids, 0.0).sum(1, keepdim=True, dtype=torch.float64)
        logr = -torch.log1p(inside / outside)
        pr = (1 - p.sum(1, keepdim=True)).clamp(min=0)
        loss = loss + torch.where(pr > 0, pr * (torch.log(pr) - logr), 0.0).squeeze(1)
        scale = 1 - pr / torch.exp(logr)
    g = s["grad_loss"].unsqueeze(1) / T
    grad = (e * (scale / total).float()).scatter_(1, ids, at.float()) * g
    return loss.float(), torch.cat((lse, logr), 1).float(), grad.to(s["grad"].dtype)


# ---- what a pass cannot do without --------------------------------------------------


def work(case):
    op = case["op"]
    if op == "dense":
        M, N, K, out = case["M"], case["N"], case["K"], 4 if case["out"] == "fp32" else 2
        return dict(bytes=2 * M * K + 2 * N * K + (4 * N if case["bias"] else 0) + M * N * out * (2 if case["residual"] else 1), flops=2 * M * N * K)
    V = case["vocab"]
    if op == "control":
        S, n = case["sequences"], case["sequences"] * case["rows"]
        return dict(bytes=n * V * 8 + n * V // 8 + S * V // 8 + S * min(case["history"], V) * 4 + S * case["biases"] * 8, flops=n * V)
    if op == "history":
        S, L = case["sequences"], case["length"]
        return dict(bytes=S * (V * 4 + V // 8) + S * L * 4, flops=S * L)
    size, n, k = 4 if case["dtype"] == "fp32" else 2, case["rows"], case["k"]
    if op == "top":
        return dict(bytes=n * (V * size + 8 * k + 12), flops=4 * n * V)
    return dict(bytes=n * (2 * V * size + 8 * k + 16), flops=8 * n * V)


# ---- the definitions in 64 bits -----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "dense":
        y = torch.mm(s["x"].double(), s["w"].double().t())
        if case["bias"]:
            y += s["bias"].double()
        if case["act"] == "relu":
            y = y.clamp(min=0)
        elif case["act"] == "silu":
            y = y * torch.special.expit(y)
        elif case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        return y + s["residual"].double() if case["residual"] else y
    V = case["vocab"]
    if op == "control":
        S, R = case["sequences"], case["rows"]
        x = s["logits"].double()
        for seq in range(S):
            rep, freq, pres = s["penalties"][seq].double()
            seen = _flags(s["seen"][seq], V)
            count = s["counts"][seq].long()
            bias = torch.zeros(V, dtype=torch.float64, device=DEV)
            for i in range(seq * case["biases"], (seq + 1) * case["biases"]):
                bias[s["bias_ids"][i].long()] = s["bias_values"][i].double()
            for j in range(R):
                row = x[seq * R + j]
                if j:
                    d = s["drafts"][seq, j - 1].long()
                    count = count.clone()
                    count[d] += 1
                    seen = seen.clone()
                    seen[d] = True
                row = torch.where(seen, torch.where(row > 0, row / rep, row * rep), row)
                row = row - freq * count - torch.where(count > 0, pres, 0.0) + bias
                m = int(s["mask_index"][seq * R + j])
                x[seq * R + j] = row if m < 0 else torch.where(_flags(s["mask"][m], V), row, s["masked"])
        return x
    if op == "history":
        toks = s["tokens"].view(case["sequences"], -1).long()
        n = torch.stack([torch.bincount(t, minlength=V) for t in toks])
        return (n if case["generated"] else torch.zeros_like(n)).int(), _bits(n > 0)
    T, n, part = case["temperature"], case["rows"], max(1, (1 << 27) // V)
    got = []
    for i in range(0, n, part):
        x = s["logits"][i:i + part].double()
        lse = torch.logsumexp(x / T, 1)
        if op == "top":
            v, at = torch.sort(x, dim=1, descending=True, stable=True)
            c = s["chosen"][i:i + part].long().unsqueeze(1)
            got.append((at[:, :case["k"]].int(), v[:, :case["k"]].clone(), lse, x.gather(1, c).squeeze(1) / T - lse))
            continue
        ids = s["teacher_ids"][i:i + part].long()
        t = s["teacher_logits"][i:i + part].double() / T
        logp = t - s["teacher_lse"][i:i + part].double().unsqueeze(1) if case["rest"] else torch.log_softmax(t, 1)
        logq = torch.log_softmax(x / T, 1)
        target = torch.zeros_like(x).scatter_(1, ids, logp.exp())
        loss = (logp.exp() * (logp - logq.gather(1, ids))).sum(1)
        logr, ratio = torch.zeros_like(lse), torch.zeros_like(lse)
        if case["rest"]:
            logr = torch.logsumexp((x / T).scatter(1, ids, -math.inf), 1) - lse
            pr = (1 - logp.exp().sum(1)).clamp(min=0)
            loss += torch.xlogy(pr, pr) - pr * logr
            ratio = pr / logr.exp()
        q = logq.exp()
        q = torch.where(torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids, True), q, q * (1 - ratio).unsqueeze(1))
        got.append((loss, torch.stack((lse, logr), 1), (q - target) * (s["grad_loss"][i:i + part].double() / T).unsqueeze(1)))
    return tuple(torch.cat(p) for p in zip(*got))
