"""The operators of a training step as programs put them together: two calls at once on two streams, forms that write in place captured
into graphs and replayed, rows and outputs as columns of one buffer. Results are compared bit for bit with plain calls, which are held
against 64 bits elsewhere."""
import pytest

import ds41_gfx950 as G
import test_gpu_ffn as F

pytestmark = pytest.mark.gpu


def policy_rows(gpu, n, V, dtype, seed):
    import torch
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.empty((n, V), device=gpu).normal_(0, 2.5, generator=g).to(dtype)
    tok = torch.randint(0, V, (n,), device=gpu, generator=g).int()
    tok[::7] = -1
    old = torch.log_softmax(x.double(), 1).gather(1, tok.clamp(min=0).long().unsqueeze(1)).squeeze(1).float() - 0.05
    return x, tok, old, torch.empty(n, device=gpu).normal_(0, 1, generator=g), torch.full((n,), 1.0 / n, device=gpu)


def test_two_streams_at_once(gpu):
    """Each stream with outputs and workspaces of its own, several calls deep."""
    import torch
    blocks = [F.make(gpu, 300, 520, 776, seed=s) for s in (1, 2)]
    rows = [policy_rows(gpu, 40, 50257, torch.float32, s) for s in (1, 2)]
    held = [policy_rows(gpu, 260, 40000, torch.bfloat16, s) for s in (3, 4)]
    lists = [[torch.randn(n, device=gpu) for n in (100003, 7, 5000)] for _ in range(2)]
    masters = [torch.randn(512, 1024, device=gpu) for _ in range(2)]

    def calls(i, stream=None):
        x, wg, wu, wd, dy = blocks[i]
        saved = G._new(stream, x, (300, 2 * 776), torch.float32)
        out = [G.ffn_forward(x, wg, wu, wd, saved=saved, stream=stream)]
        out += G.ffn_backward(x, wg, wu, wd, saved, dy, stream=stream)
        out += G.policy_step(*rows[i], stream=stream)
        out += G.policy_step(*held[i], stream=stream)
        clipped = [G._new(stream, t, t.shape, t.dtype) for t in lists[i]]
        out += [G.grad_clip(lists[i], 1.0, out=clipped, stream=stream)] + clipped
        return out + list(G.quantize_mxfp4(masters[i], values=True, stream=stream))
    want = [calls(i) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i in (0, 1):
            got[i].append(calls(i, streams[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_captured_in_place_and_added(gpu):
    """A whole step in one graph: gradients added to what is there, the policy gradient in its logits' place, clipping in place."""
    import torch
    M, H, I, V = 150, 264, 328, 3001
    x, wg, wu, wd, dy = F.make(gpu, M, H, I)
    rows = policy_rows(gpu, M, V, torch.float32, 5)
    logits, ws = rows[0].clone(), torch.empty(G.ffn_workspace_bytes(M, H, I), dtype=torch.uint8, device=gpu)
    pws = torch.empty(G.lib().ds41_policy_workspace_bytes(M, V), dtype=torch.uint8, device=gpu)
    gws, norm = torch.empty(1 << 16, dtype=torch.uint8, device=gpu), torch.empty(1, device=gpu)
    saved, y, gx = torch.empty((M, 2 * I), device=gpu), torch.empty((M, H), dtype=torch.bfloat16, device=gpu), torch.empty((M, H), dtype=torch.bfloat16, device=gpu)
    first = [torch.randn(s, device=gpu) for s in ((I, H), (I, H), (H, I))]
    grads = [t.clone() for t in first]
    out = [torch.empty(M, device=gpu), torch.empty(M, device=gpu), torch.empty((M, 3), device=gpu)]

    def step():
        G.ffn_forward(x, wg, wu, wd, limit=1.5, out=y, saved=saved, workspace=ws)
        G.policy_step(logits, *rows[1:], grad=logits, loss=out[0], logprob=out[1], stats=out[2], workspace=pws)
        G.ffn_backward(x, wg, wu, wd, saved, dy, limit=1.5, grad_x=gx, grad_gate=grads[0], grad_up=grads[1], grad_down=grads[2], accumulate=True, workspace=ws)
        G.grad_clip(grads, 3.0, norm=norm, workspace=gws)

    def start():
        logits.copy_(rows[0])
        for t, f in zip(grads, first):
            t.copy_(f)
    everything = [y, logits, gx, norm, *grads, *out]
    start()
    wants = []
    for _ in range(3):  # the gradients go on from step to step, the logits come anew
        logits.copy_(rows[0])
        step()
        wants.append([t.clone() for t in everything])
    start()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    start()
    for want in wants:
        logits.copy_(rows[0])
        for t in (y, saved, gx, norm, ws, pws, gws, *out):
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(everything, want))
        x.float().sum().item()


@pytest.mark.parametrize("M", [1, 5, 100, 700])
def test_columns_of_one_buffer(gpu, M):
    """Inputs and outputs beside each other in the rows of one buffer; what lies between them stays."""
    import torch
    H, I = 264, 328
    x, wg, wu, wd, dy = F.make(gpu, M, H, I)
    saved = torch.empty((M, 2 * I), device=gpu)
    y = G.ffn_forward(x, wg, wu, wd, saved=saved)
    want = G.ffn_backward(x, wg, wu, wd, saved, dy)
    buf = torch.full((M, 4 * H + 8), 7.0, dtype=torch.bfloat16, device=gpu)
    bx, by, bdy, bgx = (buf[:, i * H:(i + 1) * H] for i in range(4))
    bx.copy_(x)
    bdy.copy_(dy)
    G.ffn_forward(bx, wg, wu, wd, out=by, saved=saved)
    got = G.ffn_backward(bx, wg, wu, wd, saved, bdy, grad_x=bgx)
    assert torch.equal(by, y) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(bx, x) and torch.equal(bdy, dy) and (buf[:, 4 * H:] == 7).all()
    n, V = M, 1000
    rows = policy_rows(gpu, n, V, torch.float32, M)
    want = G.policy_step(*rows)
    both = torch.full((n, 2 * V + 3), 7.0, device=gpu)
    both[:, :V] = rows[0]
    got = G.policy_step(both[:, :V], *rows[1:], grad=both[:, V:2 * V])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(both[:, :V], rows[0]) and (both[:, 2 * V:] == 7).all()
