"""The operators of a training step at the ends of their sizes: offsets beyond 32 bits, the widest and the narrowest blocks, a million
rows, and workspaces of exactly the bytes asked for. Bounds: see test_gpu_ffn.py and test_gpu_policy.py."""
import pytest

import ds41_gfx950 as G
import test_gpu_ffn as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,H,I", [(33000, 64, 65536), (66000, 65536, 64)])
def test_block_offsets_beyond_32_bits(gpu, M, H, I):
    """More than 2^32 elements of the saved g and u, or of the rows and their gradients: the last rows come out as the formulas have
    them, and the weights' gradients are theirs where no other row has one."""
    import torch
    n = 40
    x, wg, wu, wd, dy = F.make(gpu, n, H, I)
    big = torch.zeros((M, H), dtype=torch.bfloat16, device=gpu)
    big[-n:] = x
    saved = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=gpu)
    y = G.ffn_forward(big, wg, wu, wd, limit=1.5, saved=saved)
    F.check_forward(x, wg, wu, wd, y[-n:], saved[-n:], 1.5)
    assert not y[:-n].any() and not saved[:1000].any() and not saved[-n - 1000:-n].any()
    del y
    grad = torch.zeros((M, H), dtype=torch.bfloat16, device=gpu)
    grad[-n:] = dy
    got = G.ffn_backward(big, wg, wu, wd, saved, grad, limit=1.5)
    F.check_backward((x, wg, wu, wd), saved[-n:], dy, 1.5, (got[0][-n:],) + got[1:])
    assert not got[0][:-n].any()


@pytest.mark.parametrize("M,H,I", [(1, 8, 65536), (1, 65536, 8), (32, 8, 65536), (32, 65536, 8), (40, 8, 65536), (40, 65536, 8), (300, 65536, 16),
                                   (300, 16, 65536), (1 << 20, 8, 8), ((1 << 20) - 1, 16, 8)])
def test_ends_of_the_blocks_sizes(gpu, M, H, I):
    import torch
    x, wg, wu, wd, dy = F.make(gpu, M, H, I)
    w = x, wg, wu, wd
    saved = torch.empty((M, 2 * I), device=gpu)
    y = G.ffn_forward(*w, limit=1.5, saved=saved)
    F.check_forward(*w, y, saved, 1.5)
    F.check_backward(w, saved, dy, 1.5, G.ffn_backward(*w, saved, dy, limit=1.5, grad_dtype=torch.float32))


@pytest.mark.parametrize("M,H,I", [(3, 264, 136), (70, 520, 1032), (405, 4096, 2880), (600, 1032, 520), (1152, 1120, 32), (2048, 5120, 2304),
                                   (2368, 1280, 6848), (2941, 6448, 1360)])
def test_a_workspace_of_the_bytes_asked_for(gpu, M, H, I):
    import torch
    x, wg, wu, wd, dy = F.make(gpu, M, H, I)
    w = x, wg, wu, wd
    n = G.ffn_workspace_bytes(M, H, I)
    buf = torch.full((n + 4096,), 255, dtype=torch.uint8, device=gpu)
    saved = torch.empty((M, 2 * I), device=gpu)
    y = G.ffn_forward(*w, saved=saved, workspace=buf[:n])
    assert torch.equal(y, G.ffn_forward(*w))
    grads = G.ffn_backward(*w, saved, dy, workspace=buf[:n])
    assert all(torch.equal(a, b) for a, b in zip(grads, G.ffn_backward(*w, saved, dy)))
    assert (buf[n:] == 255).all()


@pytest.mark.parametrize("dtype,n,V", [("bfloat16", 34000, 129280), ("float32", 33000, 131080)])
def test_policy_offsets_beyond_32_bits(gpu, dtype, n, V):
    """The last rows of more than 2^32 logits, in rows that are held and in rows that are not, come out as they do in a call of them
    alone: in place, and forward and backward apart."""
    import torch
    k = 160  # enough that a call of these rows alone goes the same way
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.zeros((n, V), dtype=getattr(torch, dtype), device=gpu)
    x[-k:] = torch.empty((k, V), device=gpu).normal_(0, 2.5, generator=g).to(x.dtype)
    few = x[-k:].clone()
    tok = torch.full((n,), -1, dtype=torch.int32, device=gpu)
    tok[-k:] = torch.randint(0, V, (k,), device=gpu, generator=g).int()
    old, A, gl = torch.full((n,), -12.0, device=gpu), torch.ones(n, device=gpu), torch.full((n,), 0.1, device=gpu)
    want = G.policy_step(few, tok[-k:], old[-k:], A[-k:], gl[-k:], clip_high=100.0)
    assert int(want[3].any(1).sum()) > k // 2
    loss, lp, stats = G.policy_forward(x, tok, old, A, clip_high=100.0)
    alone = G.policy_forward(few, tok[-k:], old[-k:], A[-k:], clip_high=100.0)
    assert torch.equal(loss[-k:], alone[0]) and torch.equal(lp[-k:], alone[1]) and torch.equal(stats[-k:], alone[2]) and not loss[:-k].any()
    apart = G.policy_backward(x, tok, old, A, stats, gl, clip_high=100.0)
    assert torch.equal(apart[-k:], G.policy_backward(few, tok[-k:], old[-k:], A[-k:], alone[2], gl[-k:], clip_high=100.0))
    assert not apart[:-k].any()
    del apart
    got = G.policy_step(x, tok, old, A, gl, grad=x, clip_high=100.0)
    assert all(torch.equal(a[-k:], b) for a, b in zip(got, want)) and not x[:-k].any()
