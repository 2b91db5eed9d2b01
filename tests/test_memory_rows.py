"""Whether two lists of rows share a byte, compiled for the host and compared with every byte marked, and the calls that
refuse outputs over their inputs: every check runs on the host before any launch, so the addresses are never read."""
import os
import subprocess

import pytest

import ds41_gfx950 as G

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "memory_rows.hpp"
using namespace ds41g;
static bool marked(const MemoryRows &a, const MemoryRows &b) {
  std::vector<char> m(4096);
  for (size_t r = 0; r < a.rows; ++r)
    for (size_t i = 0; i < a.bytes; ++i) m[a.at + r * a.stride + i] = 1;
  for (size_t r = 0; r < b.rows; ++r)
    for (size_t i = 0; i < b.bytes; ++i)
      if (m[b.at + r * b.stride + i]) return true;
  return false;
}
int main() {
  long seen = 0, meet = 0;
  for (size_t ra : {1, 2, 5}) for (size_t wa : {1, 3, 4}) for (size_t sa : {4, 6, 9})
    for (size_t rb : {1, 2, 3, 7}) for (size_t wb : {1, 2, 4}) for (size_t sb : {4, 6, 11})
      for (size_t at = 1; at < 120; ++at) {
        const MemoryRows a{40, ra, wa, sa}, b{at, rb, wb, sb};
        const bool want = marked(a, b);
        if (memory_meets(a, b) != want || memory_meets(b, a) != want) {
          std::printf("%zu %zu %zu, %zu: %zu %zu %zu\n", ra, wa, sa, at, rb, wb, sb);
          return 1;
        }
        ++seen;
        meet += want;
      }
  if (memory_meets(memory_block(nullptr, 8), memory_block(nullptr, 8))) return 2;
  const MemoryRows out[] = {memory_block((void *)100, 8), memory_block((void *)108, 8)}, in[] = {memory_block((void *)116, 8)};
  const MemoryRows over[] = {memory_block((void *)100, 9), memory_block((void *)108, 8)}, read[] = {memory_block((void *)115, 8)};
  if (memory_collides(out, in) || !memory_collides(over, in) || !memory_collides(out, read)) return 3;
  std::printf("%ld %ld\n", seen, meet);
}
"""


def test_rows_that_share_a_byte(tmp_path):
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "deepseek-v4.1-flash-pro6000_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True, timeout=120)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
    seen, meet = map(int, r.stdout.split())
    assert seen > 100000 and seen // 10 < meet < seen


INVALID = 1


def at(i):
    """Addresses far apart."""
    return (i + 1) << 32


def call(name, args, **change):
    return getattr(G.lib(), "ds41_" + name)(*dict(args, **change).values())


def accepted(name, args, **change):
    """The checks let the call pass: without a GPU its launch then fails with another error. With one it is not made, since its
    addresses are of nothing."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("no call with these addresses where there is a GPU")
    assert call(name, args, **change) not in (0, INVALID)


M, H, I = 5, 64, 40
FFN = dict(x=at(0), ldx=H, w_gate=at(1), w_up=at(2), w_down=at(3), limit=10.0)
FORWARD = dict(FFN, y=at(4), ldy=H, saved=at(5), saved_type=0, M=M, H=H, I=I, ws=at(6), ws_bytes=1 << 30, stream=None)
BACKWARD = dict(FFN, saved=at(5), saved_type=0, grad_y=at(4), ld_grad_y=H, grad_x=at(7), ld_grad_x=H, grad_gate=at(8), grad_up=at(9),
                grad_down=at(10), grad_type=1, accumulate=0, M=M, H=H, I=I, ws=at(6), ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change", [
    dict(y=at(0)), dict(y=at(0) + 2 * H * (M - 1)), dict(y=at(1)), dict(y=at(2) + 2 * I * H - 16), dict(y=at(3)), dict(y=at(5)), dict(y=at(6) + 256),
    dict(saved=at(0)), dict(saved=at(1)), dict(saved=at(3) + 16), dict(saved=at(4) + 16), dict(saved=at(6)),
    dict(saved=at(0) - 4 * 2 * I * M + 16), dict(ws=at(0)), dict(ws=at(1)), dict(ws=at(3)),
    dict(x=at(0), ldx=160, y=at(0) + 2 * 56, ldy=160)])  # rows of one buffer, eight columns shared
def test_ffn_forward_refuses_outputs_over_inputs(change):
    accepted("ffn_forward", FORWARD)
    assert call("ffn_forward", FORWARD, **change) == INVALID


@pytest.mark.parametrize("change", [
    dict(grad_x=at(4)),                                          # over the gradient that the down projection's still reads
    dict(grad_x=at(0)),                                          # over the rows that the gate's and the up projection's still read
    dict(grad_x=at(1)), dict(grad_x=at(2)), dict(grad_x=at(3)), dict(grad_x=at(5) + 16), dict(grad_x=at(6)), dict(grad_x=at(8)),
    dict(grad_gate=at(0)), dict(grad_gate=at(1)), dict(grad_gate=at(4)), dict(grad_gate=at(9)), dict(grad_up=at(2)), dict(grad_up=at(0) + 16),
    dict(grad_up=at(10)), dict(grad_down=at(3)), dict(grad_down=at(4)), dict(grad_down=at(5)), dict(grad_down=at(7) + 16),
    dict(grad_gate=at(9) - 4 * I * H + 16, grad_type=0),         # fp32 gradients reach twice as far
    dict(ws=at(0)), dict(ws=at(5)), dict(ws=at(10)),
    dict(ldx=160, grad_x=at(0) + 2 * 56, ld_grad_x=160)])
def test_ffn_backward_refuses_outputs_over_inputs(change):
    accepted("ffn_backward", BACKWARD)
    assert call("ffn_backward", BACKWARD, **change) == INVALID


def test_ffn_takes_columns_of_one_buffer():
    accepted("ffn_forward", FORWARD, ldx=2 * H, y=at(0) + 2 * H, ldy=2 * H)
    accepted("ffn_forward", FORWARD, ldx=2 * H + 8, y=at(0) + 2 * H, ldy=2 * H + 8)
    accepted("ffn_forward", FORWARD, w_up=at(1))  # inputs may be the same
    accepted("ffn_forward", FORWARD, saved=None)
    accepted("ffn_backward", BACKWARD, ldx=2 * H, grad_x=at(0) + 2 * H, ld_grad_x=2 * H)
    accepted("ffn_backward", BACKWARD, grad_gate=at(9) - 2 * I * H)
    accepted("ffn_backward", BACKWARD, grad_gate=at(9) - 4 * I * H, grad_type=0)
    accepted("ffn_backward", BACKWARD, grad_x=None, grad_up=None)
    accepted("ffn_backward", BACKWARD, grad_gate=None, grad_up=None, grad_down=None)
    # a workspace that reaches over another tensor behind what the call needs
    accepted("ffn_forward", FORWARD, ws=at(4) - (G.ffn_workspace_bytes(M, H, I) + 255) // 256 * 256)


# The refusals of the block's other arguments, each by itself: distinct addresses, so that nothing else refuses them.
BOTH = [dict(x=None), dict(w_gate=None), dict(w_up=None), dict(w_down=None), dict(ldx=63), dict(ldx=56), dict(ldx=68), dict(x=at(0) + 8),
        dict(w_gate=at(1) + 8), dict(w_up=at(2) + 2), dict(w_down=at(3) + 4), dict(limit=-1.0), dict(limit=float("nan")), dict(limit=float("inf")),
        dict(M=0), dict(M=(1 << 20) + 1), dict(H=0), dict(H=60), dict(I=0), dict(I=44), dict(I=65544), dict(ws=None), dict(ws=at(6) + 16),
        dict(ws_bytes=256), dict(saved=at(5) + 8), dict(saved_type=2), dict(saved_type=-1)]


@pytest.mark.parametrize("change", BOTH + [dict(y=None), dict(ldy=56), dict(ldy=65), dict(y=at(4) + 8)])
def test_ffn_forward_refusals_alone(change):
    assert call("ffn_forward", FORWARD, **change) == INVALID


@pytest.mark.parametrize("change", BOTH + [
    dict(saved=None), dict(grad_y=None), dict(ld_grad_y=63), dict(ld_grad_x=56), dict(grad_x=at(7) + 8), dict(grad_gate=at(8) + 8), dict(grad_up=at(9) + 4),
    dict(grad_down=at(10) + 2), dict(grad_type=2), dict(grad_type=-1)])
def test_ffn_backward_refusals_alone(change):
    assert call("ffn_backward", BACKWARD, **change) == INVALID


QUANT = dict(x=at(0), type=0, ldx=64, q=at(1), scales=at(2), values=at(3), rows=3, cols=64, stream=None)


@pytest.mark.parametrize("change", [
    dict(q=at(0)), dict(q=at(0) + 4 * 191), dict(scales=at(0) + 767), dict(values=at(0), type=1), dict(values=at(0) - 382, type=1), dict(q=at(3)),
    dict(q=at(3) + 380), dict(scales=at(1) + 95), dict(scales=at(1) - 5), dict(values=at(2)), dict(ldx=80, q=at(0) + 4 * 80),
    dict(x=at(0) + 2), dict(x=at(0) + 1, type=1)])  # an address between elements
def test_quantize_refuses_outputs_over_its_rows_and_rows_between_elements(change):
    accepted("quantize_mxfp4", QUANT)
    assert call("quantize_mxfp4", QUANT, **change) == INVALID


def test_quantize_takes_outputs_beside_its_rows():
    accepted("quantize_mxfp4", QUANT, q=at(0) + 4 * 192)
    accepted("quantize_mxfp4", QUANT, scales=at(0) - 6)
    accepted("quantize_mxfp4", QUANT, scales=at(1) + 96, values=None)
    accepted("quantize_mxfp4", QUANT, rows=1, ldx=128, q=at(0) + 256)
    accepted("quantize_mxfp4", QUANT, rows=1, cols=32, ldx=40, x=at(0) + 4, scales=at(0) + 132)
    accepted("quantize_mxfp4", QUANT, x=at(0) + 2, type=1)


@pytest.mark.parametrize("change", [dict(x=None), dict(q=None), dict(scales=None), dict(type=2), dict(type=-1), dict(ldx=63), dict(rows=0),
                                    dict(rows=-1), dict(cols=0), dict(cols=48), dict(q=at(1) + 2), dict(values=at(3) + 1)])
def test_quantize_refusals_alone(change):
    assert call("quantize_mxfp4", QUANT, **change) == INVALID


N, V = 6, 1000
POLICY = dict(logits=at(0), type=0, ld=V, rows=N, vocab=V, tokens=at(1), old=at(2), advantage=at(3), ref=at(4), kl=0.1, low=0.2, high=0.3, temperature=1.0)
P_FORWARD = dict(POLICY, loss=at(6), logprob=at(7), stats=at(8), ws=at(9), ws_bytes=1 << 20, stream=None)
P_BACKWARD = dict(POLICY, stats=at(8), grad_loss=at(5), grad=at(10), ld_grad=V, stream=None)
P_STEP = dict(POLICY, grad_loss=at(5), loss=at(6), logprob=at(7), stats=at(8), grad=at(10), ld_grad=V, ws=at(9), ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change", [
    # a row's workgroups read these after the first of them has written its loss and log-probability
    dict(logprob=at(2)), dict(loss=at(3)), dict(loss=at(2) + 4), dict(logprob=at(4) + 20), dict(stats=at(2)), dict(stats=at(1) - 4),
    dict(loss=at(7)), dict(loss=at(8) + 68), dict(logprob=at(8)), dict(ws=at(0)), dict(ws=at(2)), dict(ws=at(6)), dict(loss=at(9) + 4),
    dict(loss=at(0)), dict(logprob=at(0) + 4 * 5999), dict(stats=at(1))])
def test_policy_refuses_outputs_over_inputs(change):
    accepted("policy_forward", P_FORWARD)
    accepted("policy_step", P_STEP)
    assert call("policy_forward", P_FORWARD, **change) == INVALID
    assert call("policy_step", P_STEP, **change) == INVALID


@pytest.mark.parametrize("change", [
    dict(grad=at(0) + 4), dict(grad=at(0) - 4), dict(grad=at(0), ld=V + 1), dict(grad=at(0) + 4 * 5999), dict(grad=at(2)), dict(grad=at(5)), dict(grad=at(4)),
    dict(grad=at(1)), dict(grad=at(8)), dict(ld=2 * V, grad=at(0) + 4 * (V - 1), ld_grad=2 * V), dict(ld=V + 8, grad=at(0) + 4 * V, ld_grad=V + 8)])
def test_policy_refuses_gradients_over_inputs(change):
    accepted("policy_backward", P_BACKWARD)
    assert call("policy_backward", P_BACKWARD, **change) == INVALID
    assert call("policy_step", P_STEP, **change) == INVALID


def test_policy_takes_gradients_in_place_and_beside():
    for name, args in (("policy_backward", P_BACKWARD), ("policy_step", P_STEP)):
        accepted(name, args, grad=at(0))
        accepted(name, args, type=1, grad=at(0))
        accepted(name, args, ld=2 * V, grad=at(0) + 4 * V, ld_grad=2 * V)
        accepted(name, args, ref=None, kl=0.0)
    accepted("policy_step", P_STEP, ref=at(6), kl=0.0)  # not read
    accepted("policy_forward", P_FORWARD, old=at(4))


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(type=2), dict(type=-1), dict(ld=999), dict(rows=0), dict(rows=65536), dict(vocab=0), dict(vocab=(1 << 20) + 1, ld=1 << 21),
    dict(tokens=None), dict(old=None), dict(advantage=None), dict(ref=None), dict(kl=-0.1), dict(kl=float("nan")), dict(kl=float("inf")), dict(low=-0.1),
    dict(low=1.1), dict(low=float("nan")), dict(high=-0.1), dict(high=float("inf")), dict(temperature=0.0), dict(temperature=1000.0), dict(stats=None)])
def test_policy_refusals_alone(change):
    for name, args in (("policy_forward", P_FORWARD), ("policy_backward", P_BACKWARD), ("policy_step", P_STEP)):
        assert call(name, args, **change) == INVALID, name


def test_policy_refusals_of_outputs_alone():
    for change in (dict(loss=None), dict(logprob=None), dict(ws=None), dict(ws=at(9) + 8), dict(ws_bytes=1)):
        assert call("policy_forward", P_FORWARD, **change) == INVALID
        assert call("policy_step", P_STEP, **change) == INVALID
    for change in (dict(grad=None), dict(grad_loss=None), dict(ld_grad=999), dict(grad=at(0), ld_grad=1001)):
        assert call("policy_backward", P_BACKWARD, **change) == INVALID
        assert call("policy_step", P_STEP, **change) == INVALID


def grads(*entries):
    a = (G.GradDesc * len(entries))(*(G.GradDesc(*e) for e in entries))
    a.n = len(entries)
    return a


def grad_call(name, entries, *rest):
    import ctypes
    a = grads(*entries)
    return getattr(G.lib(), "ds41_" + name)(ctypes.addressof(a), a.n, *rest, None)


LIST = [(at(0), None, 100, 0, 0), (at(1), at(2), 51, 1, 0), (None, None, 0, 0, 0)]


def grad_accepted(name, *rest):
    import torch
    if torch.cuda.is_available():
        pytest.skip("no call with these addresses where there is a GPU")
    assert grad_call(name, LIST, *rest) not in (0, INVALID)


@pytest.mark.parametrize("norm", [at(0), at(0) + 396, at(2) + 100])
def test_clip_refuses_a_norm_inside_its_outputs(norm):
    """A workgroup would scale it while others still read it."""
    grad_accepted("grad_clip", at(5), 1.0)
    grad_accepted("grad_clip", at(0) + 400, 1.0)
    grad_accepted("grad_clip", at(1), 1.0)  # read, not written
    assert grad_call("grad_clip", LIST, norm, 1.0) == INVALID


@pytest.mark.parametrize("norm,square,ws", [
    (at(0), None, at(6)), (at(5), at(0) + 392, at(6)), (at(1) + 100, None, at(6)), (at(5), None, at(0)), (at(5), None, at(1)),
    (at(5), None, at(0) - 2048 * 8), (at(6) + 8, None, at(6)), (at(5), at(6), at(6)), (at(5), at(5), at(6)), (at(5) + 4, at(5), at(6))])
def test_grad_norm_refuses_outputs_over_gradients_or_each_other(norm, square, ws):
    grad_accepted("grad_norm", at(5), at(5) + 8, at(6), 1 << 20)
    grad_accepted("grad_norm", at(0) + 400, at(5), at(6), 1 << 20)
    grad_accepted("grad_norm", at(2), None, at(6), 1 << 20)  # clipping's outputs are not this call's
    change = 0 if ws != at(0) - 2048 * 8 else 256  # reaches over the first gradient by 256 bytes
    assert grad_call("grad_norm", LIST, norm, square, ws + change, 1 << 20) == INVALID


@pytest.mark.parametrize("entries,limit,norm,square,ws", [
    (LIST, 1.0, at(0), None, at(6)), (LIST, 1.0, at(2) + 100, None, at(6)), (LIST, 1.0, at(5), at(2), at(6)), (LIST, 1.0, at(5), None, at(2)),
    (LIST, 1.0, at(5), None, at(2) - 2048 * 8), (LIST, 1.0, at(1), None, at(6)), (LIST, 1.0, at(6), None, at(6)), (LIST, 1.0, at(5), at(5), at(6)),
    (LIST, -1.0, at(5), None, at(6)), (LIST, float("nan"), at(5), None, at(6)), (LIST, float("inf"), at(5), None, at(6)), (LIST, 1.0, None, None, at(6)),
    (LIST, 1.0, at(5), None, None), (LIST, 1.0, at(5), None, at(6) + 8), (LIST + LIST[:1], 1.0, at(5), None, at(6)),
    ([(at(0), at(1), 100, 0, 0), (at(1), at(0), 100, 0, 0)], 1.0, at(5), None, at(6)), ([(at(0), None, 100, 2, 0)], 1.0, at(5), None, at(6))])
def test_norm_and_clip_refusals(entries, limit, norm, square, ws):
    grad_accepted("grad_norm_clip", 1.0, at(5), at(5) + 8, at(6), 1 << 20)
    grad_accepted("grad_norm_clip", 1.0, at(5), None, at(6), G.lib().ds41_grad_workspace_bytes(len(LIST)))
    assert grad_call("grad_norm_clip", entries, limit, norm, square, ws, 1 << 20) == INVALID
    assert grad_call("grad_norm_clip", entries, 1.0, at(5), None, at(6), G.lib().ds41_grad_workspace_bytes(len(entries)) - 1) == INVALID


def test_binding_refuses_a_sum_of_a_known_norm():
    import torch
    one = torch.zeros(1)
    with pytest.raises(ValueError, match="no sum"):
        G.grad_clip([torch.zeros(3)], 1.0, norm=one, known=True, square_sum=one.double())
