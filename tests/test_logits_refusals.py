"""Refusals of the dense, control, top-logits and distillation entries: every check runs on the host before any
launch, so none of these calls needs a GPU (the addresses are never read)."""
import pytest

import ds41_gfx950 as G

P = 1 << 20  # an address: aligned, never read
INVALID = 1


def call(name, args, **change):
    a = dict(args, **change)
    return getattr(G.lib(), "ds41_" + name)(*a.values())


DENSE = dict(x=P, ldx=64, w=P, ldw=64, bias=P, residual=P, ldr=32, y=P + 4096, ldy=32, y_type=1, M=4, N=32, K=64, act=0, ws=None,
             ws_bytes=0, stream=None)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(w=None), dict(y=None), dict(M=0), dict(N=0), dict(K=0), dict(M=-1), dict(M=(1 << 20) + 1), dict(N=(1 << 20) + 1),
    dict(K=(1 << 20) + 1), dict(ldx=63), dict(ldw=63), dict(ldy=31), dict(ldr=31), dict(y_type=2), dict(y_type=-1), dict(act=-1), dict(act=4),
    dict(residual=P + 4096, ldr=40),  # in place with another stride
])
def test_dense_refusals(change):
    assert call("dense_bf16", DENSE, **change) == INVALID


def test_workspace_sizes_of_refused_shapes():
    L = G.lib()
    for bad in ((0, 8, 8), (8, 0, 8), (8, 8, 0), (1 << 21, 8, 8)):
        assert L.ds41_dense_bf16_workspace_bytes(*bad) == 0
    for bad in ((0, 100, 1), (1, 0, 1), (1, 100, 0), (1, 100, 101), (1, 100, 129), (65536, 100, 1), (1, (1 << 20) + 1, 1)):
        assert L.ds41_top_logits_workspace_bytes(*bad) == 0
    assert L.ds41_top_logits_workspace_bytes(3, 100, 100) > 0
    for bad in ((0, 100), (1, 0), (65536, 100), (1, (1 << 20) + 1)):
        assert L.ds41_distill_workspace_bytes(*bad) == 0
    assert L.ds41_distill_workspace_bytes(65535, 1 << 20) > 0


COUNTS = dict(counts=P, seen=P, table_rows=4, vocab=100, index=None)


@pytest.mark.parametrize("change", [dict(counts=None), dict(seen=None), dict(table_rows=0), dict(vocab=0), dict(vocab=(1 << 20) + 1)])
def test_token_table_refusals(change):
    assert call("token_counts_clear", dict(COUNTS, n=4, stream=None), **change) == INVALID
    add = dict(COUNTS, tokens=P, offsets=P, n=4, total=10, generated=1, stream=None)
    assert call("token_counts_add", add, **change) == INVALID
    assert call("token_counts_commit", dict(COUNTS, results=P, n=4, stream=None), **change) == INVALID


def test_token_table_refusals_of_sequences():
    for n in (0, 5, 65536):  # 5 sequences without an index need 5 table rows
        assert call("token_counts_clear", dict(COUNTS, n=n, stream=None)) == INVALID
        assert call("token_counts_add", dict(COUNTS, tokens=P, offsets=P, n=n, total=10, generated=1, stream=None)) == INVALID
        assert call("token_counts_commit", dict(COUNTS, results=P, n=n, stream=None)) == INVALID
    add = dict(COUNTS, tokens=P, offsets=P, n=4, total=10, generated=1, stream=None)
    for change in (dict(tokens=None), dict(offsets=None), dict(total=-1)):
        assert call("token_counts_add", add, **change) == INVALID
    assert call("token_counts_add", add, total=0) == 0  # nothing to add, nothing launched
    assert call("token_counts_commit", dict(COUNTS, results=None, n=4, stream=None)) == INVALID


CONTROL = dict(logits=P, ld_in=100, out=P + (1 << 16), ld_out=100, sequences=2, rows=4, vocab=100, counts=P, seen=P, table_rows=2, index=None,
               drafts=P, draft_ld=3, penalties=P, bias_ids=P, bias_values=P, bias_offsets=P, bias_total=5, mask=P, mask_ld=4, mask_rows=8,
               mask_index=None, masked=-3.0e38, stream=None)


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(out=None), dict(sequences=0), dict(sequences=65536), dict(rows=0), dict(rows=65), dict(vocab=0),
    dict(vocab=(1 << 20) + 1, ld_in=1 << 21, ld_out=1 << 21), dict(ld_in=99), dict(ld_out=99), dict(out=P, ld_out=101), dict(table_rows=0),
    dict(table_rows=1), dict(draft_ld=0), dict(bias_values=None), dict(bias_offsets=None), dict(bias_total=-1), dict(mask_ld=3),
    dict(mask_rows=0), dict(mask_rows=7), dict(masked=0.0), dict(masked=float("nan")), dict(masked=-1e29), dict(masked=float("inf")),
])
def test_control_refusals(change):
    assert call("logits_control", CONTROL, **change) == INVALID


TOP = dict(logits=P, type=0, ld=1000, rows=3, vocab=1000, k=20, temperature=1.0, ids=P, values=P, lse=P, chosen=P, logprob=P, ws=P,
           ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(type=2), dict(ld=999), dict(rows=0), dict(rows=65536), dict(vocab=0), dict(k=0), dict(k=129), dict(vocab=10, k=11),
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(ids=None),
    dict(values=None), dict(chosen=None), dict(logprob=None), dict(ids=None, values=None, lse=None, chosen=None, logprob=None), dict(ws=None),
    dict(ws=P + 16), dict(ws_bytes=64),
])
def test_top_refusals(change):
    assert call("top_logits", TOP, **change) == INVALID


TEACHER = dict(logits=P, type=1, ld=1000, rows=3, vocab=1000, ids=P, tlogits=P, k=20, tlse=None, temperature=1.0)
FORWARD = dict(TEACHER, loss=P, stats=P, ws=P, ws_bytes=1 << 20, stream=None)
BACKWARD = dict(TEACHER, stats=P, grad_loss=P, grad=P + (1 << 16), ld_grad=1000, stream=None)
STEP = dict(TEACHER, grad_loss=P, loss=P, stats=P, grad=P + (1 << 16), ld_grad=1000, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(type=2), dict(type=-1), dict(ld=999), dict(rows=0), dict(rows=65536), dict(vocab=0), dict(ids=None),
    dict(tlogits=None), dict(k=0), dict(k=129), dict(temperature=0.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
    dict(temperature=0.001), dict(temperature=1000.0), dict(temperature=-1.0), dict(stats=None),
])
def test_distill_refusals(change):
    for name, args in (("distill_forward", FORWARD), ("distill_backward", BACKWARD), ("distill_step", STEP)):
        assert call(name, args, **change) == INVALID, name


def test_distill_refusals_of_outputs():
    for change in (dict(loss=None), dict(ws=None), dict(ws=P + 8), dict(ws_bytes=1)):
        assert call("distill_forward", FORWARD, **change) == INVALID
        assert call("distill_step", STEP, **change) == INVALID
    for change in (dict(grad=None), dict(grad_loss=None), dict(ld_grad=999), dict(grad=P, ld_grad=1001)):
        assert call("distill_backward", BACKWARD, **change) == INVALID
        assert call("distill_step", STEP, **change) == INVALID


def test_binding_refuses_wrong_tensors():
    """Types, shapes and strides that the C entries cannot see."""
    import torch
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    for bad in (dict(x=x.float()), dict(w=w[:, :63]), dict(x=x.t()), dict(bias=torch.zeros(31)), dict(bias=torch.zeros(32, dtype=torch.bfloat16)),
                dict(residual=torch.zeros(4, 32)), dict(out=torch.zeros(4, 31))):
        with pytest.raises(ValueError):
            G.dense_bf16(**dict(dict(x=x, w=w), **bad))
    z = torch.zeros(4, 100)
    for bad in (dict(rows=3), dict(logits=z.double()), dict(out=z[:2]), dict(penalties=torch.zeros(3)), dict(mask=torch.zeros(4, 4)),
                dict(counts=torch.zeros(4, 100)), dict(seen=torch.zeros(4, 3, dtype=torch.int32)), dict(drafts=torch.zeros(4, 3)),
                dict(bias_ids=torch.zeros(2, dtype=torch.int32), bias_values=torch.zeros(1), bias_offsets=torch.zeros(5, dtype=torch.int32))):
        with pytest.raises(ValueError):
            G.logits_control(**dict(dict(logits=z, rows=1), **bad))
    ids, t = torch.zeros(4, 5, dtype=torch.int32), torch.zeros(4, 5)
    for bad in (dict(logits=z.half()), dict(teacher_ids=ids.long()), dict(teacher_logits=t[:3]), dict(grad=torch.zeros(4, 99)),
                dict(grad=torch.zeros(4, 100, dtype=torch.bfloat16)), dict(grad_loss=torch.zeros(3))):
        with pytest.raises(ValueError):
            G.distill_step(**dict(dict(logits=z, teacher_ids=ids, teacher_logits=t, grad_loss=torch.zeros(4), workspace=torch.zeros(1)), **bad))
    with pytest.raises(ValueError):
        G.top_logits(z, 5, ids=torch.zeros(4, 5), workspace=torch.zeros(1))
    with pytest.raises(ValueError):
        G.token_counts_commit(torch.zeros(1, 9, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), 9, torch.zeros(9, dtype=torch.int32))


@pytest.mark.parametrize("temperature", [1e-38, 1e-45, 2e38, 3.4e38])
def test_top_refuses_temperatures_whose_scale_is_not_normal(temperature):
    """log2(e) / T is infinite below FLT_MIN's reach and not a normal number above 1e38."""
    assert call("top_logits", TOP, temperature=temperature) == INVALID


def test_binding_refuses_host_tensors():
    """A host address in a kernel's arguments would fault: well-formed calls on host tensors raise before the entry."""
    import torch
    bf16, i32 = torch.bfloat16, torch.int32
    z, counts, seen = torch.zeros(4, 96), torch.zeros(4, 96, dtype=i32), torch.zeros(4, 3, dtype=i32)
    ids, t, one = torch.zeros(4, 5, dtype=i32), torch.zeros(4, 5), torch.zeros(4)
    for f in (lambda: G.dense_bf16(torch.zeros(4, 64, dtype=bf16), torch.zeros(32, 64, dtype=bf16)),
              lambda: G.logits_control(z, counts=counts, seen=seen), lambda: G.token_counts_clear(counts, seen, 96),
              lambda: G.token_counts_add(counts, seen, 96, ids.flatten(), torch.zeros(5, dtype=i32)),
              lambda: G.token_counts_commit(counts, seen, 96, torch.zeros(40, dtype=torch.uint8)), lambda: G.top_logits(z, 5),
              lambda: G.distill_forward(z, ids, t), lambda: G.distill_backward(z, ids, t, torch.zeros(4, 2), one),
              lambda: G.distill_step(z, ids, t, one)):
        with pytest.raises(ValueError, match="tensors on cpu"):
            f()


def test_binding_refuses_rows_of_another_width():
    """Enough elements, but in rows of another width, which would be read as other rows' elements. The calls are refused by
    shape, before the tensors' device is looked at."""
    import torch
    i32 = torch.int32
    z, ids, t, one = torch.zeros(4, 96), torch.zeros(4, 5, dtype=i32), torch.zeros(4, 5), torch.zeros(4)
    counts, seen, bits = torch.zeros(4, 96, dtype=i32), torch.zeros(4, 3, dtype=i32), torch.zeros(4, 6, dtype=i32)
    padded, padded_seen = torch.zeros(4, 101, dtype=i32), torch.zeros(4, 4, dtype=i32)  # of a padded vocabulary
    tokens, offsets, results = torch.zeros(5, dtype=i32), torch.zeros(5, dtype=i32), torch.zeros(160, dtype=torch.uint8)
    wrong = [lambda: G.logits_control(z, counts=padded, seen=seen), lambda: G.logits_control(z, counts=counts, seen=padded_seen),
             lambda: G.logits_control(z, counts=padded), lambda: G.logits_control(z, seen=padded_seen),
             lambda: G.logits_control(z, counts=counts.flatten()), lambda: G.logits_control(z, penalties=torch.zeros(4, 4)),
             lambda: G.logits_control(z, penalties=torch.zeros(13)), lambda: G.logits_control(z, mask=bits[:, :2]),
             lambda: G.top_logits(z, 5, ids=torch.zeros(4, 8, dtype=i32)), lambda: G.top_logits(z, 5, values=torch.zeros(5, 6)),
             lambda: G.distill_forward(z, ids, torch.zeros(4, 8)), lambda: G.distill_forward(z, torch.zeros(4, 8, dtype=i32), t),
             lambda: G.distill_forward(z, ids, t, stats=torch.zeros(4, 3)), lambda: G.distill_backward(z, ids, t, torch.zeros(4, 3), one),
             lambda: G.distill_step(z, ids, torch.zeros(4, 8), one), lambda: G.distill_step(z, ids, t, one, stats=torch.zeros(3, 4))]
    for c, s in ((padded, seen), (counts, padded_seen)):
        wrong += [lambda c=c, s=s: G.token_counts_clear(c, s, 96), lambda c=c, s=s: G.token_counts_add(c, s, 96, tokens, offsets),
                  lambda c=c, s=s: G.token_counts_commit(c, s, 96, results, n=4)]
    for f in wrong:
        with pytest.raises(ValueError) as e:
            f()
        assert "tensors on" not in str(e.value)
    # more rows than the call has, and rows in one dimension, are what they were; the tensors' device is what is refused then
    for f in (lambda: G.logits_control(z[:2], counts=counts, seen=seen, penalties=torch.zeros(4, 3)),
              lambda: G.logits_control(z, penalties=torch.zeros(12), mask=bits), lambda: G.distill_step(z[:1], ids[0], t[0], one),
              lambda: G.distill_step(z[:3], ids, t, one), lambda: G.top_logits(z[:3], 5, ids=ids, values=t)):
        with pytest.raises(ValueError, match="tensors on cpu"):
            f()
