"""What the operators over rows of logits make of tensors that are more than their bytes: no GPU needed."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from multimodal_seq2seq_gscan_amd import logits as ops


@pytest.fixture()
def on_host(monkeypatch):
    """The Python layer with CPU tensors; the library's calls are left out."""
    from multimodal_seq2seq_gscan_amd import build
    build.build()
    calls = []
    monkeypatch.setattr(ops, "_require", lambda names, *tensors: 0)
    monkeypatch.setattr(ops, "_call", lambda name, device, *args: calls.append((name, args)))
    return calls


@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_a_forward_mode_derivative_is_refused(on_host, leaf, grad):
    """The loss has a backward pass only: logits with a tangent raise, whether or not a gradient is asked for as well, and do
    not come back as a loss without a derivative."""
    x = torch.randn(2, 3, 10, requires_grad=leaf)
    index, teacher = torch.zeros(2, 3, 4, dtype=torch.int32), torch.zeros(2, 3, 4)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="jvp"):
            ops.distillation_loss(dual, index, teacher)
        assert not ops.distillation_loss(x.detach(), index, teacher).requires_grad      # others are taken in its place
    assert ops.distillation_loss(x, index, teacher).requires_grad == leaf


def conjugated(n, *shape):
    """A lazily negated view of n floats and lazily conjugated complex numbers, in these shapes."""
    x = torch.complex(torch.randn(*shape, generator=torch.Generator().manual_seed(n)), torch.randn(*shape))
    assert x.conj().is_conj() and x.conj().imag.is_neg()
    return x.conj(), x.conj().imag


def copy_states(calls):
    """What gscan_beam_reorder does with a table of states, on the host."""
    def call(name, device, B, W, order, table, count):
        import ctypes as C
        parents = (C.c_int32 * (B * W)).from_address(order)
        for s in table[:count]:
            for o in range(s.outer):
                for r in range(B * W):
                    for m in range(s.mid):
                        C.memmove(s.dst + o * s.out_outer + r * s.out_row + m * s.out_mid,
                                  s.src + o * s.in_outer + (r // W * W + parents[r]) * s.in_row + m * s.in_mid, s.bytes)
        calls.append((name, ()))
    return call


def test_lazily_conjugated_and_negated_states_are_moved_by_value(on_host, monkeypatch):
    monkeypatch.setattr(ops, "_call", copy_states(on_host))
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]], dtype=torch.int32)
    rows = (torch.arange(2)[:, None] * 3 + parents).reshape(-1)
    for state in conjugated(1, 6, 5):
        got = ops.beam_reorder(parents, state)
        assert not got.is_conj() and not got.is_neg() and torch.equal(got, state[rows])
        cache = torch.zeros(6, 9, dtype=state.dtype)
        ops.beam_reorder(parents, [state], out=[cache[:, :5]])
        assert torch.equal(cache[:, :5], state[rows]) and (cache[:, 5:] == 0).all()
    strided = conjugated(2, 4, 6, 3, 8)[1][::2, :, 1:, ::2]             # copied first: the strides are no one dimension's
    assert torch.equal(ops.beam_reorder(parents, strided, dim=1), strided[:, rows])
    assert len(on_host) == 5


def test_outputs_that_are_written_through_a_conjugation_are_refused(on_host):
    parents = torch.zeros(2, 3, dtype=torch.int32)
    for out in conjugated(3, 6, 5):
        with pytest.raises(ValueError, match="conjugat"):
            ops.beam_reorder(parents, torch.zeros(6, 5, dtype=out.dtype), out=out)
    assert not on_host


def floats_at(address, like):
    import ctypes as C
    return torch.tensor(list((C.c_float * like.numel()).from_address(address))).view(like.shape)


def test_lazily_negated_logits_scores_and_gradients_are_read_by_value(on_host, monkeypatch):
    """Everything that the library reads as floats: what lies at the addresses that it is given."""
    seen = []

    def call(name, device, rows, *args):
        rows = rows._obj
        took = [floats_at(rows.data, torch.empty(rows.outer, rows.inner, rows.V))]
        if name == "gscan_distillation_loss":
            terms, upstream = args[0]._obj, args[1]
            took.append(floats_at(terms.teacher, torch.empty(rows.outer, rows.inner, terms.K)))
            if upstream:
                took.append(floats_at(upstream, torch.empty(())))
        if name == "gscan_beam_select":
            took.append(floats_at(args[0], torch.empty(rows.outer, rows.inner)))
        seen.append(took)
    monkeypatch.setattr(ops, "_call", call)
    # adjacent words: the imaginary parts of complex numbers lie two floats apart
    logits, teacher, scores = (torch._neg_view(torch.randn(*shape)) for shape in ((2, 3, 10), (2, 3, 4), (2, 3)))
    index = torch.zeros(2, 3, 4, dtype=torch.int32)
    ops.top_logits(logits, 2)
    ops.distillation_loss(logits, index, teacher)
    ops.distillation_loss_and_gradient(logits, index, teacher)
    ops.beam_select(logits, scores, torch.zeros(2, 3, dtype=torch.bool), eos_idx=2, pad_idx=0)
    assert len(seen) == 4
    for took, want in zip(seen, ([logits], [logits, teacher], [logits, teacher], [logits, scores])):
        assert all(torch.equal(a, b) for a, b in zip(took, want)) and len(took) == len(want)
    # a gradient that arrives negated: that of the imaginary part of a conjugated number
    leaf = torch.randn(2, 3, 10, requires_grad=True)
    loss = ops.distillation_loss(leaf, index, teacher)
    torch.complex(torch.zeros(()), loss).conj().backward(torch.complex(torch.tensor(0.0), torch.tensor(3.0)))
    assert seen[-1][2].item() == -3.0
    # and from the operator's own entry to a number of other strides
    x = conjugated(4, 2, 3, 10)[1]
    ops.top_logits(x, 2)
    assert torch.equal(seen[-1][0], x)
    grad = torch.zeros(2, 3, 10)
    with pytest.raises(ValueError, match="negated"):
        ops.distillation_loss_and_gradient(logits, index, teacher, out=torch._neg_view(grad))
