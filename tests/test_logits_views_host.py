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
