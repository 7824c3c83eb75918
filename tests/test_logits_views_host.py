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
