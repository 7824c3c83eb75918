"""Tensors that are more than their bytes, on the device: lazily conjugated and negated views, forward-mode tangents."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_logits_gpu import gen, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def test_lazily_conjugated_and_negated_views(ops):  # noqa: F811
    g = gen(97)
    x = torch.complex(torch.randn(6, 70, generator=g), torch.randn(6, 70, generator=g)).cuda()
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]], dtype=torch.int32).cuda()
    rows = (torch.arange(2, device="cuda")[:, None] * 3 + parents).reshape(-1)
    for state in (x.conj(), x.conj().imag, x.imag, x):
        assert torch.equal(ops.beam_reorder(parents, state), state.resolve_conj().resolve_neg()[rows])
    z = x.conj().imag                                                   # words two floats apart, of the other sign
    plain = z.resolve_neg().contiguous()
    for a, b in zip(ops.top_logits(z, 5, return_lse=True), ops.top_logits(plain, 5, return_lse=True)):
        assert torch.equal(a, b)
    index, teacher = torch.randint(0, 70, (6, 4), generator=g).cuda(), torch.randn(6, 4, generator=g).cuda()
    for a, b in zip(ops.distillation_loss_and_gradient(z, index, torch._neg_view(teacher), temperature=2.0),
                    ops.distillation_loss_and_gradient(plain, index, -teacher, temperature=2.0)):
        assert torch.equal(a, b)
    scores, none = -torch.rand(2, 3, generator=g).cuda(), torch.zeros(2, 3, dtype=torch.bool).cuda()
    for a, b in zip(ops.beam_select(z.view(2, 3, 70), torch._neg_view(-scores), none, eos_idx=2, pad_idx=0),
                    ops.beam_select(plain.view(2, 3, 70), scores, none, eos_idx=2, pad_idx=0)):
        assert torch.equal(a, b)
    leaf = plain.clone().requires_grad_()
    loss = ops.distillation_loss(leaf, index, teacher)
    torch.complex(torch.zeros_like(loss), loss).conj().backward(torch.complex(torch.tensor(0.0), torch.tensor(3.0)).cuda())
    assert torch.equal(leaf.grad, torch.autograd.grad(ops.distillation_loss(again := plain.clone().requires_grad_(), index, teacher) * -3.0, again)[0])


def test_tangents_are_refused(ops):  # noqa: F811
    x, index, teacher = torch.randn(6, 70).cuda(), torch.zeros(6, 4, dtype=torch.int32).cuda(), torch.randn(6, 4).cuda()
    with forward_ad.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            with pytest.raises(NotImplementedError, match="jvp"):
                ops.distillation_loss(forward_ad.make_dual(leaf, torch.ones_like(x)), index, teacher)
        assert torch.isfinite(ops.distillation_loss(x, index, teacher))
