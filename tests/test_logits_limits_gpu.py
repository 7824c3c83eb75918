"""The operators over rows of logits at the largest sizes that they take: offsets beyond 32 bits, rows of 2^28 words, 2^23 - 1
rows; and a backward pass that is captured with its forward pass."""
import math

import pytest
import torch

from test_logits_gpu import NEG, TYPES, gen, ops, top_oracle  # noqa: F401

pytestmark = pytest.mark.gpu


def test_offsets_beyond_32_bits(ops):  # noqa: F811
    """70001 rows of 32008 words of 16 bits: 4.5 GB of logits, as many of gradient.  The last rows are checked one by one, the
    others are copies of the first."""
    n, V, K = 70001, 32008, 20
    g = gen(n, V)
    first, last = (torch.randn(4, V, generator=g) * 2).bfloat16(), (torch.randn(4, V, generator=g) * 2).bfloat16()
    logits = torch.empty(n, V, dtype=torch.bfloat16, device="cuda")
    logits[:] = first[0].cuda()
    logits[:4], logits[-4:] = first.cuda(), last.cuda()
    assert logits.numel() * 2 > 1 << 32
    values, index, lse = ops.top_logits(logits, K, return_lse=True)
    v, i, s = top_oracle(torch.cat([first, last]), K)
    assert torch.equal(torch.cat([index[:4], index[-4:]]).cpu().long(), i)
    assert torch.equal(torch.cat([values[:4], values[-4:]]).cpu().double(), v)
    assert ((torch.cat([lse[:4], lse[-4:]]).cpu().double() - s).abs() <= (math.log(V) + 4 + V / 256) * 2.0 ** -23 + s.abs() * 2.0 ** -24).all()
    assert torch.equal(index[4:-4], index[:1].expand(n - 8, K))
    labels = index[:, 3].long()
    labels[-2] = -100
    loss, grad = ops.distillation_loss_and_gradient(logits, index, values, labels, temperature=2.0, hard_weight=0.5, reduction="sum")
    some = [0, 1, 4, n - 5, n - 4, n - 3, n - 2, n - 1]
    alone = ops.distillation_loss_and_gradient(logits[some], index[some], values[some], labels[some], temperature=2.0, hard_weight=0.5,
                                               reduction="sum")[1]
    assert torch.equal(grad[some], alone)                        # a row's gradient of a sum is its own
    assert torch.equal(grad[5:-4], grad[4:5].expand(n - 9, V)) and (grad[-2] == 0).all()
    assert math.isfinite(loss.item())
    state = logits[:70001 // 3 * 3].view(-1, 3, V)               # slices of 192 KB, the last one's offset beyond 2^32
    beams = state.shape[0]
    parents = torch.arange(beams - 1, -1, -1, dtype=torch.int32).view(1, beams).cuda()
    moved = ops.beam_reorder(parents, state)
    assert torch.equal(moved[0], state[-1]) and torch.equal(moved[-1], state[0]) and torch.equal(moved[beams // 2], state[beams - 1 - beams // 2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, (1 << 28) + 3), (3, (1 << 24) + 9)])
def test_rows_of_many_words(ops, dtype, rows, V):  # noqa: F811
    """Small words with a few large ones among them, some in the last words and at the joints of chunks."""
    logits = torch.full((rows, V), -4.0, dtype=dtype, device="cuda")
    at = torch.tensor([0, 1, 5, 4096, 65535, 1 << 20, (1 << 23) - 1, 1 << 23, V // 2, V // 2 + 1, V // 512, V // 512 + 1, V - 4, V - 2, V - 1])
    k = len(at)
    large = torch.arange(k, 0, -1).to(dtype)[torch.randperm(k, generator=gen(V))]
    logits[:, at.cuda()] = large.cuda()
    logits[:, 7] = NEG
    logits[:, 9] = float("nan")
    values, index, lse = ops.top_logits(logits, k + 3, return_lse=True)
    order = torch.sort(large.float(), descending=True)[1]
    rest = [v for v in range(20) if v not in at.tolist() + [7, 9]][:3]           # of the equal ones the first
    assert index.cpu().tolist() == [at[order].tolist() + rest] * rows
    assert values[0].cpu().tolist() == large[order].tolist() + [-4.0] * 3
    want = math.log(math.fsum([math.exp(x) for x in large.tolist()] + [(V - k - 2) * math.exp(-4.0)]))
    # a thread adds up at most 2^12 words that are all alike, each off by 2^-22, in 2^-24 steps of its sum
    assert (lse.cpu().double() - want).abs().max() <= ((1 << 12) + 8) * 2.0 ** -24 + want * 2.0 ** -23


def test_a_beam_step_over_2_to_the_24_words(ops):  # noqa: F811
    V = 1 << 24
    logits = torch.zeros(1, 3, V, device="cuda")
    logits[0, 0, V - 1], logits[0, 1, 12345], logits[0, 2, V - 2] = 30.0, 29.0, 31.0
    scores = torch.tensor([[-1.0, -0.5, -3.0]]).cuda()
    got = ops.beam_select(logits, scores, torch.zeros(1, 3, dtype=torch.bool).cuda(), eos_idx=12345, pad_idx=0)
    assert got[1].tolist() == [[1, 0, 2]] and got[2].tolist() == [[12345, V - 1, V - 2]] and got[3].tolist() == [[True, False, False]]
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros(1, 1, 1, device="cuda").expand(1, 1, V + 1), scores[:, :1], torch.zeros(1, 1, dtype=torch.bool).cuda(),
                        eos_idx=2, pad_idx=0)


@pytest.mark.parametrize("V,k", [(9, 2), (100, 3), (600, 65), (5000, 1)])
def test_as_many_rows_as_there_may_be(ops, V, k):  # noqa: F811
    """2^23 - 1 rows that are all the same one (a stride of zero)."""
    n = (1 << 23) - 1
    row = torch.randn(V, generator=gen(V, 95)) * 2
    rows = row.cuda().expand(n, V)
    values, index = ops.top_logits(rows, k)
    v, i, _ = top_oracle(row[None], k)
    assert torch.equal(index[0].cpu().long(), i[0]) and torch.equal(values[0].cpu().double(), v[0])
    assert torch.equal(index, index[:1].expand(n, k)) and torch.equal(values, values[:1].expand(n, k))
    labels = torch.full((n,), V - 1, device="cuda")
    labels[::2] = -100
    loss = ops.distillation_loss(rows, index, values, labels, temperature=2.0, hard_weight=0.5)
    alone = ops.distillation_loss(rows[:1], index[:1], values[:1], labels[1:2], temperature=2.0, hard_weight=0.5)
    # 2^22 equal numbers added up in 64 bits, the one of them rounded once, the mean once
    assert abs(loss.item() - alone.item()) <= 2.0 ** -23 * abs(alone.item())
    with pytest.raises(Exception, match="rows"):
        ops.top_logits(row.cuda().expand(n + 1, V), k)


@pytest.mark.parametrize("V", [9, 700, 40000])
def test_a_backward_pass_captured_with_its_forward_pass(ops, V):  # noqa: F811
    """Replayed on new inputs, with eager calls between the replays, against the eager gradient."""
    B, T, K = 3, 4, 5
    static = dict(logits=torch.zeros(B, T, V, device="cuda"), index=torch.zeros(B, T, K, dtype=torch.int64, device="cuda"),
                  teacher=torch.zeros(B, T, K, device="cuda"), labels=torch.ones(B, T, dtype=torch.int64, device="cuda"))
    kw = dict(temperature=2.0, hard_weight=0.5, ignore_index=0, shift_labels=True)

    def both(s):
        leaf = s["logits"].detach().requires_grad_()
        loss = ops.distillation_loss(leaf * 1.5, s["index"], s["teacher"], s["labels"], **kw)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both(static)
    for k in range(4):
        g = gen(V, k, 96)
        fresh = dict(logits=torch.randn(B, T, V, generator=g), index=torch.randint(0, V, (B, T, K), generator=g),
                     teacher=torch.randn(B, T, K, generator=g), labels=torch.randint(0, V, (B, T), generator=g))
        for name, t in fresh.items():
            static[name].copy_(t)
        eager = both({name: t.cuda() for name, t in fresh.items()})
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))
