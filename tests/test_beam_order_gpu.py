"""The order of a beam step's candidates where their scores do not tell: scores of -inf, NaN and +inf, rows without a log-softmax,
scores so far out that those of one beam round to the same number.  Every vocabulary size has the same answer, whichever kernel
it is that takes it."""
import pytest
import torch

from test_logits_gpu import NEG, TYPES, gen, ops  # noqa: F401

pytestmark = pytest.mark.gpu

SIZES = [(3, 4, 9), (2, 16, 9), (2, 8, 5), (3, 7, 30), (2, 20, 9), (1, 4, 64), (2, 4, 200), (1, 4, 1000), (2, 3, 9000), (1, 6, 40003)]


def ordered(logits, scores, finished, eos, pad):
    """Every candidate by (score in 64 bits descending, beam, logit descending, word); logits do not count where they order
    nothing."""
    B, W, V = logits.shape
    answers = []
    for b in range(B):
        candidates = []
        for w in range(W):
            score = scores[b, w].double()
            if finished[b, w]:
                candidates.append((-score.item(), w, 0.0, pad))
                continue
            z = logits[b, w].double()
            z = torch.where(z.isnan(), torch.full_like(z, NEG), z)
            lse = torch.logsumexp(z, -1)
            if score > NEG and torch.isfinite(lse):
                total = score + (z - lse)
                total = torch.where(total.isnan(), torch.full_like(total, NEG), total)
            else:
                total, z = torch.full_like(z, NEG), torch.zeros_like(z)
            best = torch.sort(z, descending=True, stable=True)[1][:W].tolist()
            candidates += [(-total[v].item(), w, -z[v].item(), v) for v in best]
        answers.append([(-s, w, v, bool(finished[b, w]) or v == eos) for s, w, _, v in sorted(candidates)[:W]])
    return [torch.tensor([[c[i] for c in row] for row in answers], dtype=t)
            for i, t in enumerate((torch.float64, torch.int32, torch.int64, torch.bool))]


def check_order(ops, logits, scores, finished, eos=2, pad=0):  # noqa: F811
    got = [x.cpu() for x in ops.beam_select(logits.cuda(), scores.cuda(), finished.cuda(), eos_idx=eos, pad_idx=pad)]
    want = ordered(logits, scores, finished, eos, pad)
    assert torch.equal(got[1], want[1]), (got[1], want[1])
    assert torch.equal(got[2], want[2]), (got[2], want[2])
    assert torch.equal(got[3], want[3])
    far = ~torch.isfinite(want[0]) | (want[0].abs() > 1e20)
    # far out the log-softmax is less than half a step of the score's last bit
    assert torch.equal(got[0][far], want[0][far].float())


def inputs(B, W, V, dtype, key):
    g = gen(B, W, V, key)
    return (torch.randn(B, W, V, generator=g) * 2).to(dtype), -torch.rand(B, W, generator=g) * 5, torch.zeros(B, W, dtype=torch.bool)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V", SIZES)
def test_beams_without_a_log_softmax_come_last_in_the_order_of_their_words(ops, dtype, B, W, V):  # noqa: F811
    logits, scores, none = inputs(B, W, V, dtype, 80)
    logits[:, :, V // 2] = float("inf")
    check_order(ops, logits, scores, none)                              # every beam
    check_order(ops, logits, scores, torch.arange(W).expand(B, W) % 2 == 1)
    logits, scores, none = inputs(B, W, V, dtype, 81)
    logits[:, 0, V - 1] = float("inf")                                  # the best beam
    scores[:, 0] = 0.0
    check_order(ops, logits, scores, none)
    logits[:, :, 2:] = NEG                                              # and the others have two words left each
    logits[:, 0, V - 1] = float("inf")
    check_order(ops, logits, scores, none)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V", SIZES)
def test_scores_that_are_no_numbers_count_as_minus_infinity(ops, dtype, B, W, V):  # noqa: F811
    logits, scores, none = inputs(B, W, V, dtype, 82)
    check_order(ops, logits, torch.full_like(scores, float("nan")), none)
    scores[:, 1:] = float("nan")
    check_order(ops, logits, scores, none)
    logits[:, :, 2:] = NEG
    check_order(ops, logits, scores, none)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V", SIZES)
@pytest.mark.parametrize("out", [torch.finfo(torch.float32).min, -1e30, float("inf")])
def test_scores_that_round_to_the_same_number(ops, dtype, B, W, V, out):  # noqa: F811
    """A search that is started with a large negative score in the place of -inf: such beams come after what the first one has,
    by beam, logit and word."""
    logits, scores, none = inputs(B, W, V, dtype, 83)
    check_order(ops, logits, torch.full_like(scores, out), none)
    scores[:, 1:] = out
    check_order(ops, logits, scores, none)
    logits[:, 0, 2:] = NEG                                              # two words left to the first
    check_order(ops, logits, scores, none)
    logits[:, 1:, ::3] = logits[:, 1:, :1]                              # and equal logits among the others'
    check_order(ops, logits, scores, none)
