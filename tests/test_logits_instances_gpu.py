"""The operators over rows of logits at the sizes that decide which kernel runs: every compiled form of the long-row kernels is
launched here, on both sides of each rule, against statements in 64 bits."""
import math

import pytest
import torch

import test_logits_gpu as plain
from test_logits_gpu import HALF_STEP, LEAST, NEG, TYPES, check_beams, gen, ops, student, top_oracle  # noqa: F401

pytestmark = pytest.mark.gpu

F32, BF16, F16 = TYPES


# ---------------------------------------------------------------------------------------------------------------------
# the top K of rows that are not split: 512 of them
# ---------------------------------------------------------------------------------------------------------------------
def check_many(ops, x, k, lse):  # noqa: F811
    """`x` [n, V], n a divisor of 512, as 512 rows that repeat it (a stride of zero): every copy has the same answer."""
    n, V = x.shape
    got = ops.top_logits(x.cuda().expand(512 // n, n, V), k, return_lse=lse)
    v, i, s = top_oracle(x, k)
    for g, want in zip(got, (v, i)):
        first = g[0].cpu()
        assert torch.equal(first.to(want.dtype), want)
        assert torch.equal(g, g[:1].expand_as(g))
    if lse:
        g = got[2][0].cpu().double()
        assert torch.equal(got[2], got[2][:1].expand_as(got[2]))
        live = torch.isfinite(s)
        assert torch.equal(g[~live], s[~live])
        # each term is off by 2^-23 |distance| (weighted: at most log V) + 2^-22, a thread's partial sum by 2^-24 a term
        tol = (math.log(V) + 4 + V / 256) * 2.0 ** -23 + s.abs() * 2.0 ** -24
        assert ((g - s).abs() <= tol)[live].all(), (g - s).abs().max()


# 256 threads a row: pieces of 16 bytes in registers up to 1024, their maxima kept one by one up to 4096 and 8192 of them, by groups
# of two and three pieces beyond
LONG = [(F32, 4096), (F32, 4097), (F32, 16384), (F32, 16385), (F32, 32768), (F32, 32772), (F32, 70001),
        (BF16, 8192), (BF16, 8193), (BF16, 20003), (BF16, 32768), (BF16, 32769), (BF16, 65536), (BF16, 65544), (BF16, 131075),
        (F16, 8192), (F16, 8200), (F16, 32001), (F16, 40000), (F16, 65543), (F16, 65545), (F16, 140001)]


EDGES = [(F32, 4097), (F32, 16385), (F32, 32772), (BF16, 8193), (F16, 40000), (BF16, 65544)]


@pytest.mark.parametrize("dtype,V,k,lse", [(*size, *how) for size in LONG for how in ((64, True), (256, False))]
                         + [(*size, *how) for size in EDGES for how in ((1, False), (65, True))])
def test_top_of_long_rows(ops, dtype, V, k, lse):  # noqa: F811
    g = gen(V, k, 90)
    x = (torch.randn(16, V, generator=g) * 3).to(dtype)
    x[1] = torch.sort(x[1])[0]                                          # the best words in the last groups
    x[2] = torch.sort(x[2], descending=True)[0]
    x[3] = torch.randint(-2, 3, (V,), generator=g).to(dtype)            # many equal
    x[4] = torch.where(torch.rand(V, generator=g) < 0.5, x[4], torch.tensor(NEG, dtype=dtype))
    x[5, torch.rand(V, generator=g) < 0.9] = float("nan")
    x[6, 1:] = NEG                                                      # one word
    x[7] = NEG                                                          # none
    x[8, :-3] = float("nan")                                            # three, behind the last whole piece
    x[9] = torch.finfo(dtype).min
    x[10, V // 2] = float("inf")
    x[11, -min(k + 2, V):] += 40.0                                      # the best k + 2 at the row's end
    x[12, :k + 2] += 40.0
    x[13] = 0.0
    x[13, V - 1], x[13, V // 3] = 1.0, 1.0                              # two above many equal
    step = 256 * (4 if dtype == F32 else 8)
    x[14, torch.arange(V) % step < 4] += 30.0                           # one thread's words
    x[15, (V - 1) // step * step:] += 30.0                              # the last round, which not every thread has a piece of
    check_many(ops, x, k, lse)


@pytest.mark.parametrize("dtype,V", [(F32, 513), (F32, 1024), (F32, 1025), (F32, 2048), (BF16, 1025), (F16, 2047), (BF16, 2048)])
@pytest.mark.parametrize("k,lse", [(1, False), (63, True), (64, True)])
def test_top_of_rows_of_one_wave(ops, dtype, V, k, lse):  # noqa: F811
    test_top_of_long_rows(ops, dtype, V, k, lse)


# ---------------------------------------------------------------------------------------------------------------------
# beams whose lists would not fit, and long rows behind a batch's beams
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V", [(1, 64, 9001), (1, 32, 40003), (1, 16, 131075), (2, 33, 20001)])
def test_beams_whose_rows_are_split_less_for_their_lists(ops, dtype, B, W, V):  # noqa: F811
    """W lists of W words and a row's chunks: 4096 entries are joined at most."""
    g = gen(B, W, V, 91)
    logits = (torch.randn(B, W, V, generator=g) * 2).to(dtype)
    scores = -torch.rand(B, W, generator=g) * 5
    finished = torch.rand(B, W, generator=g) < 0.2
    check_beams(ops, logits, scores, torch.zeros_like(finished))
    scores[:, 3::5] = NEG
    logits[finished] = float("nan")
    check_beams(ops, logits, scores, finished)
    start = torch.full((B, W), NEG)
    start[:, 0] = 0.0
    check_beams(ops, logits[:, :1].nan_to_num(0.0).expand(B, W, V).contiguous(), start, torch.zeros_like(finished))
    logits[:, :, 5:V - 4] = NEG                                         # nine words a beam, in its first and its last chunk
    check_beams(ops, logits, scores, finished)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V", [(3, 5, 17), (65, 3, 25), (2, 8, 32), (1, 1, 31)])
def test_beams_over_32_lanes(ops, dtype, B, W, V):  # noqa: F811
    plain.test_beam_step(ops, dtype, B, W, V)


def test_beams_of_a_batch_over_a_long_vocabulary(ops):  # noqa: F811
    """32 x 8 rows of float in two chunks each, three pieces to a group, with the softmax sum."""
    g = gen(92)
    B, W, V = 32, 8, 131075
    logits = torch.randn(2, W, V, generator=g) * 2
    logits[0, :, -20:] += 12.0
    logits[1, 3] = torch.sort(logits[1, 3])[0]
    scores, finished = -torch.rand(2, W, generator=g) * 5, torch.rand(2, W, generator=g) < 0.2
    many = lambda t: t.repeat(16, *[1] * (t.dim() - 1))  # noqa: E731
    got = ops.beam_select(many(logits).cuda(), many(scores).cuda(), many(finished).cuda(), eos_idx=2, pad_idx=0)
    alone = check_beams(ops, logits, scores, finished)
    want = [many(t) for t in alone]
    assert got[0].shape == (B, W)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got[1:], want[1:]))
    # the sums of other chunks are added up in another order
    assert ((got[0].cpu() - want[0]).abs() <= 2 * (math.log(V) + 4 + V / 256) * 2.0 ** -23 + want[0].abs() * 2.0 ** -23).all()


# ---------------------------------------------------------------------------------------------------------------------
# distillation: rows in registers and rows that are streamed
# ---------------------------------------------------------------------------------------------------------------------
# 8 pieces a thread of 64, 256 and 512 threads, 16 of 512 threads, then streamed; first and last size of each
HELD = [(F32, 2051), (F32, 2052), (F32, 8195), (F32, 8196), (F32, 16387), (F32, 16388), (F32, 25001), (F32, 32771),
        (BF16, 4103), (BF16, 4104), (BF16, 16391), (BF16, 16392), (BF16, 32775), (BF16, 32776), (BF16, 50001), (BF16, 65543),
        (F16, 4103), (F16, 4104), (F16, 16391), (F16, 16392), (F16, 32775), (F16, 32776), (F16, 50001), (F16, 65543)]
STREAMED = [(F32, 32772), (F32, 70001), (F32, 131072), (BF16, 65544), (BF16, 131075), (F16, 65544), (F16, 100003)]


def formula(z, index, teacher, labels, temperature, soft_weight, hard_weight):
    """Loss (sum), gradient and the size of what it is a difference of, in 64 bits."""
    z, teacher = z.double(), teacher.double()
    logp, logq, logs = (torch.log_softmax(t, -1) for t in (teacher / temperature, z / temperature, z))
    target = torch.zeros_like(z).scatter_add_(1, index, logp.exp())
    pick = torch.zeros_like(z).scatter_(1, labels[:, None], 1.0)
    loss = (soft_weight * temperature ** 2 * (logp.exp() * (logp - logq.gather(1, index))).sum()
            - hard_weight * logs.gather(1, labels[:, None]).sum())
    soft, hard = soft_weight * temperature, hard_weight
    grad = soft * (logq.exp() - target) + hard * (logs.exp() - pick)
    size = soft * (logq.exp() + target) + hard * (logs.exp() + pick)
    return loss.item(), grad, size


@pytest.mark.parametrize("dtype,V", HELD + STREAMED)
@pytest.mark.parametrize("temperature,soft,hard", [(2.0, 1.0, 0.0), (1.0, 0.5, 0.5), (2.0, 0.5, 0.5), (3.0, 0.5, 0.5), (4.0, 0.5, 0.5),
                                                   (3.5, 0.5, 0.5)])
def test_distillation_of_long_rows(ops, dtype, V, temperature, soft, hard):  # noqa: F811
    """One exponential a word, one and its power (temperatures 2, 3, 4), two; a row at the type's lowest value, which is uniform."""
    K = 33
    z, index, teacher, labels = student((4,), V, K, dtype, int(4 * temperature), torch.int64)
    z[1] = torch.finfo(dtype).min
    index[2, :5] = V - 1 - torch.arange(5)                              # words of the last piece and behind it
    index[2, 5] = V - 1                                                 # one of them twice
    labels[2], labels[3] = V - 1, index[3, 0]
    kw = dict(temperature=temperature, soft_weight=soft, hard_weight=hard)
    want, grad, size = formula(z, index, teacher, labels, **kw)
    args = (z.cuda(), index.cuda(), teacher.cuda(), labels.cuda())
    loss, got = ops.distillation_loss_and_gradient(*args, reduction="sum", **kw)
    # A density is an exponential over a sum.  The exponent, X = 1.45 D in base 2 at the most (D: the largest distance from the
    # maximum), is off by 5 roundings of itself (1 / tau, log2 e, their product, the distance, the product), the exponential by
    # 2^-22 of it, the power of it that gives the other temperature's by as many times that and 3 roundings; the sum by a rounding
    # a term (pieces of 16 bytes shared by the workgroup's threads, then eight waves; half as many again where a streamed row's
    # maximum grows) and what its terms are off by, the quotient and the mixing by 8 roundings more.
    D = (z.double().amax(-1, keepdim=True) - z.double()).max().item()
    X = 1.45 * D / (1.0 if hard else temperature)
    threads = 64 if V * z.element_size() < 8208 else 256 if V * z.element_size() < 32784 else 512
    terms = -(-V // threads) + 8 * (16 // z.element_size()) + 16
    rel = (2 * (0.7 * 5 * X + 4 * max(1, temperature if hard else 1)) + 1.5 * terms + 16) * 2.0 ** -24
    tol = rel * size + HALF_STEP[dtype] * grad.abs() + LEAST[dtype] / 2 * 1.0001
    far = (got.double().cpu() - grad).abs()
    assert (far <= tol).all(), (far / tol).max()
    # the loss: the logarithms of two sums, and K products of shares and distances
    weight = 4 * (soft * temperature ** 2 + hard)
    near = weight * (rel + (K + 8) * 2.0 ** -24 * (2 * D / temperature + 8)) + abs(want) * 2.0 ** -23
    assert abs(loss.item() - want) <= near, (loss.item(), want, near)
    alone = ops.distillation_loss(*args, reduction="sum", **kw)
    assert abs(alone.item() - want) <= near, (alone.item(), want, near)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [2100, 9000, 40000, 70000])
def test_training_against_shifted_labels_in_sums(ops, dtype, V):  # noqa: F811
    """What a training step asks for: the gradient of the sum, with the statistics that data-parallel ranks add up."""
    z, index, teacher, labels = student((2, 3), V, 4, dtype, 93, torch.int64)
    labels[0, 2], labels[1, 1] = 0, 0
    shifted = torch.cat([labels[:, 1:], torch.zeros_like(labels[:, :1])], 1)
    live = (shifted != 0).flatten()
    device, logits, rows, terms, kept = ops._distillation(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), 2.0, 0.5, 0.25, 0, True, "sum")
    stats, grad = torch.full((4,), 7.0, device="cuda"), torch.empty_like(logits)
    loss = ops._launch_distillation(device, logits, rows, terms, None, grad, stats=stats)
    flat = [t.reshape(6, -1)[live] for t in (z, index, teacher)] + [shifted.flatten()[live]]
    soft, hard = (formula(*flat, 2.0, *w)[0] for w in ((1.0, 0.0), (0.0, 1.0)))
    want = torch.tensor([0.5 * soft + 0.25 * hard, live.sum().item(), hard, soft / 4], dtype=torch.float64)      # divergences without tau^2
    # of every term at most 2e-5, as in test_logits_gpu.py
    assert ((stats.cpu().double() - want).abs() <= 2e-5 * 6 * 4 * (2 + math.log(V))).all(), (stats, want)
    assert stats[1].item() == live.sum().item() and loss.item() == stats[0].item()
    assert (grad.cpu().reshape(6, V)[~live] == 0).all()
    _, want, size = formula(*flat, 2.0, 0.5, 0.25)
    far = (grad.double().cpu().reshape(6, V)[live] - want).abs()
    assert (far <= 4e-5 * size + HALF_STEP[dtype] * want.abs() + LEAST[dtype]).all()
