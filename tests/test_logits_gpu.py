"""The operators over rows of logits against plain statements in 64 bits (on the CPU), at the sizes, masks, strides and orders
where they can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

NEG = float("-inf")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}     # the least subnormal


@pytest.fixture(scope="module")
def ops():
    from multimodal_seq2seq_gscan_amd import _lib, logits
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    _lib.load()
    return logits


def gen(*key):
    return torch.Generator().manual_seed(hash(key) % (1 << 40))


# ---------------------------------------------------------------------------------------------------------------------
# the top K
# ---------------------------------------------------------------------------------------------------------------------
def top_oracle(x, k):
    """x [N, V] on the CPU: NaN as -inf, stable sort."""
    clean = torch.where(x.isnan(), torch.full_like(x, NEG), x)
    v, i = torch.sort(clean.double(), dim=-1, descending=True, stable=True)
    return v[:, :k], i[:, :k], torch.logsumexp(clean.double(), -1)


def check_top(ops, x, k, lse=True):
    got = ops.top_logits(x, k, return_lse=lse)
    flat = x.reshape(-1, x.shape[-1]).cpu()
    v, i, s = top_oracle(flat, k)
    assert got[0].dtype == x.dtype and got[1].dtype == torch.int32 and got[0].shape == got[1].shape == (*x.shape[:-1], k)
    assert torch.equal(got[1].reshape(-1, k).cpu().long(), i)
    assert torch.equal(got[0].reshape(-1, k).cpu().double(), v)
    if lse:
        g = got[2].reshape(-1).cpu().double()
        live = torch.isfinite(s)
        assert torch.equal(g[~live], s[~live])
        # log of a sum of exponentials: each term is off by 2^-23 |distance| (weighted: at most log V) + 2^-22, a thread's
        # partial sum by 2^-24 a term, the result by half a step
        n = x.shape[-1]
        tol = (math.log(n) + 4 + n / 256) * 2.0 ** -23 + s.abs() * 2.0 ** -24
        assert ((g - s).abs() <= tol)[live].all(), (g - s).abs().max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (130, 7, 3), (5, 8, 8), (33, 9, 4), (7, 16, 16), (5, 17, 5), (9, 63, 40),
                                      (4, 64, 64), (3, 65, 65), (3, 65, 7), (5, 255, 33), (5, 257, 256), (3, 1000, 64), (6, 1000, 65),
                                      (2, 2048, 64), (2, 2049, 1), (2, 4097, 256), (1, 8191, 50), (3, 32003, 64), (1, 131072, 256),
                                      (1, 100001, 1), (530, 4099, 17), (600, 70, 3)])
def test_top_matches_a_stable_sort(ops, dtype, rows, V, k):
    g = gen(rows, V, k)
    check_top(ops, (torch.randn(rows, V, generator=g) * 3).to(dtype).cuda(), k)
    # many equal values
    check_top(ops, torch.randint(-2, 3, (rows, V), generator=g).to(dtype).cuda(), k, lse=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,k", [(3, 9, 9), (5, 64, 20), (3, 300, 64), (3, 300, 200), (513, 5000, 60), (2, 40000, 200)])
def test_top_of_awkward_rows(ops, dtype, rows, V, k):
    g = gen(rows, V, k, 1)
    least = torch.finfo(dtype).min
    for fill in (0.0, -0.0, least, NEG, float("nan")):
        check_top(ops, torch.full((rows, V), fill, dtype=dtype).cuda(), k)
    x = (torch.randn(rows, V, generator=g) * 3).to(dtype)
    for bad in (NEG, least, float("nan")):                  # a few words left, in every row others
        y = torch.full_like(x, bad)
        at = torch.randint(0, V, (rows, 3), generator=g)
        y.scatter_(1, at, torch.gather(x, 1, at))
        check_top(ops, y.cuda(), k)
    y = x.clone()
    y[:, ::3] = NEG
    y[:, 1::5] = float("nan")
    check_top(ops, y.cuda(), k)
    y = x.clone()
    y[:, V // 2] = float("inf")
    check_top(ops, y.cuda(), k)
    signed = torch.where(torch.rand(rows, V, generator=g) < 0.5, 0.0, -0.0).to(dtype)      # zeros of both signs are equal
    check_top(ops, signed.cuda(), k)
    for order in (False, True):                             # best words first, best words last
        check_top(ops, torch.sort(x, dim=-1, descending=order)[0].cuda(), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,k", [(19, 65, 32), (16, 100, 1), (5, 127, 20), (33, 128, 4), (7, 129, 16), (17, 256, 32), (3, 257, 5),
                                      (18, 500, 31), (2, 512, 33), (35, 513, 8), (17, 1000, 32), (5, 1024, 2), (3, 1025, 32), (3, 700, 100), (5, 2000, 200), (2, 2100, 256),
                                      (3, 4000, 256)])
def test_top_of_short_rows(ops, dtype, rows, V, k):
    """Rows that share a wave with others (up to 512 words of 32 bits, 1024 of 16, at most 64 looked for) and those behind; many looked
    for among few pieces."""
    test_top_matches_a_stable_sort(ops, dtype, rows, V, k)
    test_top_of_awkward_rows(ops, dtype, rows, V, k)
    x = torch.zeros(rows, V)                               # a few above many equal ones, in some of the rows
    x[::2, V // 3:V // 3 + min(5, k)] = 7.0
    x[1::2] = torch.randn(rows, V, generator=gen(rows, V, 3))[1::2]
    check_top(ops, x.to(dtype).cuda(), k)
    values, index = ops.top_logits(x.to(dtype).cuda()[:, 1:][::3], min(k, V - 1))       # strided, any alignment
    want = top_oracle(x.to(dtype)[:, 1:][::3], min(k, V - 1))
    assert torch.equal(index.cpu().long(), want[1]) and torch.equal(values.cpu().double(), want[0])


@pytest.mark.parametrize("dtype,k", [(torch.float32, 256), (torch.bfloat16, 256), (torch.float16, 100)])
def test_top_of_rows_laid_out_against_the_grouping(ops, dtype, k):
    """Rows whose large words share the threads that keep one maximum each: more candidates than the list holds."""
    vec = 4 if dtype == torch.float32 else 8
    V, g = 64 * 1024 * vec // 8, gen(k, 2)
    x = torch.randn(520, V, generator=g)
    word = torch.arange(V) % (1024 * vec)
    x[:, word < (k - 1) * vec] += 50.0
    check_top(ops, x[:1].to(dtype).expand(520, V).cuda(), k, lse=False)
    check_top(ops, x.to(dtype).cuda(), k, lse=False)
    x[:, word < (k - 1) * vec] = 60.0                      # and all of those equal
    check_top(ops, x.to(dtype).cuda(), k, lse=False)
    x = torch.zeros(520, V)                                # a few above many equal ones
    x[:, V // 3:V // 3 + 5] = 7.0
    check_top(ops, x.to(dtype).cuda(), k, lse=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_top_of_strided_and_unaligned_logits(ops, dtype):
    x = (torch.randn(3, 4, 6, 1003, generator=gen(3)) * 3).to(dtype).cuda()
    for view in (x[:, 0, :5], x[:, :3, 1:3], x[..., 1:], x[..., 3:990], x[1, 2], x[2, 3, 4], x[:, :1, :1].expand(3, 4, 6, 1003), x.transpose(2, 3)):
        check_top(ops, view, 6)


# ---------------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------------
def distill_oracle(z, index, teacher, labels, *, temperature=1.0, soft_weight=1.0, hard_weight=0.0, ignore_index=-100, shift_labels=False,
                   reduction="mean", upstream=1.0):
    """Row by row in 64 bits on the CPU: (loss, gradient, size of what the gradient is a difference of)."""
    V, K = z.shape[-1], index.shape[-1]
    lead = z.shape[:-1]
    if labels is not None and shift_labels:
        labels = torch.cat([labels[..., 1:], torch.zeros_like(labels[..., :1])], -1)
    zs, ids, ts = z.reshape(-1, V).double(), index.reshape(-1, K).long(), teacher.reshape(-1, K).double()
    ys = None if labels is None else labels.reshape(-1).tolist()
    grad, size = torch.zeros_like(zs), torch.zeros_like(zs)
    live = [r for r in range(zs.shape[0]) if ys is None or (ys[r] != ignore_index and 0 <= ys[r] < V)]
    scale = 1.0 if reduction == "sum" else 1.0 / max(1, len(live))
    loss = 0.0
    for r in live:
        if soft_weight:
            entry = (ids[r] >= 0) & (ids[r] < V) & (ts[r] != NEG)
            if entry.any():
                logp = torch.log_softmax(ts[r][entry] / temperature, -1)
                logq = torch.log_softmax(zs[r] / temperature, -1)
                p = logp.exp()
                loss += scale * soft_weight * temperature ** 2 * (p * (logp - logq[ids[r][entry]])).sum().item()
                target = torch.zeros(V, dtype=torch.float64).index_add_(0, ids[r][entry], p)
                grad[r] += scale * soft_weight * temperature * (logq.exp() - target)
                size[r] += scale * soft_weight * temperature * (logq.exp() + target)
        if hard_weight:
            logs = torch.log_softmax(zs[r], -1)
            loss += -scale * hard_weight * logs[ys[r]].item()
            pick = torch.zeros(V, dtype=torch.float64)
            pick[ys[r]] = 1.0
            grad[r] += scale * hard_weight * (logs.exp() - pick)
            size[r] += scale * hard_weight * (logs.exp() + pick)
    return loss, (grad * upstream).view(*lead, V), (size * abs(upstream)).view(*lead, V)


def check_gradient(got, want, size, dtype):
    """The densities are off by at most 2e-5 of themselves — an exponent of up to 87 below the maximum by 87 2^-23 = 1.1e-5,
    the sums of up to 128 terms a thread by 128 2^-24 = 7.7e-6, a few roundings — and the result by half a step."""
    got = got.double().cpu()
    tol = 2e-5 * size + HALF_STEP[dtype] * want.abs() + LEAST[dtype] / 2 * 1.0001
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


def check_loss(got, want, terms_size):
    # every term of a row is a sum of numbers of at most `terms_size` in 32 bits
    assert abs(got.item() - want) <= 2e-5 * max(terms_size, abs(want)), (got.item(), want)


def student(lead, V, K, dtype, key, index_dtype=torch.int32):
    g = gen(*lead, V, K, key)
    z = (torch.randn(*lead, V, generator=g) * 2).to(dtype)
    index = torch.randint(0, V, (*lead, K), generator=g).to(index_dtype)
    teacher = (torch.randn(*lead, K, generator=g) * 2 + 3).to(dtype)
    labels = torch.randint(0, V, lead, generator=g)
    return z, index, teacher, labels


OPTIONS = [dict(), dict(hard_weight=0.5, temperature=2.0), dict(hard_weight=1.0, soft_weight=0.3, temperature=1.0, reduction="sum"),
           dict(soft_weight=0.0, hard_weight=2.0, temperature=3.0), dict(temperature=0.25), dict(hard_weight=0.7, soft_weight=0.7, temperature=40.0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,V,K", [((1, 1), 1, 1), ((3, 5), 2, 2), ((2, 40), 8, 3), ((4, 9), 9, 256), ((33,), 16, 5), ((5,), 17, 17),
                                      ((3, 2), 64, 70), ((4,), 65, 1), ((2, 3), 127, 60), ((3,), 1000, 256), ((2,), 2048, 16),
                                      ((2,), 2052, 16), ((2,), 4096, 8), ((2,), 4104, 65), ((1, 2), 16385, 31), ((2,), 32770, 64)])
@pytest.mark.parametrize("options", range(len(OPTIONS)))
def test_distillation_matches_its_formula(ops, dtype, lead, V, K, options):
    kw = OPTIONS[options]
    index_dtype = (torch.int32, torch.int64)[options % 2]
    z, index, teacher, labels = student(lead, V, K, dtype, options, index_dtype)
    kw = dict(kw, ignore_index=int(labels.reshape(-1)[0]) if labels.numel() > 2 else -100)      # some rows are not live
    want, grad, size = distill_oracle(z, index, teacher, labels, **kw)
    zd, idd, td, yd = z.cuda(), index.cuda(), teacher.cuda(), labels.cuda()
    loss, got = ops.distillation_loss_and_gradient(zd, idd, td, yd, **kw)
    assert got.dtype == dtype and got.shape == z.shape
    rows = 1 if kw.get("reduction") != "sum" else labels.numel()
    weight = kw.get("soft_weight", 1.0) * kw.get("temperature", 1.0) ** 2 + kw.get("hard_weight", 0.0)
    check_loss(loss, want, rows * weight * (2 + math.log(V)))
    check_gradient(got, grad, size, dtype)
    alone = ops.distillation_loss(zd, idd, td, yd, **kw)      # without the gradient a row's sums are taken in another order
    check_loss(alone, want, rows * weight * (2 + math.log(V)))
    leaf = zd.clone().requires_grad_()
    up = ops.distillation_loss(leaf, idd, td, yd, **kw)
    assert up.requires_grad and torch.equal(up.detach(), alone)
    (up * -2.5).backward()
    check_gradient(leaf.grad, grad * -2.5, size * 2.5, dtype)
    assert torch.equal(ops.distillation_loss_and_gradient(zd, idd, td, yd, **kw)[1], got)       # the same bits again


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,V,K", [((67,), 5, 3), ((40,), 9, 100), ((35,), 9, 130), ((33,), 31, 70), ((18,), 33, 2), ((17,), 129, 130),
                                      ((5, 3), 257, 9), ((17,), 511, 1), ((3,), 513, 33), ((18,), 1023, 7), ((3,), 1025, 5)])
def test_distillation_of_short_rows(ops, dtype, lead, V, K):
    """Rows that share a wave with others (up to 512 words of 32 bits, 1024 of 16) and those just behind; the last workgroup
    has fewer rows than places, some of its rows are not live, more entries than words."""
    for options in (1, 2, 5):
        kw = dict(OPTIONS[options], ignore_index=0)
        z, index, teacher, labels = student(lead, V, K, dtype, options + 70, (torch.int64, torch.int32)[options % 2])
        labels.view(-1)[1::3] = 0
        want, grad, size = distill_oracle(z, index, teacher, labels, **kw)
        zd, idd, td, yd = z.cuda(), index.cuda(), teacher.cuda(), labels.cuda()
        loss, got = ops.distillation_loss_and_gradient(zd, idd, td, yd, **kw)
        rows = 1 if kw.get("reduction") != "sum" else labels.numel()
        weight = kw.get("soft_weight", 1.0) * kw.get("temperature", 1.0) ** 2 + kw.get("hard_weight", 0.0)
        check_loss(loss, want, rows * weight * (2 + math.log(V)))
        check_gradient(got, grad, size, dtype)
        assert (got.cpu()[labels == 0] == 0).all()
        check_loss(ops.distillation_loss(zd, idd, td, yd, **kw), want, rows * weight * (2 + math.log(V)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [2, 4, 31, 60, 250])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.5])
def test_a_student_that_agrees_has_no_divergence(ops, dtype, V, temperature):
    """A teacher that names every word and a student with the same logits: equal exponentials, summed in 64 bits in two orders —
    2 V steps of 2^-53 at most, times temperature^2."""
    z = (torch.randn(5, V, generator=gen(V, 71)) * 2).to(dtype)
    index = torch.stack([torch.randperm(V, generator=gen(V, r)) for r in range(5)]).int()
    teacher = z.gather(1, index.long())
    loss = ops.distillation_loss(z.cuda(), index.cuda(), teacher.cuda(), temperature=temperature)
    assert abs(loss.item()) <= 2 * (V + 4) * 2.0 ** -53 * temperature ** 2


@pytest.mark.parametrize("n,V", [(8193, 1030), (131200, 70)])
def test_sums_of_many_rows(ops, n, V):
    """More workgroups than one launch adds up; the mean is counted by a launch of its own."""
    g = gen(n, V)
    z, labels = torch.randn(n, V, generator=g), torch.randint(0, V, (n,), generator=g)
    index = torch.stack([labels, (labels + 1) % V], 1).int()
    teacher = torch.randn(n, 2, generator=g)
    live = labels != 0
    logp, logq, logs = (torch.log_softmax(t.double(), -1) for t in (teacher / 2, z / 2, z))
    rows = 0.5 * 4 * (logp.exp() * (logp - logq.gather(1, index.long()))).sum(1) - 0.25 * logs.gather(1, labels[:, None])[:, 0]
    want = rows[live].mean().item()
    kw = dict(temperature=2.0, soft_weight=0.5, hard_weight=0.25, ignore_index=0)
    loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), **kw)
    check_loss(loss, want, 2.25 * (2 + math.log(V)))
    check_loss(ops.distillation_loss(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), **kw), want, 2.25 * (2 + math.log(V)))
    target = torch.zeros(n, V, dtype=torch.float64).scatter_(1, index.long(), logp.exp())
    pick = torch.zeros(n, V, dtype=torch.float64).scatter_(1, labels[:, None], 1.0)
    scale = live.double()[:, None] / live.sum()
    check_gradient(got, scale * (logq.exp() - target + 0.25 * (logs.exp() - pick)),
                   scale * (logq.exp() + target + 0.25 * (logs.exp() + pick)), torch.float32)
    assert (got.cpu()[~live] == 0).all()


# (Every size here is streamed: 512 threads hold rows of up to 32771 words of float and 65543 of 16 bits.  Those sizes, and both
# sides of the rule, are in test_logits_instances_gpu.py.)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [66000, 131075])
def test_distillation_over_large_vocabularies(ops, dtype, V):
    """Rows of 1024 threads' registers, and (float32 from 65540 words, 16 bits from 131080) rows that are read again."""
    for extra in (0, 5, 131072):
        n = V + extra
        z, index, teacher, labels = student((2,), n, 20, dtype, extra)
        for kw in (dict(hard_weight=0.5, temperature=2.0), dict()):
            want, grad, size = distill_oracle(z, index, teacher, labels, **kw)
            loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), **kw)
            check_loss(loss, want, 5 * (2 + math.log(n)))
            check_gradient(got, grad, size, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,K", [(9, 4), (64, 8), (300, 40), (5000, 70)])
def test_rows_that_are_not_live_are_not_read(ops, dtype, V, K):
    z, index, teacher, labels = student((3, 7), V, K, dtype, 9)
    labels[0, 2], labels[1, 0], labels[2, 6], labels[2, 5] = 3, -1, V, 1 << 40
    clean, kw = z.clone(), dict(hard_weight=0.5, temperature=2.0, ignore_index=3)
    dead = (labels == 3) | (labels < 0) | (labels >= V)
    for bad in (float("nan"), float("inf"), NEG):
        z, t = clean.clone(), teacher.clone()
        z[dead], t[dead] = bad, bad
        want, grad, size = distill_oracle(clean, index, teacher, labels, **kw)
        loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), t.cuda(), labels.cuda(), **kw)
        check_loss(loss, want, 4.5 * (2 + math.log(V)))
        check_gradient(got, grad, size, dtype)
        assert (got.cpu()[dead] == 0).all()
    none = torch.full_like(labels, 3)                  # no live row at all
    for reduction in ("mean", "sum"):
        loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), t.cuda(), none.cuda(), reduction=reduction, **kw)
        assert loss.item() == 0.0 and (got == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,K", [(9, 6), (40, 6), (700, 6), (9000, 6)])
def test_absent_and_repeated_entries(ops, dtype, V, K):
    z, index, teacher, labels = student((2, 3), V, K, dtype, 10, torch.int64)
    index[0, 0, 2:] = -1                               # two entries
    teacher[0, 0, 2:] = float("nan")
    index[0, 1] = torch.tensor([-1, V, V + 5, 1 << 40, -(1 << 40), -7])         # none
    teacher[0, 1] = float("nan")
    index[0, 2] = 5 % V                                # one word six times
    index[1, 0, :4] = torch.tensor([1, 2, 1, 2])
    teacher[1, 1, 1:] = NEG                            # all but one of probability 0
    teacher[1, 2] = NEG                                # all of them
    labels[0, 2] = 5 % V                               # the label is that word too
    for kw in (dict(), dict(hard_weight=0.5, temperature=2.0)):
        want, grad, size = distill_oracle(z, index, torch.where(teacher.isnan(), torch.full_like(teacher, NEG), teacher), labels, **kw)
        loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), **kw)
        check_loss(loss, want, 4.5 * (2 + math.log(V)))
        check_gradient(got, grad, size, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [9, 50, 900, 9000])
def test_barred_words_and_lowest_values(ops, dtype, V):
    z, index, teacher, labels = student((4,), V, 3, dtype, 11)
    z[0, ::2] = NEG
    index[0] = torch.tensor([1, 3, 5], dtype=torch.int32)
    labels[0] = 1
    z[1] = torch.finfo(dtype).min                      # a row whose every word is at the type's lowest value: uniform
    z[2, 1:] = torch.finfo(dtype).min                  # and one with a single word left
    index[2], labels[2] = 0, 0
    kw = dict(hard_weight=0.5, temperature=2.0)
    want, grad, size = distill_oracle(z, index, teacher, labels, **kw)
    loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), **kw)
    check_loss(loss, want, 4.5 * (2 + math.log(V)))
    check_gradient(got, grad, size, dtype)
    z[3, int(labels[3])] = NEG                         # the label itself is barred
    loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), **kw)
    assert loss.item() == float("inf") and torch.isfinite(got).all()
    z[3] = NEG                                         # nothing left in a live row: no softmax, as log_softmax says
    loss, got = ops.distillation_loss_and_gradient(z.cuda(), index.cuda(), teacher.cuda(), labels.cuda(), **kw)
    assert math.isnan(loss.item()) and got[3].isnan().all() and torch.isfinite(got[:3]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [9, 1003])
def test_distillation_of_strided_logits_and_shifted_labels(ops, dtype, V):
    z, index, teacher, labels = student((4, 5), V, 3, dtype, 12)
    big = torch.randn(3, 4, 7, V + 3, generator=gen(13)).to(dtype).cuda()
    view = big[1, :, 1:6, 1:V + 1]
    view.copy_(z)
    spread = torch.zeros(4, 5, 6, dtype=torch.int32, device="cuda")[..., ::2]
    spread.copy_(index)
    for kw in (dict(hard_weight=0.5, temperature=2.0, shift_labels=True, ignore_index=0), dict(hard_weight=0.2, shift_labels=True)):
        want, grad, size = distill_oracle(z, index, teacher, labels, **kw)
        other = torch.empty(5, 4, dtype=torch.int64, device="cuda").t()
        other.copy_(labels)
        out = torch.full_like(z, 7.0).cuda()
        loss, got = ops.distillation_loss_and_gradient(view, spread, teacher.cuda(), other, out=out, **kw)
        assert got is out
        check_loss(loss, want, 4.5 * (2 + math.log(V)))
        check_gradient(got, grad, size, dtype)
    wide = z[:1].cuda().expand(4, 5, V)                # one row's logits for all: the gradient is summed by autograd
    leaf = z[:1].cuda().requires_grad_()
    loss = ops.distillation_loss(leaf.expand(4, 5, V), index.cuda(), teacher.cuda(), labels.cuda(), hard_weight=0.5)
    loss.backward()
    want, grad, size = distill_oracle(wide.cpu(), index, teacher, labels, hard_weight=0.5)
    check_loss(loss, want, 1.5 * (2 + math.log(V)))
    got, tol = leaf.grad.double().cpu(), 2e-5 * size.sum(0) + 8 * HALF_STEP[dtype] * size.sum(0) + 4 * LEAST[dtype]
    assert ((got - grad.sum(0, keepdim=True)).abs() <= tol).all()


@pytest.mark.parametrize("V", [9, 200, 5000])
def test_distillation_gradient_against_differences(ops, V):
    z, index, teacher, labels = student((1, 2), V, 4, torch.float32, 14)
    kw = dict(hard_weight=0.5, temperature=1.5, reduction="sum")
    zd, args = z.cuda(), (index.cuda(), teacher.cuda(), labels.cuda())
    _, grad = ops.distillation_loss_and_gradient(zd, *args, **kw)
    h = 2.0 ** -5
    for word in {int(index[0, 0, 0]), int(index[0, 1, 1]), int(labels[0, 0]), V // 2, V - 1}:
        for row in (0, 1):
            up, down = zd.clone(), zd.clone()
            up[0, row, word] += h
            down[0, row, word] -= h
            slope = (ops.distillation_loss(up, *args, **kw) - ops.distillation_loss(down, *args, **kw)).item() / (2 * h)
            # a third derivative of at most soft tau^2 / tau^3 + hard < 1.5: h^2 / 6 of it; and two losses of about 40 in 32 bits
            assert abs(slope - grad[0, row, word].item()) < 1.5 * h * h / 6 + 2 * 40 * 2.0 ** -23 / (2 * h), (word, row)


@pytest.mark.parametrize("V", [9, 300, 5000])
def test_backward_with_tensors_saved_elsewhere(ops, V):
    """Hooks on saved tensors (kept on the host, copied back for the backward pass, with other strides and addresses) change
    nothing; logits changed in place between the passes raise."""
    z, index, teacher, labels = student((3, 4), V, 5, torch.float32, 77)
    z, index, teacher, labels = z.cuda(), index.cuda(), teacher.cuda(), labels.cuda()
    kw = dict(hard_weight=0.5, temperature=2.0)
    want = ops.distillation_loss_and_gradient(z, index, teacher, labels, **kw)[1]
    for view in (z, torch.stack([z, z], 1)[:, 0]):
        leaf = view.detach().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
            loss = ops.distillation_loss(leaf, index, teacher, labels, **kw)
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)
        leaf = view.detach().requires_grad_()
        loss = ops.distillation_loss(leaf, index, teacher, labels, **kw)
        assert torch.equal(torch.autograd.grad(loss, leaf, retain_graph=True)[0], want)
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)
    leaf = (z * 1.0).requires_grad_()
    moved = leaf * 1.0
    loss = ops.distillation_loss(moved, index, teacher, labels, **kw)
    moved.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---------------------------------------------------------------------------------------------------------------------
# beam search
# ---------------------------------------------------------------------------------------------------------------------
def beam_oracle(logits, scores, finished, eos, pad):
    B, W, V = logits.shape
    out = []
    for b in range(B):
        z = torch.where(logits[b].isnan(), torch.full_like(logits[b], NEG), logits[b]).double()
        total = scores[b].double()[:, None] + (z - torch.logsumexp(z, -1, keepdim=True))
        cand = []
        for w in range(W):
            if finished[b, w]:
                cand.append((-scores[b, w].double().item(), w, pad))
            else:
                s = torch.where(total[w].isnan(), torch.full_like(total[w], NEG), total[w])
                order = torch.sort(s, descending=True, stable=True)[1][:W].tolist()
                cand += [(-s[v].item(), w, v) for v in order]
        cand = sorted(cand)[:W]
        out.append([(-s, w, v, bool(finished[b, w]) or v == eos) for s, w, v in cand])
    t = lambda i, dt: torch.tensor([[c[i] for c in row] for row in out], dtype=dt)      # noqa: E731
    return t(0, torch.float64), t(1, torch.int32), t(2, torch.int64), t(3, torch.bool)


def check_beams(ops, logits, scores, finished, eos=2, pad=0):
    got = [x.cpu() for x in ops.beam_select(logits.cuda(), scores.cuda(), finished.cuda(), eos_idx=eos, pad_idx=pad)]
    want = beam_oracle(logits, scores, finished, eos, pad)
    assert torch.equal(got[1], want[1]), (got[1], want[1])
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    live = torch.isfinite(want[0])
    assert torch.equal(got[0].double()[~live], want[0][~live])
    # scores in 64 bits but for the softmax sum's terms (2^-22 and the distance from the maximum), then one rounding
    n = logits.shape[-1]
    tol = (math.log(n) + 4 + n / 256) * 2.0 ** -23 + want[0].abs() * 2.0 ** -24
    assert ((got[0].double() - want[0]).abs() <= tol)[live].all()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V", [(1, 1, 3), (5, 1, 9), (7, 4, 9), (3, 5, 6), (300, 3, 8), (2, 8, 4), (3, 16, 16), (2, 33, 5), (2, 4, 64), (2, 5, 64),
                                   (2, 64, 3), (3, 4, 65), (2, 7, 257), (1, 16, 1000), (2, 64, 130), (2, 3, 4099), (1, 4, 32003), (40, 2, 700),
                                   (1, 1, 100001), (150, 4, 2100)])
def test_beam_step(ops, dtype, B, W, V):
    g = gen(B, W, V)
    logits = (torch.randn(B, W, V, generator=g) * 2).to(dtype)
    scores = -torch.rand(B, W, generator=g) * 5
    finished = torch.rand(B, W, generator=g) < 0.25
    check_beams(ops, logits, scores, torch.zeros_like(finished))
    got = check_beams(ops, logits, scores, finished)
    assert (got[2][torch.gather(finished, 1, got[1].long())] == 0).all()
    logits[finished] = float("nan")                        # a finished beam's logits are not looked at
    check_beams(ops, logits, scores, finished, eos=1, pad=V - 1)
    check_beams(ops, logits, scores, torch.ones_like(finished))
    start = torch.full((B, W), NEG)                        # the first step: equal states, one beam counts
    start[:, 0] = 0.0
    first = (torch.randn(B, 1, V, generator=g) * 2).to(dtype).expand(B, W, V)
    check_beams(ops, first, start, torch.zeros_like(finished))
    check_beams(ops, first, torch.full((B, W), -1.5), torch.zeros_like(finished))        # equal beams: ties
    check_beams(ops, first, torch.full((B, W), NEG), torch.zeros_like(finished))         # no beam counts


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,W,V", [(3, 4, 9), (2, 6, 200), (2, 4, 9000)])
def test_beam_step_with_barred_words(ops, dtype, B, W, V):
    g = gen(B, W, V, 1)
    logits = (torch.randn(B, W, V, generator=g) * 2).to(dtype)
    scores = -torch.rand(B, W, generator=g) * 5
    none = torch.zeros(B, W, dtype=torch.bool)
    logits[:, :, 1::2] = NEG
    check_beams(ops, logits, scores, none)
    logits[0, :, 1:] = NEG                                  # one word left per beam
    logits[1, 1] = NEG                                      # and none
    logits[1, 2, 0] = float("nan")
    check_beams(ops, logits, scores, none)
    logits[:] = NEG
    check_beams(ops, logits, scores, none)
    logits[:] = torch.finfo(dtype).min                      # all alike, if lowest
    check_beams(ops, logits, scores, none)
    logits[0, 0, 0] = float("inf")                          # no softmax there: in range all the same
    got = ops.beam_select(logits.cuda(), scores.cuda(), none.cuda(), eos_idx=2, pad_idx=0)
    assert ((got[1] >= 0) & (got[1] < W)).all() and ((got[2] >= 0) & (got[2] < V)).all() and not got[0].isnan().any()


def test_beam_step_of_strided_logits(ops):
    big = torch.randn(3, 2, 5, 301, generator=gen(20))
    for view in (big[:, 0, :4, 1:], big[:, 1, ::2], big[:1, 0].expand(3, 5, 301), big[0, :, :3].transpose(0, 1)):
        B, W = view.shape[:2]
        got = ops.beam_select(big.cuda().as_strided(view.size(), view.stride(), view.storage_offset()), torch.zeros(B, W).cuda(),
                              torch.zeros(B, W, dtype=torch.bool).cuda(), eos_idx=2, pad_idx=0)
        want = beam_oracle(view, torch.zeros(B, W), torch.zeros(B, W, dtype=torch.bool), 2, 0)
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])


REORDERED = [torch.float32, torch.bfloat16, torch.float16, torch.int64, torch.int32, torch.uint8, torch.bool, torch.float64]


def filled(shape, dtype, key):
    return torch.randint(0, 2 if dtype == torch.bool else 100, shape, generator=gen(*shape, key)).to(dtype)


@pytest.mark.parametrize("dtype", REORDERED)
def test_reorder_moves_every_type_and_width(ops, dtype):
    for B, W, inner in ((1, 1, 1), (3, 4, 1), (2, 5, 3), (4, 3, 100), (2, 2, 8193), (1, 64, 5000)):
        parents = torch.randint(0, W, (B, W), generator=gen(B, W, inner), dtype=torch.int32)
        state = filled((B * W, inner), dtype, 0)
        rows = (torch.arange(B)[:, None] * W + parents).reshape(-1)
        assert torch.equal(ops.beam_reorder(parents.cuda(), state.cuda()).cpu(), state[rows])
        shifted = filled((B * W * inner + 1,), dtype, 1)         # an unaligned beginning
        assert torch.equal(ops.beam_reorder(parents.cuda(), shifted.cuda()[1:].view(B * W, inner)).cpu(), shifted[1:].view(B * W, inner)[rows])


def test_reorder_of_strided_caches_and_many_states(ops):
    B, W = 2, 3
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]], dtype=torch.int32)
    rows = (torch.arange(B)[:, None] * W + parents).reshape(-1)
    cache = filled((3, 6, 4, 10, 8), torch.bfloat16, 2)              # layers, beams, heads, positions, width
    got = ops.beam_reorder(parents.cuda(), cache.cuda(), dim=1)
    assert torch.equal(got.cpu(), cache[:, rows])
    got = ops.beam_reorder(parents.cuda(), cache.cuda()[:, :, :, :7], dim=-4)
    assert got.is_contiguous() and torch.equal(got.cpu(), cache[:, rows][:, :, :, :7])
    out = filled(tuple(cache.shape), torch.bfloat16, 3)              # what lies behind the used positions is left alone
    dev = out.cuda()
    ops.beam_reorder(parents.cuda(), cache.cuda()[:, :, :, :7], out=dev[:, :, :, :7], dim=1)
    out[:, :, :, :7] = cache[:, rows][:, :, :, :7]
    assert torch.equal(dev.cpu(), out)
    odd = cache.cuda()[::2, :, 1:3, ::2]                             # an input that is copied first
    assert torch.equal(ops.beam_reorder(parents.cuda(), odd, dim=1).cpu(), cache[:, rows][::2, :, 1:3, ::2])
    many = [filled((6, n), t, 4) for n, t in zip(range(1, 21), REORDERED * 3)]
    for s, d in zip(many, ops.beam_reorder(parents.cuda(), [s.cuda() for s in many])):
        assert torch.equal(d.cpu(), s[rows])
    bad = torch.tensor([[-1, 3, 1], [1 << 30, -(1 << 31), 0]], dtype=torch.int32)       # parents that are none
    got = ops.beam_reorder(bad.cuda(), cache.cuda(), dim=1).cpu()
    assert torch.equal(got[:, 2], cache[:, 1]) and torch.equal(got[:, 5], cache[:, 3]) and (got[:, [0, 1, 3, 4]] == 0).all()
    assert ops.beam_reorder(parents.cuda(), []) == []


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs, use together
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("V", [9, 700, 40000])
def test_captured_and_replayed(ops, V):
    """Every operator in one graph, replayed on new inputs between eager calls of the same, against the eager results."""
    B, W, K = 3, 4, 5
    static = dict(logits=torch.zeros(B, W, V, device="cuda"), scores=torch.zeros(B, W, device="cuda"),
                  finished=torch.zeros(B, W, dtype=torch.bool, device="cuda"), state=torch.zeros(B * W, 50, device="cuda"),
                  labels=torch.ones(B, W, dtype=torch.int64, device="cuda"))

    def everything(s):
        values, index, lse = ops.top_logits(s["logits"], K, return_lse=True)
        loss, grad = ops.distillation_loss_and_gradient(s["logits"], index, values, s["labels"], temperature=2.0, hard_weight=0.5, ignore_index=0)
        scores, parents, words, done = ops.beam_select(s["logits"], s["scores"], s["finished"], eos_idx=2, pad_idx=0)
        return [values, index, lse, loss, grad, scores, parents, words, done, ops.beam_reorder(parents, s["state"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything(static)
    for k in range(4):
        g = gen(V, k, 30)
        fresh = dict(logits=torch.randn(B, W, V, generator=g) * 2, scores=-torch.rand(B, W, generator=g), finished=torch.rand(B, W, generator=g) < 0.3,
                     state=torch.randn(B * W, 50, generator=g), labels=torch.randint(0, V, (B, W), generator=g))
        for name, t in fresh.items():
            static[name].copy_(t)
        eager = everything({name: t.cuda() for name, t in fresh.items()})
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_two_streams_at_once(ops):
    """Calls in flight on two streams share nothing: the same as one after the other."""
    g = gen(40)
    inputs = [(torch.randn(4, 60000, generator=g) * 2).cuda() for _ in range(4)]
    alone = [ops.top_logits(x, 20, return_lse=True) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for i in range(16):
        with torch.cuda.stream(streams[i % 2]):
            results.append((i % 4, ops.top_logits(inputs[i % 4], 20, return_lse=True)))
    torch.cuda.synchronize()
    for i, got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, alone[i]))


def test_a_whole_search(ops):
    """Beam search over a table of transition logits with a state per beam, against every sequence scored one by one."""
    V, W, steps, eos, pad = 7, 5, 4, 2, 0
    g = gen(50)
    table = (torch.randn(V, V, V, generator=g) * 1.5)          # logits of the next word by the last two
    logp = torch.log_softmax(table.double(), -1)
    beams = [(0.0, [1], False)]                                # (score, words, finished)
    for _ in range(steps):
        cand = []
        for w, (s, words, done) in enumerate(beams):
            last, before = words[-1], words[-2] if len(words) > 1 else 0
            cand += [(-s, w, pad, words, True)] if done else [(-(s + logp[before, last, v].item()), w, v, words, v == eos) for v in range(V)]
        cand.sort(key=lambda c: c[:3])
        beams = [(-s, words + [v], done) for s, _, v, words, done in cand[:W]]
    dev = table.cuda()
    last, before = torch.ones(W, dtype=torch.int64, device="cuda"), torch.zeros(W, dtype=torch.int64, device="cuda")
    scores = torch.full((1, W), NEG, device="cuda")
    scores[0, 0] = 0.0
    finished = torch.zeros(1, W, dtype=torch.bool, device="cuda")
    history = torch.ones(W, 1, dtype=torch.int64, device="cuda")
    for _ in range(steps):
        scores, parents, words, finished = ops.beam_select(dev[before, last].view(1, W, V), scores, finished, eos_idx=eos, pad_idx=pad)
        history, before = ops.beam_reorder(parents, [history, last])
        last = words.view(-1)
        history = torch.cat([history, last.unsqueeze(1)], 1)
    assert history.tolist() == [words for _, words, _ in beams]
    assert finished[0].tolist() == [done for _, _, done in beams]
    assert torch.allclose(scores[0].cpu().double(), torch.tensor([s for s, _, _ in beams], dtype=torch.float64), atol=1e-5)


def test_a_student_learns_from_its_teacher(ops):
    """top_logits of a teacher, distillation of a student: the gradient vanishes where they agree on a whole vocabulary."""
    z = (torch.randn(3, 50, generator=gen(60)) * 2).cuda()
    values, index = ops.top_logits(z, 50)
    loss, grad = ops.distillation_loss_and_gradient(z, index, values, temperature=2.0)
    assert abs(loss.item()) < 1e-5 and grad.abs().max().item() < 1e-6
    values, index = ops.top_logits(z, 10)
    lead = ops.distillation_loss(z, index, values).item()
    assert lead == pytest.approx(-(torch.softmax(z, -1).gather(1, index.long()).sum(-1)).log().mean().item(), rel=1e-4)
