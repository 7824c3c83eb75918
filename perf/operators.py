"""Operators over rows of logits: top-logits selection, distillation from a teacher's top logits, the beam search step.

Each case is one call (or, for a beam step, the two calls) that a training or decoding loop makes per step.  With
`own = False` the operators are written in elementary torch operations; with `own = True` the framework's entry points
(`multimodal_seq2seq_gscan_amd.logits`) are called on the same inputs."""
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
INDEX = {"int32": torch.int32, "int64": torch.int64}
PAD, EOS = 0, 2
NEG_INF = float("-inf")


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _distill(name, mode, outer, inner, V, K, dtype, **more):
    case = dict(op="distill", mode=mode, outer=outer, inner=inner, V=V, K=K, dtype=dtype, index="int32", temperature=2.0,
                soft=0.5, hard=0.5, shift=False, strided=False)
    case.update(more)
    return dict(case, name=name) if name else case


def _top(name, rows, V, K, dtype, lse):
    case = dict(op="top", rows=rows, V=V, K=K, dtype=dtype, lse=lse)
    return dict(case, name=name) if name else case


def _beam(name, B, W, V, dtype, states, heads, length, width, first=False):
    case = dict(op="beam", B=B, W=W, V=V, dtype=dtype, states=states, heads=heads, length=length, width=width, first=first)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the student's log-probabilities of one training batch of the compositional configuration, teacher's top 4
        _distill("distill_step_compositional", "step", 256, 20, 9, 4, "fp32", shift=True),
        # the same for the long targets (120 steps), as many words as the teacher has kept
        _distill("distill_step_long_targets", "step", 256, 120, 8, 3, "fp32", shift=True, temperature=3.5),
        # one training step's rows over a subword vocabulary: loss and gradient in one call
        _distill("distill_step_subwords_bf16", "step", 8, 511, 32000, 64, "bf16"),
        # through autograd (forward, then backward), logits a slice of a longer batch, odd vocabulary
        _distill("distill_autograd_fp32", "autograd", 4, 255, 50001, 16, "fp32", strided=True, temperature=1.0, index="int64"),
        # validation: the loss alone, soft term only
        _distill("distill_eval_fp16", "eval", 2, 1000, 65537, 32, "fp16", hard=0.0, soft=1.0),
        # the largest vocabulary and batch
        _distill("distill_step_largest_bf16", "step", 4, 1024, 131072, 128, "bf16"),
        # what a teacher leaves for its student: one compositional batch, one subword batch
        _top("top_logits_compositional", 5120, 9, 4, "fp32", False),
        _top("top_logits_teacher_bf16", 4088, 32000, 64, "bf16", True),
        # one position's alternatives, for an answer in progress
        _top("top_logits_one_row", 1, 131072, 50, "fp32", True),
        # one step of beam search over a batch of the compositional configuration: selection, then h and c reordered
        _beam("beam_step_compositional", 256, 4, 9, "fp32", 2, 1, 1, 100),
        # one request over a subword vocabulary: latency
        _beam("beam_step_one_request", 1, 4, 32000, "bf16", 2, 8, 129, 64),
        # a batch of requests, the largest vocabulary, keys and values of two layers behind it
        _beam("beam_step_batch_fp32", 32, 8, 131072, "fp32", 4, 8, 512, 64),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    import math
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(sorted(TYPES))
    op = rng.choice(["distill", "distill", "top", "beam"])
    if op == "beam":
        W = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
        V = _log(rng, 9, 131072)
        B = _log(rng, 1, max(1, min(256, (1 << 25) // (W * V))))
        heads, width = rng.choice([1, 2, 5, 8]), rng.choice([33, 64, 100, 128])
        length = _log(rng, 1, max(1, min(1024, (1 << 26) // (B * W * heads * width))))
        return _beam(None, B, W, V, dtype, rng.choice([1, 2, 4]), heads, length, width, rng.random() < 0.2)
    V = _log(rng, 2, 131072)
    K = _log(rng, 1, min(V, 256))
    if op == "top":
        return _top(None, _log(rng, 1, min(65536, (1 << 27) // V)), V, K, dtype, rng.random() < 0.5)
    rows = _log(rng, 1, min(65536, (1 << 28) // V))
    outer = _log(rng, 1, rows)
    return _distill(None, rng.choice(["step", "step", "autograd", "eval"]), outer, max(1, rows // outer), V, K, dtype,
                    index=rng.choice(sorted(INDEX)), temperature=rng.choice([1.0, 2.0, 3.5]), soft=rng.choice([0.5, 0.9]),
                    hard=rng.choice([0.0, 0.5]), shift=rng.random() < 0.3, strided=rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device="cuda", generator=g)
    state = dict(case=case)
    V, dtype = case["V"], TYPES[case["dtype"]]
    if case["op"] == "top":
        logits = torch.randn(case["rows"], V, **kw).mul_(2.5).to(dtype)
        if V > 64:      # words that the vocabulary bars
            logits[:, torch.randint(0, V, (V // 64,), **kw)] = NEG_INF
        state["logits"] = logits
        return state
    if case["op"] == "beam":
        B, W = case["B"], case["W"]
        if case["first"]:   # the first step: every beam holds the same state, one of them counts
            logits = torch.randn(B, 1, V, **kw).mul_(2.5).to(dtype).expand(B, W, V).contiguous()
            scores = torch.full((B, W), NEG_INF, device="cuda")
            scores[:, 0] = 0.0
            finished = torch.zeros(B, W, dtype=torch.bool, device="cuda")
        else:
            logits = torch.randn(B, W, V, **kw).mul_(2.5).to(dtype)
            scores = torch.rand(B, W, **kw).mul_(-6.0).sort(dim=1, descending=True)[0]
            finished = torch.rand(B, W, **kw) < 0.1
        state.update(logits=logits, scores=scores, finished=finished)
        shape = (B * W, case["heads"], case["length"], case["width"])
        state["states"] = [torch.randn(shape, **kw).to(dtype) for _ in range(case["states"])]
        return state
    outer, inner, K = case["outer"], case["inner"], case["K"]
    rows = outer * inner
    full = torch.randn(outer, inner + int(case["strided"]), V, **kw).mul_(2.0).to(dtype)
    # the teacher's K best words of a row: all different, spread over the vocabulary; the student gives them more than others
    at = torch.randint(0, V, (outer, inner, 1), **kw)
    index = (at + torch.arange(K, device="cuda") * (V // K)) % V
    teacher = torch.randn(outer, inner, K, **kw).mul_(1.5).add_(5.0).sort(dim=-1, descending=True)[0]
    logits = full[:, :inner]
    logits.scatter_(-1, index, (teacher + torch.randn(outer, inner, K, **kw)).to(dtype))
    lengths = torch.randint((inner + 1) // 2, inner + 1, (outer, 1), **kw)
    words = torch.randint(1, V, (outer, inner), **kw)
    best = index[..., 0]
    labels = torch.where(torch.rand(outer, inner, **kw) < 0.6, best, words)
    labels = torch.where(torch.arange(inner, device="cuda") < lengths, labels, torch.full_like(labels, PAD))
    state.update(logits=logits, index=index.to(INDEX[case["index"]]), teacher=teacher.to(dtype), labels=labels, rows=rows)
    return state


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _order_keys(x):
    """Whole numbers that order a row by value, the lowest index first among equals (a NaN counts as -inf)."""
    x = torch.where(x.isnan(), torch.full_like(x, NEG_INF), x).float() + 0.0
    bits = x.view(torch.int32)
    ordered = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    return (ordered << 32) + (0xFFFFFFFF - torch.arange(x.shape[-1], device=x.device))


def _top_plain(logits, K):
    index = 0xFFFFFFFF - (torch.topk(_order_keys(logits), K, dim=-1, largest=True, sorted=True)[0] & 0xFFFFFFFF)
    return torch.gather(logits, -1, index), index


def _lse_plain(x, dtype=torch.float32):
    x = x.to(dtype)
    top = x.amax(-1, keepdim=True)
    return (x - top).exp().sum(-1).log() + top.squeeze(-1)


def _labels_plain(case, labels):
    if not case["shift"]:
        return labels
    return torch.cat([labels[:, 1:], torch.zeros_like(labels[:, :1])], dim=1)


def _distill_plain(s):
    case = s["case"]
    tau, soft, hard = case["temperature"], case["soft"], case["hard"]
    labels = _labels_plain(case, s["labels"])
    live = labels != PAD
    count = live.sum().clamp(min=1)
    z, index = s["logits"].float(), s["index"].long()
    top = z.amax(-1, keepdim=True)
    t = s["teacher"].float()
    t = (t - t.amax(-1, keepdim=True)) / tau
    logp = t - t.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    zt = (z - top) / tau
    et = zt.exp()
    sum_t = et.sum(-1, keepdim=True)
    soft_rows = (p * (logp - (torch.gather(zt, -1, index) - sum_t.log()))).sum(-1) * (tau * tau)
    soft_sum = torch.where(live, soft_rows, torch.zeros_like(soft_rows)).double().sum()
    scale = live.unsqueeze(-1) / count
    grad = None
    if case["mode"] != "eval":
        grad = et.mul_(scale * (soft * tau) / sum_t)
        grad.scatter_add_(-1, index, -p * scale * (soft * tau))
    loss = soft * soft_sum
    if hard:
        z = z - top
        e = z.exp()
        sum_1 = e.sum(-1, keepdim=True)
        hard_rows = sum_1.log().squeeze(-1) - torch.gather(z, -1, labels.unsqueeze(-1)).squeeze(-1)
        loss = loss + hard * torch.where(live, hard_rows, torch.zeros_like(hard_rows)).double().sum()
        if grad is not None:
            grad += e.mul_(scale * hard / sum_1)
            grad.scatter_add_(-1, labels.unsqueeze(-1), -hard * scale)
    loss = (loss / count).float()
    return (loss,) if grad is None else (loss, grad.to(s["logits"].dtype))


def _beam_plain(s):
    """Scores in 64 bits: candidates of different beams come close to each other."""
    case, logits, scores, finished = s["case"], s["logits"], s["scores"], s["finished"]
    B, W, V = logits.shape
    n = min(W, V)
    value, word = _top_plain(logits, n)
    total = scores.double().unsqueeze(-1) + (value.double() - _lse_plain(logits, torch.float64).unsqueeze(-1))
    first = torch.arange(n, device=logits.device).expand(B, W, n)
    # a finished beam goes on as itself, with padding; one without a score comes last, its words in order
    total = torch.where(finished.unsqueeze(-1), torch.where(first == 0, scores.double().unsqueeze(-1), NEG_INF), total)
    dead = (scores == NEG_INF) & ~finished
    word = torch.where(dead.unsqueeze(-1), first, torch.where(finished.unsqueeze(-1), torch.full_like(word, PAD), word))
    total, at = total.reshape(B, W * n).sort(dim=-1, descending=True, stable=True)
    total, at = total[:, :W], at[:, :W]
    parents = at // n
    words = torch.gather(word.reshape(B, W * n), 1, at)
    done = torch.gather(finished, 1, parents) | (words == EOS)
    rows = (torch.arange(B, device=logits.device).unsqueeze(1) * W + parents).reshape(-1)
    return (total.float(), parents.to(torch.int32), words, done, *[x[rows] for x in s["states"]])


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["op"] == "top":
        values, index = _top_plain(state["logits"], case["K"])
        out = (values, index.to(torch.int32))
        return (*out, _lse_plain(state["logits"])) if case["lse"] else out
    return _distill_plain(state) if case["op"] == "distill" else _beam_plain(state)


def _run_own(s):
    from multimodal_seq2seq_gscan_amd import logits as ops
    case = s["case"]
    if case["op"] == "top":
        return ops.top_logits(s["logits"], case["K"], return_lse=case["lse"])
    if case["op"] == "beam":
        scores, parents, words, done = ops.beam_select(s["logits"], s["scores"], s["finished"], eos_idx=EOS, pad_idx=PAD)
        return (scores, parents, words, done, *ops.beam_reorder(parents, s["states"]))
    kw = dict(labels=s["labels"], temperature=case["temperature"], soft_weight=case["soft"], hard_weight=case["hard"],
              ignore_index=PAD, shift_labels=case["shift"])
    if case["mode"] == "eval":
        return (ops.distillation_loss(s["logits"], s["index"], s["teacher"], **kw),)
    if case["mode"] == "step":
        return ops.distillation_loss_and_gradient(s["logits"], s["index"], s["teacher"], **kw)
    leaf = s["logits"].detach().requires_grad_()
    loss = ops.distillation_loss(leaf, s["index"], s["teacher"], **kw)
    return loss.detach(), torch.autograd.grad(loss, leaf)[0]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    V = case["V"]
    if case["op"] == "top":
        n = case["rows"]
        return dict(bytes=n * (V * size + case["K"] * (size + 4) + (4 if case["lse"] else 0)),
                    flops=n * V * (4 if case["lse"] else 1))
    if case["op"] == "beam":
        n = case["B"] * case["W"]
        moved = 2 * case["states"] * n * case["heads"] * case["length"] * case["width"] * size
        return dict(bytes=n * (V * size + 4 + 1 + 4 + 4 + 8 + 1) + moved, flops=n * V * 4)
    n = case["outer"] * case["inner"]
    terms = int(case["soft"] > 0) + int(case["hard"] > 0)
    grads = 0 if case["mode"] == "eval" else 1
    return dict(bytes=n * (V * size * (1 + grads) + case["K"] * (size + (4 if case["index"] == "int32" else 8)) + 8),
                flops=n * V * terms * (3 + 3 * grads))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "top":
        x = s["logits"]
        order = torch.sort(x, dim=-1, descending=True, stable=True)
        out = (order[0][:, :case["K"]].double(), order[1][:, :case["K"]].to(torch.int32))
        if not case["lse"]:
            return out
        return (*out, torch.cat([torch.logsumexp(c.double(), -1) for c in x.split(512)]))
    if case["op"] == "beam":
        B, W, V = s["logits"].shape
        results = []
        for b in range(B):
            total = torch.log_softmax(s["logits"][b].double(), -1) + s["scores"][b].double()[:, None]
            for w in torch.nonzero(s["finished"][b]).flatten().tolist():
                total[w] = NEG_INF
                total[w, PAD] = s["scores"][b, w].double()
            results.append(torch.sort(total.flatten(), descending=True, stable=True)[0][:W])
        return (torch.stack(results), None, None, None, *[None] * case["states"])
    tau, K = case["temperature"], case["K"]
    flat = s["logits"].flatten(0, 1)
    index, teacher = s["index"].flatten(0, 1).long(), s["teacher"].flatten(0, 1)
    labels = s["labels"]
    if case["shift"]:
        labels = torch.nn.functional.pad(labels[:, 1:], (0, 1))
    labels = labels.flatten()
    count = int((labels != PAD).sum())
    if not count:
        return None
    loss, grads = 0.0, []
    step = max(1, (1 << 26) // case["V"])
    for lo in range(0, flat.shape[0], step):
        x = flat[lo:lo + step].double()
        p = torch.softmax(teacher[lo:lo + step].double() / tau, -1)
        live = (labels[lo:lo + step] != PAD).double()
        logq = torch.log_softmax(x / tau, -1)
        target = torch.zeros_like(x).scatter_add_(-1, index[lo:lo + step], p)
        kl = (torch.xlogy(p, p) - p * torch.gather(logq, -1, index[lo:lo + step])).sum(-1)
        loss = loss + case["soft"] * tau ** 2 * (kl * live).sum()
        d = case["soft"] * tau * (logq.exp() - target)
        if case["hard"]:
            ls = torch.log_softmax(x, -1)
            pick = labels[lo:lo + step, None]
            loss = loss - case["hard"] * (torch.gather(ls, -1, pick)[:, 0] * live).sum()
            d += case["hard"] * (ls.exp() - torch.zeros_like(x).scatter_(-1, pick, 1.0))
        if case["mode"] != "eval":
            grads.append((d * (live / count)[:, None]).float())
    if case["mode"] == "eval":
        return (loss / count,)
    return loss / count, torch.cat(grads).view(s["logits"].shape)
