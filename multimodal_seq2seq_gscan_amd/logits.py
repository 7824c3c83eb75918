"""Operators over rows of logits, on libgscan_hip.so: the top K of every row, distillation from a teacher's top logits, the
step of a beam search.

The framework builds on them (`Model.get_distillation_loss`, `train.TrainStep(teacher=...)`, `predict.beam_decode`); they take
any vocabulary, in float32, bfloat16 or float16.  Logits are read where they are: `[..., V]` with adjacent words and any strides
in front of them (a slice of a longer batch, an expanded dimension).  Every call runs on the current stream of its tensors'
device, allocates what it returns and its workspace from torch's allocator, and neither synchronises nor keeps anything between
calls, so it can be captured in a graph.  CPU tensors raise: there is no CPU path in this package."""
from __future__ import annotations

import ctypes as C
import functools
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_INDEX_BITS = {torch.int32: 32, torch.int64: 64}


def _require(names: str, *tensors: Optional[torch.Tensor]) -> int:
    """The index of the device that all of the tensors are on; raises for a CPU tensor or two devices."""
    index = tensors[0].get_device()
    for i, t in enumerate(tensors):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{names.split()[i]} is on {t.device}: this operator runs on the HIP device only (there is no CPU "
                               "fallback in this package)")
        if t.get_device() != index:
            raise ValueError(f"{names.split()[i]} is on {t.device}, {names.split()[0]} is on {tensors[0].device}")
    return index


def _call(name: str, device: int, *args) -> None:
    """One library call on the current stream of `device`, with that device current."""
    fn = getattr(_lib.load(), name)
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _lib.check(rc, name)


def _float_type(t: torch.Tensor, name: str) -> int:
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return _TYPES[t.dtype]


def _rows(logits: torch.Tensor) -> Tuple[torch.Tensor, _lib.Rows]:
    """The rows of `logits` [..., V] as the library takes them: the last leading dimension is `inner`, those before it one
    `outer` dimension.  Copies only where no pair of strides describes them (or the words of a row are not adjacent)."""
    kind = _float_type(logits, "logits")
    if logits.is_neg():          # the library reads memory: a sign that only the view knows of would be lost
        logits = logits.resolve_neg()
    shape, stride = logits.shape, logits.stride()
    n = len(shape)
    if n == 0 or shape[-1] == 0:
        raise ValueError(f"logits must be [..., V] with at least one word, got {tuple(shape)}")
    V = shape[-1]
    if stride[-1] != 1 and V > 1:
        return _rows(logits.contiguous())
    inner, si = (shape[-2], stride[-2]) if n > 1 else (1, 0)
    if n <= 3:
        outer, so = (shape[0], stride[0]) if n == 3 else (1, 0)
        return logits, _lib.Rows(logits.data_ptr(), kind, V, outer, inner, so, si)
    outer, so = 1, 0
    for size, step in zip(reversed(shape[:-2]), reversed(stride[:-2])):
        if size == 1:
            continue
        if outer == 1:
            outer, so = size, step
        elif step == outer * so:
            outer *= size
        else:
            return _rows(logits.contiguous())
    return logits, _lib.Rows(logits.data_ptr(), kind, V, outer, inner, so, si)


def _workspace(size: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


# ---------------------------------------------------------------------------------------------------------------------
# the top K of every row
# ---------------------------------------------------------------------------------------------------------------------
def top_logits(logits: torch.Tensor, k: int, return_lse: bool = False) -> Tuple[torch.Tensor, ...]:
    """The k best words of every row of `logits` [..., V], best first: (values [..., k] of the logits' type, indices [..., k]
    int32) and, with `return_lse`, the rows' log-sum-exp [...] in float32 (`values - lse` are log-probabilities).

    Value descending, the lowest index first among equals.  A NaN counts as -inf, and is returned as -inf.
    1 <= k <= min(V, 256).  No gradient flows through it."""
    device = _require("logits", logits)
    logits, rows = _rows(logits)
    k = int(k)
    if not 1 <= k <= min(rows.V, _lib.MAX_TOP):
        raise ValueError(f"k must be 1 to {min(rows.V, _lib.MAX_TOP)} for rows of {rows.V} words, got {k}")
    lead, where = logits.shape[:-1], logits.device
    values = torch.empty(*lead, k, dtype=logits.dtype, device=where)
    indices = torch.empty(*lead, k, dtype=torch.int32, device=where)
    lse = torch.empty(lead, dtype=torch.float32, device=where) if return_lse else None
    if values.numel():
        size = _lib.load().gscan_top_logits_workspace_bytes(C.byref(rows), k)
        ws = _workspace(size, where)
        _call("gscan_top_logits", device, C.byref(rows), k, values.data_ptr(), indices.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), size)
    return (values, indices, lse) if return_lse else (values, indices)


# ---------------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------------
def _distillation(logits, teacher_indices, teacher_logits, labels, temperature, soft_weight, hard_weight, ignore_index,
                  shift_labels, reduction):
    """Checks the arguments; (device, logits, rows, terms, tensors that the terms point at)."""
    device = _require("logits teacher_indices teacher_logits labels", logits, teacher_indices, teacher_logits, labels)
    logits, rows = _rows(logits)
    lead = logits.shape[:-1]
    if teacher_indices.dtype not in _INDEX_BITS:
        raise TypeError(f"teacher_indices must be int32 or int64, got {teacher_indices.dtype}")
    kind = _float_type(teacher_logits, "teacher_logits")
    if teacher_indices.dim() == 0 or teacher_indices.shape[:-1] != lead or teacher_indices.shape != teacher_logits.shape:
        raise ValueError(f"teacher_indices and teacher_logits must be {tuple(lead)} + [K], got {tuple(teacher_indices.shape)} "
                         f"and {tuple(teacher_logits.shape)}")
    K = teacher_indices.shape[-1]
    if not 1 <= K <= _lib.MAX_TOP:
        raise ValueError(f"1 to {_lib.MAX_TOP} teacher entries per row, got {K}")
    temperature, soft_weight, hard_weight = float(temperature), float(soft_weight), float(hard_weight)
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError(f"temperature must be 1e-3 to 1e3, got {temperature}")
    if not (0.0 <= soft_weight < 1e30 and 0.0 <= hard_weight < 1e30):
        raise ValueError(f"soft_weight and hard_weight must be finite and not negative, got {soft_weight} and {hard_weight}")
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean' or 'sum', got {reduction!r}")
    if labels is None:
        if hard_weight or shift_labels:
            raise ValueError("a hard loss (hard_weight > 0, the default is 0) and shift_labels need labels")
    else:
        if labels.dtype != torch.int64:
            raise TypeError(f"labels must be int64, got {labels.dtype}")
        if labels.shape != lead:
            raise ValueError(f"labels must be {tuple(lead)}, got {tuple(labels.shape)}")
        labels = labels.contiguous()
    indices, teacher = teacher_indices.contiguous(), teacher_logits.contiguous()
    if teacher.is_neg():
        teacher = teacher.resolve_neg()
    terms = _lib.Distillation(indices.data_ptr(), teacher.data_ptr(), _lib.ptr(labels), int(ignore_index),
                              _INDEX_BITS[indices.dtype], kind, K, int(bool(shift_labels)), temperature, soft_weight, hard_weight,
                              int(reduction == "sum"))
    return device, logits, rows, terms, (indices, teacher, labels)


def _gradient(logits: torch.Tensor) -> torch.Tensor:
    if logits.is_contiguous():
        return torch.empty_like(logits)
    return torch.empty(*logits.shape, dtype=logits.dtype, device=logits.device)


def _launch_distillation(device: int, logits, rows, terms, upstream: Optional[torch.Tensor], grad: Optional[torch.Tensor],
                         stats: Optional[torch.Tensor] = None, want_loss: bool = True) -> Optional[torch.Tensor]:
    """The loss (None where only the gradient is wanted); `stats` [4] receives [sum of the rows' losses, live rows, sum of the hard terms, sum of the divergences]."""
    where = logits.device
    if logits.numel() == 0:
        if stats is not None:
            stats.zero_()
        return torch.zeros((), dtype=torch.float32, device=where)
    loss = torch.empty_strided((), (), dtype=torch.float32, device=where) if want_loss else None
    size = _lib.load().gscan_distillation_workspace_bytes(C.byref(rows))
    ws = torch.empty(size, dtype=torch.uint8, device=where)
    _call("gscan_distillation_loss", device, C.byref(rows), C.byref(terms), _lib.ptr(upstream), _lib.ptr(grad), _lib.ptr(loss),
          _lib.ptr(stats), ws.data_ptr(), size)
    return loss


class _DistillationLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, indices, teacher, labels, options):
        device, logits, rows, terms, kept = _distillation(logits, indices, teacher, labels, *options)
        ctx.save_for_backward(logits, *kept)
        ctx.options, ctx.call = options, (device, rows, terms, logits.stride())
        return _launch_distillation(device, logits, rows, terms, None, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, indices, teacher, labels = ctx.saved_tensors
        device, rows, terms, stride = ctx.call
        if not (logits.data_ptr() == rows.data and logits.stride() == stride and indices.data_ptr() == terms.indices and teacher.data_ptr() == terms.teacher
                and (labels is None or labels.data_ptr() == terms.labels)):       # hooks on saved tensors may have moved them
            device, logits, rows, terms, _kept = _distillation(logits, indices, teacher, labels, *ctx.options)
        grad = _gradient(logits)
        _launch_distillation(device, logits, rows, terms, g.resolve_neg(), grad, want_loss=False)
        return grad, None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_indices: torch.Tensor, teacher_logits: torch.Tensor,
                      labels: Optional[torch.Tensor] = None, *, temperature: float = 1.0, soft_weight: float = 1.0,
                      hard_weight: float = 0.0, ignore_index: int = -100, shift_labels: bool = False,
                      reduction: str = "mean") -> torch.Tensor:
    """The loss of a student's `logits` [..., V] against a teacher's top logits (`top_logits` of the teacher):

        mean over the live rows of  soft_weight * temperature^2 * KL(p || q)  +  hard_weight * -log softmax(logits)[label]

    p = softmax(teacher_logits / temperature) over the row's K entries [..., K], q = softmax(logits / temperature) over all
    words.  An index outside [0, V) (say -1) is no entry, a teacher's logit of -inf has probability 0, an index that comes
    twice counts with both entries; a row without entries has no soft term.  Log-probabilities serve as logits.

    labels [...] int64: rows whose label is `ignore_index` or not a word are not live — no loss, a gradient of exactly 0,
    nothing of them is read; without labels every row is live.  `shift_labels`: labels are whole sequences and a row is
    scored against the next one, the last against 0, as `Model.get_loss` does (seq2seq/model.py:108-115).
    reduction "mean" (0 when no row is live) or "sum".  A differentiable float32 scalar; the gradient goes to `logits` only
    (backward only: logits with a forward-mode tangent raise).
    Into a graph, capture the backward pass of a loss that was captured too, with no eager loss of the same parameters alive
    (autograd adds up a parameter's gradient on the stream that it was first used on)."""
    options = (temperature, soft_weight, hard_weight, ignore_index, shift_labels, reduction)
    # a tangent too is autograd's to deal with: it raises, this function having no forward-mode derivative
    if (torch.is_grad_enabled() and logits.requires_grad) or forward_ad.unpack_dual(logits).tangent is not None:
        return _DistillationLoss.apply(logits, teacher_indices, teacher_logits, labels, options)
    device, logits, rows, terms, _kept = _distillation(logits, teacher_indices, teacher_logits, labels, *options)
    return _launch_distillation(device, logits, rows, terms, None, None)


def distillation_loss_and_gradient(logits: torch.Tensor, teacher_indices: torch.Tensor, teacher_logits: torch.Tensor,
                                   labels: Optional[torch.Tensor] = None, *, temperature: float = 1.0, soft_weight: float = 1.0,
                                   hard_weight: float = 0.0, ignore_index: int = -100, shift_labels: bool = False,
                                   reduction: str = "mean", out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`distillation_loss` and its gradient with respect to the logits in one pass over them, outside autograd: what a loop
    that issues its own backward pass calls (`train.TrainStep`).  Returns (loss, gradient [..., V] of the logits' type);
    `out`: a contiguous tensor for the gradient, which may not share memory with an argument."""
    device, logits, rows, terms, _kept = _distillation(logits, teacher_indices, teacher_logits, labels, temperature, soft_weight,
                                                       hard_weight, ignore_index, shift_labels, reduction)
    if out is None:
        out = _gradient(logits)
    else:
        _check_gradient_out(out, logits, _kept)
    return _launch_distillation(device, logits, rows, terms, None, out), out


def _check_gradient_out(out: torch.Tensor, logits: torch.Tensor, others: Sequence[Optional[torch.Tensor]]) -> None:
    _require("logits out", logits, out)
    if out.shape != logits.shape or out.dtype != logits.dtype or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {tuple(logits.shape)} tensor of {logits.dtype}")
    if out.is_neg():
        raise ValueError("out is a lazily negated view")
    if any(t is not None and _overlap(out, t) for t in (logits, *others)):
        raise ValueError("out shares memory with the logits, the teacher's entries or the labels")


def _extent(t: torch.Tensor) -> Tuple[int, int]:
    """First byte and the byte behind the last of a tensor's elements."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size() if t.numel() else t.data_ptr()


def _overlaps_itself(t: torch.Tensor) -> bool:
    """True unless every element has a place of its own (as far as strides that nest tell)."""
    end = 1
    for stride, size in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if stride < end:
            return True
        end += (size - 1) * stride
    return False


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    return a0 < b1 and b0 < a1


# ---------------------------------------------------------------------------------------------------------------------
# beam search
# ---------------------------------------------------------------------------------------------------------------------
def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor, *, eos_idx: int, pad_idx: int
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """One step of a beam search: the W best of a batch row's W * V continuations.

    logits [B, W, V] of the next word, scores [B, W] float32 (the beams' log-probabilities so far), finished [B, W] bool.
    A candidate's score is `scores[b, w] + log_softmax(logits[b, w])[v]`; a finished beam has one candidate, itself with its
    score as it is and the word `pad_idx`, and its logits are not read.  Returns, best first (scores are
    compared in 64 bits; of equal ones the lowest beam's comes first, of one beam's the largest logit, then the lowest word):
    (scores [B, W], parents [B, W] int32, words [B, W] int64, finished [B, W] bool: the parent was, or the word is `eos_idx`).
    Start a search with scores of 0 for one beam and -inf for the others: beams of -inf fill only places that nothing else
    takes.  W <= 64, V <= 2^24; a word barred with -inf (or NaN) has the score -inf, as
    have all words of a beam whose score is NaN or one of whose logits is +inf.  No gradient flows through it."""
    device = _require("logits scores finished", logits, scores, finished)
    if logits.dim() != 3:
        raise ValueError(f"logits must be [B, W, V], got {tuple(logits.shape)}")
    logits, rows = _rows(logits)
    B, W, V = logits.shape
    if tuple(scores.shape) != (B, W) or tuple(finished.shape) != (B, W):
        raise ValueError(f"scores and finished must be [{B}, {W}], got {tuple(scores.shape)} and {tuple(finished.shape)}")
    if scores.dtype != torch.float32 or finished.dtype != torch.bool:
        raise TypeError(f"scores must be float32 and finished bool, got {scores.dtype} and {finished.dtype}")
    if not 1 <= W <= _lib.MAX_BEAMS or V > 1 << 24:
        raise ValueError(f"1 to {_lib.MAX_BEAMS} beams and at most 2^24 words, got {W} and {V}")
    if not (0 <= int(eos_idx) < V and 0 <= int(pad_idx) < V):
        raise ValueError(f"eos_idx {eos_idx} or pad_idx {pad_idx} is not one of the {V} words")
    where = logits.device
    scores, finished = scores.contiguous(), finished.contiguous()
    if scores.is_neg():
        scores = scores.resolve_neg()
    new_scores = torch.empty(B, W, dtype=torch.float32, device=where)
    parents = torch.empty(B, W, dtype=torch.int32, device=where)
    words = torch.empty(B, W, dtype=torch.int64, device=where)
    done = torch.empty(B, W, dtype=torch.bool, device=where)
    if B:
        size = _lib.load().gscan_beam_select_workspace_bytes(C.byref(rows))
        ws = _workspace(size, where)
        _call("gscan_beam_select", device, C.byref(rows), scores.data_ptr(), finished.data_ptr(), int(eos_idx), int(pad_idx),
              new_scores.data_ptr(), parents.data_ptr(), words.data_ptr(), done.data_ptr(), _lib.ptr(ws), size)
    return new_scores, parents, words, done


def _slices(src: torch.Tensor, dst: torch.Tensor, dim: int) -> Optional[_lib.State]:
    """The copy src -> dst of one slice per index of `dim` (None: no such pair of strides)."""
    size = src.element_size()
    if dim == 0 and src.is_contiguous() and dst.is_contiguous():
        n = src.numel() // src.shape[0] * size
        return _lib.State(src.data_ptr(), dst.data_ptr(), 1, 1, n, 0, 0, n, n, 0, 0)
    dims = list(zip(src.shape, src.stride(), dst.stride()))
    run, behind = 1, []                       # adjacent elements of a slice, then what is left of it
    for n, a, b in reversed(dims[dim + 1:]):
        if n == 1:
            continue
        if not behind and a == b == run:
            run *= n
        elif behind and a == behind[-1][1] * behind[-1][0] and b == behind[-1][2] * behind[-1][0]:
            behind[-1] = (behind[-1][0] * n, behind[-1][1], behind[-1][2])
        else:
            behind.append((n, a, b))
    before = []
    for n, a, b in reversed(dims[:dim]):
        if n == 1:
            continue
        if before and a == before[-1][1] * before[-1][0] and b == before[-1][2] * before[-1][0]:
            before[-1] = (before[-1][0] * n, before[-1][1], before[-1][2])
        else:
            before.append((n, a, b))
    if len(behind) > 1 or len(before) > 1:
        return None
    mid = behind[0] if behind else (1, 0, 0)
    outer = before[0] if before else (1, 0, 0)
    return _lib.State(src.data_ptr(), dst.data_ptr(), outer[0], mid[0], run * size, outer[1] * size, outer[2] * size,
                      dims[dim][1] * size, dims[dim][2] * size, mid[1] * size, mid[2] * size)


@functools.lru_cache(maxsize=None)
def _table(n: int):
    """The array type of n states (ctypes makes a new class for every `State * n`)."""
    return _lib.State * n


def beam_reorder(parents: torch.Tensor, states: Union[torch.Tensor, Sequence[torch.Tensor]],
                 out: Union[None, torch.Tensor, Sequence[torch.Tensor]] = None, dim: int = 0
                 ) -> Union[torch.Tensor, List[torch.Tensor]]:
    """The beams' states in the order that `beam_select` gave: slice b * W + w of the result is slice b * W + parents[b, w] of
    the state, along `dim` (which has B * W entries).  parents [B, W] int32; states: a tensor of any type, or a sequence of
    them, all moved in one launch (16 at a time).  `out`: where to write (of the states' shapes, any strides: a slice of a
    longer cache keeps what lies behind it), in memory whose span, from its first element to its last, meets neither a state's
    nor another `out`'s; otherwise new contiguous tensors are returned.
    A parent outside [0, W) gives zeros.  No gradient flows through it."""
    single = isinstance(states, torch.Tensor)
    sources = [states] if single else list(states)
    if parents.dim() != 2 or parents.dtype != torch.int32:
        raise ValueError(f"parents must be an int32 tensor [B, W], got {parents.dtype} {tuple(parents.shape)}")
    device = _require("parents", parents)
    B, W = parents.shape
    if out is None:
        targets = [torch.empty(s.shape, dtype=s.dtype, device=parents.device) for s in sources]
    else:
        targets = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(targets) != len(sources):
            raise ValueError(f"{len(sources)} states, but {len(targets)} tensors to write them to")
    moves = []
    for i, (s, d) in enumerate(zip(sources, targets)):
        if s.get_device() != device or d.get_device() != device:
            _require(f"parents states[{i}] out[{i}]", parents, s, d)
        at = dim + s.dim() if dim < 0 else dim
        if not 0 <= at < s.dim() or s.shape[at] != B * W:
            raise ValueError(f"states[{i}] {tuple(s.shape)} has not {B} x {W} entries along dimension {dim}")
        if d.shape != s.shape or d.dtype != s.dtype:
            raise ValueError(f"out[{i}] must be {tuple(s.shape)} of {s.dtype}, got {tuple(d.shape)} of {d.dtype}")
        if s.numel() == 0:
            continue
        if s.is_neg() or s.dtype.is_complex:       # bytes are moved: a conjugation that only the view knows of would be lost
            s = s.resolve_conj().resolve_neg()
        if out is not None:
            if d.is_neg() or d.is_conj():
                raise ValueError(f"out[{i}] is a lazily conjugated or negated view")
            if any(_overlap(d, other) for other in (parents, *sources)):
                raise ValueError(f"out[{i}] shares memory with a state or with the parents")
            if _overlaps_itself(d):
                raise ValueError(f"out[{i}]: elements of {tuple(d.shape)} with the strides {tuple(d.stride())} share memory")
        move = _slices(s, d, at)
        if move is None:
            s = s.contiguous()
            move = _slices(s, d, at)
        if move is None:
            raise ValueError(f"out[{i}]: the strides {tuple(d.stride())} of {tuple(d.shape)} are not one dimension before and one "
                             f"behind dimension {dim}")
        moves.append((move, s))
    if moves:
        if len(targets) > 1 and out is not None:
            spans = sorted(_extent(d) for d in targets if d.numel())
            if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
                raise ValueError("two tensors of out share memory")
        table = _table(len(moves))(*(m for m, _ in moves))
        order = parents.contiguous()
        _call("gscan_beam_reorder", device, B, W, order.data_ptr(), table, len(moves))
    return targets[0] if single else targets
