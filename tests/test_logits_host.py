"""What the operators over rows of logits refuse, and how tensors' strides become rows and slices: no GPU needed."""
import ctypes as C

import pytest
import torch

from multimodal_seq2seq_gscan_amd import _lib, logits as ops


@pytest.fixture(scope="module")
def lib():
    from multimodal_seq2seq_gscan_amd import build
    build.build()
    return _lib.load()


@pytest.fixture()
def on_host(monkeypatch, lib):
    """The Python layer with CPU tensors and no launches: its checks only."""
    calls = []
    monkeypatch.setattr(ops, "_require", lambda names, *tensors: 0)
    monkeypatch.setattr(ops, "_call", lambda name, device, *args: calls.append(name))
    return calls


def rows(**kw):
    base = dict(data=4096, type=_lib.F32, V=100, outer=4, inner=5, stride_outer=500, stride_inner=100)
    base.update(kw)
    return _lib.Rows(**base)


def message(lib):
    return lib.gscan_last_error().decode()


@pytest.mark.parametrize("kw,word", [(dict(data=None), "NULL"), (dict(type=7), "type"), (dict(V=0), "words"), (dict(outer=0), "rows"),
                                     (dict(inner=0), "rows"), (dict(outer=1 << 13, inner=1 << 12), "rows"),
                                     (dict(stride_inner=-1), "stride"), (dict(data=4097), "aligned")])
def test_rows_that_no_kernel_takes_are_refused(lib, kw, word):
    assert lib.gscan_top_logits(C.byref(rows(**kw)), 3, 4096, 4096, None, None, 0, None) != 0
    assert word in message(lib)
    assert lib.gscan_distillation_workspace_bytes(C.byref(rows(**kw))) == 0
    assert word in message(lib)


def test_library_refuses_bad_selections(lib):
    for k in (0, -1, 101, 257):
        assert lib.gscan_top_logits(C.byref(rows()), k, 4096, 4096, None, None, 0, None) != 0
        assert "K = " in message(lib)
    assert lib.gscan_top_logits(None, 3, 4096, 4096, None, None, 0, None) != 0
    assert lib.gscan_top_logits(C.byref(rows()), 3, None, 4096, None, None, 0, None) != 0
    long = rows(V=100000, outer=1, inner=1)
    need = lib.gscan_top_logits_workspace_bytes(C.byref(long), 8)
    assert need > 0                                             # one long row is split over workgroups
    assert lib.gscan_top_logits(C.byref(long), 8, 4096, 4096, None, 4096, need - 1, None) != 0
    assert "workspace" in message(lib)
    assert lib.gscan_top_logits(C.byref(long), 8, 4096, 4096, None, None, need, None) != 0
    assert lib.gscan_top_logits_workspace_bytes(C.byref(rows()), 8) == 0


def terms(**kw):
    base = dict(indices=4096, teacher=4096, labels=4096, ignore_index=0, index_bits=32, teacher_type=_lib.F32, K=4,
                shift_labels=0, temperature=1.0, soft_weight=1.0, hard_weight=0.5, sum_reduction=0)
    base.update(kw)
    return _lib.Distillation(**base)


@pytest.mark.parametrize("kw,word", [(dict(K=0), "entries"), (dict(K=257), "entries"), (dict(indices=None), "NULL"),
                                     (dict(teacher=None), "NULL"), (dict(index_bits=16), "bits"), (dict(teacher_type=5), "type"),
                                     (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                                     (dict(temperature=float("inf")), "temperature"), (dict(soft_weight=-1.0), "weights"),
                                     (dict(hard_weight=float("inf")), "weights"), (dict(hard_weight=float("nan")), "weights"),
                                     (dict(labels=None), "labels")])
def test_library_refuses_bad_distillation(lib, kw, word):
    assert lib.gscan_distillation_loss(C.byref(rows()), C.byref(terms(**kw)), None, None, 4096, None, 4096, 1 << 20, None) != 0
    assert word in message(lib)


def test_library_refuses_missing_outputs_and_small_workspaces(lib):
    assert lib.gscan_distillation_loss(C.byref(rows()), C.byref(terms()), None, None, None, None, 4096, 1 << 20, None) != 0
    need = lib.gscan_distillation_workspace_bytes(C.byref(rows()))
    assert lib.gscan_distillation_loss(C.byref(rows()), C.byref(terms()), None, None, 4096, None, 4096, need - 1, None) != 0
    assert "workspace" in message(lib)
    assert lib.gscan_distillation_loss(C.byref(rows()), None, None, None, 4096, None, 4096, need, None) != 0
    select = [C.byref(rows(inner=4)), 4096, 4096, 2, 0, 8192, 8192, 8192, 8192, None, 0, None]
    assert lib.gscan_beam_select(*select) != 0 and "workspace" in message(lib)
    for at, bad, word in ((1, None, "NULL"), (3, 100, "eos"), (4, -1, "pad"), (5, 4096, "inputs")):
        args = list(select)
        args[at] = bad
        assert lib.gscan_beam_select(*args) != 0
        assert word in message(lib)
    args = list(select)
    args[0] = C.byref(rows(inner=65))
    assert lib.gscan_beam_select(*args) != 0 and "beams" in message(lib)
    args[0] = C.byref(rows(V=(1 << 24) + 1))
    assert lib.gscan_beam_select(*args) != 0 and "2^24" in message(lib)


def state(**kw):
    base = dict(src=4096, dst=1 << 20, outer=1, mid=1, bytes=64, in_outer=0, out_outer=0, in_row=64, out_row=64, in_mid=0, out_mid=0)
    base.update(kw)
    return _lib.State(**base)


@pytest.mark.parametrize("kw", [dict(src=None), dict(dst=None), dict(outer=0), dict(mid=0), dict(bytes=0), dict(in_row=-64),
                                dict(outer=1 << 24, mid=1 << 24), dict(bytes=1 << 41)])
def test_library_refuses_bad_states(lib, kw):
    table = (_lib.State * 2)(state(), state(**kw))
    assert lib.gscan_beam_reorder(2, 3, 4096, table, 2, None) != 0
    assert "state 1" in message(lib)
    assert lib.gscan_beam_reorder(2, 3, None, table, 1, None) != 0
    assert lib.gscan_beam_reorder(0, 3, 4096, table, 1, None) != 0
    assert lib.gscan_beam_reorder(1 << 13, 1 << 13, 4096, table, 1, None) != 0
    assert lib.gscan_beam_reorder(2, 3, 4096, table, 0, None) != 0


def test_cpu_tensors_raise():
    x = torch.randn(2, 3, 10)
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.top_logits(x, 2)
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.distillation_loss(x, torch.zeros(2, 3, 1, dtype=torch.int32), torch.zeros(2, 3, 1))
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.beam_select(x, torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool), eos_idx=2, pad_idx=0)
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.beam_reorder(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 4))


def test_python_layer_refuses(on_host):
    x = torch.randn(2, 3, 10)
    index, teacher, labels = torch.zeros(2, 3, 4, dtype=torch.int32), torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64)
    for bad in (0, 11, -1):
        with pytest.raises(ValueError):
            ops.top_logits(x, bad)
    with pytest.raises(TypeError):
        ops.top_logits(x.double(), 2)
    with pytest.raises(ValueError):
        ops.top_logits(x[:, :, :0], 1)
    cases = [(dict(index=index[:1]), ValueError), (dict(teacher=teacher[..., :3]), ValueError), (dict(index=index.to(torch.int16)), TypeError),
             (dict(teacher=teacher.double()), TypeError), (dict(labels=labels[:, :2]), ValueError),
             (dict(labels=labels.to(torch.int32)), TypeError), (dict(temperature=0.0), ValueError),
             (dict(temperature=float("nan")), ValueError), (dict(soft_weight=-0.5), ValueError),
             (dict(hard_weight=float("inf")), ValueError), (dict(reduction="none"), ValueError),
             (dict(labels=None, hard_weight=0.5), ValueError), (dict(labels=None, shift_labels=True), ValueError)]
    for change, error in cases:
        kw = dict(index=index, teacher=teacher, labels=labels)
        kw.update(change)
        args = (x, kw.pop("index"), kw.pop("teacher"), kw.pop("labels"))
        with pytest.raises(error):
            ops.distillation_loss(*args, **kw)
        with pytest.raises(error):
            ops.distillation_loss_and_gradient(*args, **kw)
    for out in (x, torch.empty(2, 3, 9), torch.empty(2, 3, 10, dtype=torch.float16), torch.empty(2, 10, 3).transpose(1, 2), x[:, :, :]):
        with pytest.raises(ValueError):
            ops.distillation_loss_and_gradient(x, index, teacher, labels, out=out)
    scores, done = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool)
    for args, kw, error in [((x[0], scores, done), {}, ValueError), ((x, scores[:1], done), {}, ValueError),
                            ((x, scores.double(), done), {}, TypeError), ((x, scores, done.to(torch.uint8)), {}, TypeError),
                            ((x, scores, done), dict(eos_idx=10), ValueError), ((x, scores, done), dict(pad_idx=-1), ValueError),
                            ((torch.zeros(1, 65, 5), torch.zeros(1, 65), torch.zeros(1, 65, dtype=torch.bool)), {}, ValueError)]:
        with pytest.raises(error):
            ops.beam_select(*args, **{**dict(eos_idx=2, pad_idx=0), **kw})
    parents, cache = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 4, 5)
    for args, kw in [((parents.long(), cache), {}), ((parents[0], cache), {}), ((parents, cache[:5]), {}), ((parents, cache), dict(dim=3)),
                     ((parents, cache), dict(dim=1)), ((parents, cache), dict(out=cache)), ((parents, cache), dict(out=torch.zeros(6, 4, 6))),
                     ((parents, cache), dict(out=cache.long())), ((parents, [cache]), dict(out=[])),
                     ((parents, cache), dict(out=torch.zeros(6, 9, 2, 5)[:, ::2].permute(0, 1, 3, 2)[:, :4, :, 0].expand(6, 4, 5).transpose(1, 2)))]:
        with pytest.raises(ValueError):
            ops.beam_reorder(*args, **kw)
    both = torch.zeros(12, 4, 5)
    with pytest.raises(ValueError):           # two results in one place
        ops.beam_reorder(parents, [cache, cache], out=[both[:6], both[3:9]])
    assert not on_host


def fields(s):
    return {f: getattr(s, f) for f, _ in s._fields_}


def test_rows_of_strided_logits(lib):
    base = torch.randn(3, 4, 6, 10)
    got, r = ops._rows(base[:, 0, :5])
    assert got.data_ptr() == base.data_ptr() and (r.outer, r.inner, r.stride_outer, r.stride_inner, r.V) == (3, 5, 240, 10, 10)
    got, r = ops._rows(base)
    assert (r.outer, r.inner, r.stride_outer, r.stride_inner) == (12, 6, 60, 10)
    got, r = ops._rows(base[:, :, :, 2:7])
    assert got.data_ptr() == base.data_ptr() + 8 and (r.outer, r.inner, r.V) == (12, 6, 5)
    got, r = ops._rows(base[:, :, 1:3])
    assert (r.outer, r.inner, r.stride_outer, r.stride_inner) == (12, 2, 60, 10)
    copied = base[:, :3, 1:3]                                   # two dimensions that no single stride describes
    got, r = ops._rows(copied)
    assert got.is_contiguous() and torch.equal(got, copied) and (r.outer, r.inner) == (9, 2)
    got, r = ops._rows(base.transpose(2, 3))                    # words that are not adjacent
    assert got.is_contiguous() and r.V == 6
    got, r = ops._rows(base[0, 0, 0])
    assert (r.outer, r.inner, r.V) == (1, 1, 10)
    got, r = ops._rows(base[:, :1, :1].expand(3, 4, 6, 10)[:, 0])
    assert (r.outer, r.inner, r.stride_outer, r.stride_inner) == (3, 6, 240, 0)


def test_slices_of_strided_states(lib):
    cache = torch.zeros(3, 12, 4, 10, 8)                        # layers, beams, heads, positions, width
    used, new = cache[:, :, :, :7], torch.empty(3, 12, 4, 7, 8)
    s = fields(ops._slices(used, new, 1))
    assert (s["outer"], s["mid"], s["bytes"]) == (3, 4, 7 * 8 * 4)
    assert (s["in_row"], s["out_row"], s["in_mid"], s["out_mid"]) == (4 * 80 * 4, 4 * 56 * 4, 80 * 4, 56 * 4)
    assert (s["in_outer"], s["out_outer"]) == (12 * 4 * 80 * 4, 12 * 4 * 56 * 4)
    s = fields(ops._slices(torch.zeros(12), torch.zeros(12), 0))
    assert (s["outer"], s["mid"], s["bytes"], s["in_row"]) == (1, 1, 4, 4)
    assert ops._slices(torch.zeros(2, 3, 5, 12, 2)[:, :2, :4], torch.zeros(2, 2, 4, 12, 2), 3) is None
    s = fields(ops._slices(torch.zeros(12, 6).t()[:, :12], torch.zeros(6, 12), 1))        # columns: one element each
    assert (s["outer"], s["bytes"], s["mid"], s["in_row"], s["out_row"]) == (6, 4, 1, 24, 4)


def test_empty_batches_launch_nothing(on_host):
    values, index, lse = ops.top_logits(torch.zeros(0, 7, 10), 3, return_lse=True)
    assert values.shape == index.shape == (0, 7, 3) and lse.shape == (0, 7)
    loss, grad = ops.distillation_loss_and_gradient(torch.zeros(0, 7, 10), torch.zeros(0, 7, 2, dtype=torch.int32), torch.zeros(0, 7, 2))
    assert loss.item() == 0.0 and grad.shape == (0, 7, 10)
    out = ops.beam_select(torch.zeros(0, 4, 10), torch.zeros(0, 4), torch.zeros(0, 4, dtype=torch.bool), eos_idx=2, pad_idx=0)
    assert all(t.shape == (0, 4) for t in out)
    assert ops.beam_reorder(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 0)).shape == (6, 0)
    assert not on_host


def test_more_threads_than_a_launch_counts_are_refused(lib):
    """512 threads a row, 256 per four segments of a state: 2^32 of them is more than a launch takes."""
    many = rows(outer=1 << 23, inner=1, stride_outer=0, stride_inner=0)
    assert lib.gscan_top_logits(C.byref(many), 3, 4096, 4096, None, None, 0, None) != 0 and "rows" in message(lib)
    assert lib.gscan_distillation_workspace_bytes(C.byref(many)) == 0 and "rows" in message(lib)
    many.outer -= 1
    assert lib.gscan_distillation_workspace_bytes(C.byref(many)) > 0
    table = (_lib.State * 1)(state(outer=1 << 12, mid=1 << 10, bytes=1 << 13))
    assert lib.gscan_beam_reorder(2, 3, 4096, table, 1, None) != 0 and "pieces" in message(lib)


def test_outputs_that_share_memory_are_refused(on_host):
    parents, cache = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 4, 5)
    for out in (torch.zeros(6, 4, 1).expand(6, 4, 5), torch.zeros(1, 4, 5).expand(6, 4, 5), torch.zeros(60).as_strided((6, 4, 5), (8, 4, 1))):
        with pytest.raises(ValueError, match="share memory"):
            ops.beam_reorder(parents, cache, out=out)
    ids = torch.zeros(6, dtype=torch.int32)
    with pytest.raises(ValueError, match="parents"):
        ops.beam_reorder(parents, ids, out=parents.view(-1))
    assert not on_host
    for out in (torch.zeros(9, 4, 5)[:6], torch.zeros(6, 4, 10)[..., :5], torch.zeros(6, 1, 4, 5)[:, 0]):
        ops.beam_reorder(parents, cache, out=out)
    assert len(on_host) == 3
    x = torch.randn(2, 3, 10)
    place = torch.zeros(2, 3, 10)
    teacher = place.view(-1)[:24].view(2, 3, 4)
    index, labels = torch.zeros(2, 3, 4, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="shares memory"):
        ops.distillation_loss_and_gradient(x, index, teacher, labels, out=place)
    assert len(on_host) == 3
