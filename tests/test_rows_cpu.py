"""What the operators over rows of scores check before they reach the library, and their entry points without a GPU."""
import ctypes as C

import numpy as np
import pytest

from rows_reference import distill, kept, sample, top


@pytest.fixture
def context(accb):
    """A context without a device: enough for the checks of arguments."""
    c = object.__new__(accb.Context)
    c.handle, c.device = None, 0
    return c


def array(accb, *shape, kind=np.float32):
    return accb.DeviceArray(1 << 20, shape, kind)


def refused(accb, call, *args, **kw):
    with pytest.raises(accb.AccbError) as e:
        call(*args, **kw)
    assert e.value.status == accb.EINVAL
    return str(e.value)


def test_arguments_are_checked(accb, context):
    a = lambda *shape, kind=np.float32: array(accb, *shape, kind=kind)  # noqa: E731
    x, i32 = a(3, 100), np.int32
    assert "float64" in refused(accb, context.top_rows, a(3, 100, kind=np.float64), a(3, 5), a(3, 5, kind=i32))
    assert "rank" in refused(accb, context.top_rows, a(100), a(3, 5), a(3, 5, kind=i32))
    assert "rank" in refused(accb, context.top_rows, x, a(5), a(3, 5, kind=i32))
    assert "shape" in refused(accb, context.top_rows, x, a(2, 5), a(3, 5, kind=i32))
    assert "shape" in refused(accb, context.top_rows, x, a(3, 5), a(3, 4, kind=i32))
    assert "type" in refused(accb, context.top_rows, x, a(3, 5, kind=np.float16), a(3, 5, kind=i32))
    assert "type" in refused(accb, context.top_rows, x, a(3, 5), a(3, 5, kind=np.int64))
    assert "lse" in refused(accb, context.top_rows, x, a(3, 5), a(3, 5, kind=i32), lse=a(4))
    for name, good in (("temperature", np.float32), ("top_k", np.int32), ("top_p", np.float32), ("min_p", np.float32), ("logprob", np.float32)):
        assert name in refused(accb, context.sample_rows, x, a(3), a(3, kind=i32), **{name: a(2, kind=good)})
        assert name in refused(accb, context.sample_rows, x, a(3), a(3, kind=i32), **{name: a(3, kind=np.float64)})
    assert "uniform" in refused(accb, context.sample_rows, x, a(3, kind=np.float64), a(3, kind=i32))
    assert "token" in refused(accb, context.sample_rows, x, a(3), a(3, kind=np.int64))
    assert "allowed" in refused(accb, context.sample_rows, x, a(3), a(3, kind=i32), allowed=a(3, 3, kind=i32))
    assert "allowed" in refused(accb, context.sample_rows, x, a(3), a(3, kind=i32), allowed=a(3, 100, kind=np.bool_))
    teacher = (a(3, 5), a(3, 5, kind=i32))
    assert "teacher" in refused(accb, context.distill_rows, x, a(2, 5), teacher[1], a(3))
    assert "teacher" in refused(accb, context.distill_rows, x, a(3, 5, kind=np.float64), teacher[1], a(3))
    assert "index" in refused(accb, context.distill_rows, x, teacher[0], a(3, 6, kind=i32), a(3))
    assert "weight" in refused(accb, context.distill_rows, x, *teacher, a(3), weight=a(1))
    assert "teacher_lse" in refused(accb, context.distill_rows, x, *teacher, a(3), teacher_lse=a(3, 1))
    assert "loss" in refused(accb, context.distill_rows, x, *teacher, a(1))
    assert "stats" in refused(accb, context.distill_rows, x, *teacher, a(3), stats=a(3, 3))
    assert "grad" in refused(accb, context.distill_rows, x, *teacher, a(3), grad=a(3, 100, kind=np.float64))
    assert "upstream" in refused(accb, context.distill_rows_backward, x, *teacher, a(3, 4), a(2), a(3, 100))


def test_tensors_elsewhere_are_refused(accb, context):
    torch = pytest.importorskip("torch")
    x = torch.zeros(3, 100)
    assert "cpu" in refused(accb, context.top_rows, x, torch.zeros(3, 5), torch.zeros(3, 5, dtype=torch.int32))
    assert "contiguous" in refused(accb, context.sample_rows, torch.zeros(100, 3).T, torch.zeros(3), torch.zeros(3, dtype=torch.int32))


def test_what_is_no_device_array_is_refused(accb, context):
    """Host arrays and things that are no arrays at all, in every place: a refusal, not an error from within."""
    a = lambda *shape, kind=np.float32: array(accb, *shape, kind=kind)  # noqa: E731
    i32 = np.int32
    calls = [(context.top_rows, dict(x=a(3, 100), values=a(3, 5), index=a(3, 5, kind=i32), lse=a(3))),
             (context.sample_rows, dict(x=a(3, 100), uniform=a(3), token=a(3, kind=i32), logprob=a(3), temperature=a(3), top_k=a(3, kind=i32),
                                        top_p=a(3), min_p=a(3), allowed=a(3, 4, kind=i32))),
             (context.distill_rows, dict(student=a(3, 100), teacher=a(3, 5), index=a(3, 5, kind=i32), loss=a(3), grad=a(3, 100), stats=a(3, 4),
                                         teacher_lse=a(3), weight=a(3))),
             (context.distill_rows_backward, dict(student=a(3, 100), teacher=a(3, 5), index=a(3, 5, kind=i32), stats=a(3, 4), upstream=a(3),
                                                  grad=a(3, 100), teacher_lse=a(3), weight=a(3)))]
    for call, good in calls:
        for name, value in good.items():
            for other in (np.zeros(value.shape, value.dtype), [[1.0] * 5] * 3, 3.0):
                with pytest.raises(TypeError, match="not a device array"):
                    call(**{**good, name: other}, stream=0)


def test_without_a_stream_where_torch_has_no_gpu(accb, context, monkeypatch):
    """Memory that is not torch's, beside a torch that has no GPU: the default stream, as for every other launch."""
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    monkeypatch.setattr(accb, "_stream_of", None)
    a = lambda *shape, kind=np.float32: array(accb, *shape, kind=kind)  # noqa: E731
    assert context._own_stream(None) == 0
    assert "null context" in refused(accb, context.top_rows, a(3, 100), a(3, 5), a(3, 5, kind=np.int32))


def test_entry_points_refuse_a_null_context(accb):
    L = accb.lib()
    a = C.byref(accb.accb_rows_array(1 << 20, 0, 8, 1, 8))
    p = C.c_void_p(1 << 20)
    assert L.accb_top_rows(None, None, a, 1.0, 1, p, p, None) == accb.EINVAL
    assert L.accb_sample_rows(None, None, a, None, 0, p, None, None, None, None, p, None) == accb.EINVAL
    assert L.accb_distill_rows(None, None, a, p, 0, p, 2, None, None, 1.0, p, None, None) == accb.EINVAL
    assert L.accb_distill_rows_backward(None, None, a, p, 0, p, 2, None, None, 1.0, p, None, a) == accb.EINVAL


def test_struct_layout_matches_the_header(accb):
    s = accb.accb_rows_array
    assert (s.ptr.offset, s.type.offset, s.cols.offset, s.rows.offset, s.pitch.offset, C.sizeof(s)) == (0, 8, 12, 16, 24, 32)


# the reference that the GPU tests compare with, on rows small enough to check by hand
def test_reference_top():
    v, i, s = top(np.array([1.0, np.nan, 3.0, 3.0, -np.inf]), 4, 1.0)
    assert v.tolist() == [3.0, 3.0, 1.0, -np.inf] and i.tolist() == [2, 3, 0, -1]
    assert abs(s - np.log(2 * np.exp(3) + np.e)) < 1e-12


def test_reference_cuts():
    row = np.log(np.array([1.0, 4.0, 2.0, 1.0]))
    on = lambda **kw: np.nonzero(kept(row, **{**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw}))[0].tolist()  # noqa: E731
    assert on() == [0, 1, 2, 3] and on(top_k=3) == [0, 1, 2] and on(top_p=0.5 - 1e-9) == [1] and on(top_p=0.6) == [1, 2]
    assert on(top_p=0.8) == [0, 1, 2] and on(min_p=0.4) == [1, 2] and on(top_p=0.0) == [1] and on(temperature=0.0) == [1]
    assert on(top_k=2, top_p=0.7) == [1, 2]  # 4 / 6 < 0.7
    assert sample(row, 0.0)[0] == 0 and sample(row, 0.13)[0] == 1 and sample(row, 0.99)[0] == 3
    assert sample(row, 0.5, allowed=np.array([True, False, True, False]))[0] == 2


def test_reference_distillation_by_differences():
    rng = np.random.default_rng(3)
    z, t, at = rng.normal(0, 1, 12), rng.normal(0, 1, 4), np.array([3, 5, 3, -1])
    for lse in (None, np.log(np.exp(t).sum()) + 0.7):
        loss, d, _ = distill(z, t, at, lse, 1.5, 2.0)
        for j in range(12):
            e = np.eye(12)[j] * 1e-5
            n = (distill(z + e, t, at, lse, 1.5, 2.0)[0] - distill(z - e, t, at, lse, 1.5, 2.0)[0]) / 2e-5
            assert abs(n - d[j]) < 1e-8
