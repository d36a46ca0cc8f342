"""CPU: the serving operators' calls on tensor objects (kq_*_tensors), their objects described by this file as
CUDA tensors over made-up addresses. The host has no device, so what passes every check ends in KQ_ERR_BACKEND
and nothing is launched."""
import ctypes as C

import pytest

P16 = 1 << 20


class DlTensor(C.Structure):
    """DLPack's DLTensor (version 1)."""
    _fields_ = [("data", C.c_void_p), ("device_type", C.c_int32), ("device_id", C.c_int32), ("ndim", C.c_int32), ("code", C.c_uint8),
                ("bits", C.c_uint8), ("lanes", C.c_uint16), ("shape", C.POINTER(C.c_int64)), ("strides", C.POINTER(C.c_int64)),
                ("byte_offset", C.c_uint64)]


class Made(object):
    """A description: shape, strides, type (DLPack's code and bits)."""

    def __init__(self, shape, strides=None, kind=(2, 32)):
        dense = [1]
        for d in reversed(shape[1:]):
            dense.insert(0, dense[0] * d)
        self.shape = (C.c_int64 * len(shape))(*shape)
        self.strides = (C.c_int64 * len(shape))(*(strides or dense))
        self.kind = kind


INT = (0, 32)


@pytest.fixture
def direct():
    """The library's calls on Made objects; the tensor library's own description is put back afterwards."""
    import kq as K
    from kq import serve
    if K.lib().kq_device_count() > 0:
        pytest.skip("a GPU is present: made-up addresses stay off it")
    known = {}

    @C.PYFUNCTYPE(C.c_int, C.c_void_p, C.c_void_p)
    def describe(obj, out):
        made = known[obj]
        C.cast(out, C.POINTER(DlTensor))[0] = DlTensor(P16, 2, 0, len(made.shape), made.kind[0], made.kind[1], 1, made.shape, made.strides, 0)
        return 0

    lib = C.PyDLL(K.LIB_PATH)
    lib.kq_tensor_source.argtypes = lib.kq_tensor_stream.argtypes = [C.c_void_p]
    lib.kq_tensor_source(C.cast(describe, C.c_void_p))

    def call(name, *args):
        f = getattr(lib, name)
        f.restype, f.argtypes = K.SIGNATURES[name]
        known.update((id(a), a) for a in args if isinstance(a, Made))
        return f(*(id(a) if isinstance(a, Made) else a for a in args))

    call.lib = lib
    yield call
    was = serve._Direct.type
    serve._Direct.type, serve._Direct._tried = None, set()
    lib.kq_tensor_source(None)
    lib.kq_tensor_stream(None)
    if was is not None:
        serve._Direct.try_type(was)


def rules(direct, vocab=200, mask=None, mask_row=None):
    z = Made((2, vocab))
    return direct("kq_logit_rules_tensors", z, z, *[None] * 9, mask, mask_row, 0)


def test_masks_too_narrow_for_the_vocabulary_are_not_taken(direct):
    """Columns of a wider array: its stride is wide enough, its rows are not."""
    import kq as K
    from kq.serve import _Direct
    assert rules(direct, mask=Made((2, 7), kind=INT)) == K.ERR_BACKEND           # ceil(200 / 32) words: taken
    assert rules(direct, mask=Made((2, 7), (5000, 1), INT)) == K.ERR_BACKEND
    for shape, strides in (((2, 6), (5000, 1)), ((2, 6), None), ((2, 1), (7, 1)), ((1, 6), (5000, 1))):
        assert rules(direct, mask=Made(shape, strides, INT), mask_row=Made((2,), kind=INT)) == _Direct.OTHER


def test_calls_ask_for_the_current_stream_where_they_are_told_to(direct):
    """KQ_STREAM_CURRENT: the tensors' library is asked, for the tensors' device; any other handle is taken as it is."""
    import kq as K
    from kq.serve import _Direct
    asked, status = [], [0]

    @C.PYFUNCTYPE(C.c_int, C.c_int, C.c_int32, C.POINTER(C.c_void_p))
    def current(kind, device, out):
        asked.append((kind, device))
        out[0] = 1234
        return status[0]

    direct.lib.kq_tensor_stream(C.cast(current, C.c_void_p))
    z = Made((2, 200))
    none = [None] * 11
    assert direct("kq_logit_rules_tensors", z, z, *none, 0) == K.ERR_BACKEND and not asked
    assert direct("kq_logit_rules_tensors", z, z, *none, 77) == K.ERR_BACKEND and not asked
    assert direct("kq_logit_rules_tensors", z, z, *none, _Direct.CURRENT) == K.ERR_BACKEND and asked == [(2, 0)]
    status[0] = -1                                       # it does not know: nothing is launched
    assert direct("kq_logit_rules_tensors", z, z, *none, _Direct.CURRENT) == _Direct.OTHER


def test_calls_without_a_stream_take_the_current_one(monkeypatch):
    """The Python face: what the library is given where no stream is named, both ways of passing tensors."""
    import kq as K
    from kq import serve
    torch = pytest.importorskip("torch")
    streams = []

    def record(*args):
        streams.append(args[-1])
        return 0

    c = object.__new__(K.PagedCache)
    c.h, c.device, c.n_kv, c.page, c.hd, c.type = 1, -1, 2, 16, 64, serve.F16
    c._free, c._append, c._attend = (lambda h: None), record, record
    k, table, i = torch.zeros((1, 2, 64)), torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def calls(**kw):
        del streams[:]
        c.append(k, k, table, i, **kw)
        c.attend(k, table, i, k, **kw)
        return streams

    for name in ("page_append", "page_attend"):
        monkeypatch.setattr(serve._Direct, name, record, raising=False)
    monkeypatch.setattr(serve._Direct, "type", torch.Tensor)
    assert calls() == [serve._Direct.CURRENT] * 2
    assert calls(stream=0) == [0, 0] and calls(stream=5) == [5, 5]
    monkeypatch.setattr(serve._Direct, "type", None)
    monkeypatch.setattr(serve, "current_stream", lambda device, *tensors: 99)
    assert calls() == [99, 99]
    assert calls(stream=0) == [0, 0] and calls(stream=5) == [5, 5]
    c.h = None
