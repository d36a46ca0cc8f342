"""CPU: refusals of the serving operators (paged K/V cache, logit rules). Every argument the host can
see is checked before the device is touched, so a made-up address is never read here: a call that
passed the checks would fail on this host with a CUDA error, not with KQ_ERR_ARG."""
import struct

import pytest

P16 = 1 << 20            # a made-up, aligned device address
DESC = dict(k=P16, v=P16, kp=8 * 16 * 128, kh=16 * 128, kr=128, vp=8 * 16 * 128, vh=16 * 128, vr=128, ks=0, vs=0, type=1,
            n_pages=4, page=16, kv=8, hd=128)


@pytest.fixture(scope="module")
def kq():
    import kq as K
    return K


def create(kq, **change):
    d = dict(DESC, **change)
    return kq.lib().kq_pages_create(struct.pack("2P6q2P5i4x", *d.values()), 0)


@pytest.mark.parametrize("change,text", [
    (dict(k=0), "16-byte"), (dict(v=0), "16-byte"), (dict(k=P16 + 2), "16-byte"), (dict(kr=124), "16-byte"),
    (dict(vh=-2048), "16-byte"), (dict(type=0), "type"), (dict(type=7), "type"), (dict(hd=96), "head_dim"),
    (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(page=2048), "power of two"),
    (dict(n_pages=0), "count"), (dict(kv=0), "count"), (dict(ks=P16), "e4m3"),
])
def test_bad_page_descriptions(kq, change, text):
    assert not create(kq, **change)
    assert text in kq.last_error()


def test_null_handles(kq):
    L = kq.lib()
    assert L.kq_pages_create(None, 0) is None
    assert L.kq_page_append(None, b"\0" * 184, None) == kq.ERR_ARG
    assert L.kq_page_attend(None, b"\0" * 112, None) == kq.ERR_ARG
    assert L.kq_logit_rules(None, 0, None) == kq.ERR_ARG
    L.kq_pages_free(None)


RULES = dict(logits=P16, out=P16, in_ld=100, out_ld=100, best=0, hist=0, hist_len=0, prompt_len=0, hist_ld=0, rep=0, freq=0,
             pres=0, bias_id=0, bias=0, bias_ld=0, mask=0, mask_row=0, mask_ld=0, n=2, vocab=100, type=0, max_hist=0, n_bias=0,
             n_masks=0)


@pytest.mark.parametrize("change", [
    dict(logits=0), dict(out=0), dict(logits=P16 + 2), dict(in_ld=99), dict(out_ld=99), dict(n=-1), dict(vocab=0),
    dict(vocab=393217, in_ld=400000, out_ld=400000), dict(type=3), dict(out_ld=101), dict(hist=P16), dict(hist_len=P16),
    dict(hist=P16, hist_len=P16, max_hist=5, hist_ld=4), dict(prompt_len=P16), dict(bias=P16), dict(bias_id=P16),
    dict(bias=P16, bias_id=P16, n_bias=3, bias_ld=2), dict(n_bias=1), dict(mask=P16, n_masks=2, mask_ld=3),
    dict(mask=P16, n_masks=1, mask_ld=4), dict(mask=P16, n_masks=0, mask_ld=4, mask_row=P16), dict(mask_row=P16),
])
def test_bad_rules(kq, change):
    a = struct.pack("2P2qP3Pq3P2Pq2Pq6i", *dict(RULES, **change).values())
    assert kq.lib().kq_logit_rules(a, 0, None) == kq.ERR_ARG
    assert "kq_logit_rules" in kq.last_error()


class Fake(object):
    """The tensor interface the operators read, over no memory."""

    def __init__(self, shape, dtype="float32", stride=None, device=0, ptr=P16):
        self.shape, self.dtype, self._device, self._ptr = shape, "torch." + dtype, device, ptr
        s = [1]
        for d in reversed(shape[1:]):
            s.insert(0, s[0] * d)
        self._stride = tuple(s if stride is None else stride)

    def data_ptr(self):
        return self._ptr

    def get_device(self):
        return self._device

    def stride(self, i=None):
        return self._stride if i is None else self._stride[i]


def test_python_refusals(kq):
    good = Fake((4, 8, 16, 128), "float16")
    for bad in (Fake((4, 8, 16, 128), "float32"), Fake((4, 8, 16), "float16"), Fake((4, 8, 16, 128), "float16", device=-1),
                Fake((4, 8, 16, 128), "float16", stride=(16384, 2048, 1, 16))):
        with pytest.raises(ValueError):
            kq.PagedCache(bad, bad)
    with pytest.raises(ValueError):
        kq.PagedCache(good, Fake((4, 8, 16, 64), "float16"))
    with pytest.raises(ValueError):
        kq.PagedCache(good, Fake((4, 8, 16, 128), "bfloat16"))
    with pytest.raises(ValueError):
        kq.PagedCache(good, Fake((4, 8, 16, 128), "float16", device=1))
    z = Fake((2, 100))
    for kw in (dict(best=Fake((3,), "int32")), dict(best=Fake((2,), "int64")), dict(hist=Fake((2, 5), "int32")),
               dict(hist_len=Fake((2,), "int32")), dict(bias=Fake((2, 5))), dict(bias_ids=Fake((2, 5), "int32")),
               dict(mask=Fake((2, 3), "int32")), dict(mask_row=Fake((2,), "int32")), dict(repetition=Fake((2,), "float16")),
               dict(presence=Fake((2,), device=1))):
        with pytest.raises(ValueError):
            kq.logit_rules(z, z, **kw)
    with pytest.raises(ValueError):
        kq.logit_rules(z, Fake((2, 99)))
    with pytest.raises(ValueError):
        kq.logit_rules(z, Fake((2, 100), "float16"))


def test_structures_match_the_header(kq):
    """The packed arguments have the C structures' sizes (all fields naturally aligned, no holes but the tail)."""
    from kq import serve
    assert struct.calcsize("2P6q2P5i4x") == 104
    assert (serve._APPEND.size, serve._ATTEND.size, serve._RULES.size) == (184, 112, 168)


def test_operators_fail_without_a_device(kq):
    if kq.lib().kq_device_count() > 0:
        pytest.skip("a GPU is present")
    assert not create(kq)
    assert kq.lib().kq_logit_rules(struct.pack("2P2qP3Pq3P2Pq2Pq6i", *RULES.values()), 0, None) == kq.ERR_BACKEND


def test_tensors_of_another_device_are_refused_by_both_ways(kq):
    """PyTorch tensors take the short way through their DLPack interface; what it cannot take ends in the checks."""
    torch = pytest.importorskip("torch")
    from kq import serve
    z = torch.zeros((2, 64))
    with pytest.raises(ValueError, match="GPU"):
        kq.logit_rules(z, z)
    if getattr(torch.Tensor, "__dlpack_c_exchange_api__", None) is not None:
        assert serve._Direct.type is torch.Tensor
        args = [id(z), id(z)] + [None] * 11
        assert serve._Direct.logit_rules(*args, 0) == serve._Direct.OTHER
    c = object.__new__(kq.PagedCache)
    c.h, c.device, c.n_kv, c.page, c.hd, c.type = 1, 0, 2, 16, 64, serve.F16
    c._free = lambda h: None
    k, table, i = torch.zeros((1, 2, 64)), torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    serve._Direct.page_attend, kept = (lambda *a: serve._Direct.OTHER), serve._Direct.page_attend
    serve._Direct.page_append, kept2 = (lambda *a: serve._Direct.OTHER), serve._Direct.page_append
    try:
        with pytest.raises(ValueError, match="not on device 0"):
            c.attend(k, table, i, k)
        with pytest.raises(ValueError, match="not on device 0"):
            c.append(k, k, table, i)
    finally:
        serve._Direct.page_attend, serve._Direct.page_append = kept, kept2
        c.h = None
