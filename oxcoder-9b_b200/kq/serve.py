"""kq.serve -- the serving operators on device tensors (include/kq.h, "serving operators"):

    cache = kq.PagedCache(k, v)                     # pages of one attention layer, the caller's tensors
    cache.append(k_new, v_new, table, pos, rope=(cos, sin), q=q, q_out=q)
    cache.attend(q, table, lens, out)
    kq.logit_rules(logits, out, best=ids, hist=..., mask=...)
    kq.check_stream()                               # waits, raises what the kernels flagged

Tensors are any objects with PyTorch's tensor interface (data_ptr, shape, stride, dtype, get_device);
this module does not import it. Calls are enqueued on `stream`, a CUDA stream handle (0: the legacy default
stream; None: the stream that PyTorch's own operations are enqueued on at the time, the legacy default where the
tensors' library does not tell), and neither wait nor allocate. Wrong types, shapes, strides or devices
raise ValueError before anything is launched."""
import ctypes as C
import struct
import sys

F32, F16, BF16, E4M3, I32 = 0, 1, 2, 3, 4
_NAMES = {"float32": F32, "float16": F16, "bfloat16": BF16, "float8_e4m3fn": E4M3, "int32": I32, "uint32": I32}
_types = {}     # dtype object -> code

_APPEND = struct.Struct("4P8q3P2P2q7i4x")
_ATTEND = struct.Struct("2P4q3Pq6if4x")
_RULES = struct.Struct("2P2qP3Pq3P2Pq2Pq6i")


class _Direct(object):
    """The library's calls on tensor objects (kq_*_tensors) for a tensor type that has DLPack's C exchange
    interface, or None of them: those calls answer OTHER for whatever they cannot take, and the checks
    below then say why. They keep Python's lock (the interface needs it)."""
    OTHER = 1
    CURRENT = C.c_void_p(-1).value                      # KQ_STREAM_CURRENT
    type = None
    current = None
    _tried = set()

    @classmethod
    def try_type(cls, t):
        if t in cls._tried:
            return
        cls._tried.add(t)
        capsule = getattr(t, "__dlpack_c_exchange_api__", None)
        if cls.type is not None or capsule is None:
            return
        from . import LIB_PATH, SIGNATURES
        get = C.pythonapi.PyCapsule_GetPointer
        get.restype, get.argtypes = C.c_void_p, [C.py_object, C.c_char_p]
        api = get(capsule, b"dlpack_exchange_api")
        if C.c_uint32.from_address(api).value != 1:     # the interface's major version
            return
        describe = C.c_void_p.from_address(api + 5 * 8).value   # dltensor_from_py_object_no_sync
        current = C.c_void_p.from_address(api + 6 * 8).value    # current_work_stream
        if not describe or not current:
            return
        lib = C.PyDLL(LIB_PATH)
        lib.kq_tensor_source.argtypes = [C.c_void_p]
        lib.kq_tensor_source(describe)
        lib.kq_tensor_stream.argtypes = [C.c_void_p]
        lib.kq_tensor_stream(current)
        cls.current = C.PYFUNCTYPE(C.c_int, C.c_int, C.c_int32, C.POINTER(C.c_void_p))(current)
        for name in ("kq_page_append_tensors", "kq_page_attend_tensors", "kq_logit_rules_tensors"):
            f = getattr(lib, name)
            f.restype, f.argtypes = SIGNATURES[name]
            setattr(cls, name[3:-8], f)
        cls.type = t


def current_stream(device, *tensors):
    """Handle of the stream on which the library of such tensors enqueues its operations on the device now (0: unknown)."""
    for t in tensors:
        if t is not None:
            _Direct.try_type(type(t))
    if _Direct.current is not None:
        s = C.c_void_p()
        return s.value or 0 if _Direct.current(2, device, C.byref(s)) == 0 else 0
    torch = sys.modules.get("torch")                    # a PyTorch without that interface
    return torch.cuda.current_stream(device).cuda_stream if torch is not None and torch.cuda.is_initialized() else 0


def _bind():
    from . import check, last_error, lib
    return lib(), check, last_error


_rule_call = []


def _rules():
    if not _rule_call:
        _rule_call.append(_bind()[0].kq_logit_rules)
    return _rule_call[0]


def _type(t):
    c = _types.get(t.dtype)
    if c is None:
        c = _types[t.dtype] = _NAMES.get(str(t.dtype).rpartition(".")[2], -1)
    return c


def _refuse(t, what, kind, shape, device):
    """Says why _rows or _vec refused a tensor."""
    if t.get_device() != device:
        raise ValueError("%s is not on device %d" % (what, device))
    if _type(t) != kind:
        raise ValueError("%s has an unsupported or another type: %s" % (what, t.dtype))
    if tuple(t.shape) != shape:
        raise ValueError("%s must have the shape %s, not %s" % (what, shape, tuple(t.shape)))
    raise ValueError("the last dimension of %s must be dense" % what)


# These checks are most of what a call costs on the host (a few tenths of a microsecond a tensor, against
# kernels of a few microseconds), so each looks a property up once.
def _rows(t, what, kind, shape, device, _codes=_types.get):
    """(pointer, strides) of a tensor of this type code, shape and device whose last dim is dense."""
    s = t.stride()
    if (_codes(t.dtype) != kind and _type(t) != kind) or t.shape != shape or t.get_device() != device or (s[-1] != 1 and shape[-1] > 1):
        _refuse(t, what, kind, shape, device)
    return t.data_ptr(), s


def _vec(t, what, kind, shape, device, _codes=_types.get):
    """Pointer of a dense vector of this type code, shape (n,) and device."""
    if (_codes(t.dtype) != kind and _type(t) != kind) or t.shape != shape or t.get_device() != device or (t.stride()[0] != 1 and shape[0] > 1):
        _refuse(t, what, kind, shape, device)
    return t.data_ptr()


class PagedCache(object):
    """K and V pages of one attention layer: tensors [n_pages, n_kv_heads, page, head_dim] of fp16, bf16
    or e4m3 (any strides with dense rows on 16-byte boundaries: a transposed view of
    [n_pages, page, n_kv_heads, head_dim] will do). k_scale, v_scale (e4m3 only): fp32 [n_kv_heads], a stored
    x stands for x * scale. The tensors stay the caller's and are kept alive by this object. Calls on
    one cache that overlap in time on different streams race: use one PagedCache for each stream. It may
    be closed or collected at any time; a graph that captured its calls needs the tensors alone."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        lib, check, error = _bind()
        self.h = None
        self._check = check
        self._free = lib.kq_pages_free
        _Direct.try_type(type(k))
        if len(k.shape) != 4:
            raise ValueError("K pages must be [n_pages, n_kv_heads, page, head_dim]")
        self.device = k.get_device()
        if self.device < 0:
            raise ValueError("the pages must be on a GPU")
        self.n_pages, self.n_kv, self.page, self.hd = shape = tuple(k.shape)
        self.type = _type(k)
        if self.type not in (F16, BF16, E4M3):
            raise ValueError("pages are float16, bfloat16 or float8_e4m3fn, not %s" % k.dtype)
        kp, k_st = _rows(k, "k", self.type, shape, self.device)
        vp, v_st = _rows(v, "v", self.type, shape, self.device)
        ks = None if k_scale is None else _vec(k_scale, "k_scale", F32, (self.n_kv,), self.device)
        vs = None if v_scale is None else _vec(v_scale, "v_scale", F32, (self.n_kv,), self.device)
        self.tensors = (k, v, k_scale, v_scale)
        d = struct.pack("2P6q2P5i4x", kp, vp, *k_st[:3], *v_st[:3], ks or 0, vs or 0, self.type, self.n_pages,
                        self.page, self.n_kv, self.hd)
        h = lib.kq_pages_create(d, self.device)
        if not h:
            raise (MemoryError if "alloc" in error() else ValueError)(error())
        self.h = C.c_void_p(h)
        self._append, self._attend = lib.kq_page_append, lib.kq_page_attend

    def close(self):
        if self.h:
            self._free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _table(self, table, seq, n):
        """Pointers of the table and of the tokens' rows, the table's row stride and shape."""
        shape = table.shape
        if len(shape) != 2:
            raise ValueError("the page table must be [sequences, pages]")
        n_seq, wide = shape
        t, s = _rows(table, "table", I32, shape, self.device)
        if seq is not None:
            return t, _vec(seq, "seq", I32, (n,), self.device), s[0] if n_seq > 1 else wide, n_seq, wide
        if n > n_seq:
            raise ValueError("more tokens than page-table rows: give seq")
        return t, 0, s[0] if n_seq > 1 else wide, n_seq, wide

    def append(self, k, v, table, pos, seq=None, rope=None, q=None, q_out=None, stream=None):
        """K/V rows k, v [n, n_kv_heads, head_dim] (fp32, fp16 or bf16) to positions pos [n] of the sequences whose
        page-table rows are seq [n] (None: row i for token i); table [sequences, pages] int32. rope: (cos, sin)
        fp32 [positions, rot / 2]: the keys are rotated on the way, and so are the queries q [n, heads,
        head_dim] into q_out (may be q). pos < 0 skips a token. Slots of one call must be distinct."""
        if not self.h:
            raise ValueError("the cache is closed")
        T = _Direct.type
        if type(k) is T and type(v) is T and type(table) is T and type(pos) is T and (seq is None or type(seq) is T) \
                and (rope is None or (type(rope[0]) is T and type(rope[1]) is T)) \
                and (q is None or (type(q) is T and type(q_out) is T)):
            rc = _Direct.page_append(self.h, id(k), id(v), id(table), id(pos), None if seq is None else id(seq),
                                     None if rope is None else id(rope[0]), None if rope is None else id(rope[1]),
                                     None if q is None else id(q), None if q_out is None else id(q_out),
                                     _Direct.CURRENT if stream is None else stream)
            if not rc:
                return
            if rc != _Direct.OTHER:
                self._check(rc)
        n, dev, hd = k.shape[0], self.device, self.hd
        kind = _type(k)
        shape = (n, self.n_kv, hd)
        kp, (k0, k1, _) = _rows(k, "k", kind, shape, dev)
        vp, (v0, v1, _) = _rows(v, "v", kind, shape, dev)
        tp, sp, ld, n_seq, wide = self._table(table, seq, n)
        pp = _vec(pos, "pos", I32, (n,), dev)
        cp = np_ = rot = rl = n_pos = 0
        if rope is not None:
            cos, sin = rope
            shape = cos.shape
            n_pos, half = shape
            cp, c_st = _rows(cos, "cos", F32, shape, dev)
            np_, s_st = _rows(sin, "sin", F32, shape, dev)
            rl, rot = c_st[0] if n_pos > 1 else half, 2 * half
            if n_pos > 1 and s_st[0] != rl:
                raise ValueError("cos and sin must have the same strides")
        qp = op = q0 = q1 = o0 = o1 = heads = 0
        if q is not None:
            if q_out is None:
                raise ValueError("queries need q_out")
            heads = q.shape[1]
            shape = (n, heads, hd)
            qp, (q0, q1, _) = _rows(q, "q", kind, shape, dev)
            op, (o0, o1, _) = _rows(q_out, "q_out", kind, shape, dev)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if not n:
            return
        if stream is None:
            stream = current_stream(dev, k)
        rc = self._append(self.h, _APPEND.pack(kp, vp, qp, op, k0, k1, v0, v1, q0, q1, o0, o1, tp, sp, pp, cp, np_, ld, rl, n,
                                               heads, kind, n_seq, wide, rot, n_pos), stream)
        if rc:
            self._check(rc)

    def attend(self, q, table, lens, out, seq=None, window=0, scale=None, stream=None):
        """out[i][h] = softmax(scale q[i][h] . K) V over positions [0, lens[i]) of the sequence with page-table row
        seq[i] (None: row i); window > 0: over its last `window` positions. q, out [n, heads, head_dim] of one
        type (fp32, fp16, bf16), scale: 1 / sqrt(head_dim) by default. A row without positions gives zeros."""
        if not self.h:
            raise ValueError("the cache is closed")
        T = _Direct.type
        if type(q) is T and type(table) is T and type(lens) is T and type(out) is T and (seq is None or type(seq) is T):
            rc = _Direct.page_attend(self.h, id(q), id(table), id(lens), id(out), None if seq is None else id(seq), window,
                                     self.hd ** -0.5 if scale is None else scale, _Direct.CURRENT if stream is None else stream)
            if not rc:
                return out
            if rc != _Direct.OTHER:
                self._check(rc)
        shape = q.shape
        n, heads, hd = shape
        dev, kind = self.device, _type(q)
        if hd != self.hd:
            raise ValueError("q has head_dim %d, the cache %d" % (hd, self.hd))
        qp, (q0, q1, _) = _rows(q, "q", kind, shape, dev)
        op, (o0, o1, _) = _rows(out, "out", kind, shape, dev)
        tp, sp, ld, n_seq, wide = self._table(table, seq, n)
        lp = _vec(lens, "lens", I32, (n,), dev)
        if not n:
            return out
        if stream is None:
            stream = current_stream(dev, q)
        rc = self._attend(self.h, _ATTEND.pack(qp, op, q0, q1, o0, o1, tp, sp, lp, ld, n, heads, kind, n_seq, wide, window,
                                               hd ** -0.5 if scale is None else scale), stream)
        if rc:
            self._check(rc)
        return out


def _rule_fields(n, vocab, dev, hist=None, hist_len=None, prompt_len=None, repetition=None, frequency=None, presence=None,
                 bias_ids=None, bias=None, mask=None, mask_row=None):
    """The rules' part of kq_rule_args, checked: 13 pointers and strides, then max_hist, n_bias, n_masks."""
    row = (n,)
    hp = hl = pl = hld = most = 0
    if hist is not None:
        if hist_len is None:
            raise ValueError("hist needs hist_len")
        most = hist.shape[1]
        hp, (hld, _) = _rows(hist, "hist", I32, (n, most), dev)
        hl = _vec(hist_len, "hist_len", I32, row, dev)
        if prompt_len is not None:
            pl = _vec(prompt_len, "prompt_len", I32, row, dev)
        if n == 1:
            hld = most
        if not most:
            hp = hl = pl = 0
    elif hist_len is not None or prompt_len is not None:
        raise ValueError("history lengths without a history")
    rp = 0 if repetition is None else _vec(repetition, "repetition", F32, row, dev)
    fp = 0 if frequency is None else _vec(frequency, "frequency", F32, row, dev)
    sp = 0 if presence is None else _vec(presence, "presence", F32, row, dev)
    ap = dp = bld = entries = 0
    if bias_ids is not None and bias is not None:
        entries = bias_ids.shape[1]
        ap, (bld, _) = _rows(bias_ids, "bias_ids", I32, (n, entries), dev)
        dp, (vld, _) = _rows(bias, "bias", F32, (n, entries), dev)
        if n == 1:
            bld = entries
        elif bld != vld:
            raise ValueError("bias_ids and bias must have the same strides")
        if not entries:
            ap = dp = 0
    elif bias_ids is not None or bias is not None:
        raise ValueError("bias_ids and bias go together")
    mp = mr = mld = masks = 0
    if mask is not None:
        wide = mask.shape
        masks, words = wide
        mp, (mld, _) = _rows(mask, "mask", I32, wide, dev)
        if masks == 1:
            mld = words
        if words < (vocab + 31) // 32:
            raise ValueError("the masks have too few words")
        if mask_row is not None:
            mr = _vec(mask_row, "mask_row", I32, row, dev)
    elif mask_row is not None:
        raise ValueError("mask_row without masks")
    return hp, hl, pl, hld, rp, fp, sp, ap, dp, bld, mp, mr, mld, most, entries, masks


def pack_rules(n, vocab, device, **rules):
    """kq_rule_args of a step that has its own logits (kq_paged_step)."""
    f = _rule_fields(n, vocab, device, **rules)
    return _RULES.pack(0, 0, 0, 0, 0, *f[:13], n, vocab, F32, *f[13:])


def logit_rules(logits, out, best=None, hist=None, hist_len=None, prompt_len=None, repetition=None, frequency=None,
                presence=None, bias_ids=None, bias=None, mask=None, mask_row=None, stream=None):
    """Penalties for repeated tokens, biases and grammar masks on logits [n, vocab] (fp32, fp16, bf16), into out
    (may be logits); best [n] int32: the greedy ids (-1 where nothing is allowed). hist [n, most] int32 with
    hist_len [n] tokens in use, of which prompt_len [n] (None: 0) are the prompt; repetition, frequency, presence:
    fp32 [n]; bias_ids int32 and bias fp32 [n, entries] (ids outside the vocabulary are padding; the last entry
    of an id stands); mask int32 or uint32 [masks, >= ceil(vocab / 32)], bit id % 32 of word id / 32 set: allowed;
    mask_row [n]: a mask for each row, -1 for none (None: mask i for row i)."""
    T = _Direct.type
    if type(logits) is not T:
        _Direct.try_type(type(logits))
        T = _Direct.type
    given = (logits, out, best, hist, hist_len, prompt_len, repetition, frequency, presence, bias_ids, bias, mask, mask_row)
    if type(logits) is T:
        ids = []
        for t in given:
            if t is None:
                ids.append(None)
            elif type(t) is T:
                ids.append(id(t))
            else:
                break
        else:
            rc = _Direct.logit_rules(*ids, _Direct.CURRENT if stream is None else stream)
            if not rc:
                return out
            if rc != _Direct.OTHER:
                _bind()[1](rc)
    shape = logits.shape
    n, vocab = shape
    dev, kind = logits.get_device(), _type(logits)
    if dev < 0:
        raise ValueError("the logits must be on a GPU")
    ip, (ild, _) = _rows(logits, "logits", kind, shape, dev)
    op, (old, _) = _rows(out, "out", kind, shape, dev)
    if n == 1:
        ild = old = vocab
    bp = 0 if best is None else _vec(best, "best", I32, (n,), dev)
    fields = _rule_fields(n, vocab, dev, hist, hist_len, prompt_len, repetition, frequency, presence, bias_ids, bias, mask, mask_row)
    if not n:
        return out
    if stream is None:
        stream = current_stream(dev, logits)
    rc = _rules()(_RULES.pack(ip, op, ild, old, bp, *fields[:13], n, vocab, kind, *fields[13:]), dev, stream)
    if rc:
        _bind()[1](rc)
    return out


def check_stream(device=0, stream=None):
    """Waits for the stream (None: as for the operators) and raises ValueError if an operator's kernel met a page id, position, length or row
    index out of range since the last check on this device (such entries are skipped, never read)."""
    lib, check, _ = _bind()
    if stream is None:
        stream = current_stream(device) if lib.kq_device_count() > device else 0
    check(lib.kq_stream_check(device, stream))
