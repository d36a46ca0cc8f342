"""GPU: the paged K/V cache (PagedCache.append / attend) against plain 64-bit formulas.

Tolerances, derived from the arithmetic include/kq.h states (32-bit sums, one rounding at the end):
  append  a rotated value is two products and a sum in 32 bits (error <= 3 * 2^-24 (|a c| + |b s|)),
          then one division by the scale and one rounding to the type: u |x| with u = 2^-24 (fp32),
          2^-11 (fp16), 2^-8 (bf16), 2^-4 (e4m3), or half the smallest subnormal step.
  attend  a score is a sum of head_dim products: |ds| <= scale (head_dim + 8) 2^-23 sum |q k|, plus 4 ulp for the
          scaling, the maximum's subtraction and the exponential; weights then carry a relative 2 ds
          and the sums over L keys (L + 64) 2^-23, both times the largest |v|. 16-bit outputs may
          take weights of 16 significant bits (2^-16), and their own rounding u |o|."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float8_e4m3fn": 2.0 ** -4}
STEP = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0, "float8_e4m3fn": 2.0 ** -10}   # half a subnormal step


@pytest.fixture(scope="module")
def env():
    import torch
    import kq as K
    assert K.lib().kq_device_count() > 0 and torch.cuda.is_available(), "no GPU"
    return K, torch


def dt(torch, name):
    return getattr(torch, name)


def f64(t):
    """Any tensor as a float64 numpy array."""
    import torch
    return t.to(torch.float32).cpu().numpy().astype(np.float64) if t.dtype != torch.float64 else t.cpu().numpy()


def make_pool(torch, g, n_pages, kv, page, hd, kind, token_major=False):
    """K and V pages with normal values; token_major: pages stored [page][row][head][dim] and viewed head-major."""
    out = []
    for _ in range(2):
        shape = (n_pages, page, kv, hd) if token_major else (n_pages, kv, page, hd)
        x = torch.randn(shape, device="cuda", generator=g)
        x = (x * 24).clamp(-448, 448).to(dt(torch, kind)) if kind == "float8_e4m3fn" else x.to(dt(torch, kind))
        out.append(x.transpose(1, 2) if token_major else x)
    return out


def scales(torch, g, kv, kind):
    if kind != "float8_e4m3fn":
        return None, None
    return tuple(torch.rand(kv, device="cuda", generator=g) * 0.02 + 0.03 for _ in range(2))


def make_table(torch, rng, n, wide, n_pages):
    """Distinct random pages for n rows of `wide` entries."""
    return torch.tensor(rng.permutation(n_pages)[:n * wide].reshape(n, wide).astype(np.int32), device="cuda")


# ----------------------------------------------------------------------------- append
def rope_tables(torch, n_pos, rot):
    inv = 1e6 ** (-2.0 * np.arange(rot // 2) / rot)
    a = np.arange(n_pos)[:, None] * inv[None, :]
    return (torch.tensor(np.cos(a).astype(np.float32), device="cuda"), torch.tensor(np.sin(a).astype(np.float32), device="cuda"))


def turned(x, cos, sin, rot):
    """Rows x [n][h][hd] and the bound on the 32-bit error of each element."""
    y, e = x.copy(), np.zeros_like(x)
    if rot:
        h = rot // 2
        a, b, c, s = x[..., :h], x[..., h:rot], cos[:, None, :], sin[:, None, :]
        y[..., :h], y[..., h:rot] = a * c - b * s, b * c + a * s
        e[..., :h] = 3 * 2.0 ** -24 * (abs(a * c) + abs(b * s))
        e[..., h:rot] = 3 * 2.0 ** -24 * (abs(b * c) + abs(a * s))
    return y, e


def within(got, want, err, kind):
    u, step = U[kind], STEP[kind]
    lim = err + (u + 2.0 ** -23) * (abs(want) + err) + step
    bad = abs(got - want) > lim
    assert not bad.any(), (int(bad.sum()), float(abs(got - want)[bad].max()))


@pytest.mark.parametrize("src,cache,hd,kv,heads,page,rot,n,seqs,token_major", [
    ("float32", "float16", 128, 8, 32, 64, 128, 1, 1, False),
    ("float32", "float16", 128, 2, 6, 16, 128, 130, 3, True),
    ("bfloat16", "bfloat16", 64, 3, 3, 16, 32, 37, 4, False),
    ("float16", "float8_e4m3fn", 128, 4, 0, 32, 128, 65, 65, False),
    ("bfloat16", "float8_e4m3fn", 256, 1, 16, 128, 64, 19, 2, True),
    ("float16", "float16", 256, 4, 28, 1024, 256, 9, 1, False),
    ("float32", "bfloat16", 64, 12, 12, 16, 16, 50, 7, True),
    ("float32", "float8_e4m3fn", 64, 1, 1, 16, 64, 3, 1, False),
    ("float16", "bfloat16", 128, 2, 2, 32, 0, 21, 5, False),
    ("float32", "float16", 128, 2, 6, 16, 64, 5000, 25, False),
    ("bfloat16", "float8_e4m3fn", 128, 8, 17, 16, 128, 5000, 25, True),
])
def test_append(env, src, cache, hd, kv, heads, page, rot, n, seqs, token_major):
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(hd * 7 + n)
    rng = np.random.default_rng(n + page)
    n_pos = 3 * page + 200
    wide = -(-n_pos // page)
    k, v = make_pool(torch, g, seqs * wide + 2, kv, page, hd, cache, token_major)
    ks, vs = scales(torch, g, kv, cache)
    table = make_table(torch, rng, seqs, wide, seqs * wide + 2)
    slots = rng.permutation(seqs * n_pos)[:n]           # distinct (sequence, position) pairs, any order
    seq, pos = (slots // n_pos).astype(np.int32), (slots % n_pos).astype(np.int32)
    pos[n // 2] = -1 if n > 2 else pos[n // 2]          # a padded token
    rows = torch.randn((n, (heads + 2 * kv) * hd), device="cuda", generator=g).to(dt(torch, src))
    q, kn, vn = (t.view(n, -1, hd) for t in rows.split([heads * hd, kv * hd, kv * hd], 1))
    cos, sin = rope_tables(torch, n_pos, rot) if rot else (None, None)
    before = [f64(k), f64(v)]
    mark = torch.full((n, heads, hd), 7.0, device="cuda", dtype=dt(torch, src)) if heads else None
    c = K.PagedCache(k, v, ks, vs)
    c.append(kn, vn, table, torch.tensor(pos, device="cuda"), seq=torch.tensor(seq, device="cuda"),
             rope=(cos, sin) if rot else None, q=q if heads else None, q_out=mark)
    K.check_stream()
    live = pos >= 0
    cs, sn = (f64(cos)[np.maximum(pos, 0)], f64(sin)[np.maximum(pos, 0)]) if rot else (None, None)
    kt, ke = turned(f64(kn), cs, sn, rot)
    pages = table.cpu().numpy()[seq, np.maximum(pos, 0) // page]
    for got, old, want, err, sc in ((k, before[0], kt, ke, ks), (v, before[1], f64(vn), np.zeros_like(f64(vn)), vs)):
        now = f64(got)
        if sc is not None:
            want, err = want / f64(sc)[None, :, None], err / f64(sc)[None, :, None]
            want = np.clip(want, -448, 448)
        new = now[pages, :, pos % page]
        within(new[live], want[live], err[live], cache)
        now[pages[live], :, pos[live] % page] = old[pages[live], :, pos[live] % page]
        assert np.array_equal(now, old)                 # no other row changed
    if heads:
        qt, qe = turned(f64(q), cs, sn, rot)
        within(f64(mark)[live], qt[live], qe[live], src)
        assert (f64(mark)[~live] == 7.0).all()


def test_append_in_place_queries_and_saturation(env):
    K, torch = env
    k = torch.zeros((2, 1, 16, 64), device="cuda").to(torch.float8_e4m3fn)
    v = torch.zeros_like(k)
    one = torch.ones(1, device="cuda")
    c = K.PagedCache(k, v, one, one)
    x = torch.tensor([1e4, -1e4, 448.0, 463.0, 2.0 ** -9, 2.0 ** -11, math.inf, -0.0], device="cuda").repeat(8).view(1, 1, 64)
    q = torch.randn((1, 2, 64), device="cuda")
    q0 = f64(q)
    cos, sin = rope_tables(torch, 5, 64)
    table, pos = torch.ones((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    c.append(x, x, table, pos, rope=(cos, sin), q=q, q_out=q)
    K.check_stream()
    want, err = turned(q0, f64(cos)[4:5], f64(sin)[4:5], 64)
    within(f64(q), want, err, "float32")
    got = f64(v)[1, 0, 4][:8]
    assert got.tolist() == [448.0, -448.0, 448.0, 448.0, 2.0 ** -9, 0.0, 448.0, 0.0]


def test_append_flags_bad_operands_and_stores_nothing(env):
    K, torch = env
    k = torch.zeros((3, 2, 16, 64), device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    c = K.PagedCache(k, v)
    kn = torch.ones((4, 2, 64), device="cuda", dtype=torch.float16)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1], [3, -1]], **i32)
    cases = [([0, 0, 0, 0], [32, 40, 2000000000, 33], "position"), ([2, -1, 5, 9], [0, 1, 2, 3], "row index"),
             ([1, 1, 1, 1], [0, 3, 17, 30], "page id")]
    for seq, pos, text in cases:
        c.append(kn, kn, table, torch.tensor(pos, **i32), seq=torch.tensor(seq, **i32))
        with pytest.raises(ValueError, match=text):
            K.check_stream()
        assert not k.any() and not v.any()
    cos, sin = rope_tables(torch, 5, 64)
    c.append(kn, kn, table, torch.tensor([5, 6, 31, 7], **i32), seq=torch.tensor([0, 0, 0, 0], **i32), rope=(cos, sin))
    with pytest.raises(ValueError, match="position"):
        K.check_stream()
    assert not k.any() and not v.any()
    K.check_stream()                                    # reported once


# ----------------------------------------------------------------------------- attention
def attend_exact(q, k, v, ks, vs, table, lens, page, window, scale):
    """(out, bound on the 32-bit error) in float64; NaN rows of unused page slots never enter."""
    n, heads, hd = q.shape
    kv = k.shape[1]
    G = heads // kv
    out, err = np.zeros(q.shape), np.zeros((n, heads, 1))
    for i in range(n):
        L = int(lens[i])
        t = np.arange(max(0, L - window) if window else 0, L)
        if not len(t):
            continue
        pg = table[i][t // page]
        for g in range(kv):
            kk, vv = k[pg, g, t % page], v[pg, g, t % page]
            if ks is not None:
                kk, vv = kk * ks[g], vv * vs[g]
            qq = q[i, g * G:(g + 1) * G]
            s = scale * (qq @ kk.T)
            ds = abs(scale) * (hd + 8) * 2.0 ** -23 * (abs(qq) @ abs(kk).T).max(1) + 4 * 2.0 ** -23 * abs(s).max(1) + 2.0 ** -21
            p = np.exp(s - s.max(1, keepdims=True))
            out[i, g * G:(g + 1) * G] = (p @ vv) / p.sum(1, keepdims=True)
            err[i, g * G:(g + 1) * G, 0] = abs(vv).max() * (2 * ds + (len(t) + 64) * 2.0 ** -23)
    return out, err


def check_attend(got, want, err, vmax, kind):
    if kind != "float32":
        err = err + 2.0 ** -16 * vmax
    within(got, want, err + np.zeros_like(want), kind)


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 511, 1000]


@pytest.mark.parametrize("qt,cache,hd,kv,G,page,window,token_major", [
    ("float32", "float16", 128, 8, 4, 64, 0, False),
    ("float32", "float16", 128, 2, 1, 16, 0, True),
    ("float16", "float16", 128, 2, 8, 16, 0, False),
    ("float16", "float16", 64, 3, 2, 32, 0, False),
    ("float16", "float16", 256, 2, 4, 32, 0, True),
    ("float32", "float16", 256, 1, 16, 16, 0, False),
    ("float32", "bfloat16", 128, 2, 3, 16, 0, False),
    ("bfloat16", "bfloat16", 128, 1, 7, 128, 0, True),
    ("bfloat16", "bfloat16", 64, 12, 1, 16, 100, False),
    ("float32", "bfloat16", 256, 2, 12, 16, 0, False),
    ("float16", "bfloat16", 64, 2, 4, 16, 0, False),
    ("bfloat16", "float16", 128, 2, 4, 16, 0, False),
    ("float32", "float8_e4m3fn", 128, 2, 4, 16, 0, False),
    ("bfloat16", "float8_e4m3fn", 256, 4, 4, 32, 0, False),
    ("float16", "float8_e4m3fn", 64, 1, 8, 1024, 0, True),
    ("float16", "float8_e4m3fn", 128, 1, 24, 64, 33, False),
    ("float32", "float16", 64, 1, 40, 16, 1, False),
    ("float32", "float16", 128, 2, 9, 16, 17, True),
])
def test_attend(env, qt, cache, hd, kv, G, page, window, token_major):
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(hd + G)
    rng = np.random.default_rng(page + G)
    n = len(LENS)
    wide = -(-max(LENS) // page) + 1
    n_pages = n * wide + 3
    k, v = make_pool(torch, g, n_pages, kv, page, hd, cache, token_major)
    ks, vs = scales(torch, g, kv, cache)
    table = make_table(torch, rng, n, wide, n_pages)
    for i, L in enumerate(LENS):                        # what lies past a sequence's end is garbage
        last = int(table[i, L // page])
        k[last, :, L % page:] = math.nan
        v[last, :, L % page:] = math.nan
        if L // page + 1 < wide:
            table[i, L // page + 1:] = -5 if i % 2 else 1 << 30
    rows = torch.randn((n, kv * G + 3, hd), device="cuda", generator=g) * 2
    q = rows.to(dt(torch, qt))[:, 1:kv * G + 1]         # strided rows
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    out = torch.full((n, kv * G, hd), math.nan, device="cuda", dtype=dt(torch, qt))
    scale = hd ** -0.5
    c = K.PagedCache(k, v, ks, vs)
    c.attend(q, table, lens, out, window=window)
    K.check_stream()
    args = (f64(q), f64(k), f64(v), None if ks is None else f64(ks), None if vs is None else f64(vs), table.cpu().numpy(),
            LENS, page, window, scale)
    want, err = attend_exact(*args)
    vmax = np.nanmax(abs(f64(v))) * (1.0 if vs is None else float(vs.max()))
    got = f64(out)
    assert (got[0] == 0).all()
    check_attend(got, want, err, vmax, qt)
    again = torch.empty_like(out)
    c.attend(q, table, lens, again, window=window)
    assert torch.equal(out, again)                      # equal calls, equal bits


@pytest.mark.parametrize("n,L,kv,G,hd,page,cache", [
    (1, 20011, 2, 4, 128, 16, "float16"), (1, 4096, 8, 4, 128, 64, "float16"), (3, 9001, 1, 1, 64, 32, "bfloat16"),
    (2, 30000, 4, 4, 256, 64, "float8_e4m3fn"), (200, 333, 2, 2, 64, 16, "float16"), (1, 65, 1, 16, 128, 16, "bfloat16"),
])
def test_attend_long_and_many(env, n, L, kv, G, hd, page, cache):
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(L)
    rng = np.random.default_rng(L)
    lens = [max(0, L - 37 * i) for i in range(n)]
    wide = -(-L // page)
    pages = n * wide
    k, v = make_pool(torch, g, pages, kv, page, hd, cache)
    ks, vs = scales(torch, g, kv, cache)
    table = make_table(torch, rng, n, wide, pages)
    q = torch.randn((n, kv * G, hd), device="cuda", generator=g) * 2
    q[0, 0] *= 8                                        # one sharp head
    out = torch.empty_like(q)
    c = K.PagedCache(k, v, ks, vs)
    c.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out)
    K.check_stream()
    want, err = attend_exact(f64(q), f64(k), f64(v), None if ks is None else f64(ks), None if vs is None else f64(vs),
                             table.cpu().numpy(), lens, page, 0, hd ** -0.5)
    check_attend(f64(out), want, err, 0.0, "float32")


def test_attend_shared_pages_seq_rows_and_scale(env):
    """Several tokens on one table row (a prompt chunk: growing lengths), rows in any order, a scale of its own."""
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = make_pool(torch, g, 20, 2, 16, 64, "float16")
    table = torch.tensor([[3, 7, 1, 9], [11, 3, 7, 2]], dtype=torch.int32, device="cuda")   # pages 3 and 7 are shared
    seq, lens = [1, 0, 0, 1, 0], [33, 1, 64, 50, 17]
    q = torch.randn((5, 6, 64), device="cuda", generator=g)
    out = torch.empty_like(q)
    c = K.PagedCache(k, v)
    t = dict(dtype=torch.int32, device="cuda")
    c.attend(q, table, torch.tensor(lens, **t), out, seq=torch.tensor(seq, **t), scale=0.3)
    K.check_stream()
    want, err = attend_exact(f64(q), f64(k), f64(v), None, None, table.cpu().numpy()[seq], lens, 16, 0, 0.3)
    check_attend(f64(out), want, err, 0.0, "float32")


def test_attend_extreme_scores(env):
    """Huge, tiny, equal and infinite scores: no overflow on the way, NaN only where the formula has it."""
    K, torch = env
    k = torch.zeros((4, 1, 16, 64), device="cuda", dtype=torch.float16)
    v = torch.arange(4 * 16 * 64, device="cuda", dtype=torch.float32).view(4, 1, 16, 64).remainder(97).half()
    k[0, 0, 3, 0], k[1, 0, 5, 0], k[2, 0, :, 1] = 60000.0, -60000.0, 6e-8
    k[3, 0, 0, 2] = math.inf
    table = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    q = torch.zeros((1, 8, 64), device="cuda")
    q[0, 0, 0], q[0, 1, 0], q[0, 2, 1], q[0, 3, 0] = 1e30, -1e4, 1e-30, 0.0
    q[0, 4, 0], q[0, 5, 0], q[0, 6, :], q[0, 7, 0] = 3e-5, 65504.0 * 8, 1e-42, math.nan
    out = torch.empty_like(q)
    c = K.PagedCache(k, v)
    c.attend(q, table, torch.tensor([48], dtype=torch.int32, device="cuda"), out)
    K.check_stream()
    kk, vv = f64(k)[:3, 0].reshape(48, 64), f64(v)[:3, 0].reshape(48, 64)
    got = f64(out)[0]
    for h in range(7):
        s = (f64(q)[0, h] @ kk.T) / 8
        p = np.exp(s - s.max())
        assert abs(got[h] - (p @ vv) / p.sum()).max() <= 97 * 2.0 ** -12, h
    assert np.isnan(got[7]).all()
    q[0, :, 2] = torch.tensor([1.0, -1.0] * 4, device="cuda")
    c.attend(q, table, torch.tensor([49], dtype=torch.int32, device="cuda"), out)
    K.check_stream()
    got = f64(out)[0]
    assert np.isnan(got[2]).all()                       # +inf score: inf - inf
    s = (f64(q)[0, 3] @ kk.T) / 8                       # -inf score: that key has no weight
    assert abs(got[3] - (np.exp(s - s.max()) @ vv) / np.exp(s - s.max()).sum()).max() <= 97 * 2.0 ** -12


def test_attend_flags_bad_operands(env):
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = make_pool(torch, g, 6, 1, 16, 128, "float16")
    c = K.PagedCache(k, v)
    t = dict(dtype=torch.int32, device="cuda")
    q = torch.randn((3, 2, 128), device="cuda", generator=g)
    out = torch.empty_like(q)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], **t)

    def want(rows, lens):
        return attend_exact(f64(q), f64(k), f64(v), None, None, rows, lens, 16, 0, 128 ** -0.5)

    c.attend(q, table, torch.tensor([20, 33, -4], **t), out)             # past the table: cut; negative: empty
    with pytest.raises(ValueError, match="length"):
        K.check_stream()
    o, e = want(table.cpu().numpy(), [20, 32, 0])
    check_attend(f64(out), o, e, 0.0, "float32")
    c.attend(q, table, torch.tensor([20, 30, 5], **t), out, seq=torch.tensor([0, 3, -1], **t))
    with pytest.raises(ValueError, match="row index"):
        K.check_stream()
    assert (f64(out)[1:] == 0).all()
    bad = torch.tensor([[6, 1], [2, -1], [7, 8]], **t)
    c.attend(q, bad, torch.tensor([32, 20, 31], **t), out)               # the bad pages' keys are left out
    with pytest.raises(ValueError, match="page id"):
        K.check_stream()
    o, e = attend_exact(f64(q)[:2], f64(k), f64(v), None, None, np.array([[1], [2]]), [16, 16], 16, 0, 128 ** -0.5)
    check_attend(f64(out)[:2], o, e, 0.0, "float32")
    assert (f64(out)[2] == 0).all()
    K.check_stream()


def test_offsets_past_32_bits(env):
    """Pages whose elements lie past 2^31: K and V of 2.2e9 8-bit elements each."""
    K, torch = env
    kv, page, hd = 8, 1024, 128
    pages = 2100
    k = torch.zeros((pages, kv, page, hd), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    v = torch.zeros((pages, kv, page, hd), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    c = K.PagedCache(k, v)
    g = torch.Generator(device="cuda").manual_seed(6)
    t = dict(dtype=torch.int32, device="cuda")
    n = 40
    kn, vn = (torch.randn((n, kv, hd), device="cuda", generator=g) for _ in range(2))
    table = torch.tensor([[pages - 1, 2060, 0]], **t)
    pos = torch.arange(1010, 1010 + n, **t)
    c.append(kn, vn, table, pos, seq=torch.zeros(n, **t))
    q = torch.randn((1, 2 * kv, hd), device="cuda", generator=g)
    out = torch.empty_like(q)
    c.attend(q, table, torch.tensor([1010 + n], **t), out, window=n)
    K.check_stream()
    kk, vv = f64(kn.to(torch.float8_e4m3fn)), f64(vn.to(torch.float8_e4m3fn))
    assert np.array_equal(f64(k[2060, :, :1050 - 1024]), kk[14:].transpose(1, 0, 2))
    o, e = attend_exact(f64(q), kk.reshape(1, n, kv, hd).transpose(0, 2, 1, 3), vv.reshape(1, n, kv, hd).transpose(0, 2, 1, 3),
                        None, None, np.zeros((1, 1), int), [n], n, 0, hd ** -0.5)
    check_attend(f64(out), o, e, 0.0, "float32")


def test_streams_and_graph_capture(env):
    """Enqueued on the caller's stream; a captured step replays with what its buffers then hold."""
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(8)
    k, v = make_pool(torch, g, 40, 2, 16, 128, "float16")
    c = K.PagedCache(k, v)
    t = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(32, **t).view(2, 16)
    pos, lens = torch.tensor([100, 7], **t), torch.tensor([101, 8], **t)
    kn, vn = (torch.randn((2, 2, 128), device="cuda", generator=g) for _ in range(2))
    q = torch.randn((2, 8, 128), device="cuda", generator=g)
    out = torch.zeros_like(q)
    c.append(kn, vn, table, pos)
    c.attend(q, table, lens, out)
    torch.cuda.synchronize()
    first = out.clone()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        c.append(kn, vn, table, pos, stream=s.cuda_stream)
        c.attend(q, table, lens, out, stream=s.cuda_stream)
    kn.normal_(generator=g)
    pos += 1
    lens += 1
    graph.replay()
    torch.cuda.synchronize()
    K.check_stream()
    assert not torch.equal(out, first)
    want, err = attend_exact(f64(q), f64(k), f64(v), None, None, table.cpu().numpy(), [102, 9], 16, 0, 128 ** -0.5)
    check_attend(f64(out), want, err, 0.0, "float32")
    assert torch.equal(k[int(table[1, 0]), :, 8], kn[1].half())


def test_refusals(env):
    K, torch = env
    k, v = (torch.zeros((4, 2, 16, 64), device="cuda", dtype=torch.float16) for _ in range(2))
    c = K.PagedCache(k, v)
    t = dict(dtype=torch.int32, device="cuda")
    table, lens = torch.zeros((2, 2), **t), torch.zeros(2, **t)
    q = torch.zeros((2, 4, 64), device="cuda")
    kn = torch.zeros((2, 2, 64), device="cuda")
    bad_attend = [dict(q=q[:, :3]), dict(q=q.half()), dict(q=q.double()), dict(out=q.transpose(1, 2)), dict(table=table[:1]),
                  dict(table=table.long()), dict(lens=lens[:1]), dict(lens=lens.cpu()), dict(window=-1),
                  dict(q=torch.zeros((2, 4, 65), device="cuda")[:, :, 1:])]
    for kw in bad_attend:
        with pytest.raises(ValueError):
            c.attend(**dict(dict(q=q, table=table, lens=lens, out=torch.empty_like(q)), **kw))
    cos = torch.zeros((8, 16), device="cuda")
    bad_append = [dict(k=kn[:, :1]), dict(v=kn.half()), dict(pos=lens[:1]), dict(rope=(cos, cos[:7])), dict(q=q), dict(q_out=q),
                  dict(rope=(cos[:, :5], cos[:, :5])), dict(rope=(torch.zeros((8, 40), device="cuda"),) * 2), dict(q=q.half(), q_out=q),
                  dict(k=kn.cpu()), dict(seq=lens[:1])]
    for kw in bad_append:
        with pytest.raises(ValueError):
            c.append(**dict(dict(k=kn, v=kn, table=table, pos=lens), **kw))
    empty = torch.zeros((0, 2, 64), device="cuda")
    c.append(empty, empty, table, torch.zeros(0, **t))                   # no token: nothing to do
    c.attend(q[:0], table, lens[:0], q[:0].clone())
    c.close()
    with pytest.raises(ValueError):
        c.attend(q, table, lens, torch.empty_like(q))
    K.check_stream()


def test_both_ways_of_passing_tensors_agree(env, monkeypatch):
    """The short way (DLPack descriptions read by the library) and the checks in Python make the same call."""
    K, torch = env
    from kq import serve
    g = torch.Generator(device="cuda").manual_seed(9)
    t = dict(dtype=torch.int32, device="cuda")
    for n, kv, G in ((1, 1, 1), (1, 2, 3), (5, 1, 4), (4, 3, 1)):
        rows = torch.randn((n, 2 * kv + kv * G + 1, 64), device="cuda", generator=g)
        kn, vn, q = rows[:, :kv], rows[:, kv:2 * kv], rows[:, 2 * kv:2 * kv + kv * G]
        big = torch.arange(40, **t).view(5, 8)
        table, seq = big[:n, 1:5], torch.arange(n, **t).flip(0).contiguous()
        pos = torch.tensor([3 + 11 * i for i in range(n)], **t)
        cos, sin = rope_tables(torch, 64, 32)
        got = []
        for direct in (True, False):
            monkeypatch.setattr(serve._Direct, "type", torch.Tensor if direct else None)
            monkeypatch.setattr(serve._Direct, "_tried", {torch.Tensor})
            k, v = (torch.zeros((40, kv, 16, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2))
            c = K.PagedCache(k, v)
            qo, out = torch.zeros_like(q), torch.zeros_like(q)
            c.append(kn, vn, table, pos, seq=seq, rope=(cos, sin), q=q, q_out=qo)
            c.attend(qo, table, pos + 1, out, seq=seq, window=9, scale=0.2)
            z, best = torch.zeros((n, 64), device="cuda"), torch.zeros(n, **t)
            K.logit_rules(rows[:, 0], z, best=best, hist=big[:n], hist_len=pos.clamp(max=8), prompt_len=seq, presence=z[:, 0] + 1,
                          bias_ids=big[:n, :3], bias=torch.ones((n, 8), device="cuda")[:, :3],
                          mask=big, mask_row=seq)
            K.check_stream()
            got.append((k, v, qo, out, z, best))
        for a, b in zip(*got):
            assert torch.equal(a, b)


def test_many_handles_and_streams(env):
    """Handles that come and go, on streams of their own that do not wait for the default one."""
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(10)
    k, v = make_pool(torch, g, 64, 2, 16, 128, "float16")
    t = dict(dtype=torch.int32, device="cuda")
    table, lens = torch.arange(64, **t).view(1, 64), torch.tensor([1000], **t)
    q = torch.randn((1, 8, 128), device="cuda", generator=g)
    want, err = attend_exact(f64(q), f64(k), f64(v), None, None, table.cpu().numpy(), [1000], 16, 0, 128 ** -0.5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(6)]
    for _ in range(3):
        caches = [K.PagedCache(k, v) for _ in streams]
        outs = [torch.empty_like(q) for _ in streams]
        torch.cuda.synchronize()
        for _ in range(4):
            for c, o, s in zip(caches, outs, streams):
                c.attend(q, table, lens, o, stream=s.cuda_stream)
        for s in streams:
            K.check_stream(stream=s.cuda_stream)
        for o in outs:
            check_attend(f64(o), want, err, 0.0, "float32")
            assert torch.equal(o, outs[0])
        for c in caches:
            c.close()
