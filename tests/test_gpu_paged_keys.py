"""GPU: which keys the paged attention counts, and how closely, in limits that one missing key or one rounding too many
would pass. (The worst-case limits of tests/test_gpu_paged.py grow with the length and cannot see either.)

  counting  queries of zeros weigh all keys alike and V marks a key by a one in a single dim, so an output times the
            length is a number of keys: whole to L * 2^-23 or so in 32 bits, and 0.25 is far from both sides.
  accuracy  errors of unit normal data are independent from key to key, so the root mean square of the output's error
            over that of the output is that of a score: fp32 queries are taken in 22 bits or more (2^-22 of scores of
            about 2), the sums of head_dim products and the exponential add a few 2^-23: below 2^-19 in all. A lost
            step of 16 keys in 20 000 moves it by 2^-5, queries rounded to fp16 by 2^-10."""
import numpy as np
import pytest

from test_gpu_paged import attend_exact, env, f64, make_pool, make_table, scales  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [  # queries, cache, head_dim, K/V heads, group, page
    ("float32", "float16", 128, 8, 4, 64), ("float32", "float16", 64, 2, 12, 16), ("float32", "float16", 256, 2, 8, 32),
    ("float32", "bfloat16", 128, 2, 7, 16), ("float32", "bfloat16", 256, 1, 16, 64), ("float32", "float8_e4m3fn", 128, 2, 4, 32),
    ("float32", "float8_e4m3fn", 256, 2, 3, 16), ("float32", "float8_e4m3fn", 64, 1, 1, 128), ("float16", "float16", 128, 4, 4, 16),
    ("bfloat16", "bfloat16", 64, 12, 1, 16), ("float16", "float8_e4m3fn", 256, 4, 4, 64), ("float16", "bfloat16", 64, 1, 9, 16),
]


def lengths(n, most, seed):
    rng = np.random.default_rng(seed)
    return [0, 1, most] + [int(v) for v in np.exp(rng.uniform(0, np.log(most), n - 3))]


@pytest.mark.parametrize("n,most,window", [(4, 20011, 0), (150, 700, 0), (37, 5001, 500), (9, 3000, 0)])
@pytest.mark.parametrize("qt,cache,hd,kv,G,page", SHAPES)
def test_every_key_counts_once(env, qt, cache, hd, kv, G, page, n, most, window):
    K, torch = env
    rng = np.random.default_rng(most + hd)
    lens = lengths(n, most, n)
    each = [-(-v // page) for v in lens]
    wide = max(each)
    pages = sum(each) + 1
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((n, wide), -1, np.int32)
    table[np.arange(wide)[None, :] < np.array(each)[:, None]] = order[:sum(each)]
    kind = getattr(torch, cache)
    k = torch.zeros((pages, kv, page, hd), device="cuda").to(kind)
    c, q = None, torch.zeros((n, kv * G, hd), device="cuda", dtype=getattr(torch, qt))
    for step in (16, 1):                                 # a dim for each 16 keys; for each key
        mark = np.zeros((pages, page, hd), np.float32)
        for i, L in enumerate(lens):
            t = np.arange(L)
            mark[table[i][t // page], t % page, t // step % hd] = 1.0
        v = torch.tensor(mark, device="cuda").to(kind)[:, None].expand(-1, kv, -1, -1).contiguous()
        c = K.PagedCache(k, v)
        out = c.attend(q, torch.tensor(table, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.empty_like(q),
                       window=window)
        K.check_stream()
        got = f64(out)
        for i, L in enumerate(lens):
            t = np.arange(max(0, L - window) if window else 0, L)
            want = np.bincount(t // step % hd, minlength=hd).astype(float)
            slack = 0.25 if qt == "float32" else 0.25 + want * 2.0 ** (-10 if qt == "float16" else -7)
            assert (abs(got[i] * max(len(t), 1) - want) <= slack).all(), (i, L, step)


@pytest.mark.parametrize("qt,cache,hd,kv,G,page", [s for s in SHAPES if s[0] == "float32"])
@pytest.mark.parametrize("lens", [[20011], [4096, 300, 64, 17], [997] * 40])
def test_accuracy_of_fp32_queries(env, qt, cache, hd, kv, G, page, lens):
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(hd + G + len(lens))
    rng = np.random.default_rng(hd + len(lens))
    n, wide = len(lens), -(-max(lens) // page)
    k, v = make_pool(torch, g, n * wide, kv, page, hd, cache)
    ks, vs = scales(torch, g, kv, cache)
    table = make_table(torch, rng, n, wide, n * wide)
    q = torch.randn((n, kv * G, hd), device="cuda", generator=g) * 2
    out = K.PagedCache(k, v, ks, vs).attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.empty_like(q))
    K.check_stream()
    want, _ = attend_exact(f64(q), f64(k), f64(v), None if ks is None else f64(ks), None if vs is None else f64(vs),
                           table.cpu().numpy(), lens, page, 0, hd ** -0.5)
    error = ((f64(out) - want) ** 2).mean((1, 2)) ** 0.5 / (want ** 2).mean((1, 2)) ** 0.5
    assert (error < 2.0 ** -19).all(), error.max()


@pytest.mark.parametrize("qt,cache,hd,kv,G,page", SHAPES[:4] + SHAPES[-3:])
def test_output_in_the_queries_place(env, qt, cache, hd, kv, G, page):
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(hd)
    rng = np.random.default_rng(hd)
    lens = lengths(20, 3000, 5)
    n, wide = len(lens), -(-3000 // page)
    k, v = make_pool(torch, g, n * wide, kv, page, hd, cache)
    ks, vs = scales(torch, g, kv, cache)
    table, lens = make_table(torch, rng, n, wide, n * wide), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((n, kv * G, hd), device="cuda", generator=g).to(getattr(torch, qt))
    c = K.PagedCache(k, v, ks, vs)
    apart = c.attend(q, table, lens, torch.empty_like(q))
    c.attend(q, table, lens, q)
    K.check_stream()
    assert torch.equal(q, apart)
