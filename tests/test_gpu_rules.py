"""GPU: kq.logit_rules against the plain formula in 64 bits.

Tolerance: a touched logit sees at most one division or product, two products, two sums and a bias,
each rounded once in 32 bits, so its error is below 6 * 2^-24 times the sum of the magnitudes that
enter; then one rounding to the type. An untouched logit is exact. The greedy id is checked against
the returned row itself (lowest id of the largest value), the rows within the tolerance."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def env():
    import torch
    import kq as K
    assert K.lib().kq_device_count() > 0 and torch.cuda.is_available(), "no GPU"
    return K, torch


def exact(z, hist, prompt, rep, freq, pres, ids, bias, allowed):
    """One row in float64: (values, magnitude that entered each)."""
    z = z.astype(np.float64).copy()
    mag = np.zeros_like(z)
    V = len(z)
    hist = np.asarray(hist)
    ok = (hist >= 0) & (hist < V)
    seen = np.unique(hist[ok])
    late = np.asarray(hist[prompt:])[ok[prompt:]]
    z[seen] = np.where(z[seen] > 0, z[seen] / rep, z[seen] * rep)
    mag[seen] += abs(z[seen])
    ul, cl = np.unique(late, return_counts=True)
    mag[ul] += abs(z[ul]) + abs(freq) * cl + abs(pres)
    z[ul] -= freq * cl + pres
    last = {int(a): float(b) for a, b in zip(ids, bias) if 0 <= a < V}
    for a, b in last.items():
        mag[a] += abs(z[a]) + abs(b)
        z[a] += b
    if allowed is not None:
        z[~allowed] = -math.inf
        mag[~allowed] = 0
    return z, mag


def unpack(mask, V):
    return np.unpackbits(mask.view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)


def check_row(got, best, want, mag, kind):
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and (got[inf] == want[inf]).all()
    w, m = want[~inf], mag[~inf]
    lim = 6 * 2.0 ** -24 * m + U[kind] * (abs(w) + 6 * 2.0 ** -24 * m) + (2.0 ** -25 if kind == "float16" else 0)
    if kind == "float32":
        lim = lim + np.where(m > 0, 2.0 ** -24 * abs(w), 0)
    bad = abs(got[~inf] - w) > lim
    assert not bad.any(), (int(bad.sum()), float(abs(got[~inf] - w)[bad].max()))
    top = int(np.argmax(got))
    assert best == (top if got[top] > -math.inf else -1)


@pytest.mark.parametrize("kind,n,V,most,entries,masks,ld,inplace", [
    ("float32", 1, 151936, 700, 5, 1, 0, False),
    ("float32", 5, 4096, 300, 20, 5, 0, True),
    ("float32", 3, 31, 64, 3, 3, 1, False),
    ("float32", 2, 1, 9, 2, 2, 0, False),
    ("float32", 9, 32003, 5000, 300, 4, 5, False),
    ("float32", 4, 1000, 1, 0, 0, 0, False),
    ("bfloat16", 7, 32003, 900, 31, 7, 0, False),
    ("float16", 6, 5001, 400, 7, 2, 3, True),
    ("bfloat16", 3, 393216, 2000, 50, 3, 0, False),
    ("float16", 2, 65537, 0, 0, 2, 0, False),
    ("float32", 1, 393216, 20000, 10, 1, 0, False),
])
def test_rules(env, kind, n, V, most, entries, masks, ld, inplace):
    K, torch = env
    rng = np.random.default_rng(V + n)
    dtype = getattr(torch, kind)
    base = torch.tensor(rng.normal(0, 3, (n, V + ld)).astype(np.float32), device="cuda").to(dtype)
    logits = base[:, :V]
    z0 = logits.float().cpu().numpy()
    hist = (rng.random((n, most + 3)) ** 4 * V).astype(np.int32)
    if most > 20:
        hist[:, 5], hist[:, 11], hist[:, 17] = -1, V, 2 ** 31 - 1          # padding in the middle
    hist_len = rng.integers(0, most + 1, n).astype(np.int32)
    hist_len[0] = most
    prompt = (hist_len * rng.random(n)).astype(np.int32)
    ids = rng.integers(0, V, (n, entries)).astype(np.int32)                 # repeated ids: the last one stands
    if entries > 4:
        ids[:, 1], ids[:, 2], ids[:, 4] = ids[:, 0], -1, V + 7
    bias = rng.normal(0, 4, (n, entries)).astype(np.float32)
    words = (V + 31) // 32 + 1
    mask = rng.integers(0, 2 ** 32, (max(masks, 1), words), dtype=np.uint64).astype(np.uint32)
    mask[0] |= 1
    row = rng.integers(-1, max(masks, 1), n).astype(np.int32)
    if masks > 1:
        mask[1] = 0                                                         # allows nothing
        row[n - 1] = 1
    rep, freq, pres = (rng.random(n).astype(np.float32) * s + o for s, o in ((0.5, 1), (0.5, 0), (1, -0.3)))
    rep, freq, pres = (x.astype(np.float32) for x in (rep, freq, pres))
    cu = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    out = logits if inplace else torch.full_like(base, 5.0)[:, :V]
    best = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    kw = dict(best=best, repetition=cu(rep), frequency=cu(freq), presence=cu(pres))
    kw.update(hist=cu(hist)[:, :most], hist_len=cu(hist_len), prompt_len=cu(prompt))
    if entries:
        kw.update(bias_ids=cu(ids), bias=cu(bias))
    if masks:
        kw.update(mask=cu(mask.view(np.int32)), mask_row=cu(row))
    K.logit_rules(logits, out, **kw)
    K.check_stream()
    got, ids_got = out.float().cpu().numpy().astype(np.float64), best.cpu().numpy()
    allowed = unpack(mask, V) if masks else None
    for i in range(n):
        a = allowed[row[i]] if masks and row[i] >= 0 else None
        want, mag = exact(z0[i], hist[i, :hist_len[i]], int(prompt[i]), float(rep[i]), float(freq[i]), float(pres[i]), ids[i],
                          bias[i], a)
        check_row(got[i], int(ids_got[i]), want, mag, kind)
    if ld and not inplace:
        tail = torch.as_strided(out, (n, ld), (V + ld, 1), V)
        assert (tail.float() == 5.0).all()                                  # nothing past a row is written


def test_absent_rules_copy_and_pick(env):
    K, torch = env
    z = torch.randn((3, 777), device="cuda")
    z[0, 300] = z[0, 40] = 9.0                                              # a tie: the lowest id
    z[1] = -math.inf
    z[2, 5], z[2, 6], z[2, 7] = math.nan, math.inf, math.inf
    out, best = torch.empty_like(z), torch.zeros(3, dtype=torch.int32, device="cuda")
    K.logit_rules(z, out, best=best)
    K.check_stream()
    assert np.array_equal(out.cpu().numpy(), z.cpu().numpy(), equal_nan=True)
    assert best.tolist() == [40, -1, 6]
    K.logit_rules(z, out)                                                   # without ids
    K.check_stream()


def test_lowest_values_and_infinite_biases(env):
    """The type's lowest value is a value like any other; an infinite bias forbids or forces."""
    K, torch = env
    low = torch.finfo(torch.float32).min
    z = torch.full((2, 50), low, device="cuda")
    z[1, 7] = 3.0
    ids = torch.tensor([[4], [7]], dtype=torch.int32, device="cuda")
    bias = torch.tensor([[math.inf], [-math.inf]], device="cuda")
    out, best = torch.empty_like(z), torch.zeros(2, dtype=torch.int32, device="cuda")
    K.logit_rules(z, out, best=best, bias_ids=ids, bias=bias)
    K.check_stream()
    assert best.tolist() == [4, 0] and float(out[0, 4]) == math.inf and float(out[1, 7]) == -math.inf
    assert float(out[1, 0]) == low


def test_lengths_are_cut_and_bad_mask_rows_allow_nothing(env):
    K, torch = env
    t = dict(dtype=torch.int32, device="cuda")
    z = torch.randn((3, 100), device="cuda")
    out, best = torch.empty_like(z), torch.zeros(3, **t)
    hist = torch.tensor([[1, 2, 3, 2]] * 3, **t)
    one = torch.ones(3, device="cuda")
    K.logit_rules(z, out, best=best, hist=hist, hist_len=torch.tensor([100, -3, 2], **t), prompt_len=torch.tensor([9, -1, -5], **t),
                  frequency=one, repetition=2 * one)
    K.check_stream()
    for i, (h, p) in enumerate((([1, 2, 3, 2], 4), ([], 0), ([1, 2], 0))):
        want, mag = exact(z[i].cpu().numpy(), np.array(h, int), p, 2.0, 1.0, 0.0, [], [], None)
        check_row(out[i].cpu().numpy().astype(np.float64), int(best[i]), want, mag, "float32")
    mask = torch.full((2, 4), -1, **t)
    K.logit_rules(z, out, best=best, mask=mask, mask_row=torch.tensor([2, 0, -2], **t))
    with pytest.raises(ValueError, match="row index"):
        K.check_stream()
    assert best.tolist()[0] == -1 and best.tolist()[2] == -1 and best.tolist()[1] == int(z[1].argmax())
    assert (out[0] == -math.inf).all() and torch.equal(out[1], z[1])
    K.check_stream()


def test_rules_refusals(env):
    K, torch = env
    z = torch.zeros((2, 64), device="cuda")
    for kw in (dict(best=torch.zeros(2, device="cuda")), dict(mask=torch.zeros((2, 1), dtype=torch.int32, device="cuda")),
               dict(hist=torch.zeros((2, 3), dtype=torch.int32, device="cuda")), dict(repetition=torch.ones(3, device="cuda")),
               dict(mask=torch.zeros((1, 2), dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            K.logit_rules(z, torch.empty_like(z), **kw)
    with pytest.raises(ValueError):
        K.logit_rules(z.cpu(), z)
    with pytest.raises(ValueError):
        K.logit_rules(z.t(), z.t())
    with pytest.raises(ValueError):
        K.logit_rules(z.double(), z.double())
    K.logit_rules(z[:0], z[:0].clone())
    K.check_stream()


@pytest.mark.parametrize("kind,V,ld", [("bfloat16", 20011, 1), ("float16", 9001, 3), ("float32", 5003, 2), ("bfloat16", 40000, 0)])
def test_equal_maxima_take_the_lowest_id(env, kind, V, ld):
    """Ties between ids anywhere in a row: its ends, its touched ids, ids of other CTAs, masked ones."""
    K, torch = env
    rng = np.random.default_rng(V)
    n = 24
    z = torch.tensor(rng.normal(0, 1, (n, V + ld)).astype(np.float32), device="cuda").to(getattr(torch, kind))[:, :V]
    want, hist, mask = [], np.full((n, 3), -1, np.int32), np.full((n, (V + 31) // 32), 0xffffffff, np.uint32)
    for i in range(n):
        ids = np.sort(rng.choice(V, 5, replace=False))
        if i % 4 == 0:
            ids[0] = i % 8
        if i % 4 == 1:
            ids[1:] = np.sort(V - 1 - rng.choice(20, 4, replace=False))
        z[i, torch.tensor(ids, device="cuda")] = 16.0
        hist[i, :2] = ids[:2] if i % 3 else ids[3:]     # touched, by rules that change nothing
        if i % 5 == 4:                                  # the lowest is masked
            mask[i, ids[0] // 32] &= ~np.uint32(1 << (ids[0] % 32))
            ids = ids[1:]
        want.append(int(ids[0]))
    cu = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    best = torch.zeros(n, dtype=torch.int32, device="cuda")
    K.logit_rules(z, torch.empty((n, V + ld), dtype=z.dtype, device="cuda")[:, :V], best=best, hist=cu(hist),
                  hist_len=torch.full((n,), 3, dtype=torch.int32, device="cuda"), repetition=torch.ones(n, device="cuda"),
                  mask=cu(mask.view(np.int32)))
    K.check_stream()
    assert best.tolist() == want


def test_long_histories_and_lists(env):
    """Histories past 16-bit counts and past what every CTA scans, more touched ids and biases than a CTA lists."""
    K, torch = env
    rng = np.random.default_rng(5)
    V, n, most, entries = 50021, 3, 40000, 3000
    z = torch.tensor(rng.normal(0, 3, (n, V)).astype(np.float32), device="cuda")
    hist = rng.integers(0, V, (n, most)).astype(np.int32)
    hist[0, :] = 77                                     # 40000 times one id
    hist_len = np.array([most, most, 16384], np.int32)
    prompt = np.array([0, 20000, 100], np.int32)
    ids = rng.integers(0, V, (n, entries)).astype(np.int32)
    bias = rng.normal(0, 4, (n, entries)).astype(np.float32)
    cu = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    one = torch.ones(n, device="cuda")
    out, best = torch.empty_like(z), torch.zeros(n, dtype=torch.int32, device="cuda")
    K.logit_rules(z, out, best=best, hist=cu(hist), hist_len=cu(hist_len), prompt_len=cu(prompt), repetition=1.25 * one,
                  frequency=0.5 * one, presence=0.25 * one, bias_ids=cu(ids), bias=cu(bias))
    K.check_stream()
    for i in range(n):
        want, mag = exact(z[i].cpu().numpy(), hist[i, :hist_len[i]], int(prompt[i]), 1.25, 0.5, 0.25, ids[i], bias[i], None)
        check_row(out[i].cpu().numpy().astype(np.float64), int(best[i]), want, mag, "float32")


def test_captured_and_on_a_stream_of_its_own(env):
    K, torch = env
    z = torch.randn((3, 70001), device="cuda")
    out, best = torch.empty_like(z), torch.zeros(3, dtype=torch.int32, device="cuda")
    ids = torch.tensor([[5], [70000], [-1]], dtype=torch.int32, device="cuda")
    bias = torch.full((3, 1), 50.0, device="cuda")
    K.logit_rules(z, out, best=best, bias_ids=ids, bias=bias)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        K.logit_rules(z, out, best=best, bias_ids=ids, bias=bias, stream=s.cuda_stream)
        K.logit_rules(out, out, best=best, bias_ids=ids, bias=bias, stream=s.cuda_stream)
    z.normal_()
    graph.replay()
    torch.cuda.synchronize()
    assert best.tolist() == [5, 70000, int(z[2].argmax())]
    assert float(out[0, 5]) == float(z[0, 5] + 50.0 + 50.0) and torch.equal(out[2], z[2])
    K.check_stream()
