"""GPU: kq.logit_rules with bias lists longer than a block keeps (512 entries of its ids): the same formula and tolerances
as tests/test_gpu_rules.py, and a time that does not grow with the square of the length."""
import numpy as np
import pytest

from test_gpu_rules import check_row, env, exact, unpack  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,n,V,entries,most,inplace", [
    ("float32", 2, 151936, 20000, 500, False),           # nearly all ids distinct
    ("float32", 3, 700, 5000, 100, True),                # every id many times
    ("bfloat16", 2, 32003, 32003, 900, True),            # an entry for every id of the vocabulary, in any order
    ("float16", 4, 9001, 1500, 0, False),
    ("float32", 2, 40000, 9000, 30000, False),           # a history that is scanned in parts
    ("float32", 1, 5, 3000, 3, False),
])
def test_long_lists(env, kind, n, V, entries, most, inplace):
    K, torch = env
    rng = np.random.default_rng(V + entries)
    z = torch.tensor(rng.normal(0, 3, (n, V)).astype(np.float32), device="cuda").to(getattr(torch, kind))
    z0 = z.float().cpu().numpy()
    ids = np.stack([rng.permutation(V) for _ in range(n)]).astype(np.int32) if entries == V else rng.integers(-1, V, (n, entries)).astype(np.int32)
    bias = rng.normal(0, 4, (n, entries)).astype(np.float32)
    hist = rng.integers(0, V, (n, max(most, 1))).astype(np.int32)
    length = rng.integers(0, most + 1, n).astype(np.int32)
    length[0] = most
    mask = rng.integers(0, 2 ** 32, (n, (V + 31) // 32), dtype=np.uint64).astype(np.uint32) | 1
    cu = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    one, best = torch.ones(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    out = z if inplace else torch.empty_like(z)
    K.logit_rules(z, out, best=best, hist=cu(hist), hist_len=cu(length), prompt_len=cu(length // 2), repetition=1.25 * one,
                  frequency=0.5 * one, presence=0.25 * one, bias_ids=cu(ids), bias=cu(bias), mask=cu(mask.view(np.int32)))
    K.check_stream()
    got, top, allowed = out.float().cpu().numpy().astype(np.float64), best.cpu().numpy(), unpack(mask, V)
    for i in range(n):
        want, mag = exact(z0[i], hist[i, :length[i]], int(length[i] // 2), 1.25, 0.5, 0.25, ids[i], bias[i], allowed[i])
        check_row(got[i], int(top[i]), want, mag, kind)


def test_time_of_long_lists(env):
    """16 rows with an entry for every one of 150 000 ids: 300 rounds of a few microseconds, where a walk through the list for
    each id would take seconds."""
    K, torch = env
    n, V = 16, 150000
    z = torch.randn((n, V), device="cuda")
    ids = torch.stack([torch.randperm(V, device="cuda") for _ in range(n)]).int()
    bias, out = torch.randn((n, V), device="cuda"), torch.empty_like(z)
    K.logit_rules(z, out, bias_ids=ids, bias=bias)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    K.logit_rules(z, out, bias_ids=ids, bias=bias)
    b.record()
    K.check_stream()
    assert torch.equal(out, z + torch.zeros_like(z).scatter_(1, ids.long(), bias))
    assert a.elapsed_time(b) < 50
