"""GPU: kq.logit_rules where logits and output rows start at different places of a 16-byte group (an odd vocabulary into a
padded output, a shifted view): the same formula and tolerances as tests/test_gpu_rules.py."""
import numpy as np
import pytest

from test_gpu_rules import check_row, env, exact, unpack  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,n,V,in_ld,in_at,out_ld,out_at", [
    ("float32", 3, 32003, 32003, 0, 32004, 0), ("float32", 2, 5, 7, 2, 9, 1), ("bfloat16", 5, 32003, 32003, 0, 32008, 0),
    ("float16", 4, 9001, 9005, 3, 9001, 0), ("bfloat16", 2, 65537, 65540, 1, 65537, 7), ("float32", 1, 40000, 40001, 1, 40000, 0),
    ("bfloat16", 9, 3, 3, 0, 8, 5),
])
def test_unlike_alignments(env, kind, n, V, in_ld, in_at, out_ld, out_at):
    K, torch = env
    rng = np.random.default_rng(V + in_ld + out_ld)
    dtype = getattr(torch, kind)

    def rows(ld, at, fill):
        base = torch.full((n * ld + 16,), fill, device="cuda", dtype=dtype)
        return base, torch.as_strided(base, (n, V), (ld, 1), at)

    _, z = rows(in_ld, in_at, 50.0)                      # what lies between the rows would win
    z.copy_(torch.tensor(rng.normal(0, 3, (n, V)).astype(np.float32), device="cuda"))
    base, out = rows(out_ld, out_at, 5.0)
    z0 = z.float().cpu().numpy()
    hist = rng.integers(0, V, (n, 200)).astype(np.int32)
    length = rng.integers(0, 201, n).astype(np.int32)
    prompt = length // 3
    ids = rng.integers(-1, V, (n, 9)).astype(np.int32)
    bias = rng.normal(0, 4, (n, 9)).astype(np.float32)
    mask = rng.integers(0, 2 ** 32, (n, (V + 31) // 32), dtype=np.uint64).astype(np.uint32)
    cu = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    one, best = torch.ones(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    K.logit_rules(z, out, best=best, hist=cu(hist), hist_len=cu(length), prompt_len=cu(prompt), repetition=1.5 * one,
                  frequency=0.25 * one, presence=0.125 * one, bias_ids=cu(ids), bias=cu(bias), mask=cu(mask.view(np.int32)))
    K.check_stream()
    got, top = out.float().cpu().numpy().astype(np.float64), best.cpu().numpy()
    allowed = unpack(mask, V)
    for i in range(n):
        want, mag = exact(z0[i], hist[i, :length[i]], int(prompt[i]), 1.5, 0.25, 0.125, ids[i], bias[i], allowed[i])
        check_row(got[i], int(top[i]), want, mag, kind)
    out.fill_(5.0)
    assert (base.float() == 5.0).all()                   # nothing beside the rows was written
