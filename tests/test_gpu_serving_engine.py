"""GPU: what paged and batched steps must hold beside their ids (tests/test_gpu_paged_engine.py): more rows than the
context has positions, pools made while other work is queued, refusals and flags of a step of its own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

CFG = dict(dim=1024, n_heads=8, n_kv_heads=2, head_dim=128, ffn=2048, vocab=4096)


@pytest.fixture(scope="module")
def env():
    import torch
    import kq as K
    assert K.lib().kq_device_count() > 0 and torch.cuda.is_available(), "no GPU"
    return K, torch


def engine(kq, ctx=512, n_layers=2):
    return kq.Engine(kq.Config.default(ctx=ctx, n_layers=n_layers, **CFG), seed=0)


def test_more_sequences_than_positions(env):
    """100 rows in contexts of 16: the ids of a step have room of their own."""
    K, _ = env
    toks = [int(v) for v in np.random.default_rng(4).integers(0, CFG["vocab"], 200)]
    got = []
    for ctx in (16, 512):
        e = engine(K, ctx)
        e.paged_caches(100, 16, max_seq=100)
        e.batch_caches(100)
        table, seqs = np.arange(100).reshape(100, 1), list(range(100))
        ids = [e.paged_step(table, seqs, toks[:100], [0] * 100), e.paged_step(table, seqs, toks[100:], [1] * 100)]
        one = [e.batch_step(seqs, toks[:100], [0] * 100), e.batch_step(seqs, toks[100:], [1] * 100)]
        got.append((ids, one))                           # the two paths round differently: each against itself
        e.close()
    assert got[0] == got[1]
