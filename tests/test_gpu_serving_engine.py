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


@pytest.mark.parametrize("kind", ["paged", "batch"])
def test_caches_made_on_a_used_engine_while_the_default_stream_is_busy(env, kind):
    """The zeroing of a new pool is over when the call returns: it cannot erase what the first step stores."""
    K, torch = env
    prompt = [int(v) for v in np.random.default_rng(6).integers(0, CFG["vocab"], 120)]

    def ids(busy):
        e = engine(K, n_layers=1)
        e.feed_batch(prompt[:64], 0)                     # the batched pass's buffers are there
        if busy:
            x = torch.randn((4096, 4096), device="cuda")
            for _ in range(200):                         # some tens of milliseconds
                x = (x @ x).clamp_(-1, 1)
        if kind == "paged":
            e.paged_caches(600, 1024, max_seq=1)
            table = np.array([[599]])
            e.paged_step(table, [0] * 119, prompt[:119], range(119), pick=False)
            got, t = [], prompt[119]
            for i in range(6):
                t = e.paged_step(table, [0], [t], [119 + i])[0]
                got.append(t)
        else:
            e.batch_caches(300)
            e.batch_feed(299, prompt[:119], 0)
            got, t = [], prompt[119]
            for i in range(6):
                t = e.batch_step([299], [t], [119 + i])[0]
                got.append(t)
        torch.cuda.synchronize()
        e.close()
        return got

    assert ids(True) == ids(False)


def test_a_step_reports_its_own_flags_alone(env):
    K, torch = env
    t = dict(dtype=torch.int32, device="cuda")
    e = engine(K, n_layers=1)
    e.paged_caches(4, 16, max_seq=2)
    table = np.arange(4).reshape(2, 2)
    step = (table, [0, 1], [5, 6], [0, 0])
    ids = e.paged_step(*step)
    K.check_stream()
    z = torch.zeros((1, 64), device="cuda")
    K.logit_rules(z, torch.empty_like(z), mask=torch.zeros((1, 2), **t), mask_row=torch.tensor([7], **t))
    assert e.paged_step(*step) == ids                    # another caller's flag is not the step's
    with pytest.raises(ValueError, match="row index"):
        K.check_stream()                                 # and is kept for that caller
    mask = torch.full((1, CFG["vocab"] // 32), -1, **t)
    with pytest.raises(ValueError, match="row index"):
        e.paged_step(*step, rules=dict(mask=mask, mask_row=torch.tensor([0, 3], **t)))
    K.check_stream()                                     # the step's flag was the step's
    assert e.paged_step(*step, rules=dict(mask=mask, mask_row=torch.tensor([0, -1], **t))) == ids
    e.close()
