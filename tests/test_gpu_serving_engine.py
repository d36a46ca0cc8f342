"""GPU: what paged and batched steps must hold beside their ids (tests/test_gpu_paged_engine.py): more rows than the
context has positions, pools made while other work is queued, refusals and flags of a step of its own.

The generated weights give scores of some hundreds, so each token attends to itself alone and no result depends on
the cache. Engines of mixing() take smaller query weights: scores of about one, attention over the whole context."""
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


def small_q4k(rows, cols, std, seed):
    """GGUF Q4_K rows of weights d (q - 7.5), q uniform in 0 .. 15: every sub-block's scale and minimum are 1."""
    rng = np.random.default_rng(seed)
    b = np.zeros((rows * cols // 256, 144), np.uint8)
    b[:, 0:2] = np.float16(std / 4.61).reshape(1).view(np.uint8)
    b[:, 2:4] = np.float16(7.5 * std / 4.61).reshape(1).view(np.uint8)
    b[:, 4:12], b[:, 12:16] = 1, 0x11
    b[:, 16:] = rng.integers(0, 256, (len(b), 128))
    return b.reshape(-1)


def mixing(kq, ctx=512, n_layers=2):
    e = engine(kq, ctx, n_layers)
    for l in range(n_layers):
        e.set_tensor(l, kq.T_Q, small_q4k(CFG["n_heads"] * CFG["head_dim"], CFG["dim"], 0.005, l))
    return e


def ranking(torch, e, table, seq, tok, pos, n):
    """The n best ids of one paged step in their order: each time the ones before are masked."""
    allowed = torch.ones(CFG["vocab"], dtype=torch.int64, device="cuda")
    bits, order = torch.arange(32, device="cuda"), []
    for _ in range(n):
        words = (allowed.view(-1, 32) << bits).sum(1).to(torch.uint32).view(torch.int32)
        order += e.paged_step(table, [seq], [tok], [pos], rules=dict(mask=words[None]))
        allowed[order[-1]] = 0
    return order


def test_paged_steps_that_depend_on_their_context(env):
    """The 12 best ids of a step after prompts fed in mixed chunks, against the logits of each prompt alone. K and V are
    rounded to fp16 by both paths (2^-11) and may round apart where the projections differ in their last bits; the
    logits are sums over many of them, so 2^-9 of their spread is a wide limit, and another context must pass it far."""
    K, torch = env
    rng = np.random.default_rng(31)
    prompts = [[int(v) for v in rng.integers(0, CFG["vocab"], n)] for n in (37, 150, 5, 90)]
    one = mixing(K)
    logits = []
    for p in prompts:
        one.reset()
        one.feed_batch(p[:-1], 0)
        one.step(p[-1], len(p) - 1)
        logits.append(one.ylog.astype(np.float64))
    one.reset()
    one.feed_batch([(t + 1) % CFG["vocab"] for t in prompts[1][:-1]], 0)
    one.step(prompts[1][-1], len(prompts[1]) - 1)
    limit = 2.0 ** -9 * logits[1].std()
    assert abs(one.ylog - logits[1]).max() > 20 * limit
    one.close()
    e = mixing(K)
    e.paged_caches(40, 16, max_seq=4)
    table = rng.permutation(40).reshape(4, 10)
    todo = [(s, t, i) for i in range(150) for s, p in enumerate(prompts) for t in p[i:i + 1] if i < len(p) - 1]
    for a in range(0, len(todo), 77):
        s, t, i = zip(*todo[a:a + 77])
        e.paged_step(table, s, t, i, pick=False)
    for s, p in enumerate(prompts):
        left = logits[s].copy()
        for i in ranking(torch, e, table, s, p[-1], len(p) - 1, 12):
            assert left[i] >= left.max() - limit, (s, i, left.max() - left[i], limit)
            left[i] = -np.inf
    e.close()


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
        e = mixing(K, n_layers=1)
        e.feed_batch(prompt[:64], 0)                     # the batched pass's buffers are there
        if busy:
            x = torch.randn((4096, 4096), device="cuda")
            for _ in range(200):                         # some tens of milliseconds
                x = (x @ x).clamp_(-1, 1)
        if kind == "paged":
            e.paged_caches(600, 1024, max_seq=1)
            table = np.array([[599]])
            e.paged_step(table, [0] * 119, prompt[:119], range(119), pick=False)
            got = ranking(torch, e, table, 0, prompt[119], 119, 30)
        else:
            e.batch_caches(300)
            e.batch_feed(299, prompt[:119], 0)
            got, t = [], prompt[119]
            for i in range(60):
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


def test_a_step_whose_rules_are_refused_feeds_nothing(env):
    """Fewer masks than rows is only seen by the library: the refused tokens must not have replaced the cached ones."""
    K, torch = env
    prompt = [int(v) for v in np.random.default_rng(8).integers(0, CFG["vocab"], 40)]
    ids = []
    for refused in (False, True):
        e = mixing(K)
        e.paged_caches(4, 16, max_seq=1)
        table = np.arange(4).reshape(1, 4)
        e.paged_step(table, [0] * 39, prompt[:39], range(39), pick=False)
        if refused:
            mask = torch.full((38, CFG["vocab"] // 32), -1, dtype=torch.int32, device="cuda")
            with pytest.raises(ValueError, match="masks"):
                e.paged_step(table, [0] * 39, [(t + 1) % CFG["vocab"] for t in prompt[:39]], range(39), rules=dict(mask=mask))
        ids.append(ranking(torch, e, table, 0, prompt[39], 39, 40))
        e.close()
    assert ids[0] == ids[1] and len(set(ids[0])) == 40
