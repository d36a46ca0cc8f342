"""GPU: batched decode over a paged cache (Engine.paged_caches / paged_step: the append, the paged
attention and the logit rules together) against each sequence decoded alone (feed_batch + step)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

CFG = dict(D=1024, NL=2, NH=8, NKV=2, HD=128, NFF=2048, vocab=4096, ctx=512)


@pytest.fixture(scope="module")
def env():
    import torch
    import kq as K
    assert K.lib().kq_device_count() > 0 and torch.cuda.is_available(), "no GPU"
    return K, torch


def engine(kq):
    t = CFG
    return kq.Engine(kq.Config.default(dim=t["D"], n_layers=t["NL"], n_heads=t["NH"], n_kv_heads=t["NKV"], head_dim=t["HD"],
                                       ffn=t["NFF"], vocab=t["vocab"], ctx=t["ctx"]), seed=0)


@pytest.fixture(scope="module")
def alone(env):
    """Prompts, and for each the greedy ids and logits of its steps on the whole-model path."""
    K, _ = env
    rng = np.random.default_rng(12)
    prompts = [[int(v) for v in rng.integers(0, CFG["vocab"], n)] for n in (37, 150, 5, 90)]
    e = engine(K)
    ids, logits = [], []
    for p in prompts:
        e.reset()
        e.feed_batch(p[:-1], 0)
        toks, zs, t = [], [], p[-1]
        for i in range(6):
            t = e.step(t, len(p) - 1 + i)
            toks.append(t)
            zs.append(e.ylog.copy())
        ids.append(toks)
        logits.append(zs)
    e.close()
    return prompts, ids, logits


def feed(e, table, prompts, chunk):
    """Every prompt but its last token, in chunks that hold tokens of several sequences."""
    todo = [(s, t, i) for s, p in enumerate(prompts) for i, t in enumerate(p[:-1])]
    for a in range(0, len(todo), chunk):
        s, t, i = zip(*todo[a:a + chunk])
        assert e.paged_step(table, s, t, i, pick=False) is None


@pytest.mark.parametrize("page,chunk", [(16, 100), (64, 128), (512, 31)])
def test_paged_steps_match_single_sequences(env, alone, page, chunk):
    K, _ = env
    prompts, ref, _ = alone
    e = engine(K)
    wide = -(-CFG["ctx"] // page)
    pages = 4 * wide if page > 64 else 40
    e.paged_caches(pages, page, max_seq=4)
    order = np.random.default_rng(page).permutation(pages)
    table = np.full((4, wide), pages + 9, np.int32)      # pages not yet given out are never looked at
    at = 0
    for s, p in enumerate(prompts):
        need = -(-(len(p) + 6) // page)
        table[s, :need] = order[at:at + need]
        at += need
    feed(e, table, prompts, chunk)
    seqs = [3, 0, 2, 1]
    cur, pos = [prompts[s][-1] for s in seqs], [len(prompts[s]) - 1 for s in seqs]
    got = [[] for _ in seqs]
    for _ in range(6):
        cur = e.paged_step(table, seqs, cur, pos)
        for j, t in enumerate(cur):
            got[j].append(t)
        pos = [p + 1 for p in pos]
    for j, s in enumerate(seqs):
        assert got[j] == ref[s], s
    e.close()


def test_shared_prefix_pages(env, alone):
    """Two sequences whose tables name the same pages for a common prompt."""
    K, _ = env
    prompts, ref, _ = alone
    p = prompts[1]
    e = engine(K)
    e.paged_caches(32, 16, max_seq=2)
    table = np.zeros((2, 12), np.int32)
    table[0] = np.arange(12)
    table[1] = np.arange(12)
    table[1, 9:] = [20, 21, 22]                          # positions 144.. of its own
    for a in range(0, 149, 50):
        e.paged_step(table, [0] * len(p[a:min(a + 50, 149)]), p[a:min(a + 50, 149)], range(a, min(a + 50, 149)), pick=False)
    e.paged_step(table, [1] * 5, p[144:149], range(144, 149), pick=False)
    cur, pos = [p[-1]] * 2, [149, 149]
    for i in range(4):
        cur = e.paged_step(table, [1, 0], cur, pos)
        assert cur == [ref[1][i]] * 2
        pos = [v + 1 for v in pos]
    e.close()


def test_rules_in_a_step(env, alone):
    K, torch = env
    prompts, ref, logits = alone
    e = engine(K)
    e.paged_caches(40, 16, max_seq=4)
    table = np.arange(40).reshape(4, 10)
    feed(e, table, prompts, 128)
    step = ([0, 1, 2, 3], [p[-1] for p in prompts], [len(p) - 1 for p in prompts])
    t = dict(dtype=torch.int32, device="cuda")
    first = [r[0] for r in ref]
    assert e.paged_step(table, *step, rules={}) == first
    # a mask without the best id: the second best; a row that allows nothing; a row without a mask
    second = [int(np.argsort(z[0])[-2]) for z in logits]
    mask = np.full((3, CFG["vocab"] // 32), 0xffffffff, np.uint32)
    for r in (0, 1):
        mask[r, first[r] // 32] &= ~np.uint32(1 << (first[r] % 32))
    mask[2] = 0
    rules = dict(mask=torch.tensor(mask.view(np.int32), device="cuda"), mask_row=torch.tensor([0, 1, 2, -1], **t))
    assert e.paged_step(table, *step, rules=rules) == [second[0], second[1], -1, first[3]]
    # a bias that forces an id, a presence penalty that rules the best one out
    hist = torch.tensor([[first[0]], [7], [first[2]], [8]], **t)
    one = torch.ones(4, device="cuda")
    rules = dict(hist=hist, hist_len=torch.ones(4, **t), presence=one * 1e6, bias_ids=torch.tensor([[-1], [99], [-1], [-1]], **t),
                 bias=torch.full((4, 1), 1e6, device="cuda"))
    assert e.paged_step(table, *step, rules=rules) == [second[0], 99, second[2], first[3]]
    assert e.paged_step(table, *step) == first
    e.close()


def test_paged_step_refusals(env):
    K, torch = env
    e = engine(K)
    tb = np.zeros((2, 4), np.int32)
    with pytest.raises(ValueError):
        e.paged_step(tb, [0], [1], [0])                  # no pool yet
    for bad in ((4, 24, 2), (0, 16, 2), (4, 16, 0), (4, 8, 2)):
        with pytest.raises(ValueError):
            e.paged_caches(*bad)
    with pytest.raises(MemoryError):
        e.paged_caches(1 << 28, 1024, 2)
    e.paged_caches(4, 16, 2)                             # a smaller pool after a failed one
    with pytest.raises(ValueError):
        e.paged_caches(5, 16, 2)
    tb[1] = [1, 2, 4, -1]
    for seqs, toks, pos in (([2], [1], [0]), ([-1], [1], [0]), ([0], [-1], [0]), ([0], [CFG["vocab"]], [0]), ([0], [1], [-1]),
                            ([0, 0], [1, 2], [3, 3]), ([1], [1], [32]), ([1], [1], [48])):
        with pytest.raises(ValueError):
            e.paged_step(tb, seqs, toks, pos)
    with pytest.raises(OverflowError):
        e.paged_step(tb, [0], [1], [64])
    with pytest.raises(ValueError):
        e.paged_step(np.zeros((3, 4)), [0], [1], [0])
    with pytest.raises(ValueError):
        e.paged_step(tb, [0], [1], [0], rules=dict(mask_row=torch.zeros(1, dtype=torch.int32, device="cuda")))
    with pytest.raises(TypeError):
        e.paged_step(tb, [0], [1], [0], rules=dict(unknown=1))
    assert len(e.paged_step(tb, [0, 1], [1, 2], [0, 31])) == 2
    e.close()
