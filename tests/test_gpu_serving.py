"""GPU: what the serving operators must hold beside their formulas (tests/test_gpu_paged.py, tests/test_gpu_rules.py):
refusals of tensors that are too small, the order of clusters, streams, captures, handles and error words."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import kq as K
    assert K.lib().kq_device_count() > 0 and torch.cuda.is_available(), "no GPU"
    return K, torch


@pytest.fixture(params=[True, False], ids=["direct", "checked"])
def way(request, env, monkeypatch):
    """Both ways of passing tensors: described to the library, or asked by the checks in Python."""
    K, torch = env
    from kq import serve
    serve._Direct.try_type(torch.Tensor)
    if not request.param:
        monkeypatch.setattr(serve._Direct, "type", None)
        monkeypatch.setattr(serve._Direct, "_tried", {torch.Tensor})
    return request.param


def test_narrow_masks_are_refused(env, way):
    """Columns of a wider mask array: its row stride would do, its rows would not."""
    K, torch = env
    z = torch.randn((2, 200), device="cuda")
    out = torch.empty_like(z)
    wide = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    K.logit_rules(z, out, mask=wide[:, 30:37])                              # seven words: enough
    K.check_stream()
    assert torch.equal(out, z)
    for mask in (wide[:, 34:40], wide[:, :6], wide[:1, 30:36]):
        with pytest.raises(ValueError, match="too few words"):
            K.logit_rules(z, out, mask=mask, mask_row=torch.zeros(2, dtype=torch.int32, device="cuda"))
    K.check_stream()


@pytest.mark.parametrize("vocab,kind", [(4097, "float32"), (6145, "float32"), (16390, "float32"), (8200, "bfloat16"), (40, "float16")])
def test_clusters_whose_last_blocks_have_little_to_do(env, vocab, kind):
    """Rows cut so that some blocks of a cluster own no id, or one group: they are done before the others begin."""
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(vocab)
    ids = torch.empty((60, 2), dtype=torch.int32, device="cuda")
    want = torch.empty_like(ids)
    for n in (1, 2):
        z = torch.randn((60, n, vocab), device="cuda", generator=g).to(getattr(torch, kind))
        out = torch.empty_like(z)
        for i in range(60):
            K.logit_rules(z[i], out[i], best=ids[i, :n])
        top = z.float().amax(2, keepdim=True)
        want[:, :n] = torch.where(z.float() == top, torch.arange(vocab, device="cuda", dtype=torch.int32), vocab).amin(2)
        K.check_stream()
        assert torch.equal(ids[:, :n], want[:, :n]) and torch.equal(out, z)


def test_flags_of_several_streams_are_all_reported(env):
    """Checks on one stream while others raise flags: each kind of flag is reported, none is lost."""
    K, torch = env
    t = dict(dtype=torch.int32, device="cuda")
    z, row = torch.zeros((1, 64), device="cuda"), torch.tensor([7], **t)
    out, mask = torch.empty_like(z), torch.zeros((1, 2), **t)
    k = torch.zeros((1, 1, 16, 64), device="cuda", dtype=torch.float16)
    cache, q, table, lens = K.PagedCache(k, k), torch.zeros((1, 1, 64), device="cuda"), torch.tensor([[3]], **t), torch.tensor([5], **t)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    K.check_stream()
    for _ in range(20):
        K.logit_rules(z, out, mask=mask, mask_row=row, stream=a.cuda_stream)
        cache.attend(q, table, lens, torch.empty_like(q), stream=b.cuda_stream)
        texts = []
        for s in (a, b):
            try:
                K.check_stream(stream=s.cuda_stream)
            except ValueError as e:
                texts.append(str(e))
        assert "row index" in " ".join(texts) and "page id" in " ".join(texts)
        K.check_stream()


def test_two_threads(env):
    """Operators of two host threads, each on a stream and a cache of its own."""
    import threading
    K, torch = env
    g = torch.Generator(device="cuda").manual_seed(21)
    t = dict(dtype=torch.int32, device="cuda")
    k, v = (torch.randn((64, 2, 16, 128), device="cuda", generator=g).half() for _ in range(2))
    table = torch.arange(64, **t).view(2, 32)
    lens = torch.tensor([500, 77], **t)
    q = torch.randn((2, 8, 128), device="cuda", generator=g)
    z = torch.randn((2, 5000), device="cuda", generator=g)
    ref = K.PagedCache(k, v).attend(q, table, lens, torch.empty_like(q))
    torch.cuda.synchronize()
    wrong = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            cache, out, o2, best = K.PagedCache(k, v), torch.empty_like(q), torch.empty_like(z), torch.zeros(2, **t)
            for _ in range(200):
                cache.attend(q, table, lens, out, stream=s.cuda_stream)
                K.logit_rules(z, o2, best=best, stream=s.cuda_stream)
            s.synchronize()
            if not (torch.equal(out, ref) and torch.equal(o2, z) and torch.equal(best, z.argmax(1).int())):
                wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not wrong
    K.check_stream()


def pool(torch, seed, pages=64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn((pages, 2, 16, 128), device="cuda", generator=g).half() for _ in range(2))
    return k, v, torch.randn((1, 8, 128), device="cuda", generator=g)


def plain(torch, k, v, q, L):
    """Attention of one token over the first L positions of pages 0, 1, ... in 64 bits."""
    kk, vv = (x.double().transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :L] for x in (k, v))
    z = torch.einsum("ghd,gtd->ght", q[0].double().view(k.shape[1], -1, q.shape[2]), kk) / q.shape[2] ** 0.5
    return torch.einsum("ght,gtd->ghd", z.softmax(-1), vv).reshape(q.shape[1:])


def test_handles_close_at_any_time(env):
    """During a capture, and while the device is busy: closing waits for nothing and calls nothing that a capture forbids."""
    K, torch = env
    k, v, q = pool(torch, 41)
    table, lens = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64), torch.tensor([1000], dtype=torch.int32, device="cuda")
    want = plain(torch, k, v, q, 1000)
    caches = [K.PagedCache(k, v) for _ in range(24)]
    outs = [torch.empty_like(q) for _ in caches]
    for c, o in zip(caches, outs):
        c.attend(q, table, lens, o)
    x = torch.randn((4096, 4096), device="cuda")
    for _ in range(200):                                 # some tens of milliseconds
        x = (x @ x).clamp_(-1, 1)
    late = torch.empty_like(q)
    caches[0].attend(q, table, lens, late)
    done = torch.cuda.Event()
    done.record()
    for c in caches[:12]:
        c.close()
    assert not done.query()
    torch.cuda.synchronize()
    s, graph, again = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph, stream=s):
        caches[23].attend(q, table, lens, again, stream=s.cuda_stream)
        for c in caches[12:23]:
            c.close()
    graph.replay()
    fresh = [K.PagedCache(k, v) for _ in range(24)]      # the first waits for the device
    more = [torch.empty_like(q) for _ in fresh]
    for c, o in zip(fresh, more):
        c.attend(q, table, lens, o)
    K.check_stream()
    for o in outs + more + [late, again]:
        assert float((o[0].double() - want).abs().max()) < 1e-5    # weights of 22 bits over unit normal values
        assert torch.equal(o, outs[0])


def test_graphs_keep_the_scratch_of_closed_handles(env):
    """Replays of a graph whose handle is gone, beside calls of handles made since: each has a scratch of its own."""
    K, torch = env
    k, v, q = pool(torch, 43)
    table, lens = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64), torch.tensor([1000], dtype=torch.int32, device="cuda")
    want = plain(torch, k, v, q, 1000)
    s, o = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        graphs, outs = [], [torch.empty_like(q) for _ in range(4)]
        for out in outs:
            cache = K.PagedCache(k, v)
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                cache.attend(q, table, lens, out, stream=s.cuda_stream)
            cache.close()
        caches = [K.PagedCache(k, v) for _ in range(4)]
        more = [torch.empty_like(q) for _ in caches]
        torch.cuda.synchronize()
        for i in range(50):
            with torch.cuda.stream(s):
                graphs[i % 4].replay()
            caches[i % 4].attend(q, table, lens, more[i % 4], stream=o.cuda_stream)
        torch.cuda.synchronize()
        K.check_stream()
        for x in outs + more:
            assert float((x[0].double() - want).abs().max()) < 1e-5
            assert torch.equal(x, outs[0])
        del graphs
        for c in caches:
            c.close()


def test_scratches_of_dropped_graphs_come_back(env):
    """40 handles captured, closed and their graphs dropped, one after another: not 40 scratches of 10 MB."""
    K, torch = env
    k, v, q = pool(torch, 44)
    table, lens = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64), torch.tensor([300], dtype=torch.int32, device="cuda")
    s, out = torch.cuda.Stream(), torch.empty_like(q)
    free = []
    for i in range(44):
        cache, graph = K.PagedCache(k, v), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            cache.attend(q, table, lens, out, stream=s.cuda_stream)
        graph.replay()
        cache.close()
        torch.cuda.synchronize()
        del graph
        if i in (3, 43):
            free.append(torch.cuda.mem_get_info()[0])
    assert free[0] - free[1] < 200 << 20


def test_calls_without_a_stream_follow_the_current_one(env, way):
    """Behind work that is still queued on PyTorch's current stream, and inside a capture of it."""
    K, torch = env
    k, v, q0 = pool(torch, 47)
    table, lens = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64), torch.tensor([1000], dtype=torch.int32, device="cuda")
    x, cache, s = torch.randn((4096, 4096), device="cuda"), K.PagedCache(k, v), torch.cuda.Stream()
    pos, kn = torch.tensor([999], dtype=torch.int32, device="cuda"), torch.empty((1, 2, 128), device="cuda")
    q, out, z, best = torch.zeros_like(q0), torch.empty_like(q0), torch.zeros((1, 3000), device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(100):                             # some tens of milliseconds
            x = (x @ x).clamp_(-1, 1)
        q.copy_(q0)
        kn.fill_(0.25)
        z[0, 1234] = 1.0
        cache.append(kn, kn, table, pos)
        cache.attend(q, table, lens, out)
        K.logit_rules(z, z, best=best)
        K.check_stream()
    first = out.clone()
    k[62, :, 7] = v[62, :, 7] = 0.25                     # position 999
    assert float((first[0].double() - plain(torch, k, v, q0, 1000)).abs().max()) < 1e-5
    assert best.tolist() == [1234]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache.append(kn, kn, table, pos)
        cache.attend(q, table, lens, out)
        K.logit_rules(z, z, best=best)
    q.mul_(0.5)
    z[0, 77] = 2.0
    graph.replay()
    torch.cuda.synchronize()
    assert float((out[0].double() - plain(torch, k, v, q0 * 0.5, 1000)).abs().max()) < 1e-5
    assert best.tolist() == [77]
