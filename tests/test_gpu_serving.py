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
