"""The decoder over an 8-bit cache (OffloadedDecoder(kv="e4m3")): prefill chunks written and attended to, the index built
from the keys read back, decode over picks (rows in HBM or in host memory) and over every key of a short context."""
import pytest
import torch

from tests.test_hf_gpu import _close, _model

pytestmark = pytest.mark.gpu


def _run(model, ids, n, steps, full=False, **kw):
    from fathom_b200.hf import OffloadedDecoder
    dec = OffloadedDecoder(model, max_new=steps + 2, prefill_chunk=512, **kw)
    try:
        out = [dec.prefill(ids[:, :n])]
        dec.offload()
        dense = dec.cache[0].kv8 is not None and dec.cache[0].store is None
        for s in range(steps):
            if full:
                dec.k = dec.context + 1
            out.append(dec.decode(ids[:, n + s:n + s + 1]))
        return out, dense, dec._graph is not None
    finally:
        dec.free()
        dec.unpatch()


def _ids(n, B=2, seed=1):
    return torch.randint(0, 512, (B, n), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


@pytest.mark.parametrize("klt", [False, True])
def test_8_bit_rows_stay_near_bf16_rows(klt):
    """Every token picked: the two decoders differ by the rounding of keys and values (2^-4 of each element) only."""
    model, n, steps = _model(), 1500, 3
    ids = _ids(n + steps)
    a, _, _ = _run(model, ids, n, steps, full=True, k=600, index="hbm", rows="hbm", klt=klt)
    b, _, _ = _run(model, ids, n, steps, full=True, k=600, index="hbm", rows="hbm", klt=klt, kv="e4m3")
    for x, y in zip(a, b):
        assert torch.nn.functional.cosine_similarity(x.float(), y.float(), dim=-1).min().item() > 0.99


def test_every_pick_is_dense_attention_over_the_same_cache():
    """A prefill of at most k tokens decodes over every key; a longer one with every token picked reads the same
    cache: the same logits up to the rounding of the attention's output."""
    model, n, steps = _model(), 700, 3
    ids = _ids(n + steps)
    a, dense, _ = _run(model, ids, n, steps, k=2000, index="hbm", rows="hbm", kv="e4m3")
    b, sparse, _ = _run(model, ids, n, steps, full=True, k=600, index="hbm", rows="hbm", kv="e4m3")
    assert dense and not sparse
    assert torch.equal(a[0], b[0])
    for x, y in zip(a, b):
        assert _close(x, y, 3e-2)


def test_host_rows_equal_hbm_rows():
    model, n, steps = _model(), 1300, 4
    ids = _ids(n + steps)
    kw = dict(k=300, sink=4, local=32, kv="e4m3")
    a, _, _ = _run(model, ids, n, steps, index="hbm", rows="hbm", **kw)
    b, _, _ = _run(model, ids, n, steps, index="hbm", rows="host", **kw)
    for s, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), s


@pytest.mark.parametrize("rows,k", [("hbm", 200), ("host", 200), ("hbm", 5000)])
def test_graph_decode_matches_eager(rows, k):
    model, n, steps = _model(), 1500, 14
    ids = _ids(n + steps, seed=7)
    kw = dict(k=k, sink=4, local=8, index="hbm", rows=rows, kv="e4m3")
    eager, _, _ = _run(model, ids, n, steps, **kw)
    graph, _, used = _run(model, ids, n, steps, graphs=True, **kw)
    assert used
    for s, (a, b) in enumerate(zip(eager, graph)):
        assert torch.equal(a, b), s


def test_load_kv_and_refusals():
    from fathom_b200.hf import OffloadedDecoder
    model = _model()
    with pytest.raises(ValueError, match="kv"):
        OffloadedDecoder(model, kv="int4")
    dec = OffloadedDecoder(model, k=200, index="hbm", rows="host", max_new=4, kv="e4m3")
    try:
        g = torch.Generator("cuda").manual_seed(5)
        for L in range(2):
            K, V = (torch.randn(1, 2, 900, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
            dec.load_kv(L, K, V, offload=True, rows_of=None if L == 0 else 0)
        assert dec.decode(_ids(1, B=1)).isfinite().all()
        dec.prefill(_ids(150, B=1))
        with pytest.raises(ValueError, match="shorter"):            # host rows need more than k tokens
            dec.offload()
    finally:
        dec.free()
        dec.unpatch()
