"""Layers that read another layer's 8-bit rows (load_kv(rows_of=)): generated tokens stay each layer's own."""
import pytest
import torch

from tests.test_hf_gpu import _model

pytestmark = pytest.mark.gpu


def _randn(*shape, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).bfloat16()


def _decoder(n, rows, share, layers=3, B=2, max_new=100, **kw):
    from fathom_b200.hf import OffloadedDecoder
    dec = OffloadedDecoder(_model(layers=layers), k=300, sink=4, local=32, index="hbm", rows=rows, max_new=max_new, kv="e4m3",
                           **kw)
    for L in range(layers):
        K, V = _randn(B, 2, n, 128, seed=L), _randn(B, 2, n, 128, seed=10 + L)
        dec.load_kv(L, K, V, offload=True, rows_of=0 if share and L else None)
    return dec


def _token(L, t, B=2):
    """q, k, v of layer L's token t; later layers' are louder, so that they would move another layer's block scale."""
    x = _randn(B, 8 + 2 + 2, 1, 128, seed=1000 * L + t)
    return 2 * x[:, :8], x[:, 8:10] * 8 ** L, x[:, 10:] * 8 ** L


@pytest.mark.parametrize("rows", ["hbm", "host"])
@pytest.mark.parametrize("n", [896, 901])
def test_the_owner_is_not_touched(rows, n):
    """The owning layer's attention over 70 generated tokens is the same with and without layers that read its rows."""
    outs = []
    for share in (False, True):
        dec = _decoder(n, rows, share)
        try:
            out = []
            for t in range(70):
                for L in range(3):
                    o = dec._decode_attn(L, *_token(L, t))
                    if L == 0:
                        out.append(o)
            outs.append(torch.stack(out))
        finally:
            torch.cuda.synchronize()
            dec.free()
            dec.unpatch()
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("rows", ["hbm", "host"])
def test_a_reader_has_its_own_tokens(rows):
    """A layer over shared rows attends to the owner's prefill rows and the tokens it generated itself."""
    from fathom_b200.kv8 import KVCache8
    n = 896                                              # whole blocks, so that no code of them is rounded again
    dec = _decoder(n, rows, True)
    try:
        ref = [KVCache8(2, 2, n + 100) for _ in range(3)]
        for c in ref:
            c.write(_randn(2, 2, n, 128, seed=0), _randn(2, 2, n, 128, seed=10))
        for t in range(70):
            for L in range(3):
                q, k, v = _token(L, t)
                out = dec._decode_attn(L, q, k, v)
                at = dec.cache[L].at
                idx = torch.where(dec._idx >= at, dec._idx - at + n, dec._idx)
                ref[L].write(k, v, n + t)
                assert torch.equal(out.view(4, 4, 128), ref[L].attend_picks(q.reshape(4, 4, 128), idx, n + t + 1)), (L, t)
    finally:
        torch.cuda.synchronize()
        dec.free()
        dec.unpatch()


def test_graph_decode_over_shared_rows_matches_eager():
    ids = torch.randint(0, 512, (2, 45), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    logits = []
    for graphs in (False, True):
        dec = _decoder(901, "hbm", True, graphs=graphs)
        try:
            logits.append(torch.stack([dec.decode(ids[:, t:t + 1]) for t in range(45)]))
            assert (dec._graph is not None) == graphs
        finally:
            torch.cuda.synchronize()
            dec.free()
            dec.unpatch()
    assert torch.equal(logits[0], logits[1])


def test_rows_of_without_offload_keeps_the_layers_own_rows():
    """As over bf16 rows: rows_of takes effect with offload=True only; offload() afterwards builds every layer's own."""
    from fathom_b200.hf import OffloadedDecoder
    outs = []
    for rows_of in (None, 0):
        dec = OffloadedDecoder(_model(), k=300, sink=4, local=32, index="hbm", rows="hbm", max_new=4, kv="e4m3")
        try:
            for L in range(2):
                dec.load_kv(L, _randn(1, 2, 700, 128, seed=L), _randn(1, 2, 700, 128, seed=10 + L), rows_of=rows_of if L else None)
            dec.offload()
            outs.append(dec.decode(torch.zeros(1, 1, dtype=torch.long, device="cuda")))
        finally:
            dec.free()
            dec.unpatch()
    assert torch.equal(outs[0], outs[1])
