"""8-bit key/value cache, CPU part: its numpy oracle against torch's float8 type, and the refusals that come before
the GPU."""
import ctypes

import numpy as np
import pytest
import torch

from fathom_b200 import _lib
from oracle import kv8_oracle as O


def test_oracle_e4m3_is_the_format():
    codes = np.arange(256, dtype=np.uint8)
    ref = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.decode(codes), ref, equal_nan=True)
    g = np.random.default_rng(0)
    y = np.concatenate([g.uniform(-448, 448, 20000), g.normal(size=20000) * 2.0 ** g.integers(-14, 6, 20000),
                        ref[~np.isnan(ref)], (ref[:-1] + ref[1:])[np.isfinite(ref[:-1] + ref[1:])] / 2]).astype(np.float32)
    y = y[np.abs(y) <= 448]
    got = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.encode(y), got)


def test_oracle_scales():
    for top, e in ((448.0, 0), (448.0001, 1), (1.75, -8), (1.7500001, -7), (1.0, -8), (0.0, -120), (3.4e38, 120),
                   (2.0 ** -149, -120)):
        assert O.scale_of([np.float32(top), -0.0, np.nan, np.inf]) == 2.0 ** e, top


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)      # never dereferenced: validation fails first
    OK16 = dict(strides=(8 * 128, 128, 128))

    def write(K=p, V=p, dtype=1, B=1, H=1, T=4, strides=OK16["strides"], start=0, dev=None, cap=128, rows=p, scales=p):
        return L.fathom_kv8_write(K, V, dtype, B, H, T, *strides, start, dev, cap, rows, scales, None)

    assert write(K=None) == write(rows=None) == write(scales=None) == _lib.FATHOM_ERR_NULL
    assert write(dtype=3) == _lib.FATHOM_ERR_UNSUPPORTED
    assert write(cap=100) == write(cap=0) == write(start=-1) == write(start=125) == write(T=129) == write(T=-1) \
        == write(B=0) == write(B=300, H=300) == _lib.FATHOM_ERR_SHAPE
    assert write(start=2 ** 62, T=2 ** 62) == _lib.FATHOM_ERR_SHAPE
    assert write(K=odd) == write(strides=(1024, 128, 132)) == _lib.FATHOM_ERR_SHAPE

    def read(rows=p, BH=1, cap=128, start=0, n=8, dtype=1, K=p):
        return L.fathom_kv8_read(rows, p, BH, cap, start, n, dtype, K, p, None)

    assert read(rows=None) == read(K=None) == _lib.FATHOM_ERR_NULL
    assert read(dtype=9) == _lib.FATHOM_ERR_UNSUPPORTED
    assert read(n=129) == read(start=121) == read(start=-1) == read(cap=65) == read(K=odd) == _lib.FATHOM_ERR_SHAPE

    def attend(q=p, dtype=1, B=1, H=1, G=4, T=1, cap=128, end=100, dev=None, ws=p, nb=1 << 40, strides=(512, 128, 128), sc=p):
        return L.fathom_kv8_attend(q, dtype, B, H, G, T, *strides, p, sc, cap, end, dev, p, 512, 128, 128, ws, nb, None)

    assert attend(q=None) == attend(ws=None) == _lib.FATHOM_ERR_NULL
    assert attend(dtype=0) == _lib.FATHOM_ERR_UNSUPPORTED
    assert attend(end=129) == attend(end=-1) == attend(G=0) == attend(T=0) == attend(cap=70) == _lib.FATHOM_ERR_SHAPE
    assert attend(q=odd) == attend(strides=(512, 130, 128)) == _lib.FATHOM_ERR_SHAPE
    assert attend(sc=ctypes.c_void_p(260)) == attend(cap=2 ** 31) == _lib.FATHOM_ERR_SHAPE
    assert attend(nb=0) == attend(ws=odd) == _lib.FATHOM_ERR_WORKSPACE
    assert b"workspace" in L.fathom_last_error()

    def picks(q=p, dtype=1, B=1, H=1, G=4, idx=p, k=10, cap=128, end=100, nb=1 << 40, host=0, sc=p):
        return L.fathom_kv8_attend_picks(q, dtype, B, H, G, idx, k, p, host, sc, cap, end, None, p, p, nb, None)

    assert picks(q=None) == picks(idx=None) == _lib.FATHOM_ERR_NULL
    assert picks(dtype=5) == _lib.FATHOM_ERR_UNSUPPORTED
    assert picks(k=0) == picks(end=129) == picks(G=0) == picks(B=70000) == picks(q=odd) == _lib.FATHOM_ERR_SHAPE
    assert picks(sc=ctypes.c_void_p(260)) == picks(k=2 ** 31) == _lib.FATHOM_ERR_SHAPE
    assert picks(nb=0) == picks(nb=1000, host=1) == _lib.FATHOM_ERR_WORKSPACE
    assert L.fathom_kv8_attend_picks_workspace_bytes(1, 8, 4, 580, 1) >= 8 * 4 * 580 * 256
    assert L.fathom_kv8_attend_picks_workspace_bytes(1, 8, 4, 580, 0) == 256


def test_python_layer_refuses_cpu_tensors_and_bad_sizes():
    from fathom_b200.kv8 import KVCache8
    with pytest.raises(ValueError, match="CUDA"):
        KVCache8(1, 2, 64, rows=torch.zeros(2, 64, 2, 128, dtype=torch.uint8), scales=torch.zeros(2, 1, 2))
    with pytest.raises(ValueError, match="together"):
        KVCache8(1, 2, 64, rows=torch.zeros(2, 64, 2, 128, dtype=torch.uint8))
    for bad in ((0, 2, 64), (1, 0, 64), (1, 2, 0)):
        with pytest.raises(ValueError, match="positive"):
            KVCache8(*bad)
