"""Calls with another CUDA device current than their tensors' (both devices and the library are stand-ins)."""
import contextlib

import torch


def test_calls_run_on_the_device_of_the_rows(monkeypatch):
    """With another device current, every call switches to the cache's before it reaches the library (both devices and the
    library are stand-ins)."""
    import fathom_b200.kv8 as kv8
    now, seen = [1], []

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d.index
        yield
        now[0] = before

    class Library:
        def __getattr__(self, name):
            def call(*args):
                seen.append((name, now[0]))
                return 256 if name.endswith("_bytes") else 0
            return call

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(kv8, "lib", Library)
    c = kv8.KVCache8.__new__(kv8.KVCache8)
    c.B, c.Hkv, c.BH, c.cap, c.nblk, c.host, c._buf, c._ws = 1, 2, 2, 128, 2, False, None, {}
    c.rows, c.scales = torch.zeros(2, 128, 2, 128, dtype=torch.uint8), torch.zeros(2, 2, 2)
    c.device, c._unused = torch.device("cpu", 0), torch.zeros(256, dtype=torch.uint8)
    c._check_on, c._stream = (lambda *a: None), (lambda: 0)
    K = torch.zeros(1, 2, 4, 128)
    c.write(K, K, 0)
    c.read(0, 4)
    c.attend(torch.zeros(1, 4, 1, 128, dtype=torch.float16), 4)
    c.attend_picks(torch.zeros(2, 2, 128), torch.zeros(2, 2, 3, dtype=torch.int64))
    assert {n for n, _ in seen} == {"fathom_kv8_write", "fathom_kv8_read", "fathom_kv8_attend",
                                    "fathom_kv8_attend_workspace_bytes", "fathom_kv8_attend_picks"}
    assert all(d == 0 for _, d in seen) and now == [1]


def test_launches_elsewhere_are_refused(monkeypatch):
    import pytest
    from fathom_b200 import _lib
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: type("Stream", (), {"cuda_stream": 7}))
    assert _lib.stream_of(torch.device("cuda", 0)) == _lib.stream_of(torch.device("cuda")) == 7
    with pytest.raises(ValueError, match="current device"):
        _lib.stream_of(torch.device("cuda", 1))
