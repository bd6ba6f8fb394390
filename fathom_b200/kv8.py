"""8-bit key/value cache: written as tokens come, read back, and attended to.

Keys and values as e4m3 codes with one power-of-two scale per 64-token block, KV head and K or V (half the
bytes of bf16 rows, in HBM or over the host link).  No counterpart in the reference, which keeps bf16 rows
(scripts/B_e2e_offload_v2.py:272-300).  The sequence's positions may be device tensors, so a decode
step over the cache can be captured in a CUDA graph.

    cache = KVCache8(B, Hkv, cap)
    cache.write(K, V, 0)                    # a prompt, or a chunk of one
    cache.write(k, v, pos)                  # one token of every sequence; pos an int, or int64 [B] on the device
    out = cache.attend(q, end)              # every key before `end`: prompt chunks, drafts, single tokens
    out = cache.attend_picks(q, idx, end)   # the listed keys of each query head
    K, V = cache.read(0, n)
"""
import operator

import torch

from . import _lib
from ._lib import check, lib, ptr, require_cuda
from .offload import MappedBuffer

BLK, D = 64, 128


def _position(x, B, device, what):
    """(number, device tensor or None) of a position given as an int or as int64 [B] (or [1]) on `device`."""
    if not isinstance(x, torch.Tensor):
        return operator.index(x), None                 # (a float is a TypeError, not a position rounded down)
    if x.dtype == torch.int64 and x.dim() == 1 and x.shape[0] == B and x.device == device and x.is_contiguous():
        return 0, x
    if x.device != device or x.dtype != torch.int64 or x.numel() not in (1, B) or x.dim() > 1:
        raise ValueError(f"{what} must be an int or an int64 [{B}] tensor on {device}")
    return 0, x.reshape(-1).expand(B).contiguous()


class KVCache8:
    """Room for `cap` tokens (rounded up to whole 64-token blocks) of B sequences with Hkv KV heads.

    rows    uint8 [B * Hkv, cap, 2, 128]: e4m3 codes of each token's key (0) and value (1)
    scales  fp32 [B * Hkv, cap / 64, 2]: powers of two; value = code * scale
    Either both may be given (contiguous, of these shapes) or they are made on `device`; host=True puts the rows
    into pinned mapped host memory (the scales stay on the device; free() or garbage collection releases
    the rows): written and read over the host link, attended to over picks only.  Tokens past the last written
    one are void: no call reads them.  Which tokens a sequence has is the caller's to know: a write says where it
    begins, a read or an attention where it ends.  Calls run on the rows' device, whichever is the current one."""

    def __init__(self, B, Hkv, cap, device="cuda", rows=None, scales=None, host=False):
        if B < 1 or Hkv < 1 or cap < 1:
            raise ValueError(f"KVCache8: B, Hkv and cap must be positive (got {B}, {Hkv}, {cap})")
        self.B, self.Hkv, self.BH = B, Hkv, B * Hkv
        self.nblk = -(-cap // BLK)
        self.cap = self.nblk * BLK
        if (rows is None) != (scales is None):
            raise ValueError("KVCache8: rows and scales come together")
        if host and rows is not None:
            raise ValueError("KVCache8: host=True makes the rows itself")
        self.host, self._buf = host, None
        if rows is None:
            if host:
                self._buf = MappedBuffer((self.BH, self.cap, 2, D), torch.uint8,
                                         None if torch.device(device).index is None else device)
                rows, device = self._buf.dev, self._buf.dev.device
            else:
                rows = torch.zeros(self.BH, self.cap, 2, D, dtype=torch.uint8, device=device)
            scales = torch.zeros(self.BH, self.nblk, 2, dtype=torch.float32, device=device)
        require_cuda(rows, scales)
        if rows.dtype != torch.uint8 or tuple(rows.shape) != (self.BH, self.cap, 2, D) or not rows.is_contiguous():
            raise ValueError(f"KVCache8: rows must be contiguous uint8 [{self.BH}, {self.cap}, 2, {D}]")
        if (scales.dtype != torch.float32 or tuple(scales.shape) != (self.BH, self.nblk, 2)
                or not scales.is_contiguous() or scales.device != rows.device):
            raise ValueError(f"KVCache8: scales must be contiguous float32 [{self.BH}, {self.nblk}, 2] beside the rows")
        self.rows, self.scales, self.device = rows, scales, rows.device
        self._ws = {}              # workspace bytes of a call's shape
        self._unused = torch.empty(256, dtype=torch.uint8, device=self.device)   # workspace of picks of rows in HBM

    def nbytes(self):
        return self.rows.numel() + self.scales.numel() * 4

    def free(self):
        """Release rows in host memory (device tensors go with their last reference)."""
        if self._buf is not None:
            self.rows = None
            self._buf.free()
            self._buf = None

    def _stream(self):
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    def _workspace(self, key, size, *args):
        """Scratch of one call, from the allocator's pool of the current stream: calls on two streams share none."""
        n = self._ws.get(key)
        if n is None:
            n = self._ws[key] = size(self.B, self.Hkv, *args)
        return torch.empty(n, dtype=torch.uint8, device=self.device), n

    def _check_on(self, what, *tensors):
        for t in tensors:
            if t.device != self.device:
                require_cuda(t)
                raise ValueError(f"{what}: expected tensors on {self.device}, got one on {t.device}")

    def write(self, K, V, start=0):
        """Write K, V [B, Hkv, T, 128] (fp32, bf16 or fp16, any strides) as tokens [start, start + T) of every
        sequence.  start: an int, or int64 [B] on the device (then a sequence with a negative start is left
        alone and tokens past cap are dropped).  The scale of a block covers every token written to it in
        this and in earlier calls; a block written from its first token on starts afresh.  NaN and infinities
        are stored as NaN and do not enter the scale."""
        if torch._C._cuda_getDevice() != self.device.index:
            with torch.cuda.device(self.device):
                return self.write(K, V, start)
        self._check_on("KVCache8.write", K, V)
        shape = K.shape
        if len(shape) != 4 or shape[0] != self.B or shape[1] != self.Hkv or shape[3] != D or V.shape != shape:
            raise ValueError(f"KVCache8.write: K and V must be [{self.B}, {self.Hkv}, T, {D}] "
                             f"(got {tuple(shape)}, {tuple(V.shape)})")
        if K.dtype not in _lib.DTYPE_CODE or V.dtype != K.dtype:
            raise TypeError(f"KVCache8.write: K and V must both be fp32, bf16 or fp16 (got {K.dtype}, {V.dtype})")
        T = shape[2]
        num, dev = _position(start, self.B, self.device, "KVCache8.write: start")
        if dev is None and not 0 <= num <= self.cap - T:
            raise ValueError(f"KVCache8.write: tokens [{num}, {num + T}) are outside the cache's {self.cap}")
        if T == 0:
            return
        (K, sb, sh, st), (V, *strides) = _rows16(K), _rows16(V)
        if strides != [sb, sh, st]:
            K, V = K.contiguous(), V.contiguous()
            sb, sh, st, _ = K.stride()
        check(lib().fathom_kv8_write(K.data_ptr(), V.data_ptr(), _lib.DTYPE_CODE[K.dtype], self.B, self.Hkv, T, sb, sh,
                                     st, num, ptr(dev), self.cap, self.rows.data_ptr(), self.scales.data_ptr(),
                                     self._stream()), "KVCache8.write")

    def read(self, start=0, n=None, dtype=torch.bfloat16):
        """Tokens [start, start + n) (to the end of the cache by default) as (K, V) [B, Hkv, n, 128] in dtype: fp32
        and bf16 hold the cached values exactly, fp16 rounds."""
        if torch._C._cuda_getDevice() != self.device.index:
            with torch.cuda.device(self.device):
                return self.read(start, n, dtype)
        n = self.cap - start if n is None else n
        if not 0 <= start <= self.cap or not 0 <= n <= self.cap - start:
            raise ValueError(f"KVCache8.read: tokens [{start}, {start + n}) are outside the cache's {self.cap}")
        if dtype not in _lib.DTYPE_CODE:
            raise TypeError(f"KVCache8.read: unsupported dtype {dtype}")
        K = torch.empty(self.B, self.Hkv, n, D, dtype=dtype, device=self.device)
        V = torch.empty_like(K)
        if n:
            check(lib().fathom_kv8_read(ptr(self.rows), ptr(self.scales), self.BH, self.cap, start, n,
                                        _lib.DTYPE_CODE[dtype], ptr(K), ptr(V), self._stream()),
                  "KVCache8.read")
        return K, V

    def attend(self, q, end):
        """softmax(q K^T / sqrt(128)) V of q [B, Hq, T, 128] (bf16 or fp16, any strides; Hq a multiple of Hkv):
        the T queries of a sequence are its last T tokens, already written, and query t sees the keys
        [0, end - (T - 1 - t)).  end: an int, or int64 [B] on the device (values above cap mean cap).  A query
        that sees no key gives 0; a NaN in a key or value reaches the queries that see it and no others.  Sums in fp32;
        q enters exactly or to 2^-21 (bf16) or 2^-25 (fp16) of its row's largest element, weights to 11 bits.  Returns
        [B, Hq, T, 128] in q's dtype, laid out as [B, T, Hq, 128]."""
        if torch._C._cuda_getDevice() != self.device.index:
            with torch.cuda.device(self.device):
                return self.attend(q, end)
        self._check_on("KVCache8.attend", q)
        if self.host:
            raise ValueError("KVCache8.attend: the rows are in host memory (attend_picks reads those)")
        shape = q.shape
        if len(shape) != 4 or shape[0] != self.B or shape[1] < 1 or shape[1] % self.Hkv or shape[3] != D:
            raise ValueError(f"KVCache8.attend: q must be [{self.B}, a multiple of {self.Hkv}, T, {D}] "
                             f"(got {tuple(shape)})")
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"KVCache8.attend: q must be bf16 or fp16 (got {q.dtype})")
        B, Hq, T, _ = shape
        num, dev = _position(end, B, self.device, "KVCache8.attend: end")
        if dev is None and not 0 <= num <= self.cap:
            raise ValueError(f"KVCache8.attend: end {num} is outside the cache's {self.cap}")
        out = torch.empty_strided(shape, (T * Hq * D, D, Hq * D, 1), dtype=q.dtype, device=self.device)
        if T == 0:
            return out
        q, sb, sh, st = _rows16(q)
        G = Hq // self.Hkv
        ws, nws = self._workspace((G, T), lib().fathom_kv8_attend_workspace_bytes, G, T)
        check(lib().fathom_kv8_attend(q.data_ptr(), _lib.DTYPE_CODE[q.dtype], B, self.Hkv, G, T, sb, sh, st,
                                      self.rows.data_ptr(), self.scales.data_ptr(), self.cap, num, ptr(dev),
                                      out.data_ptr(), T * Hq * D, D, Hq * D, ws.data_ptr(), nws, self._stream()),
              "KVCache8.attend")
        return out

    def attend_picks(self, q, idx, end=None):
        """Attention over listed tokens, as decode_attention over bf16 rows: q [BH, G, 128] (fp32, bf16 or fp16),
        idx [BH, G, k] int64.  Picks outside [0, end) are ignored (end: an int, int64 [B] on the device, or None
        for the whole cache); a pick listed twice counts twice; a head with no pick left gives 0.  Sums in fp32; q
        enters to 24 bits of its row's largest element, weights to 24 bits of the row's largest.  Returns [BH, G, 128]
        in q's dtype.  Of rows in host memory each distinct one of a KV head is fetched once over the link where
        G * k <= 16384; longer lists fetch a row for every pick."""
        if torch._C._cuda_getDevice() != self.device.index:
            with torch.cuda.device(self.device):
                return self.attend_picks(q, idx, end)
        self._check_on("KVCache8.attend_picks", q, idx)
        qs, ks = q.shape, idx.shape
        if len(qs) != 3 or qs[0] != self.BH or qs[1] < 1 or qs[2] != D:
            raise ValueError(f"KVCache8.attend_picks: q must be [{self.BH}, G, {D}] (got {tuple(qs)})")
        if q.dtype not in _lib.DTYPE_CODE:
            raise TypeError(f"KVCache8.attend_picks: q must be fp32, bf16 or fp16 (got {q.dtype})")
        BH, G, _ = qs
        if len(ks) != 3 or ks[0] != BH or ks[1] != G or idx.dtype != torch.int64:
            raise ValueError(f"KVCache8.attend_picks: idx must be int64 [{BH}, {G}, k] (got {idx.dtype} {tuple(ks)})")
        num, dev = _position(self.cap if end is None else end, self.B, self.device, "KVCache8.attend_picks: end")
        if dev is None and not 0 <= num <= self.cap:
            raise ValueError(f"KVCache8.attend_picks: end {num} is outside the cache's {self.cap}")
        k = ks[2]
        if k == 0:
            return torch.zeros(BH, G, D, dtype=q.dtype, device=self.device)
        q, idx = q.contiguous(), idx.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        out = torch.empty_like(q)
        ws, nws = self._unused, 256
        if self.host:
            ws, nws = self._workspace((G, k, "picks"), lib().fathom_kv8_attend_picks_workspace_bytes, G, k, 1)
        check(lib().fathom_kv8_attend_picks(q.data_ptr(), _lib.DTYPE_CODE[q.dtype], self.B, self.Hkv, G, idx.data_ptr(), k,
                                            self.rows.data_ptr(), int(self.host), self.scales.data_ptr(), self.cap, num,
                                            ptr(dev), out.data_ptr(), ws.data_ptr(), nws, self._stream()),
              "KVCache8.attend_picks")
        return out


def _rows16(x):
    """x with 16-byte aligned, contiguous 128-element rows (a copy where it has none), and its other strides."""
    sb, sh, st, sd = x.stride()
    if sd != 1 or (sb | sh | st) * x.element_size() % 16 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        sb, sh, st, sd = x.stride()
    return x, sb, sh, st
