"""8-bit key/value cache on the GPU against its 64-bit oracle.

Tolerances, from the arithmetic: codes and scales are exact.  An output in b-bit significand rounds by at most
2^-b of itself; a weight kept in 16 bits is off by at most 2^-11 of itself, so the sum by 2^-11 of
sum(weight * |V|); 2^-10 of it leaves room for the fp32 sums.  In fp32 throughout: 2^-17 of
sum(weight * |V|) (scores of some tens, off by 2^-22 of themselves)."""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as O

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROUND = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}


def _np(x):
    return x.detach().double().cpu().numpy()


def _kv(B, H, T, dtype, seed, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    gain = torch.exp(0.5 * torch.randn(B, H, 1, 128, generator=g))
    K, V = torch.randn(B, H, T, 128, generator=g) * gain, torch.randn(B, H, T, 128, generator=g)
    return K.to(dtype).to(dev), V.to(dtype).to(dev)


def _filled(B, H, n, seed, cap=None):
    """A cache holding n random tokens, and its rows and scales on the host.  The void tokens hold NaN codes."""
    from fathom_b200.kv8 import KVCache8
    c = KVCache8(B, H, cap or max(n, 1))
    c.rows.fill_(255)
    c.scales.fill_(float("nan"))
    if n:
        K, V = _kv(B, H, n, torch.float32, seed)
        c.write(K, V, 0)
    return c, c.rows.cpu().numpy(), np.nan_to_num(c.scales.cpu().numpy(), nan=1.0)


def _close(got, ref, mag, weights=2.0 ** -10):
    tol = ROUND[got.dtype] * np.abs(ref) + weights * mag + 1e-30
    bad = np.abs(_np(got) - ref) > tol
    assert not bad.any(), float((np.abs(_np(got) - ref) / tol).max())


# ---------------------------------------------------------------- write, read
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,start", [(1, 0), (1, 63), (1, 64), (1, 200), (2, 63), (64, 0), (65, 0), (63, 1), (130, 37),
                                     (257, 128)])
def test_write_matches_the_oracle(dtype, T, start):
    from fathom_b200.kv8 import KVCache8
    B, H = 2, 3
    c = KVCache8(B, H, 400)
    K0, V0 = _kv(B, H, 300, DT[dtype], 1)
    c.write(0.25 * K0, 0.25 * V0, 0)                   # tokens before (and some that are overwritten)
    rows, scales = c.rows.cpu().numpy(), c.scales.cpu().numpy()
    K, V = _kv(B, H, T, DT[dtype], T + start)
    K[0, 0] *= 8                                       # the begun block's scale grows in some rows only
    c.write(K, V, start)
    O.write(rows, scales, _np(K).reshape(6, T, 128), _np(V).reshape(6, T, 128), [start] * 6)
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    assert np.array_equal(c.rows.cpu().numpy(), rows)


def test_write_at_device_positions_per_sequence():
    from fathom_b200.kv8 import KVCache8
    B, H, T = 5, 2, 70
    c = KVCache8(B, H, 256)
    K0, V0 = _kv(B, H, 256, torch.bfloat16, 2)
    c.write(K0, V0, 0)
    rows, scales = c.rows.cpu().numpy(), c.scales.cpu().numpy()
    K, V = _kv(B, H, T, torch.bfloat16, 3)
    start = [0, 63, -1, 200, 255]                      # -1: left alone; 200, 255: the tokens past cap are dropped
    c.write(2 * K, V, torch.tensor(start, device="cuda"))
    O.write(rows, scales, _np(2 * K).reshape(-1, T, 128), _np(V).reshape(-1, T, 128), np.repeat(start, H))
    assert np.array_equal(c.rows.cpu().numpy(), rows) and np.array_equal(c.scales.cpu().numpy(), scales)
    c.write(K, V, torch.tensor([256, 2 ** 62, -5, -1, 10 ** 9], device="cuda"))      # nothing in range: nothing written
    assert np.array_equal(c.rows.cpu().numpy(), rows) and np.array_equal(c.scales.cpu().numpy(), scales)


def test_tokens_one_by_one_equal_the_oracle():
    """A block filled token by token, its amplitude growing, shrinking and spanning 40 binary orders."""
    from fathom_b200.kv8 import KVCache8
    c = KVCache8(1, 2, 128)
    rows, scales = c.rows.cpu().numpy(), c.scales.cpu().numpy()
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    for t in range(130 - 2):
        K, V = _kv(1, 2, 1, torch.float32, 100 + t)
        K, V = K * 2.0 ** ((t * 7) % 41 - 20), V * 2.0 ** (-t // 8)
        c.write(K, V, pos)
        pos += 1
        O.write(rows, scales, _np(K)[0], _np(V)[0], [t, t])
    assert np.array_equal(c.rows.cpu().numpy(), rows) and np.array_equal(c.scales.cpu().numpy(), scales)


def test_write_extreme_values():
    """Zeros, subnormals, the largest floats, NaN and infinities (stored as NaN, outside the scale)."""
    from fathom_b200.kv8 import KVCache8
    c = KVCache8(1, 1, 512)
    K, V = _kv(1, 1, 512, torch.float32, 5)
    K[0, 0, :64] = 0
    K[0, 0, 64:128] *= 2.0 ** -140
    K[0, 0, 128:192] = 3e38
    K[0, 0, 200, 3], K[0, 0, 201, 4], K[0, 0, 202, 5] = float("nan"), float("inf"), -float("inf")
    V[0, 0, 256:320] = float("nan")
    V[0, 0, 330, 7] = 1e30
    rows, scales = c.rows.cpu().numpy(), c.scales.cpu().numpy()
    c.write(K, V, 0)
    O.write(rows, scales, _np(K)[0], _np(V)[0], [0])
    got = c.rows.cpu().numpy()
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    nan = (rows & 127) == 127
    assert np.array_equal((got & 127) == 127, nan) and np.array_equal(got[~nan], rows[~nan])


@pytest.mark.parametrize("layout", ["bthd", "offset", "broadcast", "reversed"])
def test_write_takes_any_strides(layout):
    from fathom_b200.kv8 import KVCache8
    B, H, T = 2, 4, 100
    K, V = _kv(B, H, T, torch.bfloat16, 6)
    if layout == "bthd":
        K2, V2 = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (K, V))
    elif layout == "offset":                            # rows 2 bytes off any 16-byte boundary
        K2, V2 = (torch.empty(B * H * T * 128 + 1, dtype=K.dtype, device="cuda")[1:].view(K.shape).copy_(x)
                  for x in (K, V))
    elif layout == "broadcast":
        K, V = K[:, :1].expand(B, H, T, 128), V[:, :, :1].expand(B, H, T, 128)
        K2, V2 = K, V
    else:
        K2, V2 = (torch.stack([x, x], -1).transpose(-1, -2)[..., 0, :] for x in (K, V))
    a, b = KVCache8(B, H, T), KVCache8(B, H, T)
    a.write(K.contiguous(), V.contiguous())
    b.write(K2, V2)
    assert torch.equal(a.rows, b.rows) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("start,n", [(0, 1), (0, 320), (63, 2), (37, 203), (319, 1), (100, 0)])
def test_read_matches_the_oracle(dtype, start, n):
    c, rows, scales = _filled(2, 3, 320, 7)
    K, V = c.read(start, n, dtype=DT[dtype])
    Kr, Vr = O.values(rows, scales)
    for got, ref in ((K, Kr), (V, Vr)):
        ref = torch.from_numpy(ref[:, start:start + n]).to(DT[dtype]).view(2, 3, n, 128)
        assert got.dtype == DT[dtype] and torch.equal(got.cpu(), ref)


def test_read_beyond_32_bit_offsets():
    """A cache of 5.2 GB: tokens at its far end are written, read and attended to."""
    from fathom_b200.kv8 import KVCache8
    n = 10_200_000
    c = KVCache8(1, 2, n)
    K, V = _kv(1, 2, 200, torch.bfloat16, 8)
    c.write(K, V, n - 200)
    K2, V2 = c.read(n - 200, 200)
    small = KVCache8(1, 2, 256 + n % 64)
    small.write(K, V, (n - 200) % 64)                   # the same place within a block
    K3, V3 = small.read((n - 200) % 64, 200)
    assert torch.equal(K2, K3) and torch.equal(V2, V3)
    q = torch.randn(2, 4, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    idx = torch.randint(0, 200, (2, 4, 50), device="cuda", generator=torch.Generator("cuda").manual_seed(10))
    assert torch.equal(c.attend_picks(q, idx + n - 200), small.attend_picks(q, idx + (n - 200) % 64))
    # dense: every other key is 0 (score 0) with value 0, so the far tokens' weights come against n - 200 ones
    q = 6 * q.bfloat16().view(1, 8, 1, 128)
    out = c.attend(q, n)
    s = torch.einsum("hgd,hnd->hgn", q.double().view(2, 4, 128), K3[0].double()) / 128 ** 0.5
    w = s.exp() / (s.exp().sum(-1, keepdim=True) + (n - 200))
    ref, mag = w @ V3[0].double(), w @ V3[0].double().abs()
    _close(out.view(2, 4, 128), _np(ref), _np(mag))


# ---------------------------------------------------------------- attention over the cache
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("G,T,n", [(4, 1, 1), (4, 1, 63), (4, 1, 64), (1, 1, 65), (7, 1, 129), (8, 1, 700), (5, 1, 1111),
                                   (12, 1, 300), (33, 1, 200), (4, 2, 130), (4, 5, 387), (1, 33, 100), (7, 8, 250),
                                   (4, 64, 64), (2, 130, 257), (3, 100, 40), (4, 70, 900), (1, 300, 300),
                                   (8, 4, 300), (1, 17, 64), (32, 1, 1500), (3, 10, 11), (5, 6, 129)])
def test_attend_matches_the_oracle(dtype, G, T, n):
    B, H = 2, 2
    c, rows, scales = _filled(B, H, n, G * T + n, cap=n + 70)
    g = torch.Generator().manual_seed(n)
    q = (2 * torch.randn(B, H * G, T, 128, generator=g)).to(DT[dtype])
    ref, mag = O.attend(_np(q), rows, scales, [n] * B, H)
    out = c.attend(q.cuda(), n)
    assert out.dtype == q.dtype and out.shape == q.shape
    _close(out, ref, mag)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("G,T,n", [(4, 5, 1000), (3, 6, 777), (6, 3, 65), (8, 3, 640), (1, 24, 300), (5, 5, 901), (1, 18, 20),
                                   (1, 25, 128), (7, 4, 515), (4, 8, 2049)])
def test_attend_of_17_to_32_rows(dtype, G, T, n):
    """Rows shared by two groups of threads, at one length and at ragged ones (the first rows of which see nothing)."""
    B, H = 3, 2
    c, rows, scales = _filled(B, H, n, G + T + n, cap=n + 40)
    q = (2 * torch.randn(B, H * G, T, 128, generator=torch.Generator().manual_seed(n))).to(DT[dtype])
    for ends in ([n] * B, [n, T - 2, n // 2]):
        ref, mag = O.attend(_np(q), rows, scales, ends, H)
        _close(c.attend(q.cuda(), torch.tensor(ends, device="cuda")), ref, mag)


@pytest.mark.parametrize("T", [1, 3, 7, 40, 129])
def test_attend_at_device_lengths(T):
    """Ragged lengths on the device: none, one, fewer than the queries, a block's edge, the whole cache, above it."""
    ends = [0, 1, 2, 64, 65, 191, 192, 500, 640, 10 ** 12, -3]
    B, H, G = len(ends), 1, 4
    c, rows, scales = _filled(B, H, 640, T)
    q = (2 * torch.randn(B, H * G, T, 128, generator=torch.Generator().manual_seed(T))).bfloat16()
    ref, mag = O.attend(_np(q), rows, scales, ends, H)
    out = c.attend(q.cuda(), torch.tensor(ends, device="cuda"))
    _close(out, ref, mag)
    assert not out[0].any() and not out[-1].any()       # rows that see nothing


@pytest.mark.parametrize("T", [1, 4, 6, 80])
def test_attend_splits_a_long_context(T):
    n, G = 20011, 4
    c, rows, scales = _filled(1, 1, n, 11)
    q = (2 * torch.randn(1, G, T, 128, generator=torch.Generator().manual_seed(T))).bfloat16()
    K, V = (torch.from_numpy(x).cuda() for x in O.values(rows, scales))
    s = torch.einsum("gtd,nd->gtn", q[0].double().cuda(), K[0]) / 128 ** 0.5
    s.masked_fill_(torch.arange(c.cap, device="cuda") >= n - (T - 1 - torch.arange(T, device="cuda"))[:, None], -np.inf)
    w = torch.softmax(s, -1)
    V = torch.nan_to_num(V[0])
    _close(c.attend(q.cuda(), n)[0], _np(w @ V), _np(w @ V.abs()))


def test_attend_peaked_and_flat_weights():
    """Scores of hundreds (one key takes all), equal scores, and values of very different block scales."""
    from fathom_b200.kv8 import KVCache8
    n, G = 1000, 4
    K, V = _kv(1, 2, n, torch.float32, 12)
    K[:, 1] = 0.0
    V[0, 0, 320:384] *= 2.0 ** 14
    V[0, 0, 640:704] *= 2.0 ** -14
    V[0, 1, 64:128] = 0
    c = KVCache8(1, 2, n)
    c.write(K, V)
    for amp in (0.0, 1.0, 60.0):
        for T in (1, 3, 6, 50):
            q = (amp * torch.randn(1, 2 * G, T, 128, generator=torch.Generator().manual_seed(13))).bfloat16()
            ref, mag = O.attend(_np(q), c.rows.cpu().numpy(), c.scales.cpu().numpy(), [n], 2)
            _close(c.attend(q.cuda(), n), ref, mag)


@pytest.mark.parametrize("T", [1, 5, 64, 200])
def test_attend_reads_no_void_token_and_nan_reaches_only_who_sees_it(T):
    """Codes past `end` are NaN (set by _filled).  A NaN value at token j of the last T reaches the queries that
    see j and no other."""
    n, G = 333, 4
    c, rows, scales = _filled(1, 2, n, 14, cap=512)
    q = (2 * torch.randn(1, 2 * G, T, 128, generator=torch.Generator().manual_seed(T))).bfloat16().cuda()
    clean = c.attend(q, n)
    assert clean.isfinite().all()
    j = n - 1 - T // 2
    for which in (0, 1):
        rows = c.rows.clone()
        c.rows[:, j, which, 17] = 127
        out = c.attend(q, n)
        c.rows.copy_(rows)
        sees = n - (T - 1 - torch.arange(T, device="cuda")) > j
        assert torch.equal(out[:, :, ~sees], clean[:, :, ~sees])
        assert out[:, :, sees].isnan().any(-1).all()


def test_attend_takes_strided_queries_and_other_streams():
    c, rows, scales = _filled(2, 2, 400, 15)
    q = (2 * torch.randn(2, 8, 6, 128, generator=torch.Generator().manual_seed(1))).bfloat16().cuda()
    ref = c.attend(q, 400)
    assert torch.equal(c.attend(q.transpose(1, 2).contiguous().transpose(1, 2), 400), ref)
    wide = torch.empty(2, 8, 6, 129, dtype=q.dtype, device="cuda")
    wide[..., 1:] = q
    assert torch.equal(c.attend(wide[..., 1:], 400), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.attend(q, 400)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    for _ in range(5):                                   # the same bits every time
        assert torch.equal(c.attend(q, 400), ref)


def test_a_decode_step_in_a_cuda_graph():
    """write + attend + attend_picks with positions on the device, captured once and replayed as the sequence grows."""
    from fathom_b200.kv8 import KVCache8
    B, H, G, n0, steps = 2, 2, 4, 125, 6
    caches = [KVCache8(B, H, 256) for _ in range(2)]
    K, V = _kv(B, H, n0 + steps, torch.bfloat16, 16)
    for c in caches:
        c.write(K[:, :, :n0], V[:, :, :n0])
    k, v = torch.empty(B, H, 1, 128, dtype=K.dtype, device="cuda"), torch.empty(B, H, 1, 128, dtype=K.dtype, device="cuda")
    pos, q = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.empty(B, H * G, 1, 128, dtype=K.dtype, device="cuda")
    idx = torch.randint(0, n0, (B * H, G, 40), device="cuda")

    def step(c):
        c.write(k, v, pos)
        return c.attend(q, pos + 1), c.attend_picks(q.view(B * H, G, 128), idx, pos + 1)

    k.copy_(K[:, :, n0:n0 + 1]), v.copy_(V[:, :, n0:n0 + 1]), q.normal_(), pos.fill_(n0)
    step(caches[0])                                      # warm-up on the first position
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, p = step(caches[0])
    for s in range(steps):
        k.copy_(K[:, :, n0 + s:n0 + s + 1]), v.copy_(V[:, :, n0 + s:n0 + s + 1]), pos.fill_(n0 + s)
        q.normal_(generator=torch.Generator("cuda").manual_seed(s))
        graph.replay()
        a2, p2 = step(caches[1])
        assert torch.equal(a, a2) and torch.equal(p, p2)
    assert torch.equal(caches[0].rows, caches[1].rows)


# ---------------------------------------------------------------- attention over listed tokens
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,H,G,k", [(1, 1, 1, 1), (1, 2, 4, 33), (2, 2, 7, 580), (1, 1, 8, 64), (3, 1, 3, 7),
                                     (2, 8, 20, 50), (1, 1, 40, 130)])
def test_picks_match_the_oracle(dtype, B, H, G, k):
    n = 700
    c, rows, scales = _filled(B, H, n, k)
    g = torch.Generator().manual_seed(k)
    q = (2 * torch.randn(B * H, G, 128, generator=g)).to(DT[dtype])
    idx = torch.randint(0, n, (B * H, G, k), generator=g)
    ref, mag = O.attend_picks(_np(q), idx.numpy(), rows, scales, [n] * (B * H))
    _close(c.attend_picks(q.cuda(), idx.cuda()), ref, mag, 2.0 ** -17)


@pytest.mark.parametrize("k", [31, 32, 33, 95, 200])
def test_picks_of_wide_ranges(k):
    """Values of very different block scales, queries of very different elements, lists around whole steps of 32."""
    from fathom_b200.kv8 import KVCache8
    n, H, G = 512, 2, 3
    K, V = _kv(1, H, n, torch.float32, k)
    V[:, 0, 64:128] *= 2.0 ** 30
    V[:, 0, 256:320] *= 2.0 ** -30
    V[:, 1, :64] = 0
    K[:, 1, 128:192] *= 2.0 ** -20
    c = KVCache8(1, H, n)
    c.write(K, V)
    g = torch.Generator().manual_seed(k)
    q = 2 * torch.randn(H, G, 128, generator=g)
    q[:, 1] *= torch.exp2(torch.randint(-30, 1, (128,), generator=g).float())
    q[:, 2] = 0
    idx = torch.randint(0, n, (H, G, k), generator=g)
    rows, scales = c.rows.cpu().numpy(), c.scales.cpu().numpy()
    ref, mag = O.attend_picks(_np(q), idx.numpy(), rows, scales, [n] * H)
    _close(c.attend_picks(q.cuda(), idx.cuda()), ref, mag, 2.0 ** -17)


def test_calls_in_a_row_see_each_other():
    """Each call may be launched while the one before it ends: 40 steps whose inputs are the outputs before them give the
    same bits as with a wait after every call."""
    from fathom_b200.kv8 import KVCache8
    B, H, G, n0 = 2, 4, 4, 500
    K, V = _kv(B, H, n0, torch.bfloat16, 50)
    idx = torch.randint(0, n0, (B * H, G, 100), generator=torch.Generator().manual_seed(51)).cuda()

    def steps(wait):
        c = KVCache8(B, H, 1024)
        done = torch.cuda.synchronize if wait else (lambda: None)
        c.write(K, V, 0)
        pos = torch.full((B,), n0, device="cuda")
        out = K[:, :, -1:].repeat_interleave(G, 1)
        for t in range(40):
            c.write(out[:, ::G], out[:, 1::G], pos)
            done()
            pos += 1
            x = c.attend((out + K[:, :, t:t + 1].repeat_interleave(G, 1)).contiguous(), pos if t % 2 else n0 + t + 1)
            done()
            y = c.attend_picks(x.reshape(B * H, G, 128), idx + t, pos)
            done()
            z, _ = c.read(n0 + t, 1)
            done()
            out = x + y.view_as(x) + z.repeat_interleave(G, 1)
        return out

    assert torch.equal(steps(False), steps(True))


def test_picks_outside_are_ignored():
    B, H, G, k, n = 3, 2, 4, 45, 300
    c, rows, scales = _filled(B, H, n, 20, cap=400)
    g = torch.Generator().manual_seed(21)
    q = torch.randn(B * H, G, 128, generator=g)
    idx = torch.randint(-100, 500, (B * H, G, k), generator=g)
    idx[0, 0] = torch.arange(n, n + k)                   # nothing left: zeros
    idx[1, 1] = -1
    idx[2, 2] = 2 ** 40 + torch.arange(k)
    idx[3, 3] = 7                                        # one token listed k times
    ends = torch.tensor([n, 0, 171], device="cuda")
    for end, per in ((n, [n] * 6), (ends, [n, n, 0, 0, 171, 171])):
        ref, mag = O.attend_picks(_np(q), idx.numpy(), rows, scales, per)
        out = c.attend_picks(q.cuda(), idx.cuda(), end)
        _close(out, ref, mag, 2.0 ** -17)
        assert not out[0, 0].any() and not out[1, 1].any() and not out[2, 2].any()


@pytest.mark.parametrize("G,k", [(4, 580), (1, 1), (8, 64), (7, 3000)])       # 7 * 3000 > 16384: read in place
def test_picks_from_host_rows_equal_device_rows(G, k):
    from fathom_b200.kv8 import KVCache8
    B, H, n = 2, 2, 5000
    K, V = _kv(B, H, n + 3, torch.bfloat16, 30)
    dev, host = KVCache8(B, H, n + 50), KVCache8(B, H, n + 50, host=True)
    g = torch.Generator().manual_seed(k)
    idx = torch.randint(-5, n + 60, (B * H, G, k), generator=g).cuda()
    idx[:, :, : k // 3] = idx[:, :1, : k // 3]                  # shared picks across the group
    q = torch.randn(B * H, G, 128, generator=g).cuda()
    ends = torch.tensor([n + 3, 100], device="cuda")
    for c in (dev, host):
        c.write(K[:, :, :n], V[:, :, :n])
        for t in range(3):                                      # and token by token, over the link
            c.write(K[:, :, n + t:n + t + 1], V[:, :, n + t:n + t + 1], n + t)
    for end in (n + 3, ends):
        assert torch.equal(host.attend_picks(q, idx, end), dev.attend_picks(q, idx, end))
    for x, y in zip(host.read(0, n + 3), dev.read(0, n + 3)):
        assert torch.equal(x, y)
    with pytest.raises(ValueError, match="host"):
        host.attend(q[:, :, None].bfloat16().view(B, H * G, 1, 128), n)
    torch.cuda.synchronize()
    host.free()


def test_python_layer_refuses():
    from fathom_b200.kv8 import KVCache8
    c = KVCache8(2, 2, 100)
    assert c.cap == 128
    K, V = _kv(2, 2, 10, torch.bfloat16, 1)
    q = torch.zeros(2, 8, 1, 128, dtype=torch.bfloat16, device="cuda")
    idx = torch.zeros(4, 4, 3, dtype=torch.int64, device="cuda")
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (lambda: c.write(K, V, 119), lambda: c.write(K, V, -1), lambda: c.write(K, V[:, :, :5]),
                lambda: c.write(K[:, :1], V[:, :1]), lambda: c.write(K[..., :64], V[..., :64]),
                lambda: c.write(K, V, pos.int()), lambda: c.write(K, V, pos.cpu()), lambda: c.write(K.cpu(), V.cpu()),
                lambda: c.write(K, V, torch.zeros(3, dtype=torch.int64, device="cuda")),
                lambda: c.read(0, 129), lambda: c.read(-1, 5), lambda: c.attend(q, 129), lambda: c.attend(q[:, :3], 5),
                lambda: c.attend(q[0], 5), lambda: c.attend(q, -1), lambda: c.attend_picks(q[:, :, 0], idx),
                lambda: c.attend_picks(q.view(4, 4, 128), idx.int()), lambda: c.attend_picks(q.view(4, 4, 128), idx[:, :2]),
                lambda: c.attend_picks(q.view(4, 4, 128), idx, 129),
                lambda: KVCache8(2, 2, 128, rows=c.rows[:3], scales=c.scales)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.write(K, V.float()), lambda: c.write(K.double(), V.double()), lambda: c.attend(q.float(), 5),
                lambda: c.read(0, 5, torch.float64), lambda: c.attend_picks(q.view(4, 4, 128).double(), idx)):
        with pytest.raises(TypeError):
            bad()
    assert c.attend(q[:, :, :0], 0).shape == (2, 8, 0, 128)
    assert not c.attend_picks(q.view(4, 4, 128), idx[..., :0]).any()
    c.write(K[:, :, :0], V[:, :, :0], 128)
