"""8-bit key/value cache: attention where the ranges of values, weights and scores are wide, against the formula in 64 bits.

Tolerances as in test_kv8_gpu.py: an output's own rounding, and 2^-10 of sum(weight * |V|) for weights of 11 bits."""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as O
from tests.test_kv8_gpu import DT, ROUND

pytestmark = pytest.mark.gpu


def _exact(q, c, ends):
    """(out, sum of weight * |V|) of q [B, Hq, T, 128] over the cache c, in 64 bits on the GPU."""
    B, Hq, T, _ = q.shape
    K, V = (torch.from_numpy(np.nan_to_num(x)).cuda() for x in O.values(c.rows.cpu().numpy(), c.scales.cpu().numpy()))
    out, mag = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    at = torch.arange(c.cap, device="cuda")
    G = Hq // c.Hkv
    for b, end in enumerate(ends):
        sees = min(max(int(end), 0), c.cap) - (T - 1 - torch.arange(T, device="cuda"))
        for h in range(c.Hkv):
            bh, heads = b * c.Hkv + h, slice(h * G, (h + 1) * G)
            s = (q[b, heads].double() @ K[bh].T) / 128 ** 0.5
            s.masked_fill_(at[None] >= sees[:, None], -np.inf)
            w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            out[b, heads], mag[b, heads] = w @ V[bh], w @ V[bh].abs()
    return out, mag


def _close(got, ref, mag, weights=2.0 ** -10):
    tol = ROUND[got.dtype] * ref.abs() + weights * mag + 1e-37
    off = (got.double() - ref).abs() / tol
    assert not (off > 1).any() and not off.isnan().any(), float(off.nan_to_num(np.inf).max())


def _cache(K, V, cap=None):
    from fathom_b200.kv8 import KVCache8
    B, H, n, _ = K.shape
    c = KVCache8(B, H, cap or n)
    c.write(K, V, 0)
    return c


def _normal(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("G,T", [(4, 65), (4, 70), (4, 80), (4, 129), (1, 300)])
def test_short_last_items_between_heads_of_other_scales(G, T, ragged):
    """Query rows of a KV head that leave at most 128 for its last 256, and values 2^-20, 2^20, .. by head and sequence:
    no head's rows meet another's scale."""
    B, H, n = 2, 4, 3000
    K, V = _normal(B, H, n, 128, seed=T), _normal(B, H, n, 128, seed=T + 1)
    V *= torch.exp2(20.0 * (2 * (torch.arange(B * H, device="cuda") % 2) - 1)).view(B, H, 1, 1)
    c = _cache(K, V)
    q = _normal(B, H * G, T, 128, seed=G, dtype=torch.bfloat16)
    ends = [n, 1777] if ragged else [n, n]
    ref, mag = _exact(q, c, ends)
    for _ in range(5):
        out = c.attend(q, torch.tensor(ends, device="cuda") if ragged else n)
        _close(out, ref, mag)


def _blocks(n, exponents):
    """2^exponent of each token's 64-token block, [n, 1]."""
    e = torch.tensor(exponents, device="cuda", dtype=torch.float32).repeat_interleave(64)[:n]
    return torch.exp2(e)[:, None]


@pytest.mark.parametrize("low,high", [(-70, 0), (-60, 60), (0, 60), (-110, 110)])
@pytest.mark.parametrize("G,T", [(1, 128), (1, 20), (4, 70), (2, 1)])
def test_rows_that_see_only_small_values(G, T, low, high):
    """Values near 2^low in the first tokens and near 2^high from the 64th on: queries of both keep their own range,
    whichever the number of query rows."""
    n = 128
    K, V = _normal(1, 2, n, 128, seed=T), _normal(1, 2, n, 128, seed=T + 1)
    c = _cache(K, V * _blocks(n, [low, high]))
    q = _normal(1, 2 * G, T, 128, seed=G, dtype=torch.bfloat16)
    for end in (n, 90, 64, 70):
        ref, mag = _exact(q, c, [end])
        _close(c.attend(q, end), ref, mag)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("G,T", [(4, 70), (1, 300), (8, 16), (4, 1), (4, 6)])
def test_values_of_blocks_of_any_scale(G, T, ragged):
    """Values 2^-60 .. 2^60 by block in no order, over contexts that several CTAs share; scores of some tens, so that the
    largest weights and the largest values lie apart."""
    B, H, n = 2, 2, 2500
    K, V = _normal(B, H, n, 128, seed=T), _normal(B, H, n, 128, seed=T + 1)
    e = torch.randint(-60, 61, (-(-n // 64),), generator=torch.Generator().manual_seed(G + T)).tolist()
    c = _cache(K, V * _blocks(n, e))
    q = _normal(B, H * G, T, 128, seed=G, dtype=torch.bfloat16) * 4
    ends = [n, 1300] if ragged else [n, n]
    ref, mag = _exact(q, c, ends)
    _close(c.attend(q, torch.tensor(ends, device="cuda") if ragged else n), ref, mag)


@pytest.mark.parametrize("e", [-100, 118])
@pytest.mark.parametrize("G,T", [(4, 80), (1, 40)])
def test_split_rows_of_the_largest_and_smallest_values(G, T, e):
    """Rows that several CTAs share, with values near the ends of fp32's range: no part leaves it."""
    n = 20011
    K, V = _normal(1, 1, n, 128, seed=1), _normal(1, 1, n, 128, seed=2)
    c = _cache(K, V * 2.0 ** e)
    q = _normal(1, G, T, 128, seed=3, dtype=torch.bfloat16) * 0.1
    ref, mag = _exact(q, c, [n])
    _close(c.attend(q, n), ref, mag)


def _steps(c, q, end):
    """What weights in steps of 2^-27 of a row's largest weight times value scale can be off by, [B, Hq, T, 1]: half a step
    of a code of at most 448 for every token (the reference may be half the largest)."""
    B, Hq, T, _ = q.shape
    scales = c.scales.double()[:, :, 1].repeat_interleave(64, 1)
    K = torch.from_numpy(np.nan_to_num(O.values(c.rows.cpu().numpy(), c.scales.cpu().numpy())[0])).cuda()
    out = torch.empty(B, Hq, T, 1, dtype=torch.float64, device="cuda")
    for b in range(B):
        for h in range(Hq):
            bh = b * c.Hkv + h // (Hq // c.Hkv)
            w = torch.softmax((q[b, h].double() @ K[bh, :end].T) / 128 ** 0.5, -1)
            out[b, h] = end * 2.0 ** -27 * 448 * (w * scales[bh, :end]).amax(-1, keepdim=True)
    return out


@pytest.mark.parametrize("heads", [1, 148])             # a row in many CTAs, or whole in one
@pytest.mark.parametrize("G,T", [(4, 1), (8, 1), (16, 1), (4, 5), (32, 1), (4, 20)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_long_tail_beside_one_dominant_key(heads, G, T, dtype):
    """One key 13, 14 and 16 nats above 20k equal ones, whose values have a common mean: the tail's weights, 2^-18 .. 2^-23
    of the largest, count in numerator and denominator alike."""
    n = 20480
    for extra in (9.0, 10.0, 11.0):                      # numbers of the cache's type: the scores are what is said here
        K = torch.zeros(1, 1, n, 128, device="cuda")
        K[..., :64] = 1.0
        K[0, 0, 5, 64:] = extra
        V = 1 + 0.25 * _normal(1, 1, n, 128, seed=1)
        V[0, 0, 5] *= 0.25
        one = _cache(K, V)
        q = torch.full((1, G, T, 128), 0.25, device="cuda", dtype=DT[dtype])
        ref, mag = _exact(q, one, [n])
        tol = 2.0 ** -10 * mag + _steps(one, q, n)
        c = one if heads == 1 else _cache(K.expand(heads, 1, n, 128), V.expand(heads, 1, n, 128))
        out = c.attend(q.expand(heads, G, T, 128), n)
        for b in {0, heads // 2, heads - 1}:
            _close(out[b:b + 1], ref, tol, 1.0)


@pytest.mark.parametrize("G,T", [(4, 1), (16, 1), (4, 6), (4, 20)])
def test_split_rows_of_large_values_of_one_sign(G, T):
    """Shares of ~70 tiles whose weighted sums, unlike their means, are above fp32's range."""
    n, H = 20011, 64
    K, V = _normal(1, 1, n, 128, seed=1), (1 + 0.1 * _normal(1, 1, n, 128, seed=2)) * 2.0 ** 118
    one = _cache(K, V)
    q = _normal(1, G, T, 128, seed=3, dtype=torch.bfloat16) * 0.1
    ref, mag = _exact(q, one, [n])
    c = _cache(K.expand(1, H, n, 128), V.expand(1, H, n, 128))
    out = c.attend(q.repeat(1, H, 1, 1), n).view(H, G, T, 128)
    for h in range(0, H, 9):
        _close(out[h:h + 1], ref, mag)


@pytest.mark.parametrize("amp", [2.0 ** 14, 2.0 ** 17])
@pytest.mark.parametrize("G,T", [(4, 1), (16, 1), (4, 5), (4, 40), (1, 300)])
def test_scores_of_millions(G, T, amp):
    """Scores up to 2^21 (fp32 holds them to 2^-3): where one key leads by far the output is its value, whatever the scores'
    size.  Rows whose two largest scores are within 64, which 32-bit scores may not tell apart, are left out."""
    n, H = 1500, 2
    K, V = _normal(1, H, n, 128, seed=T), _normal(1, H, n, 128, seed=T + 1)
    c = _cache(K, V)
    q = _normal(1, H * G, T, 128, seed=G, dtype=torch.bfloat16) * amp
    ref, mag = _exact(q, c, [n])
    Kd, Vd = (torch.from_numpy(x).cuda() for x in O.values(c.rows.cpu().numpy(), c.scales.cpu().numpy()))
    s = (q.double().view(H, G * T, 128) @ Kd[:, :n].transpose(1, 2)) / 128 ** 0.5
    sees = n - (T - 1 - torch.arange(T, device="cuda")).repeat(G)
    top = s.masked_fill(torch.arange(n, device="cuda") >= sees[:, None], -np.inf).topk(2, -1).values
    lead = (top[..., 0] - top[..., 1] > 64).view(1, H * G, T)
    assert lead.float().mean() > 0.9
    _close(c.attend(q, n)[lead], ref[lead], mag[lead])
    if T == 1:
        idx = torch.arange(n, device="cuda").expand(H, G, n).contiguous()
        for dtype in (torch.float32, torch.bfloat16):
            out = c.attend_picks(q.view(H, G, 128).to(dtype), idx).view_as(ref)
            _close(out[lead], ref[lead], mag[lead], 2.0 ** -17)


@pytest.mark.parametrize("dtype,bits", [("bf16", 21), ("f16", 25)])
@pytest.mark.parametrize("G,T", [(4, 1), (16, 1), (4, 5), (1, 40), (4, 80)])
def test_queries_of_wide_ranges(G, T, dtype, bits):
    """Elements of q from 2^-16 of the row's largest on, which alone decide the scores: they enter to 2^-bits of the largest
    at least, so a score is off by 2^-bits * max|q| * sum|k| / sqrt(128) at most, and an output by e^(2 * that) - 1 of
    sum(weight * |V|)."""
    n, H = 300, 2
    K, V = torch.zeros(1, H, n, 128, device="cuda"), _normal(1, H, n, 128, seed=T)
    K[..., 1:5] = _normal(1, H, n, 4, seed=T + 1) * 2.0 ** 17
    c = _cache(K, V)
    q = _normal(1, H * G, T, 128, seed=G) * 2.0 ** -14
    q[..., 0] = 1.0
    q = q.to(DT[dtype])
    ref, mag = _exact(q, c, [n])
    Kc = torch.from_numpy(O.values(c.rows.cpu().numpy(), c.scales.cpu().numpy())[0]).cuda()[:, :n]
    off = 2.0 ** -bits * float(q.abs().max()) * float(Kc.abs().sum(-1).max()) / 128 ** 0.5
    _close(c.attend(q, n), ref, mag, 2.0 ** -10 + np.expm1(2 * off))


@pytest.mark.parametrize("G,T", [(4, 1), (8, 1), (4, 5), (4, 40), (4, 80)])
def test_more_sequences_than_a_warp_has_lanes(G, T):
    """40 sequences at their own device lengths, some empty, some a few tiles long, some in many CTAs."""
    B, H, n = 40, 2, 6000
    K, V = _normal(1, H, n, 128, seed=T), _normal(1, H, n, 128, seed=T + 1)
    c = _cache(K.expand(B, H, n, 128), V.expand(B, H, n, 128))
    q = _normal(B, H * G, T, 128, seed=G, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(T)
    ends = [0, 1, n, 128, 129] + torch.randint(0, n + 1, (B - 5,), generator=g).tolist()
    ref, mag = _exact(q, c, ends)
    _close(c.attend(q, torch.tensor(ends, device="cuda")), ref, mag)
