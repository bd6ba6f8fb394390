"""Cases of the 8-bit key/value cache: writing it, reading it back, and the attention that reads it.

The cache of B sequences with Hkv KV heads each (row bh = b * Hkv + h) holds, per token, 128 key codes
and 128 value codes in e4m3, and per 64-token block one power-of-two scale for the keys and one for the
values:

    rows    uint8 [B * Hkv, cap, 2, 128]      code bytes; 0: key, 1: value
    scales  fp32  [B * Hkv, cap / 64, 2]      value = code * scale

  write   tokens [start, start + T) from K, V [B, Hkv, T, 128].  The scale of a block is 2^e with the
          smallest e in [-120, 120] such that every finite |x| <= 448 * 2^e; a block whose first tokens
          were written before keeps its scale if that is larger, and has those tokens' codes rounded to
          the new scale where it grew.  code = e4m3(x / scale), to nearest, ties to even; NaN and
          infinities become NaN.
  read    tokens [start, start + n) as K, V [B, Hkv, n, 128]
  attend  softmax(q K^T / sqrt(128)) V of q [B, Hq, T, 128], query t seeing the keys [0, end - (T - 1 - t))
  picks   the same over the listed keys idx [B * Hkv, G, k] of each query head, q [B * Hkv, G, 128]

`run` is one such call, in elementary torch operations or, where `own` is set, by fathom_b200.
"""
import math

import torch

own = False

BLK, D = 64, 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E_MIN, E_MAX = -120, 120


def listed():
    return [
        # one generated token appended to a 40k context (decode, one sequence): latency
        dict(name="write-token", op="write", B=1, Hkv=8, T=1, start=40001, ragged=False, dtype="bf16"),
        # one generated token for each of 32 sequences at their own lengths (batched decode)
        dict(name="write-token-batch", op="write", B=32, Hkv=4, T=1, start=8191, ragged=True, dtype="f16"),
        # the keys and values of a whole 128k prompt
        dict(name="write-prompt-128k", op="write", B=1, Hkv=8, T=131072, start=0, ragged=False, dtype="bf16"),
        # the whole 128k context read back (to build an index from, or for a dense pass)
        dict(name="read-128k", op="read", B=1, Hkv=8, start=0, n=131072, dtype="bf16"),
        # a stretch that begins and ends inside blocks, in 32 bits (statistics of the keys)
        dict(name="read-stretch-f32", op="read", B=2, Hkv=4, start=37, n=4097, dtype="f32"),
        # one token over a short context: latency
        dict(name="attend-token-700", op="attend", B=1, Hkv=8, G=4, T=1, n=700, ragged=False, dtype="bf16"),
        # one token over 128k: the cache's bytes
        dict(name="attend-token-128k", op="attend", B=1, Hkv=8, G=4, T=1, n=131072, ragged=False, dtype="bf16"),
        # 8 sequences of their own lengths up to 128k, 7 query heads to a KV head
        dict(name="attend-token-batch", op="attend", B=8, Hkv=4, G=7, T=1, n=131072, ragged=True, dtype="bf16"),
        # five drafted tokens checked at once over 16k
        dict(name="attend-draft-16k", op="attend", B=1, Hkv=8, G=4, T=5, n=16387, ragged=False, dtype="f16"),
        # a 2048-token prefill chunk at 32k
        dict(name="attend-chunk-32k", op="attend", B=1, Hkv=8, G=4, T=2048, n=34816, ragged=False, dtype="bf16"),
        # 512 selected tokens + 4 sinks + 64 local ones of a 128k context, one sequence, 32-bit queries
        dict(name="picks-580", op="picks", B=1, Hkv=8, G=4, k=580, n=131072, dtype="f32"),
        # 2048 + 68 of them for 8 sequences
        dict(name="picks-2116-batch", op="picks", B=8, Hkv=4, G=7, k=2116, n=131072, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["write", "write", "read", "attend", "attend", "attend", "picks"])
    B, Hkv, G = rng.choice([1, 1, 2, 3, 8]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    BH = B * Hkv
    if op == "write":
        T = rng.choice([1, _log(rng, 1, (1 << 20) // BH)])
        start = rng.choice([0, rng.randrange(0, 20000)])
        return dict(op=op, B=B, Hkv=Hkv, T=T, start=start, ragged=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if op == "read":
        dtype = rng.choice(["bf16", "f16", "f32"])
        return dict(op=op, B=B, Hkv=Hkv, start=rng.choice([0, rng.randrange(0, 5000)]),
                    n=_log(rng, 1, (1 << (19 if dtype == "f32" else 20)) // BH), dtype=dtype)
    if op == "picks":
        k = _log(rng, 1, 2116)
        return dict(op=op, B=B, Hkv=Hkv, G=G, k=k, n=max(k, _log(rng, 1, 131072)), dtype=rng.choice(["bf16", "f16", "f32"]))
    T = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    n = _log(rng, 1, min(131072, (1 << 22) // BH, 2048 * 34816 * 32 // (T * BH * G)))
    return dict(op=op, B=B, Hkv=Hkv, G=G, T=T, n=n, ragged=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "f16"]))


def _room(tokens):
    return -(-tokens // BLK) * BLK


def _kv(gen, BH, n):
    """Keys with a spread of channel scales (a few strong channels, as rotary keys have) and values."""
    gain = torch.exp(0.5 * torch.randn(BH, 1, D, generator=gen, device="cuda"))
    return torch.randn(BH, n, D, generator=gen, device="cuda") * gain, torch.randn(BH, n, D, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, Hkv, op = case["B"], case["Hkv"], case["op"]
    BH, dt = B * Hkv, DTYPES[case["dtype"]]
    s = dict(case, cache=None)
    if op == "write":
        T, cap = case["T"], _room(case["start"] + case["T"])
        s["K"], s["V"] = (x.to(dt).view(B, Hkv, T, D) for x in _kv(gen, BH, T))
        # the tokens before: any codes but NaN, at the scales of such keys and values
        rows = torch.randint(0, 127, (BH, cap, 2, D), generator=gen, device="cuda", dtype=torch.uint8)
        rows += 128 * torch.randint(0, 2, rows.shape, generator=gen, device="cuda", dtype=torch.uint8)
        scales = torch.exp2(torch.randint(-8, -5, (BH, cap // BLK, 2), generator=gen, device="cuda").float())
        s["start"] = case["start"]
        if case["ragged"]:
            s["start"] = torch.randint(0, case["start"] + 1, (B,), generator=gen, device="cuda")
    else:
        n = case["n"] + (case["start"] if op == "read" else 0)
        rows = torch.zeros(BH, _room(n), 2, D, dtype=torch.uint8, device="cuda")
        scales = torch.ones(BH, _room(n) // BLK, 2, device="cuda")
        K, V = _kv(gen, BH, n)
        plain_write(rows, scales, K.view(B, Hkv, n, D), V.view(B, Hkv, n, D), 0)
        if op == "attend":
            T, G = case["T"], case["G"]
            s["q"] = (2 * torch.randn(B, T, Hkv * G, D, generator=gen, device="cuda")).to(dt).transpose(1, 2)
            s["end"] = n
            if case["ragged"]:
                s["end"] = torch.randint(n // 4, n + 1, (B,), generator=gen, device="cuda")
        elif op == "picks":
            s["q"] = (2 * torch.randn(BH, case["G"], D, generator=gen, device="cuda")).to(dt)
            s["idx"] = torch.rand(BH, case["G"], n, generator=gen, device="cuda").topk(case["k"], -1).indices
    s["rows"], s["scales"] = rows, scales
    if own:     # the handle on the same tensors that a user's program keeps
        from fathom_b200.kv8 import KVCache8
        s["cache"] = KVCache8(B, Hkv, rows.shape[1], rows=rows, scales=scales)
    return s


# ---------------------------------------------------------------- plain forms
def _positions(pos, B, Hkv):
    """pos (a number, or one per sequence) as [B * Hkv] on the device."""
    p = torch.as_tensor(pos, device="cuda").to(torch.int64).reshape(-1).expand(B)
    return p.repeat_interleave(Hkv)


def plain_write(rows, scales, K, V, start):
    B, Hkv, T, _ = K.shape
    BH = B * Hkv
    p = _positions(start, B, Hkv)
    first, off = p // BLK, p % BLK
    nb = -(-(T + BLK - 1) // BLK)                                   # blocks that any start can touch
    blk = first[:, None] + torch.arange(nb, device="cuda")          # [BH, nb]
    live = blk * BLK < (p + T)[:, None]
    at = torch.arange(nb * BLK, device="cuda")[None] - off[:, None]  # index into K, V of each token of the blocks
    new = (at >= 0) & (at < T)
    blk = blk.clamp(max=scales.shape[1] - 1)
    tok = (blk[:, :, None] * BLK + torch.arange(BLK, device="cuda")).view(BH, -1)
    bh = torch.arange(BH, device="cuda")[:, None]
    x = torch.stack([K.reshape(BH, T, D), V.reshape(BH, T, D)], 2).float()[bh, at.clamp(0, T - 1)]
    x = torch.where(new[:, :, None, None], x, torch.zeros((), device="cuda")).view(BH, nb, BLK, 2, D)
    top = torch.where(x.isfinite(), x.abs(), torch.zeros((), device="cuda")).amax((2, 4))   # [BH, nb, 2]
    f, e = torch.frexp(top)                                         # top = f * 2^e, f in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(top > 0, e - 9 + (f > 0.875), E_MIN).clamp(E_MIN, E_MAX)
    s = torch.exp2(e.float())
    before = (torch.arange(nb, device="cuda")[None] == 0) & (off > 0)[:, None]              # the block was begun before
    old = scales[bh, blk]
    s = torch.where(before[:, :, None], torch.maximum(s, old), s)
    kept = rows[bh, tok].view(torch.float8_e4m3fn).float().view(BH, nb, BLK, 2, D)
    x = torch.where(x.isfinite(), x / s[:, :, None, :, None], torch.full((), math.nan, device="cuda"))
    y = torch.where(new.view(BH, nb, BLK, 1, 1), x, kept * (old / s)[:, :, None, :, None])
    code = y.to(torch.float8_e4m3fn).view(torch.uint8).view(BH, -1, 2, D)
    put = new | (before.repeat_interleave(BLK, 1) & (at < 0))
    put &= live.repeat_interleave(BLK, 1)
    rows[bh.expand_as(tok)[put], tok[put]] = code[put]
    scales[bh.expand_as(blk)[live], blk[live]] = s[live]


def _values(rows, scales, which):
    """The fp32 values of keys (0) or values (1): [BH, cap, 128]."""
    return rows[:, :, which].view(torch.float8_e4m3fn).float() * scales[:, :, which].repeat_interleave(BLK, 1)[..., None]


def _softmax_rows(sc, seen, V):
    """softmax over the seen keys of sc [..., R, n], times V [..., n, 128]; rows that see none give 0."""
    sc = torch.where(seen, sc, torch.full((), -math.inf, device="cuda"))
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, torch.zeros((), device="cuda"), m))
    total = p.sum(-1, keepdim=True)
    return (p @ V) / torch.where(total == 0, torch.ones((), device="cuda"), total)


def _plain(s):
    op, B, Hkv, rows, scales = s["op"], s["B"], s["Hkv"], s["rows"], s["scales"]
    if op == "write":
        plain_write(rows, scales, s["K"], s["V"], s["start"])
        return {"rows": rows.view(torch.float8_e4m3fn), "scales": scales}
    if op == "read":
        a, b, dt = s["start"], s["start"] + s["n"], DTYPES[s["dtype"]]
        return {x: _values(rows, scales, w)[:, a:b].to(dt).view(B, Hkv, b - a, D) for w, x in enumerate("KV")}
    q = s["q"]
    if op == "picks":
        BH, G, k = s["idx"].shape
        bh = torch.arange(BH, device="cuda")[:, None, None]
        K, V = _values(rows, scales, 0)[bh, s["idx"]], _values(rows, scales, 1)[bh, s["idx"]]   # [BH, G, k, 128]
        sc = (q.float()[:, :, None] @ K.transpose(-1, -2)) / math.sqrt(D)
        return _softmax_rows(sc, torch.ones((), dtype=torch.bool, device="cuda"), V)[:, :, 0].to(q.dtype)
    Hq, T = q.shape[1], q.shape[2]
    K, V = _values(rows, scales, 0), _values(rows, scales, 1)
    sc = (q.reshape(B * Hkv, -1, D).float() @ K.transpose(-1, -2)) / math.sqrt(D)
    sees = _positions(s["end"], B, Hkv)[:, None] - (T - 1) + torch.arange(T, device="cuda")     # keys seen by query t
    sees = sees.repeat(1, Hq // Hkv)
    seen = torch.arange(K.shape[1], device="cuda") < sees[:, :, None]
    return _softmax_rows(sc, seen, V).to(q.dtype).view(B, Hq, T, D)


def run(s):
    if not own:
        return _plain(s)
    c, op = s["cache"], s["op"]
    if op == "write":
        c.write(s["K"], s["V"], s["start"])
        return {"rows": s["rows"].view(torch.float8_e4m3fn), "scales": s["scales"]}
    if op == "read":
        K, V = c.read(s["start"], s["n"], dtype=DTYPES[s["dtype"]])
        return {"K": K, "V": V}
    if op == "picks":
        return c.attend_picks(s["q"], s["idx"])
    return c.attend(s["q"], s["end"])


# ---------------------------------------------------------------- work
def work(case):
    op, BH, elem = case["op"], case["B"] * case["Hkv"], 4 if case["dtype"] == "f32" else 2
    if op == "write":
        n = BH * case["T"]
        return {"bytes": n * 2 * D * (elem + 1) + n / BLK * 8, "flops": n * 2 * D * 2}
    if op == "read":
        n = BH * case["n"]
        return {"bytes": n * 2 * D * (elem + 1) + n / BLK * 8, "flops": n * 2 * D}
    G, n = case["G"], case["n"]
    if op == "picks":
        distinct = n * (1 - (1 - case["k"] / n) ** G)              # rows that some head of the group picked
        return {"bytes": BH * (distinct * 2 * D + G * case["k"] * 8 + G * D * 2 * elem), "flops": 4 * D * BH * G * case["k"]}
    T = case["T"]
    mean = n * 0.625 if case["ragged"] else n                       # lengths are spread over [n / 4, n]
    pairs = T * mean - min(T, mean) * (min(T, mean) - 1) / 2 if T <= mean else mean * (mean + 1) / 2
    return {"bytes": BH * (mean * (2 * D + 8 / BLK) + G * T * D * 2 * elem), "flops": 4 * D * BH * G * pairs}


# ---------------------------------------------------------------- 64 bits
def _codes64(b):
    """e4m3 bytes to the numbers they stand for, from the format: sign, 4 exponent bits (bias 7), 3 of mantissa."""
    table = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if (c & 127) == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        table.append(-v if c & 128 else v)
    return torch.tensor(table, dtype=torch.float64, device=b.device)[b.long()]


def _round64(y):
    """The e4m3 number nearest to each y (|y| <= 448), ties to even: multiples of 2^(exponent - 3), of 2^-9 at least."""
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(y), e - 4)
    return torch.round(y / step) * step


def _write64(s, pos):
    rows, scales = s["rows"], s["scales"]
    T = s["T"]
    out, sc = _codes64(rows), scales.double()
    for bh in range(rows.shape[0]):
        p = int(pos[bh])
        X = torch.stack([s["K"].flatten(0, 1)[bh], s["V"].flatten(0, 1)[bh]], 1).double()       # [T, 2, 128]
        b0, b1 = p // BLK, (p + T - 1) // BLK + 1
        lead, tail = p - b0 * BLK, b1 * BLK - p - T
        top = torch.cat([X.new_zeros(lead, 2), X.abs().amax(-1), X.new_zeros(tail, 2)]).view(b1 - b0, BLK, 2).amax(1)
        e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0) - 1e-12)
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e).clamp(E_MIN, E_MAX)
        new = torch.exp2(e)
        if lead:
            new[0] = torch.maximum(new[0], sc[bh, b0])
            out[bh, b0 * BLK:p] = _round64(out[bh, b0 * BLK:p] * (sc[bh, b0] / new[0])[None, :, None])
        sc[bh, b0:b1] = new
        out[bh, p:p + T] = _round64(X / new.repeat_interleave(BLK, 0)[lead:lead + T, :, None])
    return {"rows": out, "scales": sc}


def exact(case, seed):
    s = prepare(case, seed)
    op, B, Hkv = case["op"], case["B"], case["Hkv"]
    BH = B * Hkv
    per_row = lambda p: torch.as_tensor(p).reshape(-1).expand(B).repeat_interleave(Hkv).tolist()  # noqa: E731
    if op == "write":
        return _write64(s, per_row(s["start"]))
    scale = s["scales"].double().repeat_interleave(BLK, 1)
    if op == "read":
        a, b = case["start"], case["start"] + case["n"]
        val = _codes64(s["rows"][:, a:b]) * scale[:, a:b, :, None]
        return {"K": val[:, :, 0].reshape(B, Hkv, b - a, D), "V": val[:, :, 1].reshape(B, Hkv, b - a, D)}
    q = s["q"].double()
    if op == "picks":
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        for bh in range(BH):
            for g in range(case["G"]):
                i = s["idx"][bh, g]
                kv = _codes64(s["rows"][bh, i]) * scale[bh, i][:, :, None]
                w = torch.softmax((kv[:, 0] @ q[bh, g]) / math.sqrt(D), 0)
                out[bh, g] = w @ kv[:, 1]
        return out
    T, G = case["T"], case["G"]
    out = torch.zeros(B, Hkv * G, T, D, dtype=torch.float64, device="cuda")
    for bh, end in enumerate(per_row(s["end"])):
        b, h = divmod(bh, Hkv)
        kv = _codes64(s["rows"][bh, :end]) * scale[bh, :end, :, None]
        for g in range(G):
            w = (q[b, h * G + g] @ kv[:, 0].T) / math.sqrt(D)
            t = torch.arange(T, device="cuda")[:, None] + end - (T - 1)
            w.masked_fill_(torch.arange(end, device="cuda")[None] >= t, -math.inf)
            w = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)
            out[b, h * G + g] = w @ kv[:, 1]
    return out
