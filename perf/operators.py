"""
Measured cases of the 4-bit KV cache and of attention with modified scores.

Three operators, each as a serving program calls it:

``cache``   new keys and values are written into a 4-bit paged pool, and the
            context (old rows and new ones) is read back dequantised.
``q4``      attention over a 4-bit paged pool: one-token decode, a verify run of
            a few rows, chunks of a prompt.
``scored``  attention over a 16-bit paged pool with capped scores, a bias that
            grows with distance, a sliding window, a prefix that every row sees.

The 4-bit pool of one layer is ``uint8 (blocks, kv_heads, 16 * D + 128)``: one
record for the 16 tokens of a block and one kv head.  A row x of D values is held
as codes n in 0..15 and two fp16 numbers, x ~ n * scale + base:
base is the largest fp16 not above min(x), scale the smallest fp16 with
15 * scale >= max(x) - base, n = (x - base) / scale rounded to nearest even.
A row that holds a NaN or a magnitude above 65504 has NaN for both.  A record is

* bytes 0 .. 8D-1: K codes, ``[16 tokens][D / 2]``, even dim in the low nibble;
* bytes 8D .. 16D-1: V codes, ``[C][token >> 3][8][(token >> 1) & 3][W][token & 1][2]``
  with C = max(1, D / 128) chunks and W = min(4, D / 32): chunk c, group g, word w
  hold dims c * 128 + g * 4W + 4w .. + 3, the even dim in the low nibble;
* 64 bytes of K parameters ``[16][scale, base]``, then 64 of V parameters.

``own`` selects the framework's calls; otherwise plain torch operations.
"""

import math

import torch

own = False

BLOCK = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------- cases

def listed():
    cache = dict(kind="cache")
    att = dict(softcap=0.0, window=0, slopes=False, prefix=0)
    q4 = dict(kind="q4", **att)
    sc = dict(kind="scored")
    return [
        # one decode step's write for a handful of chats, then their short contexts read back
        dict(cache, name="cache step", dtype="bf16", batch=8, lo=40, hi=300, new=1, hkv=8, d=128),
        # long prompts written at once, of an odd length
        dict(cache, name="cache prompt", dtype="bf16", batch=4, lo=4001, hi=4001, new=4001,
             hkv=8, d=128),
        # prompt chunks of many requests behind cached prefixes, small heads
        dict(cache, name="cache chunk", dtype="f16", batch=32, lo=300, hi=2100, new=129, hkv=4,
             d=64),
        # one chat's next token: latency
        dict(q4, name="q4 step", dtype="bf16", batch=1, lo=1000, hi=1000, qlo=1, qhi=1, hq=32,
             hkv=8, d=128),
        # a serving batch's decode step
        dict(q4, name="q4 decode", dtype="bf16", batch=64, lo=500, hi=4096, qlo=1, qhi=1, hq=32,
             hkv=8, d=128),
        # long contexts, eight query heads for each kv head
        dict(q4, name="q4 decode long", dtype="bf16", batch=48, lo=4096, hi=16384, qlo=1, qhi=1,
             hq=64, hkv=8, d=128),
        # drafts verified: five rows for each sequence, five query heads for each kv head
        dict(q4, name="q4 verify", dtype="f16", batch=16, lo=700, hi=6001, qlo=5, qhi=5, hq=40,
             hkv=8, d=128),
        # chunks of prompts behind cached prefixes, ragged
        dict(q4, name="q4 chunk", dtype="bf16", batch=4, lo=2000, hi=8000, qlo=300, qhi=2048,
             hq=32, hkv=8, d=128),
        # decode of a model that caps its scores and sees a sliding window
        dict(sc, name="scored decode", dtype="bf16", batch=32, lo=900, hi=12000, qlo=1, qhi=1,
             hq=16, hkv=8, d=128, softcap=50.0, window=4096, slopes=False, prefix=0),
        # decode with a bias by distance, one kv head for each query head
        dict(sc, name="scored decode bias", dtype="f16", batch=16, lo=33, hi=2047, qlo=1, qhi=1,
             hq=32, hkv=32, d=128, softcap=0.0, window=0, slopes=True, prefix=0),
        # prompt chunks with capped scores
        dict(sc, name="scored chunk", dtype="bf16", batch=2, lo=6000, hi=8192, qlo=2048, qhi=2048,
             hq=32, hkv=8, d=128, softcap=30.0, window=0, slopes=False, prefix=0),
        # ragged chunks under a window, with first tokens that stay visible
        dict(sc, name="scored chunk window", dtype="bf16", batch=8, lo=700, hi=5000, qlo=100,
             qhi=700, hq=32, hkv=8, d=128, softcap=0.0, window=1024, slopes=False, prefix=64),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "q4", "scored"])
    if kind == "cache":
        d = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        batch = _spread(rng, 1, 32)
        most = max(8, 16000 * 8 * 128 // (batch * hkv * d))
        hi = _spread(rng, 8, min(8000, most))
        lo = rng.randint(max(1, hi // 3), hi)
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), batch=batch, lo=lo, hi=hi,
                    new=_spread(rng, 1, lo), hkv=hkv, d=d)
    hkv = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8])
    long = rng.random() < 0.35
    c = dict(kind=kind, hkv=hkv, hq=hkv * group, softcap=0.0, window=0, slopes=False, prefix=0)
    c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    if long:
        c["d"] = 128
        c["batch"] = _spread(rng, 1, 8)
        qhi = _spread(rng, 20, 2048 // c["batch"])
        c["qlo"], c["qhi"] = rng.choice([(qhi, qhi), (rng.randint(1, qhi), qhi)])
        hi = qhi + _spread(rng, 1, 6000)
        c["lo"], c["hi"] = rng.randint(max(qhi, hi // 2), hi), hi
    else:
        c["d"] = rng.choice([64, 128, 128, 256]) if kind == "q4" else rng.choice([64, 128, 128])
        c["batch"] = _spread(rng, 1, 64)
        most = max(64, 48 * 10000 * 8 * 128 // (c["batch"] * hkv * c["d"]) // 4)
        hi = _spread(rng, 17, min(16000, most))
        c["lo"], c["hi"] = rng.randint(max(8, hi // 4), hi), hi
        q = rng.choice([1, 1, 1, rng.randint(2, 8)])
        c["qlo"] = c["qhi"] = q
        if kind == "q4" and rng.random() < 0.15:
            c["dtype"] = "f32"
    if kind == "scored" or rng.random() < 0.25:
        what = rng.choice(["cap", "window", "slopes", "prefix", "cap window", "window prefix"])
        c["softcap"] = rng.choice([20.0, 30.0, 50.0]) if "cap" in what else 0.0
        c["window"] = _spread(rng, 16, 4096) if "window" in what else 0
        c["slopes"] = "slopes" in what
        c["prefix"] = _spread(rng, 4, 512) if "prefix" in what else 0
    return c


def _between(lo, hi, n, phase):
    """n whole numbers spread over lo..hi; the first is hi."""
    at = [((i * 0.6180339887498949) + phase) % 1.0 for i in range(n)]
    return [hi if i == 0 else lo + int(a * (hi - lo + 1)) for i, a in enumerate(at)]


def _lengths(case):
    """Tokens in the cache and query rows of each sequence."""
    kv = _between(case["lo"], case["hi"], case["batch"], 0.37)
    if case["kind"] == "cache":
        return kv, [case["new"]] * case["batch"]
    q = _between(case["qlo"], case["qhi"], case["batch"], 0.11)
    return kv, [min(a, b) for a, b in zip(q, kv)]


def _row_bytes(d):
    return d + 8  # K and V codes, two fp16 pairs


def _elem(case):
    return 4 if case["dtype"] == "f32" else 2


def work(case):
    kv, ql = _lengths(case)
    h, d, es = case["hkv"], case["d"], _elem(case)
    if case["kind"] == "cache":
        new, ctx = sum(ql), sum(kv)
        read = new * h * d * 2 * es + (ctx - new) * h * _row_bytes(d) + 4 * (new + ctx)
        wrote = new * h * _row_bytes(d) + ctx * h * d * 2 * es
        return {"bytes": read + wrote, "flops": 8 * (new + ctx) * h * d}
    seen = pairs = 0
    for n, q in zip(kv, ql):
        pre = min(case["prefix"], n)
        w = case["window"]
        first = n - q  # position of the first row
        low = max(0, first - w + 1) if w else 0
        seen += n - max(0, low - pre)
        for i in range(q):
            a = max(0, first + i - w + 1) if w else 0
            pairs += first + i + 1 - max(0, a - pre) + max(0, pre - max(first + i + 1, 0))
    rows = sum(ql) * case["hq"] * d
    kvb = _row_bytes(d) if case["kind"] == "q4" else 2 * d * es
    tables = 4 * sum((n + BLOCK - 1) // BLOCK for n in kv)
    return {"bytes": seen * h * kvb + 2 * rows * es + tables, "flops": 4 * pairs * case["hq"] * d}


# ------------------------------------------------------------------- 4 bits

def _views(pool, d):
    """K codes (blocks, H, 16, D/2), V codes (blocks, 2, 4, 2, H, C, 8, W, 2), parameters
    (blocks, H, K or V, 16, scale or base) of one layer's pool, as views of it."""
    n, h, rec = pool.shape
    c, w = max(1, d // 128), min(4, d // 32)
    k = pool[:, :, :8 * d].unflatten(2, (16, d // 2))
    v = pool[:, :, 8 * d:16 * d].unflatten(2, (c, 2, 8, 4, w, 2, 2))
    par = pool[:, :, 16 * d:].view(torch.float16).unflatten(2, (2, 16, 2))
    return k, v.permute(0, 3, 5, 7, 1, 2, 4, 6, 8), par


def _step(h, k):
    """The fp16 number k steps above h >= 0 (below it for k < 0)."""
    return (h.view(torch.int16) + k).view(torch.float16)


def _below(x):
    """The largest fp16 not above x (x in fp32, within +-65504)."""
    h = x.to(torch.float16)
    bits = h.view(torch.int16)
    down = torch.where(h > 0, bits - 1, torch.where(h < 0, bits + 1, torch.full_like(bits, -32767)))
    return torch.where(h.to(torch.float32) > x, down.view(torch.float16), h)


def _quantise(x):
    """Codes (uint8), scale and base (fp16) of the rows of x; borders are decided in 64 bits."""
    x = x.to(torch.float32)
    bad = ~(x.abs() <= 65504).all(-1)
    x = torch.where(bad[..., None], 0.0, x)
    base = _below(x.amin(-1))
    span = x.amax(-1).double() - base.double()
    scale = (span / 15).float().to(torch.float16)
    scale = torch.where(scale.double() * 15 < span, _step(scale, 1), scale)
    less = _step(scale, -1)
    scale = torch.where((scale > 0) & (less.double() * 15 >= span), less, scale)
    away = (x.double() - base.double()[..., None]) / scale.double()[..., None]
    code = torch.where((scale > 0)[..., None], torch.round(away), 0.0).to(torch.uint8)
    nan = torch.full_like(scale, math.nan)
    return code, torch.where(bad, nan, scale), torch.where(bad, nan, base)


def _dequantise(code, par):
    par = par.to(torch.float32)
    return code.to(torch.float32) * par[..., 0, None] + par[..., 1, None]


def _split(b):
    """Bytes (..., n) to codes (..., 2n)."""
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _rows(pool, d, blk, slot):
    """Dequantised K and V rows (..., H, D) at (block, slot)."""
    k, v, par = _views(pool, d)
    kc = _split(k.transpose(1, 2)[blk, slot])
    vc = _split(v[blk, slot >> 3, (slot >> 1) & 3, slot & 1].flatten(-4))
    kp = par[:, :, 0].transpose(1, 2)[blk, slot]
    vp = par[:, :, 1].transpose(1, 2)[blk, slot]
    return _dequantise(kc, kp), _dequantise(vc, vp)


# ------------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _tables(kv, gen, dev):
    need = [(n + BLOCK - 1) // BLOCK for n in kv]
    blocks = sum(need) + sum(need) // 16 + 3
    perm = torch.randperm(blocks, generator=gen, device=dev)
    width = max(need)
    tables = torch.zeros((len(kv), width), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n].int()
        at += n
    return tables, blocks


def _random_q4(blocks, h, d, gen, dev):
    """A pool of stale and live rows: codes heavier in the middle, as of a bell's rows."""
    rec = 16 * d + 128
    pool = torch.randint(0, 256, (blocks, h, rec), dtype=torch.uint8, generator=gen, device=dev)
    two = torch.randint(0, 256, (blocks, h, rec), dtype=torch.uint8, generator=gen, device=dev)
    pool = (((pool & 15) + (two & 15)) >> 1) | ((((pool >> 4) + (two >> 4)) >> 1) << 4)
    scale = 0.3 + 0.15 * torch.rand((blocks, h, 2, 16), generator=gen, device=dev)
    base = -7.0 * scale + 0.1 * torch.randn((blocks, h, 2, 16), generator=gen, device=dev)
    _views(pool, d)[2].copy_(torch.stack((scale, base), -1))
    return pool


def _randn(shape, dtype, gen, dev):
    return torch.randn(shape, generator=gen, device=dev).to(dtype)


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 1000003 + 17)
    kv, ql = _lengths(case)
    h, d, dt = case["hkv"], case["d"], DTYPES[case["dtype"]]
    tables, blocks = _tables(kv, gen, dev)
    s = dict(case=case, tables=tables)
    if case["kind"] == "cache":
        s["pool"] = _random_q4(blocks, h, d, gen, dev)[None]
        t = sum(ql)
        # the model's projections: rows of one fused tensor, read with its strides
        fused = _randn((1, t, 2 * h, d), dt, gen, dev).transpose(1, 2)
        s["keys"], s["values"] = fused[:, :h], fused[:, h:]
        at, new = [], []
        for i, (n, q) in enumerate(zip(kv, ql)):
            p = torch.arange(n, device=dev)
            flat = tables[i, p // BLOCK].long() * BLOCK + p % BLOCK
            at.append(flat)
            new.append(flat[n - q:])
        s["index"], s["slots"] = torch.cat(at), torch.cat(new)
        return s
    s["kv"] = torch.tensor(kv, dtype=torch.int32, device=dev)
    s["q"] = _randn((sum(ql), case["hq"], d), dt, gen, dev) * 1.25
    s["scale"] = 1.0 / math.sqrt(d)
    uniform = min(ql) == max(ql)
    s["q_per_seq"] = ql[0] if uniform else 0
    cu = torch.tensor([0] + ql, dtype=torch.int32, device=dev).cumsum(0, dtype=torch.int32)
    s["cu"] = cu
    s["max_q"] = max(ql)
    hq = case["hq"]
    s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev) / hq)).float() \
        if case["slopes"] else None
    s["prefix"] = torch.tensor([min(case["prefix"], n) for n in kv], dtype=torch.int32,
                               device=dev) if case["prefix"] else None
    if case["kind"] == "q4":
        pool = _random_q4(blocks, h, d, gen, dev)
        # slots behind the last token hold whatever was there: here NaN
        par = _views(pool, d)[2]
        for i, n in enumerate(kv):
            if n % BLOCK:
                par[tables[i, n // BLOCK].long(), :, :, n % BLOCK:] = math.nan
        s["pool"] = pool[None]
    else:
        s["kp"] = _randn((1, blocks, BLOCK, h, d), dt, gen, dev)
        s["vp"] = _randn((1, blocks, BLOCK, h, d), dt, gen, dev)
        for i, n in enumerate(kv):
            if n % BLOCK:
                s["kp"][0, tables[i, n // BLOCK].long(), n % BLOCK:] = math.nan
                s["vp"][0, tables[i, n // BLOCK].long(), n % BLOCK:] = math.nan
    return s


# ---------------------------------------------------------------------- run

def run(s):
    if own:
        return _run_own(s)
    return _plain_cache(s) if s["case"]["kind"] == "cache" else _plain_attention(s)


def _run_own(s):
    c = s["case"]
    if c["kind"] == "cache":
        from memforge_b200.quant_cache import gather_kv_q4, scatter_kv_q4
        scatter_kv_q4(s["pool"], 0, s["slots"], s["keys"], s["values"])
        return gather_kv_q4(s["pool"], 0, s["index"], s["keys"].dtype)
    rows = dict(q_per_seq=s["q_per_seq"]) if s["q_per_seq"] else dict(cu_seqlens_q=s["cu"],
                                                                      max_q_len=s["max_q"])
    mods = dict(softcap=c["softcap"], window=c["window"], alibi_slopes=s["slopes"],
                prefix_lens=s["prefix"])
    if c["kind"] == "q4":
        from memforge_b200.quant_cache import paged_attention_q4
        return paged_attention_q4(s["q"], s["pool"], 0, s["tables"], s["kv"], scale=s["scale"],
                                  **rows, **mods)
    from memforge_b200.scored_attention import paged_attention_scored
    return paged_attention_scored(s["q"], s["kp"], s["vp"], 0, s["tables"], s["kv"],
                                  scale=s["scale"], **rows, **mods)


def _plain_cache(s):
    c, pool = s["case"], s["pool"][0]
    d = c["d"]
    k, v, par = _views(pool, d)
    blk, slot = s["slots"] // BLOCK, s["slots"] % BLOCK
    for which, x in enumerate((s["keys"], s["values"])):
        code, scale, base = _quantise(x[0].transpose(0, 1))
        byte = code[..., 0::2] | (code[..., 1::2] << 4)
        if which == 0:
            k.transpose(1, 2)[blk, slot] = byte
        else:
            v[blk, slot >> 3, (slot >> 1) & 3, slot & 1] = byte.unflatten(-1, v.shape[5:])
        par[:, :, which].transpose(1, 2)[blk, slot] = torch.stack((scale, base), -1)
    kr, vr = _rows(pool, d, s["index"] // BLOCK, s["index"] % BLOCK)
    dt = s["keys"].dtype
    return (kr.to(dt).transpose(0, 1)[None].contiguous(),
            vr.to(dt).transpose(0, 1)[None].contiguous())


def _plain_attention(s):
    c = s["case"]
    b, h, hq, d = c["batch"], c["hkv"], c["hq"], c["d"]
    dev = s["q"].device
    n = s["tables"].shape[1] * BLOCK
    pos = torch.arange(n, device=dev)
    live = pos[None] < s["kv"][:, None]
    if c["kind"] == "q4":
        k, v = _rows(s["pool"][0], d, s["tables"][:, pos // BLOCK].long(), (pos % BLOCK)[None])
    else:
        k, v = (x[0][s["tables"].long()].flatten(1, 2).float() for x in (s["kp"], s["vp"]))
    k = torch.where(live[..., None, None], k, 0.0)
    v = torch.where(live[..., None, None], v, 0.0)
    # rows padded to the longest run
    ql = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(s["max_q"], device=dev)
    real = i[None] < ql[:, None]
    at = torch.where(real, s["cu"][:-1, None] + i[None], 0).long()
    q = s["q"].float()[at].unflatten(2, (h, hq // h))
    qpos = (s["kv"] - ql)[:, None] + i[None]
    score = torch.einsum("bqhgd,bnhd->bhgqn", q, k) * s["scale"]
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    back = qpos[:, :, None] - pos
    if c["slopes"]:
        score = score - s["slopes"].view(1, h, hq // h, 1, 1) * back[:, None, None].float()
    sees = back >= 0
    if c["window"]:
        sees = sees & (back < c["window"])
    if c["prefix"]:
        sees = sees | (pos < s["prefix"][:, None, None])
    sees = sees & live[:, None]
    score = torch.where(sees[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True)
    out = torch.einsum("bhgqn,bnhd->bqhgd", p, v).flatten(2, 3)
    return out[real].to(s["q"].dtype)


# -------------------------------------------------------------------- exact

def _exact_rows(pool, d, flat):
    """K and V rows (T, H, D) in 64 bits, by the byte address of each value."""
    dev = pool.device
    blocks, h, rec = pool.shape
    blk, tok = (flat // BLOCK)[:, None], (flat % BLOCK)[:, None]
    dim = torch.arange(d, device=dev)[None]
    w = min(4, d // 32)
    chunk, inside = dim // 128, dim % 128
    group, word, nib = inside // (4 * w), (inside // 4) % w, dim % 4
    ka = tok * (d // 2) + dim // 2
    va = 8 * d + ((((chunk * 2 + tok // 8) * 8 + group) * 4 + (tok // 2) % 4) * w + word) * 4 \
        + (tok % 2) * 2 + nib // 2
    out = []
    for addr, par in ((ka, 16 * d), (va, 16 * d + 64)):
        rows = []
        for head in range(h):
            byte = pool[:, head][blk, addr].int()
            code = torch.where(dim % 2 == 0, byte % 16, byte // 16).double()
            pair = pool[:, head, par:par + 64].contiguous().view(torch.float16).double()
            pair = pair.view(blocks, 16, 2)[blk[:, 0], tok[:, 0]]
            rows.append(code * pair[:, :1] + pair[:, 1:])
        out.append(torch.stack(rows, 1))
    return out


def _halves(dev):
    """Every finite fp16 number, in order, in 64 bits."""
    up = torch.arange(0, 31744, dtype=torch.int16, device=dev).view(torch.float16).double()
    return torch.cat((-up.flip(0)[:-1], up))


def exact(case, seed):
    s = prepare(case, seed)
    kv, ql = _lengths(case)
    if case["kind"] == "cache":
        halves = _halves(s["index"].device)
        kr, vr = _exact_rows(s["pool"][0], case["d"], s["index"])
        inv = torch.full((s["pool"].shape[1] * BLOCK,), -1, dtype=torch.long,
                         device=s["index"].device)
        inv[s["index"]] = torch.arange(s["index"].numel(), device=s["index"].device)
        where = inv[s["slots"]]
        for old, x in ((kr, s["keys"]), (vr, s["values"])):
            x = x[0].transpose(0, 1).double()
            low, high = x.min(-1).values, x.max(-1).values
            base = halves[torch.searchsorted(halves, low.contiguous(), right=True) - 1]
            scale = halves[torch.searchsorted(halves, ((high - base) / 15).contiguous())]
            away = (x - base[..., None]) / scale[..., None]
            old[where] = torch.where(scale[..., None] > 0, away.round(), 0.0) * scale[..., None] \
                + base[..., None]
        return kr.transpose(0, 1)[None].contiguous(), vr.transpose(0, 1)[None].contiguous()
    if work(case)["flops"] > 4e12:
        return None
    group = case["hq"] // case["hkv"]
    outs, at = [], 0
    for b, (n, q) in enumerate(zip(kv, ql)):
        p = torch.arange(n, device=s["q"].device)
        flat = s["tables"][b, p // BLOCK].long() * BLOCK + p % BLOCK
        if case["kind"] == "q4":
            k, v = _exact_rows(s["pool"][0], case["d"], flat)
        else:
            k, v = (s[x][0].flatten(0, 1)[flat].double() for x in ("kp", "vp"))
        x = s["q"][at:at + q].double()
        at += q
        me = torch.arange(n - q, n, device=p.device)[:, None]
        ok = p[None] <= me
        if case["window"]:
            ok = ok & (me - p[None] < case["window"])
        if case["prefix"]:
            ok = ok | (p[None] < case["prefix"])
        heads = []
        for j in range(case["hq"]):
            sc = (x[:, j] @ k[:, j // group].T) * s["scale"]
            if case["softcap"]:
                sc = (sc / case["softcap"]).tanh() * case["softcap"]
            if case["slopes"]:
                sc = sc - float(s["slopes"][j]) * (me - p[None])
            w = torch.softmax(sc.masked_fill(~ok, -math.inf), -1)
            heads.append(w @ v[:, j // group])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
