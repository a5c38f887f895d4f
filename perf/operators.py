"""Paged chunk attention and the 8-bit K/V cache: the work that is measured, in plain form and through the package.

Five operators over a paged K/V pool (``[T, Hkv, 128]`` rows, a per-token table ``req_to_token``):

* ``attn16`` -- attention of a chunk of new tokens (prompt chunks, drafted tokens, single tokens) over the
  bf16 pool, with an optional trailing window; output and natural-log LSE.
* ``attn8``  -- the same over an e4m3 pool with one power-of-two scale per (token, KV head) row.
* ``ropeq``  -- decode step before attention: rotate q and k, write k and v into the e4m3 pool.
* ``write``  -- write rows of k and v into the e4m3 pool.
* ``read``   -- read rows of the e4m3 pool back into a bf16 pool.

A row of 128 values x is held as e4m3(x / s) with s the smallest power of two (at least 2**-124) for which
max|x| / s <= 448; the pool keeps s as its biased exponent, one byte.
"""
import functools
import math
import random

import torch

own = False

DIM = 128
PAGE = 16                      # consecutive positions of a request that lie together in the pool
LIMIT = 1 << 29                # score elements held at once by the plain form
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


# ------------------------------------------------------------------------------------------ cases
def _attn(name, op, batch, n, ctx, heads, kv_heads, window=-1):
    """n and ctx: (shortest, longest) of a ragged batch; ctx counts the chunk's own tokens too."""
    return dict(name=name, op=op, batch=batch, n_lo=n[0], n_hi=n[1], ctx_lo=ctx[0], ctx_hi=ctx[1],
                heads=heads, kv_heads=kv_heads, window=window)


def _rows(name, op, rows, heads, kv_heads, pool):
    return dict(name=name, op=op, rows=rows, heads=heads, kv_heads=kv_heads, pool=pool)


def listed():
    return [
        # a few short conversations, one to five drafted tokens each: latency of the call
        _attn("attn16_draft_b3_ctx1k", "attn16", 3, (1, 5), (700, 1300), 32, 8),
        # plain decode of long contexts, one token a request: the cache's bytes
        _attn("attn16_decode_b16_ctx32k", "attn16", 16, (1, 1), (30000, 32768), 32, 8),
        # one long prompt in chunks, the last of them: the products
        _attn("attn16_chunk4k_ctx32k", "attn16", 1, (4096, 4096), (32768, 32768), 32, 8),
        # whole prompts of about 2k tokens, attention of the trailing window (the band state of the ring build)
        _attn("attn16_band1k_b8_len2k", "attn16", 8, (1500, 2048), (1500, 2048), 64, 8, 1024),
        # decode of long contexts from the 8-bit pool
        _attn("attn8_decode_b16_ctx32k", "attn8", 16, (1, 1), (30000, 32768), 32, 8),
        # chunked prefill of two requests from the 8-bit pool
        _attn("attn8_chunk1k_b2_ctx8k", "attn8", 2, (900, 1024), (7000, 8192), 64, 8),
        # one decode token, and a full decode batch, rotated and written
        _rows("ropeq_n1", "ropeq", 1, 32, 8, 4096),
        _rows("ropeq_n64", "ropeq", 64, 64, 8, 4096),
        # rows of a short prompt, and of a large prefill batch
        _rows("write_n333", "write", 333, 32, 8, 4096),
        _rows("write_n32k", "write", 32768, 32, 8, 40000),
        # a parked request of 1k tokens, and one of 100k tokens, brought back into the bf16 pool
        _rows("read_n1k", "read", 1001, 32, 8, 4096),
        _rows("read_n100k", "read", 100000, 32, 8, 120000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attn16", "attn16", "attn16", "attn8", "attn8", "ropeq", "write", "read"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 16] if kv_heads < 8 else [1, 2, 4, 5, 8])
    if op in ("attn16", "attn8"):
        batch = _log(rng, 1, 48)
        n_hi = rng.choice([1, _log(rng, 2, 16), _log(rng, 16, 4096)])
        n_lo = rng.choice([n_hi, max(1, n_hi // 3)])
        ctx_hi = _log(rng, n_hi + 7, max(n_hi + 64, 49152))
        while batch > 1 and (batch * n_hi * ctx_hi * heads * 512 > 5e11 or batch * ctx_hi * kv_heads > 4e6):
            batch = (batch + 1) // 2
        if batch * n_hi * ctx_hi * heads * 512 > 1e12:
            ctx_hi = n_hi + 7
        ctx_lo = max(n_lo, rng.choice([ctx_hi, ctx_hi // 2, n_lo]))
        window = rng.choice([-1, -1, _log(rng, 1, 4096)])
        c = _attn(None, op, batch, (n_lo, n_hi), (ctx_lo, ctx_hi), heads, kv_heads, window)
    else:
        hi = 512 if op == "ropeq" else 60000
        rows = _log(rng, 1, hi)
        c = _rows(None, op, rows, heads, kv_heads, rows + rng.randrange(1, 5000))
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, cached tokens) of each request: the case's own, whatever the seed."""
    r = random.Random("%(batch)d %(n_lo)d %(n_hi)d %(ctx_lo)d %(ctx_hi)d" % case)
    n = [r.randint(case["n_lo"], case["n_hi"]) for _ in range(case["batch"])]
    kv = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    n[0], kv[0] = case["n_hi"], case["ctx_hi"]
    return n, [max(a, b) for a, b in zip(n, kv)]


def work(case):
    h, hkv = case["heads"], case["kv_heads"]
    if case["op"] in ("attn16", "attn8"):
        n, kv = _lengths(case)
        w = case["window"] if case["window"] >= 0 else 1 << 60
        row = 256 if case["op"] == "attn16" else 129
        keys = sum(min(b, a - 1 + w) for a, b in zip(n, kv))
        pairs = 0
        for a, b in zip(n, kv):                       # row at position p attends min(p + 1, w) keys
            full = max(0, min(a, b - w))              # rows whose window is full
            part = a - full
            pairs += full * w + part * (b - a + 1) + part * (part - 1) // 2
        return {"bytes": 2 * keys * hkv * row + sum(n) * h * (2 * 256 + 4), "flops": pairs * h * 4 * DIM}
    n = case["rows"]
    held = 2 * n * hkv * (DIM + 1)
    if case["op"] == "ropeq":
        return {"bytes": n * (2 * h + 2 * hkv) * 256 + n * DIM * 4 + held, "flops": n * (h + hkv) * DIM * 3}
    return {"bytes": 2 * n * hkv * 256 + held, "flops": 2 * n * hkv * DIM}


# ----------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    x = torch.empty(shape, dtype=BF16, device="cuda")
    for part in x.view(-1, shape[-1]).split(1 << 21):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    return x


def _codes(g, tokens, kv_heads):
    """An 8-bit pool as earlier writes left it: codes that reach 448 / 2 and exponents around 2**-7."""
    x = _normal(g, tokens, kv_heads, DIM)
    pool = torch.empty(tokens, kv_heads, DIM, dtype=torch.float8_e4m3fn, device="cuda")
    for a, b in zip(pool.split(1 << 16), x.split(1 << 16)):
        a.copy_((b.float() * 80).clamp(-448, 448).to(torch.float8_e4m3fn))
    return pool, torch.randint(119, 122, (tokens, kv_heads), generator=g, device="cuda", dtype=torch.uint8)


def _table(g, kv):
    """Pages of 16 positions, scattered over the pool; entries behind a request's end point nowhere."""
    pages = [(k + PAGE - 1) // PAGE for k in kv]
    perm = torch.randperm(sum(pages), generator=g, device="cuda")
    table = torch.full((len(kv) + 2, max(kv) + 5), -1, dtype=I32, device="cuda")
    ids = torch.randperm(len(kv) + 2, generator=g, device="cuda")[:len(kv)].to(I32)
    inside = torch.arange(PAGE, device="cuda")
    for row, p, k in zip(ids.tolist(), perm.split(pages), kv):
        table[row, :k] = (p[:, None] * PAGE + inside).reshape(-1)[:k].to(I32)
    return table, ids, sum(pages) * PAGE


def prepare(case, seed):
    g = _generator(seed)
    h, hkv = case["heads"], case["kv_heads"]
    s = {"case": case}
    if case["op"] in ("attn16", "attn8"):
        n, kv = _lengths(case)
        s["table"], s["ids"], tokens = _table(g, kv)
        s["offsets"] = torch.tensor([0] + n, device="cuda").cumsum(0).to(I32)
        s["kv_lens"] = torch.tensor(kv, dtype=I32, device="cuda")
        s["n_max"], s["kv_max"] = max(n), max(kv)       # a scheduler knows its longest request
        s["q"] = _normal(g, sum(n), h, DIM)
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(sum(n), h, dtype=F32, device="cuda")
        if case["op"] == "attn16":
            s["k"], s["v"] = _normal(g, tokens, hkv, DIM), _normal(g, tokens, hkv, DIM)
        else:
            (s["k"], s["k_exp"]), (s["v"], s["v_exp"]) = _codes(g, tokens, hkv), _codes(g, tokens, hkv)
        return s
    n, pool = case["rows"], case["pool"]
    s["locs"] = torch.randperm(pool, generator=g, device="cuda")[:n].to(I32)
    if case["op"] == "read":
        (s["k_pool"], s["k_exp"]), (s["v_pool"], s["v_exp"]) = _codes(g, pool, hkv), _codes(g, pool, hkv)
        s["k_buffer"] = torch.zeros(n, hkv, DIM, dtype=BF16, device="cuda")
        s["v_buffer"] = torch.zeros_like(s["k_buffer"])
        s["to"] = torch.randperm(n, generator=g, device="cuda").to(I32)
        return s
    # q, k, v: column slices of one projection's output, some channels much larger than the others
    qkv = _normal(g, n, (h + 2 * hkv) * DIM)
    qkv *= torch.exp2(torch.randn(qkv.shape[1], generator=g, device="cuda")).to(BF16)
    s["q"], s["k"], s["v"] = qkv.split([h * DIM, hkv * DIM, hkv * DIM], dim=1)
    s["k_pool"] = torch.zeros(pool, hkv, DIM, device="cuda").to(torch.float8_e4m3fn)
    s["v_pool"] = s["k_pool"].clone()
    s["k_exp"] = torch.zeros(pool, hkv, dtype=torch.uint8, device="cuda")
    s["v_exp"] = torch.zeros_like(s["k_exp"])
    if case["op"] == "ropeq":
        at = torch.arange(8192, device="cuda", dtype=F32)[:, None]
        turn = at / 500000.0 ** (torch.arange(0, DIM, 2, device="cuda", dtype=F32) / DIM)
        s["cos_sin"] = torch.cat([turn.cos(), turn.sin()], dim=1)
        s["positions"] = torch.randint(0, 8192, (n,), generator=g, device="cuda", dtype=torch.int64)
        s["q_post"] = torch.zeros(n, h, DIM, dtype=BF16, device="cuda")
    return s


# ------------------------------------------------------------------------------------- plain forms
def _scale(e):
    """2**(e - 127) of a byte e, NaN for 255."""
    return torch.where(e == 255, math.nan, torch.ldexp(torch.ones_like(e, dtype=F32), e.to(I32) - 127))


def _plain_attention(s):
    case, table = s["case"], s["table"]
    h, hkv, (nm, km), b = case["heads"], case["kv_heads"], (s["n_max"], s["kv_max"]), case["batch"]
    g = h // hkv
    dev = table.device
    t = torch.arange(nm, device=dev)
    n = s["offsets"].diff()[:, None]
    at = (s["offsets"][:-1, None] + t).clamp(max=s["q"].shape[0] - 1)            # [b, nm] row of q
    p = s["kv_lens"][:, None] - n + t                                            # [b, nm] position
    j = torch.arange(km, device=dev)
    first = (p + 1 - case["window"]).clamp(min=0) if case["window"] >= 0 else torch.zeros_like(p)
    see = (j <= p[:, :, None]) & (j >= first[:, :, None]) & (t < n)[:, :, None]  # [b, nm, km]
    loc = table[s["ids"].long(), :km].clamp(min=0).long()                        # [b, km]
    out, lse = s["out"], s["lse"]
    # so many (request, KV head) pairs at a time that their scores fit
    for pair in torch.arange(b * hkv, device=dev).split(max(1, LIMIT // (g * nm * km))):
        r, kh = pair // hkv, pair % hkv
        q = s["q"].view(-1, hkv, g, DIM)[at[r], kh[:, None]].float()             # [P, nm, g, D]
        k = s["k"][loc[r], kh[:, None]].float()                                  # [P, km, D]
        v = s["v"][loc[r], kh[:, None]].float()
        if case["op"] == "attn8":
            k = k * _scale(s["k_exp"][loc[r], kh[:, None]])[..., None]
            v = v * _scale(s["v_exp"][loc[r], kh[:, None]])[..., None]
        x = torch.bmm(q.flatten(1, 2), k.transpose(1, 2)) * DIM ** -0.5          # [P, nm * g, km]
        x = x.view(-1, nm, g, km).masked_fill_(~see[r][:, :, None], -math.inf)
        top = x.amax(-1, keepdim=True).clamp(min=-3e38)
        x = x.sub_(top).exp_()
        total = x.sum(-1, keepdim=True)
        o = torch.bmm(x.flatten(1, 2), v).view(-1, nm, g, DIM) / total.clamp(min=1e-38)
        ls = (total.log() + top)[..., 0]
        live = (t < n[r])                                                        # [P, nm]
        where = (at[r][live], kh[:, None].expand(-1, nm)[live])
        out.view(-1, hkv, g, DIM)[where] = o[live].to(BF16)
        lse.view(-1, hkv, g)[where] = ls[live]
    return out, lse


def _hold(x):
    """(codes, exponent bytes) of rows x [n, heads, 128] in 32 bits."""
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)                                  # top = m * 2**e, 0.5 <= m < 1; 448 = 0.875 * 2**9
    e = torch.where(top > 0, e - 9 + (m > 0.875).to(I32), -124).clamp(min=-124)
    codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def _plain_write(s, k, v):
    at = s["locs"].long()
    for name, x in (("k", k), ("v", v)):
        codes, e = _hold(x)
        s[name + "_pool"].view(torch.uint8)[at] = codes
        s[name + "_exp"][at] = e
    return s["k_pool"], s["v_pool"], s["k_exp"], s["v_exp"]


def _turn(x, c):
    a, b = x.chunk(2, dim=-1)
    cos, sin = c[:, None].chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_read(s):
    at, to = s["locs"].long(), s["to"].long()
    for name in ("k", "v"):
        x = s[name + "_pool"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        s[name + "_buffer"][to] = (x * _scale(s[name + "_exp"][at])[..., None]).to(BF16)
    return s["k_buffer"], s["v_buffer"]


# ------------------------------------------------------------------------------------------- a pass
@functools.lru_cache(maxsize=1)
def _program():
    """What a serving program keeps for its life: the loaded operators and one attention workspace."""
    import mac_attention_b200 as mac

    return (mac.load_mac_chunk_attention_extension(), mac.load_mac_quantized_cache_extension(),
            mac.make_chunk_attention_workspace())


def run(s):
    op, hkv = s["case"]["op"], s["case"]["kv_heads"]
    if op in ("attn16", "attn8"):
        if own:
            ext, _, workspace = _program()
            w = s["case"]["window"] if s["case"]["window"] >= 0 else None
            rest = (s["table"], s["ids"], s["offsets"], s["kv_lens"], s["out"], s["lse"], workspace)
            if op == "attn16":
                ext.mac_chunk_attention_bf16(s["q"], s["k"], s["v"], *rest, window=w)
            else:
                ext.mac_chunk_attention_e4m3(s["q"], s["k"], s["v"], s["k_exp"], s["v_exp"], *rest, window=w)
            return s["out"], s["lse"]
        return _plain_attention(s)
    if op == "read":
        if own:
            _program()[1].mac_dequantize_kv_e4m3(s["k_pool"], s["v_pool"], s["k_exp"], s["v_exp"], s["locs"],
                                                 s["k_buffer"], s["v_buffer"], s["to"])
            return s["k_buffer"], s["v_buffer"]
        return _plain_read(s)
    pool = (s["k_pool"], s["v_pool"], s["k_exp"], s["v_exp"])
    if op == "write":
        if own:
            _program()[1].mac_quantize_kv_e4m3(s["k"], s["v"], *pool, s["locs"])
            return pool
        return _plain_write(s, s["k"].unflatten(1, (hkv, DIM)).float(), s["v"].unflatten(1, (hkv, DIM)).float())
    if own:
        _program()[1].mac_decode_rope_quantize_kv_e4m3(s["q"], s["k"], s["v"], s["q_post"], *pool, s["cos_sin"],
                                                       s["positions"], s["locs"], DIM, True)
        return (s["q_post"], *pool)
    c = s["cos_sin"][s["positions"]]
    s["q_post"].copy_(_turn(s["q"].unflatten(1, (-1, DIM)).float(), c))
    k = _turn(s["k"].unflatten(1, (hkv, DIM)).float(), c)
    return (s["q_post"], *_plain_write(s, k, s["v"].unflatten(1, (hkv, DIM)).float()))


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op, h, hkv = case["op"], case["heads"], case["kv_heads"]
    f64 = torch.float64
    two = lambda e: 2.0 ** (e.to(f64) - 127.0)  # noqa: E731
    if op in ("attn16", "attn8"):
        g = h // hkv
        out = torch.zeros(s["q"].shape, dtype=f64, device="cuda")
        lse = torch.zeros(s["lse"].shape, dtype=f64, device="cuda")
        for i, (n, kv) in enumerate(zip(*_lengths(case))):
            o0 = int(s["offsets"][i])
            at = s["table"][int(s["ids"][i])][:kv].long()
            for kh in range(hkv):
                k, v = s["k"][at, kh].to(f64), s["v"][at, kh].to(f64)
                if op == "attn8":
                    k, v = k * two(s["k_exp"][at, kh])[:, None], v * two(s["v_exp"][at, kh])[:, None]
                step = max(1, (1 << 27) // (kv * g))
                for t0 in range(0, n, step):
                    t1 = min(n, t0 + step)
                    p1 = kv - n + t1                                     # keys from here on are masked for all
                    q = s["q"][o0 + t0:o0 + t1, kh * g:(kh + 1) * g].to(f64)
                    x = torch.einsum("tgd,kd->tgk", q, k[:p1]) / math.sqrt(DIM)
                    pos = torch.arange(kv - n + t0, p1, device="cuda")[:, None, None]
                    key = torch.arange(p1, device="cuda")
                    hide = key > pos
                    if case["window"] >= 0:
                        hide = hide | (key <= pos - case["window"])
                    x = torch.where(hide, -math.inf, x)
                    ls = torch.logsumexp(x, -1)
                    w = torch.where(hide, 0.0, torch.exp(x - ls[..., None]))
                    out[o0 + t0:o0 + t1, kh * g:(kh + 1) * g] = torch.einsum("tgk,kd->tgd", w, v[:p1])
                    lse[o0 + t0:o0 + t1, kh * g:(kh + 1) * g] = ls
        return out, lse
    at = s["locs"].long()
    if op == "read":
        res = []
        for name in ("k", "v"):
            y = torch.zeros(s[name + "_buffer"].shape, dtype=f64, device="cuda")
            y[s["to"].long()] = s[name + "_pool"].to(f64)[at] * two(s[name + "_exp"][at])[..., None]
            res.append(y)
        return tuple(res)

    def held(x):
        """x [n, hkv, 128] in 64 bits as unrounded codes: rounding is what the other side does."""
        top = x.abs().amax(-1)
        e = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -130) / 448.0)).clamp(min=-124)
        e = torch.where(top > 448.0 * 2.0 ** e, e + 1, e)                # the logarithm's rounding next to a power
        e = torch.where((top <= 448.0 * 2.0 ** (e - 1)) & (e > -124), e - 1, e)
        y = torch.zeros(s["k_pool"].shape, dtype=f64, device="cuda")
        y[at] = x / 2.0 ** e[..., None]
        return y

    v = held(s["v"].unflatten(1, (hkv, DIM)).to(f64))
    if op == "write":
        return held(s["k"].unflatten(1, (hkv, DIM)).to(f64)), v, None, None
    c = s["cos_sin"].to(f64)[s["positions"]][:, None]
    cos, sin = c[..., :DIM // 2], c[..., DIM // 2:]

    def rotated(x):
        x = x.unflatten(1, (-1, DIM)).to(f64)
        lo, hi = x[..., :DIM // 2], x[..., DIM // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    return rotated(s["q"]), held(rotated(s["k"])), v, None, None
