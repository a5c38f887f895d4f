"""Inputs and 64-bit references of the chunk attention and 8-bit pool tests."""
import math

import torch

D = 128


def make_chunk(lens, kv_lens, Hq, Hkv, *, seed=0, lead=0, tail=0, gain=1.0, device="cuda", table_cols=None,
               pool_extra=37):
    """Ragged chunks over a scattered pool.  ``lead`` / ``tail``: rows of q before the first and
    behind the last request.  Pool rows that no request lists hold NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    T = sum(kv_lens) + pool_extra
    perm = torch.randperm(T, generator=g)
    cols = table_cols or max(max(kv_lens), 1) + 3
    table = torch.full((B + 2, cols), T - 1, dtype=torch.int32)
    ids = torch.randperm(B + 2, generator=g)[:B].to(torch.int32)
    k = torch.full((T, Hkv, D), math.nan)
    v = torch.full((T, Hkv, D), math.nan)
    at = 0
    for b in range(B):
        rows = perm[at:at + kv_lens[b]]
        table[ids[b], :kv_lens[b]] = rows.to(torch.int32)
        k[rows] = torch.randn(kv_lens[b], Hkv, D, generator=g)
        v[rows] = torch.randn(kv_lens[b], Hkv, D, generator=g)
        at += kv_lens[b]
    rows = lead + sum(lens) + tail
    q = torch.randn(rows, Hq, D, generator=g) * gain
    offsets = torch.tensor([lead] + list(lens)).cumsum(0).to(torch.int32)
    t = dict(q=q.to(torch.bfloat16), k=k.to(torch.bfloat16), v=v.to(torch.bfloat16), table=table, ids=ids,
             offsets=offsets, kv_lens=torch.tensor(list(kv_lens), dtype=torch.int32))
    return {n: x.to(device) for n, x in t.items()}


def chunk_reference(t, window=None, sm_scale=D ** -0.5, k=None, v=None):
    """Per row in 64 bits: (out, lse, sum of weight * |v|, largest sum of |q*k| * scale)."""
    q = t["q"].double()
    k = (t["k"] if k is None else k).double()
    v = (t["v"] if v is None else v).double()
    rows, Hq = q.shape[:2]
    Hkv = k.shape[1]
    G = Hq // Hkv
    out = torch.zeros(rows, Hq, D, dtype=torch.float64, device=q.device)
    mass, lse, size = torch.zeros_like(out), out[..., 0] - math.inf, torch.zeros_like(out[..., 0])
    for b, (o0, o1) in enumerate(zip(t["offsets"].tolist(), t["offsets"].tolist()[1:])):
        n, kv = o1 - o0, int(t["kv_lens"][b])
        if n <= 0 or kv == 0:
            continue
        tok = t["table"][int(t["ids"][b])][:kv].long()
        pos = torch.arange(kv - n, kv, device=q.device)[:, None]
        j = torch.arange(kv, device=q.device)[None]
        see = (j <= pos) & ((j > pos - window) if window is not None else True)
        for h in range(Hq):
            qq, kk, vv = q[o0:o1, h], k[tok, h // G], v[tok, h // G]
            # values of keys that a row does not attend are left out, whatever they hold
            s = torch.where(see, (qq @ kk.T) * sm_scale, -math.inf)
            ls = torch.logsumexp(s, -1)
            w = torch.where(see, torch.exp(s - torch.where(see.any(-1), ls, 0.0)[:, None]), 0.0)
            bad = ~torch.isfinite(vv)
            o = w @ torch.where(bad, 0.0, vv)
            if bad.any():
                o = o + torch.where(see[:, :, None] & bad[None], w[:, :, None] * vv[None], 0.0).sum(1)
            out[o0:o1, h], lse[o0:o1, h] = o, ls
            mass[o0:o1, h] = w @ torch.where(bad, 0.0, vv).abs()
            a = torch.where(see, (qq.abs() @ kk.abs().T) * sm_scale, 0.0)
            size[o0:o1, h] = a.amax(-1)
    return out, lse, mass, size


def assert_chunk_close(out, lse, ref, rows=slice(None)):
    """The kernel rounds each weight to bf16 (half a step, 2^-8) and the result once more; its fp32
    products, exponentials and sums are allowed 2^-16 of the largest sum of products in a logit
    (128 terms, a few units of 2^-24 each) and 2^-18 beside it."""
    want, wl, mass, size = (x[rows] for x in ref)
    out, lse = out[rows].double(), lse[rows].double()
    live = torch.isfinite(wl)
    assert torch.equal(torch.isfinite(lse), live)
    assert (lse[~live] == -math.inf).all() and (out[~live] == 0).all()
    slack = 2.0 ** -16 * size + 2.0 ** -18
    err = (lse - wl).abs()[live]
    lim = (slack + 2.0 ** -20 * wl.abs())[live]
    assert (err <= lim).all(), f"lse off by {err.max().item():.3g}, {(err / lim).max().item():.2f} of the limit"
    err = (out - want).abs()
    lim = 2.0 ** -8 * (want.abs() + mass) + 2 * slack[..., None] * mass + 1e-30
    assert (err <= lim)[live].all(), f"out off by {(err / lim)[live].max().item():.2f} of the limit"


def hold_reference(x):
    """(codes as fp64 values, exponent bytes) of finite rows x [..., 128]: the definition in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1)
    e = torch.full(top.shape, -124, dtype=torch.int64, device=x.device)
    for _ in range(256):                                     # smallest power of two that holds the row
        e = torch.where(top > 448.0 * torch.exp2(e.double()), e + 1, e)
    y = x / torch.exp2(e.double())[..., None]
    # nearest e4m3, ties to even: the step is 2^(floor(log2|y|) - 3), at least 2^-9
    _, ex = torch.frexp(y.abs())                              # |y| = m 2^ex, m in [0.5, 1)
    step = torch.exp2((ex.double() - 4).clamp(min=-9))
    y = torch.round(y / step) * step
    y = torch.where((e == 120)[..., None], y.clamp(-240, 240), y)      # 256 * 2^120 is no bf16 number
    return y, (e + 127).to(torch.uint8)
