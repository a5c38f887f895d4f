"""GPU: rows of the 8-bit K/V pool, written (plain and behind the decode rotation) and read back."""
import math

import pytest
import torch

import mac_attention_b200 as mac
from mac_attention_b200 import ops
from tests.chunk_cases import D, hold_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ext():
    return mac.load_mac_quantized_cache_extension()


def values(pool):
    """What the rows of a pool stand for, in 64 bits."""
    k, v, ke, ve = pool
    two = lambda e: torch.where(e == 255, math.nan, torch.exp2(e.double() - 127))  # noqa: E731
    return k.double() * two(ke)[..., None], v.double() * two(ve)[..., None]


def rows_of_every_size(n, Hkv, seed):
    """Rows whose sizes run over the whole bf16 range, with outlier channels, zeros and exact powers."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, Hkv, D, generator=g)
    x *= torch.exp2(torch.randint(-140, 120, (n, Hkv, 1), generator=g).double()).float()
    x[::3] = torch.randn(x[::3].shape, generator=g) * torch.exp2(4 * torch.randn(D, generator=g))
    x[n // 2] = 0
    x[n // 3] = 448.0
    x[n // 4, :, 1:] = 0.01
    x[n // 4, :, 0] = 449.0
    x[n - 1, :, 0], x[n - 1, :, 1:] = 3.3e38, 1e30
    return x.to(torch.bfloat16).cuda()


@pytest.mark.parametrize("n,Hkv", [(1, 1), (5, 8), (64, 3), (333, 8), (1000, 2)])
@pytest.mark.parametrize("loc_dtype", [torch.int32, torch.int64])
def test_written_rows_and_reading_back(ext, n, Hkv, loc_dtype):
    k, v = rows_of_every_size(n, Hkv, n), rows_of_every_size(n, Hkv, n + 1)
    T = n + 50
    locs = torch.randperm(T, generator=torch.Generator().manual_seed(n))[:n].to(loc_dtype).cuda()
    pool = mac.make_quantized_pool(T, Hkv)
    for t in pool:
        t.view(torch.uint8).fill_(0x55)
    ext.mac_quantize_kv_e4m3(k.view(n, -1), v.view(n, -1), *pool, locs)
    at = locs.long()
    for x, codes, e in ((k, pool[0], pool[2]), (v, pool[1], pool[3])):
        want, we = hold_reference(x)
        assert torch.equal(e[at], we)
        assert torch.equal(codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).double(), want)
        rest = torch.ones(T, dtype=torch.bool, device="cuda")
        rest[at] = False
        assert (codes.view(torch.uint8)[rest] == 0x55).all() and (e[rest] == 0x55).all()
    # half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale among the subnormal codes
    vals = values(pool)
    for x, y, e in ((k, vals[0], pool[2]), (v, vals[1], pool[3])):
        s = torch.exp2(e[at].double() - 127)[..., None]
        assert ((y[at] - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * s)).all()
    # back: exactly the values, into the rows that are named
    kb, vb = torch.full((T + 3, Hkv, D), 9.0, dtype=torch.bfloat16, device="cuda"), None
    vb = kb.clone()
    to = torch.randperm(T + 3, generator=torch.Generator().manual_seed(n + 9))[:n].to(loc_dtype).cuda()
    ext.mac_dequantize_kv_e4m3(*pool, locs, kb, vb, to)
    for got, want in ((kb, vals[0]), (vb, vals[1])):
        assert torch.equal(got[to.long()].double(), want[at])
        rest = torch.ones(T + 3, dtype=torch.bool, device="cuda")
        rest[to.long()] = False
        assert (got[rest] == 9).all()
    ext.mac_dequantize_kv_e4m3(*pool, locs, kb, vb)
    assert torch.equal(kb[:n].double(), vals[0][at]) and torch.equal(vb[:n].double(), vals[1][at])
    assert ops.query_status() == 0


def test_every_code_and_exponent_reads_back(ext):
    """All 256 codes under all 256 exponent bytes, against code * 2^(e-127) rounded to bf16."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(2, D).repeat(256, 1).view(512, 1, D)
    e = torch.arange(256, dtype=torch.uint8, device="cuda").repeat_interleave(2).view(512, 1)
    pool = (codes.view(torch.float8_e4m3fn).contiguous(), codes.flip(0).contiguous().view(torch.float8_e4m3fn),
            e.contiguous(), e.flip(0).contiguous())
    kb = torch.zeros(512, 1, D, dtype=torch.bfloat16, device="cuda")
    vb = torch.zeros_like(kb)
    ext.mac_dequantize_kv_e4m3(*pool, torch.arange(512, device="cuda"), kb, vb)
    for got, want in zip((kb, vb), values(pool)):
        want = want.float().to(torch.bfloat16)          # 3 mantissa bits: the fp32 step rounds nothing
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])


def test_rows_with_infinities_or_nan_read_back_as_nan(ext):
    k = torch.randn(6, 2, D, device="cuda").to(torch.bfloat16)
    v = k.clone()
    k[1, 0, 5], k[2, 1, 127], v[3, 0, 0], v[4, 1, 64] = math.inf, -math.inf, math.nan, -math.nan
    pool = mac.make_quantized_pool(6, 2)
    locs = torch.arange(6, device="cuda")
    ext.mac_quantize_kv_e4m3(k.view(6, -1), v.view(6, -1), *pool, locs)
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    ext.mac_dequantize_kv_e4m3(*pool, locs, kb, vb)
    for x, got in ((k, kb), (v, vb)):
        bad = ~torch.isfinite(x).all(-1)
        assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
        assert bad.sum() == 2


@pytest.mark.parametrize("loc_dtype", [torch.int32, torch.int64])
def test_padding_is_skipped(ext, loc_dtype):
    k = torch.randn(9, 2 * D, device="cuda").to(torch.bfloat16)
    pool = mac.make_quantized_pool(5, 2)
    before = [t.clone() for t in pool]
    big = 2**31 - 1 if loc_dtype == torch.int32 else 2**40
    locs = torch.tensor([-1, 2, 5, big, -big, 4, 100, -7, 6], dtype=loc_dtype, device="cuda")
    ext.mac_quantize_kv_e4m3(k, k, *pool, locs)
    for i in (0, 1, 3):
        assert all(torch.equal(a.view(torch.uint8)[i], b.view(torch.uint8)[i]) for a, b in zip(pool, before))
    want, we = hold_reference(k.view(9, 2, D)[[1, 5]])
    assert torch.equal(pool[2][[2, 4]], we)
    kb = torch.full((3, 2, D), 9.0, dtype=torch.bfloat16, device="cuda")
    vb = kb.clone()
    src = torch.tensor([-1, 2, 5, 4, 0], dtype=loc_dtype, device="cuda")
    dst = torch.tensor([0, 1, 2, big, -1], dtype=loc_dtype, device="cuda")
    ext.mac_dequantize_kv_e4m3(*pool, src, kb, vb, dst)
    assert (kb[[0, 2]] == 9).all() and (vb[[0, 2]] == 9).all()
    assert torch.equal(kb[1].double(), values(pool)[0][2])
    ext.mac_quantize_kv_e4m3(k[:0], k[:0], *pool, locs)
    ext.mac_dequantize_kv_e4m3(*pool, src[:0], kb, vb)


def test_row_strides_and_alignment(ext):
    """k and v as slices of a projection's output, at offsets that forbid 16-byte loads too."""
    for width, off in ((10 * D, 2 * D), (10 * D + 3, 5), (4 * D + 8, 8)):
        wide = torch.randn(33, width, device="cuda").to(torch.bfloat16)
        k, v = wide[:, off:off + 2 * D], wide[:, off + 2 * D - 8:off + 4 * D - 8]
        if v.shape[1] < 2 * D:
            v = k
        a, b = mac.make_quantized_pool(40, 2), mac.make_quantized_pool(40, 2)
        locs = torch.arange(33, device="cuda", dtype=torch.int32)
        ext.mac_quantize_kv_e4m3(k, v, *a, locs)
        ext.mac_quantize_kv_e4m3(k.contiguous(), v.contiguous(), *b, locs)
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
        want, we = hold_reference(k.reshape(33, 2, D))
        assert torch.equal(a[2][:33], we) and torch.equal(a[0].view(torch.uint8)[:33].view(torch.float8_e4m3fn).double(), want)


def rotated(x, cos_sin, positions, neox):
    """x [N, H, 128] fp32: each product and sum rounded by itself, as the operator states."""
    r = cos_sin.shape[1]
    c = cos_sin[positions.long()]
    cos, sin = c[:, None, :r // 2], c[:, None, r // 2:]
    x = x.float()
    y = x.clone()
    if neox:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    return y


@pytest.mark.parametrize("N,Hq,Hkv", [(1, 32, 8), (64, 8, 2), (7, 5, 1)])
@pytest.mark.parametrize("rot,neox", [(128, True), (128, False), (64, True), (64, False), (2, True), (6, False)])
@pytest.mark.parametrize("aligned", [True, False])
def test_decode_rotation_and_write(ext, N, Hq, Hkv, rot, neox, aligned):
    g = torch.Generator().manual_seed(N + rot)
    pad = 0 if aligned else 3
    qkv = torch.randn(N, (Hq + 2 * Hkv) * D + pad, generator=g).to(torch.bfloat16).cuda()[:, pad:]
    q, k, v = qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1)
    kept = qkv.clone()
    ang = torch.rand(500, rot // 2, generator=g) * 6.3
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1).cuda()
    positions = torch.randint(0, 500, (N + 1,), generator=g).to(torch.int64 if aligned else torch.int32).cuda()
    locs = torch.randperm(N + 9, generator=g)[:N].to(torch.int32 if aligned else torch.int64).cuda()
    q_post = torch.full((N + 2, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    pool = mac.make_quantized_pool(N + 9, Hkv)
    ext.mac_decode_rope_quantize_kv_e4m3(q, k, v, q_post, *pool, cos_sin, positions, locs, D, neox)
    assert torch.equal(qkv, kept)
    assert torch.equal(q_post[:N], rotated(q.reshape(N, Hq, D), cos_sin, positions[:N], neox).to(torch.bfloat16))
    assert (q_post[N:] == 7).all()
    at = locs.long()
    for x, codes, e in ((rotated(k.reshape(N, Hkv, D), cos_sin, positions[:N], neox), pool[0], pool[2]),
                        (v.reshape(N, Hkv, D), pool[1], pool[3])):
        want, we = hold_reference(x)
        assert torch.equal(e[at], we)
        assert torch.equal(codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).double(), want)
    assert ops.query_status() == 0


def test_rotation_agrees_with_the_bf16_operator(ext):
    """The same decode step through the bf16 pool's operator: the rotated queries differ by a
    rounding of the fp32 sum at most, so by one bf16 step, and seldom."""
    N, Hq, Hkv = 32, 16, 4
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(N, h * D, generator=g).to(torch.bfloat16).cuda() for h in (Hq, Hkv, Hkv))
    ang = torch.rand(100, 64, generator=g) * 6.3
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1).cuda()
    pos, locs = torch.randint(0, 100, (N,), generator=g).cuda(), torch.arange(N).cuda()
    q_post, pool = torch.zeros(N, Hq, D, dtype=torch.bfloat16, device="cuda"), mac.make_quantized_pool(N, Hkv)
    ext.mac_decode_rope_quantize_kv_e4m3(q, k, v, q_post, *pool, cos_sin, pos, locs, D, True)
    q_pre = torch.zeros_like(q_post)
    kb = torch.zeros(N, Hkv, D, dtype=torch.bfloat16, device="cuda")
    vb = torch.zeros_like(kb)
    qq, kk = q.clone(), k.clone()
    ops.mac_decode_rope_preserve_q_bf16(qq, kk, v, q_pre, kb, vb, cos_sin, pos, locs, D, True)
    assert torch.equal(q_pre.view(N, -1), q)
    a, b = q_post.view(N, -1).float(), qq.float()
    # near zero the two fp32 results differ by a rounding of their products (at most 2^-23 * 6)
    assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -20).all() and (a != b).float().mean() < 1e-3


def test_positions_outside_the_table_are_skipped_and_reported(ext):
    N, Hq, Hkv = 4, 4, 2
    x = [torch.randn(N, h * D, device="cuda").to(torch.bfloat16) for h in (Hq, Hkv, Hkv)]
    cos_sin = torch.cat([torch.ones(10, 64), torch.zeros(10, 64)], 1).cuda()
    for bad in (10, -1, 2**31 - 1, 2**40):
        pos = torch.tensor([0, bad, 3, 9], dtype=torch.int64, device="cuda")
        q_post = torch.full((N, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
        pool = mac.make_quantized_pool(N, Hkv)
        ext.mac_decode_rope_quantize_kv_e4m3(*x, q_post, *pool, cos_sin, pos, torch.arange(N, device="cuda"), D, True)
        assert ops.query_status() & 0x2 and ops.query_status() == 0
        assert (q_post[1] == 7).all() and torch.equal(q_post[[0, 2, 3]].view(3, -1), x[0][[0, 2, 3]])
        assert (pool[2][1] == 3).all() and (pool[0].view(torch.uint8)[1] == 0).all() and (pool[3][1] == 3).all()


def test_large_pool_offsets(ext):
    """Rows whose byte offsets pass 2^31 and 2^32."""
    T, Hkv = 4_300_000, 8
    pool = mac.make_quantized_pool(T, Hkv)
    k = rows_of_every_size(20, Hkv, 4)
    locs = torch.arange(T - 20, T, device="cuda")
    ext.mac_quantize_kv_e4m3(k.view(20, -1), k.view(20, -1), *pool, locs)
    want, we = hold_reference(k)
    for i in (0, 1):
        assert torch.equal(pool[i].view(torch.uint8)[-20:].view(torch.float8_e4m3fn).double(), want)
        assert torch.equal(pool[2 + i][-20:], we)
    kb = torch.zeros(20, Hkv, D, dtype=torch.bfloat16, device="cuda")
    vb = torch.zeros_like(kb)
    ext.mac_dequantize_kv_e4m3(*pool, locs, kb, vb)
    assert torch.equal(kb.double(), want * torch.exp2(we.double() - 127)[..., None]) and torch.equal(kb, vb)


def test_captured_decode_step(ext):
    """The write captured into a graph and replayed with other rows."""
    N, Hkv = 5, 2
    k = torch.randn(N, Hkv * D, device="cuda").to(torch.bfloat16)
    v, locs, pool = k.clone(), torch.arange(N, device="cuda"), mac.make_quantized_pool(20, Hkv)
    ext.mac_quantize_kv_e4m3(k, v, *pool, locs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.mac_quantize_kv_e4m3(k, v, *pool, locs)
    k.mul_(3), v.mul_(-0.3), locs.add_(7)
    graph.replay()
    for x, i in ((k, 0), (v, 1)):
        want, we = hold_reference(x.view(N, Hkv, D))
        assert torch.equal(pool[2 + i][locs], we)
        assert torch.equal(pool[i].view(torch.uint8)[locs].view(torch.float8_e4m3fn).double(), want)
