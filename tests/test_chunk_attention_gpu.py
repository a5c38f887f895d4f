"""GPU: attention of a chunk of new tokens over the paged pool, bf16 and 8-bit, against a plain
64-bit reference."""
import math

import pytest
import torch

import mac_attention_b200 as mac
from mac_attention_b200 import ops
from tests.chunk_cases import D, assert_chunk_close, chunk_reference, make_chunk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ext():
    return mac.load_mac_chunk_attention_extension()


@pytest.fixture(scope="module")
def workspace():
    return mac.make_chunk_attention_workspace()


def quantized(t, device="cuda"):
    """The chunk's pool in 8 bits and the same read back: (8-bit pool, k, v)."""
    q8 = mac.load_mac_quantized_cache_extension()
    T, Hkv = t["k"].shape[:2]
    pool = mac.make_quantized_pool(T, Hkv, device=device)
    locs = torch.arange(T, device=device, dtype=torch.int64)
    q8.mac_quantize_kv_e4m3(t["k"].view(T, -1), t["v"].view(T, -1), *pool, locs)
    k, v = torch.empty_like(t["k"]), torch.empty_like(t["v"])
    q8.mac_dequantize_kv_e4m3(*pool, locs, k, v)
    return pool, k, v


def run(ext, t, ws, window=None, sm_scale=None, pool=None):
    out = torch.full(t["q"].shape, 7.0, dtype=torch.bfloat16, device=t["q"].device)
    lse = torch.full(t["q"].shape[:2], 3.0, device=t["q"].device)
    rest = (t["table"], t["ids"], t["offsets"], t["kv_lens"], out, lse, ws, sm_scale, window)
    if pool is None:
        ext.mac_chunk_attention_bf16(t["q"], t["k"], t["v"], *rest)
    else:
        ext.mac_chunk_attention_e4m3(t["q"], *pool, *rest)
    return out, lse


def check(ext, ws, t, window=None, sm_scale=None, both=True, rows=slice(None)):
    """Both pools against 64 bits; the 8-bit pool against its own values."""
    scale = D ** -0.5 if sm_scale is None else sm_scale
    assert_chunk_close(*run(ext, t, ws, window, sm_scale), chunk_reference(t, window, scale), rows)
    if both:
        pool, k, v = quantized(t)
        got = run(ext, t, ws, window, sm_scale, pool)
        assert_chunk_close(*got, chunk_reference(t, window, scale, k, v), rows)
    assert ops.query_status() == 0


@pytest.mark.parametrize("kv", [1, 2, 15, 16, 127, 128, 129, 255, 256, 257, 384, 385, 640, 1000])
def test_single_tokens(ext, workspace, kv):
    check(ext, workspace, make_chunk([1], [kv], 8, 2, seed=kv))


@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8, 11, 16])
@pytest.mark.parametrize("Hkv", [1, 3])
def test_head_layouts(ext, workspace, G, Hkv):
    check(ext, workspace, make_chunk([1, 9, 70, 130 // G + 1], [300, 9, 211, 517], G * Hkv, Hkv, seed=G))


@pytest.mark.parametrize("n", [2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 97, 128, 129, 200])
def test_chunk_lengths(ext, workspace, n):
    """Around the sizes at which a chunk fills one and two tiles of rows, with and without a past."""
    check(ext, workspace, make_chunk([n, n], [n, n + 333], 8, 2, seed=n))


@pytest.mark.parametrize("window", [0, 1, 2, 63, 127, 128, 129, 300, 2**31 - 1, 2**40])
def test_windows(ext, workspace, window):
    check(ext, workspace, make_chunk([1, 40, 200, 3], [700, 500, 200, 4], 8, 2, seed=3), window)


def test_empty_rows_and_requests(ext, workspace):
    """Requests without rows, without a cache, and with fewer cached tokens than rows."""
    t = make_chunk([0, 3, 0, 5, 200, 1, 0], [10, 0, 0, 2, 150, 1, 5], 8, 2, seed=5)
    check(ext, workspace, t)
    check(ext, workspace, t, 3)
    # nothing at all
    for lens, kv in (([0, 0], [0, 9]), ([], [])):
        t = make_chunk(lens or [0], kv or [0], 8, 2, tail=2)
        if not lens:
            t["ids"], t["kv_lens"], t["offsets"] = t["ids"][:0], t["kv_lens"][:0], t["offsets"][:1]
        out, lse = run(ext, t, workspace)
        assert (out == 7).all() and (lse == 3).all()
    assert ops.query_status() == 0


def test_rows_outside_the_batch_stay(ext, workspace):
    t = make_chunk([3, 50, 1], [90, 400, 600], 16, 2, lead=5, tail=9, seed=6)
    for pool in (None, quantized(t)[0]):
        out, lse = run(ext, t, workspace, pool=pool)
        for part in (slice(0, 5), slice(59, 68)):
            assert (out[part] == 7).all() and (lse[part] == 3).all()
    check(ext, workspace, t, rows=slice(5, 59))


@pytest.mark.parametrize("lens,kv", [([1], [5000]), ([1, 1, 1], [9000, 100, 3000]), ([4] * 5, [2100] * 5),
                                     ([300], [3000]), ([700, 90], [700, 2500])])
def test_split_work(ext, workspace, lens, kv):
    """Few rows over a long cache: the work of a tile is cut along the keys and joined."""
    check(ext, workspace, make_chunk(lens, kv, 8, 2, seed=len(lens)))
    check(ext, workspace, make_chunk(lens, kv, 8, 1, seed=len(lens)), 1500)


def test_many_requests(ext, workspace):
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 4, (700,), generator=g).tolist()
    kv = [n + int(e) for n, e in zip(lens, torch.randint(0, 90, (700,), generator=g))]
    check(ext, workspace, make_chunk(lens, kv, 4, 2, seed=2))


@pytest.mark.parametrize("gain,scale", [(40.0, None), (0.01, None), (1.0, 1.0), (6.0, 0.5)])
def test_logit_ranges(ext, workspace, gain, scale):
    """One key far above the rest, and all alike; later keys that raise the running maximum."""
    t = make_chunk([1, 33, 140], [400, 900, 140], 8, 2, gain=gain, seed=8)
    k = t["k"].clone()
    tok = t["table"][t["ids"][1].long()][:900].long()
    k[tok] *= torch.linspace(0.1, 3.0, 900, device="cuda")[:, None, None].to(torch.bfloat16)
    t["k"] = k
    check(ext, workspace, t, sm_scale=scale)


def test_values_that_a_row_does_not_attend_do_not_reach_it(ext, workspace):
    """NaN and infinity in keys and values of later tokens, and of tokens before the window."""
    t = make_chunk([40, 1, 170], [300, 257, 400], 8, 2, seed=9)
    table, ids = t["table"], t["ids"].long()
    for b, poison in ((0, 280), (2, 330)):
        at = table[ids[b]].long()
        t["k"][at[poison]], t["v"][at[poison]] = math.inf, math.nan
        t["v"][at[poison + 3], :, 5], t["v"][at[poison + 3], :, 6] = math.inf, -math.inf
    # rows before the poisoned token are clean, later ones are not
    clean = torch.zeros(211, dtype=torch.bool)
    clean[:20], clean[40], clean[41:41 + 100] = True, True, True
    out, lse = run(ext, t, workspace)
    assert_chunk_close(out, lse, chunk_reference(t), clean.nonzero()[:, 0].cuda())
    assert torch.isnan(out[~clean]).all() and torch.isnan(lse[~clean]).all()
    # values only: infinities come through where they are attended
    t = make_chunk([40, 170], [300, 400], 8, 2, seed=10)
    at = t["table"][t["ids"][1].long()].long()
    t["v"][at[350], 0, 5], t["v"][at[360], 0, 5], t["v"][at[390], 0, 9] = math.inf, math.inf, -math.inf
    t["v"][at[395], 0, 5] = -math.inf
    out, lse = run(ext, t, workspace)
    ref = chunk_reference(t)
    got, want = out.double(), ref[0]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got == math.inf, want == math.inf)
    fin = torch.isfinite(want)
    lim = 2.0 ** -8 * (want.abs() + ref[2]) + 2.0 ** -10 * ref[2]
    assert ((got - want).abs() <= lim)[fin].all()
    # before the window
    t = make_chunk([90], [500], 8, 2, seed=11)
    at = t["table"][t["ids"][0].long()].long()
    t["k"][at[300]], t["v"][at[300]], t["v"][at[410]] = math.nan, math.nan, math.nan
    out, lse = run(ext, t, workspace, window=64)
    clean = torch.ones(90, dtype=torch.bool)
    clean[0:64] = False                                   # positions 410..473 see token 410
    assert_chunk_close(out, lse, chunk_reference(t, 64), clean.nonzero()[:, 0].cuda())
    assert torch.isnan(out[:64]).all()


def test_held_nan_rows(ext, workspace):
    """A row held as NaN in the 8-bit pool acts like a NaN row of the bf16 pool."""
    t = make_chunk([30, 2], [200, 100], 8, 2, seed=12)
    at = t["table"][t["ids"][0].long()].long()
    t["v"][at[190], 1, 3] = math.inf
    pool, k, v = quantized(t)
    assert torch.isnan(v[at[190], 1]).all() and torch.isfinite(v[at[190], 0]).all()
    out, lse = run(ext, t, workspace, pool=pool)
    assert torch.isnan(out[20:30, 4:]).all() and torch.isfinite(out[20:30, :4]).all()
    assert torch.isfinite(out[:20]).all() and torch.isfinite(out[30:]).all() and torch.isfinite(lse).all()


def test_tables_that_lead_outside_are_reported(ext, workspace):
    base = make_chunk([4, 6, 130], [200, 300, 400], 8, 2, seed=13)
    want = chunk_reference(base)
    rows = [slice(0, 4), slice(4, 10), slice(10, 140)]

    def others_fine(out, lse, b):
        for i in range(3):
            if i != b:
                assert_chunk_close(out, lse, want, rows[i])

    for name, value, b in (("ids", 5, 0), ("ids", -1, 1), ("kv_lens", 10**6, 2), ("kv_lens", -4, 1)):
        t = dict(base)
        t[name] = base[name].clone()
        t[name][b] = value
        for pool in (None, quantized(base)[0]):
            out, lse = run(ext, t, workspace, pool=pool)
            if pool is None:
                others_fine(out, lse, b)
            assert (out[rows[b]] == 0).all() and (lse[rows[b]] == -math.inf).all()
            assert ops.query_status() & 0x2
            assert ops.query_status() == 0
    # offsets that leave the rows: the request is left out
    for off in ([0, 4, 10, 141], [-1, 4, 10, 140], [0, 4, 2, 140], [0, 2**31 - 1, 10, 140]):
        t = dict(base, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
        out, lse = run(ext, t, workspace)
        assert ops.query_status() & 0x2
        if off[3] == 141:
            others_fine(out, lse, 2)
            assert (out[10:] == 7).all()
    # entries outside the pool count as rows of zeros
    t = dict(base, table=base["table"].clone())
    row = t["table"][base["ids"][1].long()]
    row[[3, 250, 299]] = torch.tensor([-1, base["k"].shape[0], 2**31 - 1], dtype=torch.int32, device="cuda")
    t["table"][base["ids"][1].long()] = row
    zero = base["k"].shape[0]                               # the reference's own row of zeros
    with_zeros = lambda x: torch.cat([x, torch.zeros_like(x[:1])])  # noqa: E731
    ref = dict(base, table=t["table"].clone(), k=with_zeros(base["k"]), v=with_zeros(base["v"]))
    ref["table"][base["ids"][1].long(), [3, 250, 299]] = zero
    for pool in (None, quantized(base)[0]):
        out, lse = run(ext, t, workspace, pool=pool)
        assert ops.query_status() & 0x2
        if pool is None:
            assert_chunk_close(out, lse, chunk_reference(ref))
        else:
            _, k, v = quantized(base)
            assert_chunk_close(out, lse, chunk_reference(ref, k=with_zeros(k), v=with_zeros(v)))


def test_row_strides_and_missing_lse(ext, workspace):
    """q as a column slice of one projection's output."""
    t = make_chunk([5, 60], [90, 200], 8, 2, seed=14)
    wide = torch.full((65, 12 * D), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, 2 * D:10 * D] = t["q"].view(65, -1)
    t["q"] = wide[:, 2 * D:10 * D].view(65, 8, D)
    assert t["q"].stride(0) == 12 * D
    out, lse = run(ext, t, workspace)
    assert_chunk_close(out, lse, chunk_reference(t))
    again = torch.zeros_like(out)
    ext.mac_chunk_attention_bf16(t["q"], t["k"], t["v"], t["table"], t["ids"], t["offsets"], t["kv_lens"],
                                 again, None, workspace)
    assert torch.equal(again, out)


def test_shared_prefix_and_repeated_requests(ext, workspace):
    """Two requests that list the same pool rows, and one table row named twice."""
    t = make_chunk([8, 8, 3], [300, 300, 120], 8, 2, seed=15)
    t["table"][t["ids"][1].long()] = t["table"][t["ids"][0].long()]
    t["ids"][2] = t["ids"][0]
    check(ext, workspace, t)


def test_calls_repeat_bit_for_bit(ext, workspace):
    t = make_chunk([1, 1, 200, 40], [3000, 500, 900, 40], 16, 2, seed=16)
    for pool in (None, quantized(t)[0]):
        first = run(ext, t, workspace, pool=pool)
        for _ in range(3):
            again = run(ext, t, workspace, pool=pool)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_captured_call_replays_with_other_lengths(ext, workspace):
    t = make_chunk([1, 90, 6], [2500, 700, 333], 8, 2, seed=17, table_cols=4000)
    other = make_chunk([60, 1, 36], [60, 1500, 2000], 8, 2, seed=18, table_cols=4000)
    T = max(t["k"].shape[0], other["k"].shape[0])
    for s in (t, other):
        for n in ("k", "v"):
            s[n] = torch.cat([s[n], s[n].new_full((T - s[n].shape[0], 2, D), math.nan)])
    pools = [quantized(s) for s in (t, other)]
    live = {n: x.clone() for n, x in t.items()}
    live8 = [x.clone() for x in pools[0][0]]
    out, lse = torch.zeros_like(t["q"]), torch.zeros(t["q"].shape[:2], device="cuda")
    out8, lse8 = torch.zeros_like(out), torch.zeros_like(lse)
    ws2 = mac.make_chunk_attention_workspace()
    rest = (live["table"], live["ids"], live["offsets"], live["kv_lens"])

    def calls():
        ext.mac_chunk_attention_bf16(live["q"], live["k"], live["v"], *rest, out, lse, ws2)
        ext.mac_chunk_attention_e4m3(live["q"], *live8, *rest, out8, lse8, ws2, window=70)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for s, (pool, k, v) in ((t, pools[0]), (other, pools[1]), (t, pools[0])):
        for n, x in s.items():
            live[n].copy_(x)
        for a, b in zip(live8, pool):
            a.copy_(b)
        graph.replay()
        assert_chunk_close(out, lse, chunk_reference(s))
        assert_chunk_close(out8, lse8, chunk_reference(s, 70, k=k, v=v))
    assert ops.query_status() == 0


def test_two_streams_with_their_own_workspaces(ext):
    ts = [make_chunk([1, 1, 1], [4000, 900, 2500], 8, 2, seed=19 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in ts]
    spaces = [mac.make_chunk_attention_workspace() for _ in ts]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i] = run(ext, ts[i], spaces[i])
    torch.cuda.synchronize()
    for t, o in zip(ts, outs):
        assert_chunk_close(*o, chunk_reference(t))


def test_pool_rows_past_32_bit_offsets(ext, workspace):
    """Rows whose byte and element offsets pass 2^32 and 2^31."""
    T, Hkv = 2_300_000, 8
    t = make_chunk([1, 30], [130, 200], 32, Hkv, seed=20)
    small = t["k"].shape[0]
    for bits in (16, 8):
        if bits == 16:
            k = torch.zeros(T, Hkv, D, dtype=torch.bfloat16, device="cuda")
            v = torch.zeros_like(k)
            k[-small:], v[-small:] = t["k"], t["v"]
            big = dict(t, k=k, v=v, table=(t["table"] + (T - small)).to(torch.int32))
            out, lse = run(ext, big, workspace)
            assert_chunk_close(out, lse, chunk_reference(t))
        else:
            pool, rk, rv = quantized(t)
            big8 = mac.make_quantized_pool(T, Hkv)
            for a, b in zip(big8, pool):
                a.view(torch.uint8)[-small:] = b.view(torch.uint8)
            big = dict(t, table=(t["table"] + (T - small)).to(torch.int32))
            out, lse = run(ext, big, workspace, pool=big8)
            assert_chunk_close(out, lse, chunk_reference(t, k=rk, v=rv))
        del big
        torch.cuda.empty_cache()
    assert ops.query_status() == 0


def test_random_shapes(ext, workspace):
    g = torch.Generator().manual_seed(77)
    ri = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    for i in range(40):
        Hkv, G, B = ri(1, 4), ri(1, 16), ri(1, 6)
        lens = [ri(0, [1, 8, 90, 400][ri(0, 3)]) for _ in range(B)]
        kv = [max(0, n + ri(-2, [3, 100, 1500][ri(0, 2)])) for n in lens]
        window = [None, None, ri(1, 40), ri(40, 900)][ri(0, 3)]
        check(ext, workspace, make_chunk(lens, kv, G * Hkv, Hkv, seed=1000 + i, gain=[0.5, 1, 3][ri(0, 2)]), window,
              both=i % 2 == 0)
