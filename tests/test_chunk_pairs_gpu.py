"""GPU: chunk attention in calls with enough tiles of rows for every multiprocessor to take two, the way of
a prompt: both softmax streams of a unit read the same blocks.  Both pools, head layouts that leave rows of
a tile empty, windows, tokens cached before, infinities and NaN in values that only some rows attend."""
import math

import pytest
import torch

import mac_attention_b200 as mac
from mac_attention_b200 import ops
from tests.chunk_cases import assert_chunk_close, chunk_reference, make_chunk
from tests.test_chunk_attention_gpu import quantized, run

pytestmark = pytest.mark.gpu

# (heads a KV head, KV heads, new tokens, cached tokens): whole prompts, prompts behind a cache, remainders
# of one tile and of a few rows beside them
SHAPES = [(8, 8, [700, 37], [1900, 37]), (3, 8, [1000, 600, 5], [1300, 600, 800]), (5, 8, [900, 130], [900, 1500]),
          (1, 16, [2400, 130], [2600, 130]), (16, 4, [650], [1000]), (4, 8, [260] * 6, [300, 260, 261, 900, 387, 512])]


@pytest.fixture(scope="module")
def ext():
    return mac.load_mac_chunk_attention_extension()


@pytest.fixture(scope="module")
def workspace():
    return mac.make_chunk_attention_workspace()


def pairs(G, Hkv, lens, kv, seed):
    """A chunk whose tiles are taken in pairs: 128 // G tokens a tile, two tiles a multiprocessor at least."""
    tiles = Hkv * sum(-(-n // (128 // G)) for n in lens)
    assert tiles >= 2 * torch.cuda.get_device_properties(0).multi_processor_count
    return make_chunk(lens, kv, G * Hkv, Hkv, seed=seed)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window", [None, 1, 100, 256, 700])
def test_pairs_of_tiles(ext, workspace, shape, window):
    t = pairs(*shape, seed=len(shape[2]) + (window or 0))
    assert_chunk_close(*run(ext, t, workspace, window), chunk_reference(t, window))
    pool, k, v = quantized(t)
    assert_chunk_close(*run(ext, t, workspace, window, pool=pool), chunk_reference(t, window, k=k, v=v))
    assert ops.query_status() == 0


def check_poisoned(got, ref):
    """Infinities and NaN where the definition has them; the rest within the usual limits."""
    (out, lse), (want, wl, mass, _) = got, ref
    out, lse = out.double(), lse.double()
    assert torch.equal(torch.isnan(lse), torch.isnan(wl)) and torch.equal(torch.isnan(out), torch.isnan(want))
    for side in (math.inf, -math.inf):
        assert torch.equal(out == side, want == side)
    fin = torch.isfinite(want)
    lim = 2.0 ** -8 * (want.abs() + mass) + 2.0 ** -10 * mass       # weights and result rounded to bf16
    assert ((out - want).abs() <= lim)[fin].all()
    ok = torch.isfinite(wl)
    assert ((lse - wl).abs() <= 2.0 ** -12)[ok].all()               # fp32 sums of 128 products a logit


@pytest.mark.parametrize("window", [None, 100, 256])
@pytest.mark.parametrize("shape", [(8, 8, [700, 37], [900, 37]), (5, 8, [900, 130], [900, 400])])
def test_values_that_some_rows_of_a_pair_attend(ext, workspace, shape, window):
    """Infinite and NaN values of every kind of block: before the chunk, on the diagonal of either tile, at both
    edges of the window."""
    t = pairs(*shape, seed=40)
    kv, n = shape[3][0], shape[2][0]
    at = t["table"][t["ids"][0].long()].long()
    for i, pos in enumerate([kv - n - 1 if kv > n else 0, kv - n + 1, 300, 333, 401, 402, 460, 555, kv - 90, kv - 1]):
        h, d = i % 2, (7 * i) % 128                          # the low and the high half of a word
        t["v"][at[pos], h, d] = [math.inf, -math.inf, math.nan][i % 3]
        t["v"][at[pos], h, d ^ 1] = [-math.inf, math.inf, 3.0][i % 3]
    for _ in range(3):
        check_poisoned(run(ext, t, workspace, window), chunk_reference(t, window))
    # single codes of NaN, and whole rows that are held as NaN
    clean = pairs(*shape, seed=40)
    clean["v"][at[500], 1, 9] = math.inf
    pool, _, _ = quantized(clean)
    for i, pos in enumerate([0, kv - n + 1, 333, 402, 555, kv - 90, kv - 1]):
        pool[1].view(torch.uint8)[at[pos], i % 2, 11 * i] = [0x7f, 0xff][i % 2]
    k, v = torch.empty_like(clean["k"]), torch.empty_like(clean["v"])
    mac.load_mac_quantized_cache_extension().mac_dequantize_kv_e4m3(
        *pool, torch.arange(k.shape[0], device="cuda"), k, v)
    assert torch.isnan(v[at[500], 1]).all() and torch.isnan(v[at[kv - 90]]).sum() == 1
    for _ in range(3):
        check_poisoned(run(ext, clean, workspace, window, pool=pool), chunk_reference(clean, window, k=k, v=v))
    assert ops.query_status() == 0


def test_keys_that_some_rows_of_a_pair_attend(ext, workspace):
    """NaN and infinite keys of later tokens reach the rows behind them only."""
    t = pairs(8, 8, [700, 37], [900, 37], seed=41)
    at = t["table"][t["ids"][0].long()].long()
    t["k"][at[640], 0], t["k"][at[700], 1, 4] = math.nan, math.nan
    for window in (None, 100):
        ref = chunk_reference(t, window)
        assert torch.isnan(ref[1]).any() and torch.isfinite(ref[1][700:]).all()
        check_poisoned(run(ext, t, workspace, window), ref)
        pool, k, v = quantized(t)
        check_poisoned(run(ext, t, workspace, window, pool=pool), chunk_reference(t, window, k=k, v=v))


def test_pairs_repeat_bit_for_bit(ext, workspace):
    t = pairs(8, 8, [700, 37], [1900, 37], seed=42)
    for pool in (None, quantized(t)[0]):
        for window in (None, 256):
            first = run(ext, t, workspace, window, pool=pool)
            for _ in range(5):
                again = run(ext, t, workspace, window, pool=pool)
                assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
