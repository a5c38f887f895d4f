"""GPU: what the chunk attention and the 8-bit pool's operators refuse, and calls at the edge of what
they allow: exponents at odd addresses, graphs that share a workspace, workspaces of any contents."""
import math

import pytest
import torch

import mac_attention_b200 as mac
from mac_attention_b200 import ops
from tests.chunk_cases import D, assert_chunk_close, chunk_reference, make_chunk

from tests.test_chunk_attention_gpu import quantized, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ext():
    return mac.load_mac_chunk_attention_extension()


@pytest.fixture(scope="module")
def q8():
    return mac.load_mac_quantized_cache_extension()


def chunk_args():
    t = make_chunk([5, 2], [70, 40], 8, 2, seed=31)
    a = dict(q=t["q"], k=t["k"], v=t["v"], table=t["table"], ids=t["ids"], offsets=t["offsets"],
             kv_lens=t["kv_lens"], out=torch.full_like(t["q"], 7.0),
             lse=torch.full(t["q"].shape[:2], 3.0, device="cuda"), ws=mac.make_chunk_attention_workspace())
    return a


@pytest.mark.parametrize("change,text", [
    (lambda a: dict(q=a["q"].half()), "q has wrong dtype"),
    (lambda a: dict(q=a["q"][0]), "q must be"),
    (lambda a: dict(q=a["q"][..., :64]), "q must be"),
    (lambda a: dict(q=a["q"].transpose(0, 1).contiguous().transpose(0, 1)), "q rows must be contiguous"),
    (lambda a: dict(q=a["q"][:1].expand(7, -1, -1)), "stride"),
    (lambda a: dict(k=a["k"].float(), v=a["v"].float()), "k_buffer has wrong dtype"),
    (lambda a: dict(v=a["v"][:-1]), "must match"),
    (lambda a: dict(k=a["k"].flip(0).transpose(0, 1)), "k_buffer must be contiguous"),
    (lambda a: dict(k=a["k"].repeat(1, 2, 1)[:, :3].contiguous(), v=a["v"].repeat(1, 2, 1)[:, :3].contiguous()),
     "divisible"),
    (lambda a: dict(table=a["table"].long()), "req_to_token"),
    (lambda a: dict(table=a["table"][:, :-1]), "req_to_token"),
    (lambda a: dict(ids=a["ids"].long()), "req_ids"),
    (lambda a: dict(offsets=a["offsets"][:-1].contiguous()), "offsets must be"),
    (lambda a: dict(kv_lens=a["kv_lens"].cpu()), "kv_lens must be CUDA"),
    (lambda a: dict(kv_lens=a["kv_lens"][:1]), "kv_lens must be"),
    (lambda a: dict(out=a["out"].float()), "out has wrong dtype"),
    (lambda a: dict(out=a["out"][:-1]), "out must be contiguous and match q"),
    (lambda a: dict(out=a["q"]), "share memory"),
    (lambda a: dict(lse=a["lse"].double()), "lse has wrong dtype"),
    (lambda a: dict(lse=a["lse"].t().contiguous()), "lse must be"),
    (lambda a: dict(ws=a["ws"][:-1]), "workspace"),
    (lambda a: dict(ws=a["ws"][8:]), "aligned"),
    (lambda a: dict(window=-1), "window"),
    (lambda a: dict(sm_scale=0.0), "sm_scale"),
])
def test_chunk_attention_refuses(ext, change, text):
    a = dict(chunk_args(), window=None, sm_scale=None)
    out, lse = a["out"], a["lse"]
    a.update(change(a))
    with pytest.raises(RuntimeError, match=text):
        ext.mac_chunk_attention_bf16(a["q"], a["k"], a["v"], a["table"], a["ids"], a["offsets"], a["kv_lens"],
                                     a["out"], a["lse"], a["ws"], a["sm_scale"], a["window"])
    torch.cuda.synchronize()
    assert (out == 7).all() and (lse == 3).all() and ops.query_status() == 0


@pytest.mark.parametrize("change,text", [
    (lambda a: dict(k=a["k"].float()), "k has wrong dtype"),
    (lambda a: dict(v=a["v"][:, :128]), "v must be"),
    (lambda a: dict(v=a["v"][:-1]), "batch mismatch"),
    (lambda a: dict(k=a["k"].t().contiguous().t()), "contiguous last"),
    (lambda a: dict(locs=a["locs"][:-1]), "shorter"),
    (lambda a: dict(locs=a["locs"].float()), "int32 or int64"),
    (lambda a: dict(positions=a["positions"][:1]), "shorter"),
    (lambda a: dict(q=a["q"][:, :-64]), "q must be"),
    (lambda a: dict(q_post=a["q_post"][:-1]), "q_post must be"),
    (lambda a: dict(q_post=a["q"].view(4, 8, D)), "share memory"),
    (lambda a: dict(cs=a["cs"][:, :63]), "rotary_dim"),
    (lambda a: dict(cs=a["cs"].double()), "cos_sin_cache has wrong dtype"),
    (lambda a: dict(k_exp=a["pool"][2][:-1]), "k_exp must be"),
    (lambda a: dict(head_dim=64), "head_dim"),
])
def test_writes_refuse(q8, change, text):
    pool = mac.make_quantized_pool(16, 2)
    x = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)  # noqa: E731
    a = dict(q=x(4, 8 * D), k=x(4, 2 * D), v=x(4, 2 * D), q_post=torch.zeros(4, 8, D, dtype=torch.bfloat16, device="cuda"),
             pool=pool, cs=torch.zeros(32, D, device="cuda"), positions=torch.arange(4, device="cuda"),
             locs=torch.arange(4, device="cuda"), head_dim=D)
    a["k_exp"] = pool[2]
    before = [p.view(torch.uint8).clone() for p in pool]
    a.update(change(a))
    with pytest.raises(RuntimeError, match=text):
        q8.mac_decode_rope_quantize_kv_e4m3(a["q"], a["k"], a["v"], a["q_post"], pool[0], pool[1], a["k_exp"], pool[3],
                                            a["cs"], a["positions"], a["locs"], a["head_dim"], True)
    torch.cuda.synchronize()
    assert all(torch.equal(b, p.view(torch.uint8)) for b, p in zip(before, pool)) and ops.query_status() == 0


@pytest.mark.parametrize("change,text", [
    (lambda a: dict(dst=a["dst"][:-1]), "shorter"),
    (lambda a: dict(dst=None, k=a["k"][:2], v=a["v"][:2]), "shorter"),
    (lambda a: dict(k=a["k"][:, :1].contiguous(), v=a["v"][:, :1].contiguous()), "heads"),
    (lambda a: dict(src=a["src"].to(torch.int16)), "int32 or int64"),
    (lambda a: dict(k=a["k"].half(), v=a["v"].half()), "wrong dtype"),
])
def test_reads_refuse(q8, change, text):
    pool = mac.make_quantized_pool(16, 2)
    full = lambda: torch.full((8, 2, D), 7.0, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    a = dict(src=torch.arange(4, device="cuda"), dst=torch.arange(4, device="cuda"), k=full(), v=full())
    k, v = a["k"], a["v"]
    a.update(change(a))
    with pytest.raises(RuntimeError, match=text):
        q8.mac_dequantize_kv_e4m3(*pool, a["src"], a["k"], a["v"], a["dst"])
    torch.cuda.synchronize()
    assert (k == 7).all() and (v == 7).all()


@pytest.mark.parametrize("shift", [1, 7, 15])
@pytest.mark.parametrize("Hkv", [1, 3])
def test_exponents_at_odd_addresses(ext, q8, shift, Hkv):
    """The exponent arrays are views into a larger one: at any address, and with bytes of others on
    both sides of them, which stand for NaN here."""
    t = make_chunk([3, 70, 1], [50, 300, 129], 4 * Hkv, Hkv, seed=32)
    (kp, vp, ke, ve), k, v = quantized(t)
    n = ke.numel()
    wide = torch.full((2, n + 64), 255, dtype=torch.uint8, device="cuda")
    exps = [wide[i, shift:shift + n].view(ke.shape) for i in range(2)]
    exps[0].copy_(ke)
    exps[1].copy_(ve)
    ws = mac.make_chunk_attention_workspace()
    got = run(ext, t, ws, pool=(kp, vp, *exps))
    assert_chunk_close(*got, chunk_reference(t, k=k, v=v))
    assert ops.query_status() == 0


@pytest.mark.parametrize("lens,kv", [([3, 70, 1], [50, 300, 129]), ([1], [3000]), ([400] * 40, [400] * 40)])
def test_results_that_start_between_sectors(ext, lens, kv):
    """out at an address that is a multiple of 16 bytes but not of 32, inside a larger array."""
    t = make_chunk(lens, kv, 16, 2, seed=36)
    n = t["q"].numel()
    wide = torch.full((n + 32,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[8:8 + n].view(t["q"].shape)
    assert out.data_ptr() % 32 == 16
    lse = torch.zeros(t["q"].shape[:2], device="cuda")
    ws = mac.make_chunk_attention_workspace()
    ext.mac_chunk_attention_bf16(t["q"], t["k"], t["v"], t["table"], t["ids"], t["offsets"], t["kv_lens"], out, lse, ws)
    assert_chunk_close(out, lse, chunk_reference(t))
    assert (wide[:8] == 7).all() and (wide[8 + n:] == 7).all()
    other, other_lse = run(ext, t, ws)
    assert torch.equal(out, other) and torch.equal(lse, other_lse) and ops.query_status() == 0


def test_rows_read_back_between_sectors(q8):
    """Buffers at an address that is a multiple of 16 bytes but not of 32, inside a larger array."""
    t = make_chunk([9], [200], 8, 2, seed=37)
    (kp, vp, ke, ve), k, v = quantized(t)
    n = k.numel()
    wide = torch.full((2, n + 32), 7.0, dtype=torch.bfloat16, device="cuda")
    bufs = [wide[i, 8 + 16 * i:8 + 16 * i + n].view(k.shape) for i in range(2)]
    assert all(b.data_ptr() % 32 == 16 for b in bufs)
    q8.mac_dequantize_kv_e4m3(kp, vp, ke, ve, torch.arange(k.shape[0], device="cuda"), *bufs)
    for i, (b, want) in enumerate(zip(bufs, (k, v))):
        assert torch.equal(b.view(torch.int16), want.view(torch.int16))
        assert (wide[i, :8 + 16 * i] == 7).all() and (wide[i, 8 + 16 * i + n:] == 7).all()


def test_workspace_contents_do_not_matter(ext):
    t = make_chunk([1, 1, 150], [3000, 700, 2000], 8, 2, seed=33)
    ws = mac.make_chunk_attention_workspace()
    want = chunk_reference(t)
    pool, k, v = quantized(t)
    want8 = chunk_reference(t, k=k, v=v)
    for byte in (0, 1, 0x7f, 0xff):
        ws.fill_(byte)
        assert_chunk_close(*run(ext, t, ws), want)
        ws.fill_(byte)
        assert_chunk_close(*run(ext, t, ws, pool=pool), want8)
    assert ops.query_status() == 0


def test_graphs_in_order_share_a_workspace(ext):
    """Two graphs captured with one workspace, replayed one after the other on a side stream, with
    calls outside of them in between."""
    ws = mac.make_chunk_attention_workspace()
    ts = [make_chunk([1, 1], [2500, 600], 8, 2, seed=34), make_chunk([90, 7, 1], [400, 7, 5000], 8, 2, seed=35)]
    outs = [(torch.zeros_like(t["q"]), torch.zeros(t["q"].shape[:2], device="cuda")) for t in ts]

    def call(i):
        t = ts[i]
        ext.mac_chunk_attention_bf16(t["q"], t["k"], t["v"], t["table"], t["ids"], t["offsets"], t["kv_lens"],
                                     *outs[i], ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call(i)
        graphs.append(g)
    with torch.cuda.stream(side):
        for _ in range(4):
            for o in outs:
                o[0].fill_(math.nan)
            graphs[1].replay()
            call(0)
            graphs[0].replay()
            graphs[1].replay()
    side.synchronize()
    for t, o in zip(ts, outs):
        assert_chunk_close(*o, chunk_reference(t))
    assert ops.query_status() == 0
