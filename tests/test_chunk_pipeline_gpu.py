"""GPU: the chunk attention and the 8-bit pool as a serving step uses them, next to the ring build and
the decode step."""
import torch

import pytest

import mac_attention_b200 as mac
from mac_attention_b200 import ops, synth
from oracle import mac_oracle as O
from tests.chunk_cases import D, assert_chunk_close, chunk_reference
from tests.helpers import run_cuda
from tests.prefill_cases import make_prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spec", [dict(lens=[200, 37, 300], L0s=[0, 150, 90], Hq=8, Hkv=2, S=16, M=256),
                                  dict(lens=[330, 5], L0s=[0, 700], Hq=16, Hkv=2, S=64, M=64)])
def test_prompt_states_feed_the_ring_build(spec):
    """Full-prefix and band states of a chunked prompt from the chunk attention, turned into ring rows:
    the ring that the 64-bit states of the same prompt give, within the roundings of both."""
    lens, L0s, Hq, Hkv, S, M = (spec[n] for n in ("lens", "L0s", "Hq", "Hkv", "S", "M"))
    t = {k: v.cuda() for k, v in make_prompts(lens, L0s, Hq, Hkv, S, 0, M, seed=3).items()}
    ext, ws = mac.load_mac_chunk_attention_extension(), mac.make_chunk_attention_workspace()
    kv_lens = torch.tensor([a + b for a, b in zip(lens, L0s)], dtype=torch.int32, device="cuda")
    states = {}
    for name, window in (("full", None), ("band", S)):
        out, lse = torch.zeros_like(t["q_post"]), torch.zeros(t["q_post"].shape[:2], device="cuda")
        ext.mac_chunk_attention_bf16(t["q_post"], t["k"], t["v"], t["req_to_token"], t["req_ids"], t["offsets"],
                                     kv_lens, out, lse, ws, window=window)
        states[name] = (out, lse)
        # against the prompt's own 64-bit states: two roundings to bf16 (weights, result), 2^-8 each,
        # on values of a few units
        want_o, want_l = t[name + "_attn"].double(), t[name + "_lse"].double()
        assert (lse.double() - want_l).abs().max() <= 1e-4
        assert O.rel_l2(out.double(), want_o) <= 2.0 ** -7
    rings = []
    for full, band in ((states["full"], states["band"]),
                       ((t["full_attn"], t["full_lse"]), (t["band_attn"], t["band_lse"]))):
        r = {n: t[n].clone() for n in ("q_cache", "attn_cache", "lse_cache", "request_length", "ready", "cache_epoch")}
        ops.mac_prefill_downdate_update_cache(
            r["q_cache"], r["attn_cache"], r["lse_cache"], r["request_length"], t["req_ids"], t["src_q"], *full, *band,
            t["offsets"], t["lens"], M, Hq, D, ready=r["ready"], cache_epoch=r["cache_epoch"],
            request_epoch=t["request_epoch"])
        rings.append(r)
    got, want = rings
    assert torch.equal(got["q_cache"], want["q_cache"]) and bool(got["ready"].all())
    # The states differ by 2^-7 each (above); what is left after the subtraction is at least e^-3 of
    # the mass that the whole has at e^0 and more here, so that grows to a few times 2^-7.
    # A row whose window is its whole prefix has nothing left; its two LSEs, equal in exact arithmetic,
    # decide by their last bits whether a ring row is empty, so rows near that are left out.
    keep = torch.isfinite(want["lse_cache"]) & torch.isfinite(got["lse_cache"]) & (want["lse_cache"] > -3)
    assert keep.float().mean() > 0.3
    assert O.rel_l2(got["attn_cache"][keep].double(), want["attn_cache"][keep].double()) <= 3e-2
    assert ops.query_status() == 0


def test_single_tokens_agree_with_the_decode_step():
    """A decode step that finds nothing to reuse attends the whole context: the same as a chunk of one."""
    case = synth.make_decode_case(batch=3, ctx=0, ctx_list=[2300, 900, 3100], hq=32, hkv=8, capacity=256, seed=4)
    cfg = O.DecodeConfig(max_context=4096, semantic_pos_ahead=128)
    cu = run_cuda(case, cfg)
    c = case.to("cuda")
    N = 3
    table = torch.cat([c.req_to_token, torch.zeros_like(c.req_to_token[:, :1])], dim=1)
    for n in range(N):
        table[c.req_ids[n].long(), c.past_lens[n].long()] = c.out_cache_loc[n].to(torch.int32)
    out, lse = torch.zeros_like(c.q_post), torch.zeros(N, 32, device="cuda")
    ext = mac.load_mac_chunk_attention_extension()
    ext.mac_chunk_attention_bf16(c.q_post, c.k, c.v, table, c.req_ids, torch.arange(N + 1, dtype=torch.int32, device="cuda"),
                                 (c.past_lens + 1).to(torch.int32), out, lse, mac.make_chunk_attention_workspace(),
                                 sm_scale=cfg.sm_scale)
    assert int(cu.ws[3][:N].sum()) == 0                        # no head found a match
    assert O.rel_l2(out.float().cpu(), cu.out.float().cpu()) <= 1e-2
    assert (lse - cu.lse).abs().max() <= 2e-2
    assert ops.query_status() == 0


def test_decode_steps_over_the_8_bit_pool_and_a_parked_request():
    """Tokens rotated and written one step at a time, attention from the 8-bit pool after each; then the
    rows are brought back into a bf16 pool, where the same query gives the same result bit for bit."""
    B, Hq, Hkv, T, steps = 3, 16, 4, 700, 5
    g = torch.Generator().manual_seed(5)
    q8, chunk = mac.load_mac_quantized_cache_extension(), mac.load_mac_chunk_attention_extension()
    ws = mac.make_chunk_attention_workspace()
    lens = [200, 1, 133]                                       # tokens cached before
    table = torch.randperm(T, generator=g)[: B * 230].view(B, 230).to(torch.int32).cuda()
    pool = mac.make_quantized_pool(T, Hkv)
    past_k, past_v = (torch.randn(sum(lens), Hkv * D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    locs = torch.cat([table[b, :n] for b, n in enumerate(lens)])
    q8.mac_quantize_kv_e4m3(past_k, past_v, *pool, locs)
    ang = torch.rand(512, 64, generator=g) * 6.3
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1).cuda()
    ids = torch.arange(B, dtype=torch.int32, device="cuda")
    offsets = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    back = [torch.full((T, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    all_rows = torch.arange(T, device="cuda")
    for step in range(steps):
        pos = torch.tensor([n + step for n in lens], dtype=torch.int64, device="cuda")
        at = table[ids.long(), pos]
        qkv = torch.randn(B, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16).cuda()
        q, k, v = qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1)
        q_post = torch.zeros(B, Hq, D, dtype=torch.bfloat16, device="cuda")
        q8.mac_decode_rope_quantize_kv_e4m3(q, k, v, q_post, *pool, cos_sin, pos, at, D, True)
        out, lse = torch.zeros_like(q_post), torch.zeros(B, Hq, device="cuda")
        kv_lens = (pos + 1).to(torch.int32)
        chunk.mac_chunk_attention_e4m3(q_post, *pool, table, ids, offsets, kv_lens, out, lse, ws)
        q8.mac_dequantize_kv_e4m3(*pool, all_rows, *back)
        t = dict(q=q_post, k=back[0], v=back[1], table=table, ids=ids, offsets=offsets, kv_lens=kv_lens)
        assert_chunk_close(out, lse, chunk_reference(t))
        again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
        chunk.mac_chunk_attention_bf16(q_post, *back, table, ids, offsets, kv_lens, again, lse2, ws)
        assert torch.equal(again, out) and torch.equal(lse2, lse)
    assert ops.query_status() == 0
