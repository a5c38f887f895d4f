"""GPU: the sticky status word is taken once, whoever asks for it and whatever runs meanwhile."""
import re
import threading
from pathlib import Path

import pytest
import torch

import mac_attention_b200 as mac
from mac_attention_b200 import ops
from tests.chunk_cases import make_chunk

CSRC = Path(__file__).resolve().parents[1] / "mac_attention_b200" / "csrc"


def test_no_status_word_is_read_and_cleared_in_two_steps():
    """A kernel on another stream may set a bit between a copy out and a copy of zero, and that bit would be
    lost.  Every kernel file's word goes through the one exchange."""
    words = set()
    for path in sorted(CSRC.glob("*.cu")):
        text = path.read_text()
        words |= set(re.findall(r"__device__ unsigned (g_\w*status)\b", text))
        assert not re.search(r"cudaMemcpy(To|From)Symbol(Async)?\(&?\w*,?\s*g_\w*status", text), path.name
        assert not re.search(r"cudaMemcpyToSymbol\(g_\w*status", text), path.name
    assert words == {"g_status", "g_build_status", "g_tc_status", "g_chunk_status", "g_kv8_status"}
    taken = "".join(p.read_text() for p in CSRC.glob("*.cu"))
    for word in words:
        assert re.search(rf"cudaGetSymbolAddress\([^;]*\b{word}\)", taken), word


@pytest.mark.gpu
def test_a_bit_is_reported_once():
    """One thread makes calls that set one bit each and asks after each; another asks all the time.  Each bit
    is reported by exactly one of the two."""
    ext = mac.load_mac_chunk_attention_extension()
    t = make_chunk([1], [20], 8, 2, seed=1)
    t["ids"][0] = 10**6                                      # no such row of the table: one bit a call
    ws = mac.make_chunk_attention_workspace()
    out, lse = torch.zeros_like(t["q"]), torch.zeros(1, 8, device="cuda")
    torch.cuda.synchronize()
    assert ops.query_status() == 0
    calls, seen, failed, stop = 400, [0, 0], [], threading.Event()

    def ask():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while not stop.is_set():
                    seen[1] += ops.query_status() != 0
        except BaseException as exc:                          # noqa: BLE001
            failed.append(exc)

    other = threading.Thread(target=ask)
    other.start()
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(calls):
                ext.mac_chunk_attention_bf16(t["q"], t["k"], t["v"], t["table"], t["ids"], t["offsets"],
                                             t["kv_lens"], out, lse, ws)
                torch.cuda.current_stream().synchronize()
                seen[0] += ops.query_status() != 0
    finally:
        stop.set()
        other.join(60)
    assert not failed and not other.is_alive()
    assert sum(seen) == calls, seen
    assert ops.query_status() == 0
