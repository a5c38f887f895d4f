"""CPU: the chunk attention and 8-bit pool operators' host side -- exported symbols, struct
layouts, refusals -- without a GPU."""
import ctypes as C
import re
import subprocess
from pathlib import Path

import pytest
import torch

import mac_attention_b200 as pkg
from mac_attention_b200 import _abi, build, ops
from tests.chunk_cases import hold_reference

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "mac_b200_chunk.h"


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _abi.load_library()


def test_header_functions_are_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(mac_b200_[a-z0-9_]+)\s*\(", text)))
    assert sorted(_abi.CHUNK_PROTOTYPES) == names
    assert all(hasattr(lib, n) for n in names)


def test_struct_layouts_match_c(tmp_path):
    structs = [_abi.MacB200ChunkArgs, _abi.MacB200QuantizeKvArgs, _abi.MacB200DequantizeKvArgs]
    lines, want = [], []
    for s in structs:
        lines.append(f'printf("%zu ", sizeof({s.__name__}));')
        want.append(C.sizeof(s))
        for name, _ in s._fields_:
            lines.append(f'printf("%zu ", offsetof({s.__name__}, {name}));')
            want.append(getattr(s, name).offset)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{HEADER}"\nint main(void) {{ '
                   + "\n".join(lines) + " return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


def test_loaders_offer_the_operators():
    chunk = pkg.load_mac_chunk_attention_extension()
    assert chunk.mac_chunk_attention_bf16 is ops.mac_chunk_attention_bf16
    assert chunk.mac_chunk_attention_e4m3 is ops.mac_chunk_attention_e4m3
    q8 = pkg.load_mac_quantized_cache_extension()
    for name in ("mac_quantize_kv_e4m3", "mac_decode_rope_quantize_kv_e4m3", "mac_dequantize_kv_e4m3"):
        assert getattr(q8, name) is getattr(ops, name)
    with pytest.raises(RuntimeError, match="CUDA device"):
        pkg.make_chunk_attention_workspace("cpu")


def _chunk(**change):
    """Arguments that pass every check up to the device: the pointers are never followed here."""
    a = _abi.MacB200ChunkArgs()
    a.B, a.Hq, a.Hkv, a.D, a.q_rows = 1, 8, 2, 128, 4
    a.req_to_token_rows, a.req_to_token_stride, a.window = 1, 64, -1
    a.kv_tokens, a.q_stride0, a.workspace_bytes, a.sm_scale = 64, 1024, 1 << 40, 0.1
    for name, kind in a._fields_:
        if kind is _abi.ptr:
            setattr(a, name, 4096)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(D=64), b"D=128"), (dict(Hq=7), b"Hkv times"), (dict(Hq=34), b"Hkv times"), (dict(Hkv=0), b"Hkv times"),
    (dict(Hq=0), b"Hkv times"), (dict(Hq=4096, Hkv=2048), b"1024"), (dict(B=-1), b"negative"),
    (dict(q_rows=-3), b"negative"), (dict(sm_scale=0.0), b"sm_scale"), (dict(sm_scale=-1.0), b"sm_scale"),
    (dict(sm_scale=float("nan")), b"sm_scale"), (dict(sm_scale=float("inf")), b"sm_scale"),
    (dict(q=None), b"null"), (dict(workspace=None), b"null"), (dict(kv_lens=None), b"null"), (dict(out=None), b"null"),
    (dict(kv_tokens=0), b"pool"), (dict(kv_tokens=1 << 31), b"pool"), (dict(req_to_token_rows=0), b"req_to_token"),
    (dict(q_stride0=1023), b"stride"), (dict(q_stride0=1028), b"stride"), (dict(q_stride0=8), b"stride"),
    (dict(q=4104), b"aligned"), (dict(k=4097), b"aligned"), (dict(out=4100), b"aligned"), (dict(workspace=4104), b"aligned"),
])
def test_chunk_refusals(lib, change, text):
    a = _chunk(**change)
    for fn in (lib.mac_b200_chunk_attention_bf16, lib.mac_b200_chunk_attention_e4m3):
        assert fn(C.byref(a), None) == -1
        assert text in lib.mac_b200_last_error()


def test_chunk_null_empty_and_exponents(lib):
    assert lib.mac_b200_chunk_attention_bf16(None, None) == -1
    assert lib.mac_b200_chunk_attention_bf16(C.byref(_chunk(B=0)), None) == 0
    assert lib.mac_b200_chunk_attention_bf16(C.byref(_chunk(q_rows=0)), None) == 0
    assert lib.mac_b200_chunk_attention_e4m3(C.byref(_chunk(k_exp=None)), None) == -1
    assert b"exponents" in lib.mac_b200_last_error()
    assert lib.mac_b200_chunk_attention_workspace_bytes(None) == -1


def _quant(**change):
    a = _abi.MacB200QuantizeKvArgs()
    a.N, a.Hq, a.Hkv, a.D, a.rotary_dim, a.max_positions, a.kv_pool_tokens = 2, 8, 2, 128, 128, 10, 64
    for name, kind in a._fields_:
        if kind is _abi.ptr:
            setattr(a, name, 4096)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(D=64), b"D=128"), (dict(N=-1), b"negative"), (dict(Hkv=0), b"Hkv"), (dict(k=None), b"null"),
    (dict(v_exp=None), b"null"), (dict(k_pool=4104), b"aligned"), (dict(positions=None), b"rope"),
    (dict(Hq=0), b"Hq"), (dict(rotary_dim=3), b"rotary_dim"), (dict(rotary_dim=130), b"rotary_dim"),
    (dict(rotary_dim=0), b"rotary_dim"), (dict(q_post=4104), b"aligned"), (dict(N=1 << 40), b"too many"),
    (dict(kv_pool_tokens=-1), b"negative"),
])
def test_quantize_refusals(lib, change, text):
    assert lib.mac_b200_quantize_kv_e4m3(C.byref(_quant(**change)), None) == -1
    assert text in lib.mac_b200_last_error()


def test_results_that_share_memory_with_their_inputs_are_refused(lib):
    """Rows are read by other threads than those that write them: an overlap would race."""
    q, held = 1 << 20, 4 * 8 * 256                         # four rows of eight heads
    for out in (q, q + 2048, q + held - 16, q - held + 16):
        assert lib.mac_b200_chunk_attention_bf16(C.byref(_chunk(q=q, out=out)), None) == -1
        assert b"share memory" in lib.mac_b200_last_error()
    for change in (dict(), dict(q=1 << 20, v=1 << 21), dict(k=1 << 20, v=1 << 21), dict(k=1 << 20, q=1 << 21)):
        a = _quant(q_stride0=1024, k_stride0=256, v_stride0=256, **change)
        assert lib.mac_b200_quantize_kv_e4m3(C.byref(a), None) == -1
        assert b"q_post must not share memory" in lib.mac_b200_last_error()


def _dequant(**change):
    a = _abi.MacB200DequantizeKvArgs()
    a.N, a.Hkv, a.D, a.src_tokens, a.dst_tokens = 2, 2, 128, 64, 64
    for name, kind in a._fields_:
        if kind is _abi.ptr:
            setattr(a, name, 4096)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(D=64), b"D=128"), (dict(N=-1), b"negative"), (dict(Hkv=0), b"Hkv"), (dict(k_buffer=None), b"null"),
    (dict(v_buffer=4104), b"aligned"), (dict(k_pool=4104), b"aligned"), (dict(N=1 << 40), b"too many"),
    (dict(src_tokens=-1), b"negative"),
])
def test_dequantize_refusals(lib, change, text):
    assert lib.mac_b200_dequantize_kv_e4m3(C.byref(_dequant(**change)), None) == -1
    assert text in lib.mac_b200_last_error()


def test_empty_writes_and_reads_do_nothing(lib):
    assert lib.mac_b200_quantize_kv_e4m3(C.byref(_quant(N=0)), None) == 0
    assert lib.mac_b200_dequantize_kv_e4m3(C.byref(_dequant(N=0)), None) == 0


def test_operators_refuse_cpu_tensors():
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="q must be CUDA"):
        ops.mac_chunk_attention_bf16(q, k, k, i.view(1, 2), i[:1], i, i[:1], q, None, i)
    pool = pkg.make_quantized_pool(4, 2, device="cpu")
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.mac_chunk_attention_e4m3(q, *pool, i.view(1, 2), i[:1], i, i[:1], q, None, i)
    with pytest.raises(RuntimeError, match="k must be CUDA"):
        ops.mac_quantize_kv_e4m3(k.view(4, 256), k.view(4, 256), *pool, i)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.mac_decode_rope_quantize_kv_e4m3(q.view(2, -1), k.view(4, 256), k.view(4, 256), q, *pool,
                                             torch.zeros(4, 128), i, i, 128, True)
    with pytest.raises(RuntimeError, match="k_pool must be CUDA"):
        ops.mac_dequantize_kv_e4m3(*pool, i, k, k)


def test_an_empty_pool_holds_zeros():
    k, v, ke, ve = pkg.make_quantized_pool(3, 2, device="cpu")
    assert k.dtype == torch.float8_e4m3fn and tuple(k.shape) == (3, 2, 128) and tuple(ke.shape) == (3, 2)
    codes, e = hold_reference(torch.zeros(3, 2, 128))
    assert torch.equal(ke, e) and torch.equal(ve, e) and torch.equal(k.double(), codes) and (v.double() == 0).all()
