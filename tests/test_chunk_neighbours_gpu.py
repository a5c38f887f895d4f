"""GPU: requests beside one that cannot be run keep their results, over the 8-bit pool as over the bf16 pool."""
import math

import pytest
import torch

import mac_attention_b200 as mac
from mac_attention_b200 import ops
from tests.chunk_cases import assert_chunk_close, chunk_reference, make_chunk
from tests.test_chunk_attention_gpu import quantized, run

pytestmark = pytest.mark.gpu

ROWS = [slice(0, 4), slice(4, 10), slice(10, 140)]


@pytest.fixture(scope="module")
def ext():
    return mac.load_mac_chunk_attention_extension()


@pytest.fixture(scope="module")
def workspace():
    return mac.make_chunk_attention_workspace()


@pytest.mark.parametrize("name,value,bad", [("ids", 5, 0), ("ids", -1, 1), ("kv_lens", 10**6, 2), ("kv_lens", -4, 1)])
@pytest.mark.parametrize("window", [None, 50])
def test_requests_beside_a_bad_one(ext, workspace, name, value, bad, window):
    base = make_chunk([4, 6, 130], [200, 300, 400], 8, 2, seed=13)
    pool, k, v = quantized(base)
    t = dict(base)
    t[name] = base[name].clone()
    t[name][bad] = value
    for held, want in ((None, chunk_reference(base, window)), (pool, chunk_reference(base, window, k=k, v=v))):
        out, lse = run(ext, t, workspace, window, pool=held)
        for i, rows in enumerate(ROWS):
            if i != bad:
                assert_chunk_close(out, lse, want, rows)
        assert (out[ROWS[bad]] == 0).all() and (lse[ROWS[bad]] == -math.inf).all()
        assert ops.query_status() & 0x2
        assert ops.query_status() == 0


@pytest.mark.parametrize("offsets,bad", [([0, 4, 10, 141], 2), ([-1, 4, 10, 140], 0)])
def test_offsets_that_leave_the_rows(ext, workspace, offsets, bad):
    """The request is left out and its rows stay as they were."""
    base = make_chunk([4, 6, 130], [200, 300, 400], 8, 2, seed=13)
    pool, k, v = quantized(base)
    t = dict(base, offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    for held, want in ((None, chunk_reference(base)), (pool, chunk_reference(base, k=k, v=v))):
        out, lse = run(ext, t, workspace, pool=held)
        for i, rows in enumerate(ROWS):
            if i != bad:
                assert_chunk_close(out, lse, want, rows)
            else:
                assert (out[rows] == 7).all() and (lse[rows] == 3).all()
        assert ops.query_status() & 0x2
