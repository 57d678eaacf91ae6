"""What the block over a paged cache refuses, it refuses before anything is launched: its attention's
conditions, answered without a device."""
import pytest

from beacon_b200 import _lib
from test_paged_cpu import H, INV, call


@pytest.mark.parametrize("which", ["block", "attn"])
@pytest.mark.parametrize("off", [1, 4, 8, 16])
def test_workspace_that_partial_rows_cannot_be_stored_in(which, off):
    assert call(which, ws=H + off, wsb=1 << 40) == INV
    assert "32-byte aligned" in _lib.last_error()


@pytest.mark.parametrize("change", [dict(max_q=-1), dict(tokens=1 << 20, heads=1 << 12, kv=1 << 12),
                                    dict(tokens=100000, seqs=100000, max_pages=1 << 24, table_stride=1 << 24)])
def test_block_refuses_what_its_attention_refuses(change):
    assert call("block", **change) == INV, _lib.last_error()
    assert "llama_block_paged_fwd" in _lib.last_error()
